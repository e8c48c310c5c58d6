"""clip_grad_norm_ and grad_norm: the norm of all gradients together, and the
gradients scaled down to a largest one, for what AdamW does not step (it clips
inside its own step). No counterpart in the reference's surface.
"""
from __future__ import annotations

import math

import numpy as np
import torch
from torch.autograd.graph import increment_version

from .._lib import NORM_2, NORM_LARGEST, check, lib
from ..ops import TYPE_CODES
from .context import RasterizeHipContext
from .optim import _dense

# an entry of the table of tensors (dressi_clip_tensor)
_ENTRY = np.dtype([("data", "<u8"), ("n", "<u8"), ("type", "<u4"), ("unused", "<u4")])
_KINDS = {2.0: NORM_2, math.inf: NORM_LARGEST}


def _clip(ctx: RasterizeHipContext, grads: list[torch.Tensor], kind: int,
          max_norm: float) -> torch.Tensor:
    """Dense gradients' norm, and what is above max_norm scaled."""
    table = np.zeros(len(grads), _ENTRY)
    table["data"] = [g.data_ptr() for g in grads]
    table["n"] = [g.numel() for g in grads]
    table["type"] = [TYPE_CODES[g.dtype] for g in grads]
    with ctx.lock:
        norm = torch.empty((), device=ctx.device)
        scratch = torch.empty(lib.dressi_clip_norm_scratch(), dtype=torch.uint8, device=ctx.device)
        ctx._ctx.use_torch_stream()
        check(lib.dressi_clip_norm(ctx._ctx.handle, table.ctypes.data, len(grads), kind, max_norm,
                                   scratch.data_ptr(), norm.data_ptr()))
    return norm


def _apart(t: torch.Tensor) -> bool:
    """Whether no two of t's elements share memory, by strides that each reach
    past all that the smaller ones span."""
    end = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride < end:
            return False
        end += stride * (size - 1)
    return True


def _gradients(ctx: RasterizeHipContext, parameters) -> list[torch.Tensor]:
    """Those that there are, checked."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    dev = ctx.device.index
    for g in grads:
        if g.layout is not torch.strided:
            raise RuntimeError("clip_grad_norm_: sparse gradients are not supported")
        if g.dtype not in TYPE_CODES:
            raise TypeError(f"a gradient must be float32, bfloat16 or float16, got {g.dtype}")
        if g.get_device() != dev:
            raise ValueError(f"a gradient is on {g.device}, the context on {ctx.device}")
    return grads


def _kind(norm_type) -> int:
    kind = _KINDS.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    return kind


def grad_norm(ctx: RasterizeHipContext, parameters, norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all the parameters' gradients together, as a float32 scalar
    on the context's device: the square root of their sum of squares, added in
    float64, or (norm_type inf) their largest magnitude. Without gradients it
    is zero; a NaN among them makes it NaN."""
    kind = _kind(norm_type)
    grads = [g if _dense(g) else g.contiguous() for g in _gradients(ctx, parameters)]
    return _clip(ctx, grads, kind, math.inf)


def clip_grad_norm_(ctx: RasterizeHipContext, parameters, max_norm: float,
                    norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the parameters' gradients, in place, by
    min(1, max_norm / (norm + 1e-6)), norm that of all of them together
    (grad_norm), without a host round trip, and returns the norm from before.

    `parameters` is an iterable of tensors, or one; those whose grad is None
    are passed over. Gradients are float32, bfloat16 or float16, mixed as they
    come, on the context's device; no two share memory (a parameter must not be there
    twice). max_norm inf leaves all gradients as they are. Where the norm is not
    finite, the gradients become NaN or zero, as the formula says;
    error_if_nonfinite waits for the norm and raises instead, with the
    gradients as they were."""
    kind = _kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    grads = _gradients(ctx, parameters)
    packed = [g if _dense(g) else g.contiguous() for g in grads]
    views = [g for g, q in zip(grads, packed) if q is not g]
    if views and (not all(map(_apart, views)) or
                  len({g.data_ptr() for g in grads if g.numel()}) < sum(g.numel() > 0 for g in grads)):
        raise ValueError("gradients are the same or share memory")
    if error_if_nonfinite:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("error_if_nonfinite waits for the norm, which a captured call cannot")
        norm = _clip(ctx, packed, kind, math.inf)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"the gradients' norm is {float(norm)}: they are not clipped")
    norm = _clip(ctx, packed, kind, max_norm)
    if max_norm < math.inf:
        with torch.no_grad():
            for g, q in zip(grads, packed):
                if q is not g:
                    g.copy_(q)
        increment_version(grads)  # written in place
    return norm
