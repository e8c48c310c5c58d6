"""clip_grad_norm_ and grad_norm: the norm of all gradients together, and the
gradients scaled down to a largest one, for what AdamW does not step (it clips
inside its own step). No counterpart in the reference's surface.
"""
from __future__ import annotations

import math
import operator
from array import array
from itertools import chain

import torch
from torch.autograd.graph import increment_version

from .._lib import NORM_2, NORM_LARGEST, check, lib
from ..ops import TYPE_CODES, _addr
from .context import RasterizeHipContext
from .optim import _dense
from .strides import apart as _apart, shared

_KINDS = {2.0: NORM_2, math.inf: NORM_LARGEST}


def _all_contiguous(grads) -> bool:
    try:
        return all(map(torch.Tensor.is_contiguous, grads))
    except RuntimeError:  # some sparse layouts raise
        return False


def _refuse(ctx, g) -> None:
    """Raises for a gradient that a call does not take."""
    if g.layout is not torch.strided:
        raise RuntimeError("clip_grad_norm_: sparse gradients are not supported")
    if g.dtype not in TYPE_CODES:
        raise TypeError(f"a gradient must be float32, bfloat16 or float16, got {g.dtype}")
    if g.get_device() != ctx.device.index:
        raise ValueError(f"a gradient is on {g.device}, the context on {ctx.device}")


class _Gradients:
    """The parameters' gradients, checked, and the table of them that a call
    takes: an address, a count and a type for each."""

    def __init__(self, ctx: RasterizeHipContext, parameters):
        if isinstance(parameters, torch.Tensor):
            parameters = [parameters]
        self.grads = grads = [g for p in parameters if (g := p.grad) is not None]
        kinds = [g.dtype for g in grads]
        for g in grads if not set(kinds) <= TYPE_CODES.keys() or \
                not set(map(torch.Tensor.get_device, grads)) <= {ctx.device.index} else ():
            _refuse(ctx, g)
        self.views = views = []  # those not densely stored, with their packed copies
        packed = grads
        if not _all_contiguous(grads):
            packed = []
            for g in grads:
                _refuse(ctx, g)
                if not _dense(g):
                    views.append((g, g.contiguous()))
                    g = views[-1][1]
                packed.append(g)
        self.dense = map(operator.is_, grads, packed)  # of each, whether it is its own packed copy
        # three words an entry, as in dressi_clip_tensor
        self.table = array("Q", chain.from_iterable(zip(
            map(torch.Tensor.data_ptr, packed), map(torch.Tensor.numel, packed),
            map(TYPE_CODES.__getitem__, kinds))))

    def clip(self, ctx: RasterizeHipContext, kind: int, max_norm: float) -> torch.Tensor:
        """Their norm; those above max_norm are scaled."""
        at, n = self.table.buffer_info()[0], len(self.grads)
        norm = self.grads[0].new_empty((), dtype=torch.float32) if n else \
            torch.empty((), device=ctx.device)
        size = lib.dressi_clip_norm_scratch(at, n)
        scratch = norm.new_empty(size, dtype=torch.uint8) if size else None
        with ctx.lock:
            ctx._ctx.use_torch_stream()
            check(lib.dressi_clip_norm(ctx._ctx.handle, at, n, kind, max_norm, _addr(scratch),
                                       norm.data_ptr()))
        return norm


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
    return _Gradients(ctx, parameters).clip(ctx, _kind(norm_type), math.inf)


def clip_grad_norm_(ctx: RasterizeHipContext, parameters, max_norm: float,
                    norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the parameters' gradients, in place, by
    min(1, max_norm / (norm + 1e-6)), norm that of all of them together
    (grad_norm), without a host round trip, and returns the norm from before.

    `parameters` is an iterable of tensors, or one; those whose grad is None
    are passed over. Gradients are float32, bfloat16 or float16, mixed as they
    come, on the context's device; no two share memory (a parameter must not
    be there twice). max_norm inf leaves all gradients as they are, and takes
    those that do. Where the norm is not finite, the gradients become NaN or
    zero, as the formula says; error_if_nonfinite waits for the norm and raises
    instead, with the gradients as they were."""
    kind = _kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    g = _Gradients(ctx, parameters)
    # packed ones are looked at by the call
    if max_norm < math.inf and g.views and (not all(_apart(v) for v, _ in g.views) or
                                            shared(g.grads, g.dense)):
        raise ValueError("gradients are the same or share memory")
    if error_if_nonfinite:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("error_if_nonfinite waits for the norm: not in a captured call")
        norm = g.clip(ctx, kind, math.inf)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"the gradients' norm is {float(norm)}: they are not clipped")
    norm = g.clip(ctx, kind, max_norm)
    if max_norm < math.inf:
        with torch.no_grad():
            for v, packed in g.views:
                v.copy_(packed)
        increment_version(g.grads)  # written in place
    return norm
