"""group_norm and layer_norm: the normalisation layers of a neural shader over
the surface's channels-last images. No counterpart in the reference's surface.
"""
from __future__ import annotations

import torch
from torch.autograd.forward_ad import unpack_dual

from .. import ops as K
from .context import RasterizeHipContext


def _check_tensors(x, weight, bias) -> None:
    for t, name in ((x, "x"), (weight, "weight"), (bias, "bias")):
        if not isinstance(t, torch.Tensor) and (t is not None or name == "x"):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")


class _GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(fctx, x, weight, bias, vctx, groups, eps, activation):
        dev = vctx.device
        x_d, w_d, b_d = (None if t is None else t.detach().to(dev) for t in (x, weight, bias))
        w_d, b_d = (None if t is None else t.contiguous() for t in (w_d, b_d))
        with vctx.lock:
            y, mean, rstd = K.group_norm(vctx._ctx, x_d, groups, w_d, b_d, eps, activation)
        fctx.dressi = (vctx, groups, activation)
        fctx.save_for_backward(x, weight, bias, mean, rstd)
        return y.to(x.device)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(fctx, grad_out):
        vctx, groups, activation = fctx.dressi
        x, weight, bias, mean, rstd = fctx.saved_tensors
        dev = vctx.device
        x_d, w_d, b_d, g_d = (None if t is None else t.detach().to(dev)
                              for t in (x, weight, bias, grad_out))
        w_d, b_d = (None if t is None else t.contiguous() for t in (w_d, b_d))
        with vctx.lock:
            grads = K.group_norm_bwd(vctx._ctx, g_d, x_d, mean, rstd, groups, w_d, b_d,
                                     activation, fctx.needs_input_grad[:3])
        grads = [None if g is None else g.to(t.device) for g, t in zip(grads, (x, weight, bias))]
        return (*grads, None, None, None, None)


def group_norm(ctx: RasterizeHipContext, x: torch.Tensor, groups: int, weight=None, bias=None,
               eps: float = 1e-5, activation: str = "none") -> torch.Tensor:
    """Group normalisation of channels-last images and an activation.

    x is [N, ..., C] (an image batch [N, H, W, C], or pixels [N, P, C]) in
    float32, bfloat16 or float16; weight and bias are [C], of one type of the
    three, or None. Returns act((x - mean) / sqrt(var + eps) * weight + bias),
    with the mean and variance over the pixels and the C / groups channels of
    each group of each item, computed in float32; activation is "none",
    "relu", "silu" or "gelu". Differentiable w.r.t. x, weight and bias."""
    _check_tensors(x, weight, bias)
    return _GroupNormFn.apply(x, weight, bias, ctx, int(groups), float(eps), activation)


def _moved(dev, x, weight, bias):
    """The three on the context's device, the last two packed; for where
    autograd does not look."""
    x = x.to(dev)
    return x, *(None if t is None else t.to(dev).contiguous() for t in (weight, bias))


def _followed(*tensors) -> bool:
    """Whether autograd follows one of them. A tangent of forward mode, which a
    Function refuses, would be lost on the short way past it."""
    reverse = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and (reverse and t.requires_grad or unpack_dual(t).tangent is not None):
            return True
    return False


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(fctx, x, weight, bias, vctx, eps, activation):
        with vctx.lock:
            x_d, w_d, b_d = _moved(vctx.device, x, weight, bias)
            y, mean, rstd = K.layer_norm(vctx._ctx, x_d, w_d, b_d, eps, activation)
        fctx.dressi = (vctx, activation)
        fctx.save_for_backward(x, weight, bias, mean, rstd)
        return y.to(x.device)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(fctx, grad_out):
        vctx, activation = fctx.dressi
        x, weight, bias, mean, rstd = fctx.saved_tensors
        with vctx.lock:
            x_d, w_d, b_d = _moved(vctx.device, x, weight, bias)
            grads = K.layer_norm_bwd(vctx._ctx, grad_out.detach().to(vctx.device), x_d, mean, rstd,
                                     w_d, b_d, activation, fctx.needs_input_grad[:3])
        grads = [None if g is None else g.to(t.device) for g, t in zip(grads, (x, weight, bias))]
        return (*grads, None, None, None)


def layer_norm(ctx: RasterizeHipContext, x: torch.Tensor, weight=None, bias=None,
               eps: float = 1e-5, activation: str = "none") -> torch.Tensor:
    """Layer normalisation of the channels of each pixel and an activation.

    x is [..., C] (an image batch [N, H, W, C], vertices' or rays' features
    [V, C], one row [C]) in float32, bfloat16 or float16; weight and bias are
    [C], of one type of the three, or None. Returns
    act((x - mean) / sqrt(var + eps) * weight + bias), with the mean and
    variance over the C channels of each pixel, computed in float32;
    activation is "none", "relu", "silu" or "gelu". Differentiable w.r.t. x,
    weight and bias, in reverse mode; forward mode's dual tensors are refused."""
    _check_tensors(x, weight, bias)
    if _followed(x, weight, bias):
        return _LayerNormFn.apply(x, weight, bias, ctx, float(eps), activation)
    with ctx.lock:
        return K.layer_norm(ctx._ctx, *_moved(ctx.device, x, weight, bias), float(eps), activation,
                            stats=False)[0].to(x.device)
