"""Layer norm, clipping and an optimizer together, as a neural shader is trained with them."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24  # half a step of float32


def _example():
    spec = importlib.util.spec_from_file_location(
        "neural_shading", os.path.join(ROOT, "examples", "neural_shading.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("sgd", [False, True])
def test_the_example_runs(sgd):
    """Finite losses, and the same ones from the same seed: every sum runs in a fixed order."""
    a, b = (_example().train(steps=6, size=64, views=2, level=2, norm="layer", sgd=sgd)
            for _ in range(2))
    print(f"[neural shading] {a}", flush=True)
    assert torch.tensor(a).isfinite().all() and a == b


def _loss(decoder, norm, params, x, want):
    """The decoder's loss with weights `params` (linear, scale, shift) in any type."""
    n = len(decoder.scale)
    linear, scale, shift = params[:n + 1], params[n + 1:2 * n + 1], params[2 * n + 1:]
    y = x.reshape(-1, x.shape[-1])
    for w, a, b in zip(linear, scale, shift):
        z = norm(y @ w.t(), a, b)
        y = z * torch.sigmoid(z)
    return ((torch.sigmoid(y @ linear[-1].t()) - want) ** 2).sum()


def _norm(x, weight, bias):
    d = x - x.mean(-1, keepdim=True)
    return d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-5) * weight + bias


@pytest.mark.parametrize("max_norm", [0.05, 1e3])
def test_a_step_against_float64(max_norm):
    """A decoder's gradients, clipped, and a step of SGD, against the same in float64. Eight stages
    of products with up to 64 terms, each off by 64 roundings of its terms at most and passed on
    eightfold: 4096 roundings of a tensor's norm."""
    import opendressi_amd.torch as dr
    ctx = dr.RasterizeHipContext(0)
    torch.manual_seed(3)
    decoder = _example().Decoder(ctx, 11, norm="layer").to("cuda")
    params = [*decoder.linear, *decoder.scale, *decoder.shift]
    x, want = torch.randn(2, 17, 23, 11, device="cuda"), torch.rand(782, 3, device="cuda")
    exact = [p.detach().cpu().double().requires_grad_() for p in params]
    _loss(decoder, _norm, exact, x.cpu().double(), want.cpu().double()).backward()
    total = torch.cat([p.grad.reshape(-1) for p in exact]).norm()
    factor = min(1.0, max_norm / (float(total) + 1e-6))
    opt = torch.optim.SGD(params, lr=0.25)
    ((decoder(x).view(-1, 3) - want) ** 2).sum().backward()
    before = [p.detach().clone() for p in params]
    norm = dr.clip_grad_norm_(ctx, decoder.parameters(), max_norm)
    opt.step()
    assert abs(float(norm) / float(total) - 1) <= 4096 * U
    for p, q, old in zip(params, exact, before):
        g = q.grad * factor
        assert float((p.grad.cpu().double() - g).norm()) <= 4096 * U * float(g.norm())
        step = (p.detach() - old).cpu().double()
        assert float((step + 0.25 * g).norm()) <= 4096 * U * float(g.norm()) \
            + 2 * U * float(old.double().norm())


def test_features_of_rays_and_of_pixels_are_the_same():
    """Layer norm knows rows alone: an image, a list of its pixels and a slice of its channels'
    buffer give the same bits."""
    import opendressi_amd.torch as dr
    ctx = dr.RasterizeHipContext(0)
    wide = torch.randn(3, 20, 30, 70, device="cuda", dtype=torch.bfloat16)
    w, b = torch.rand(50, device="cuda"), torch.rand(50, device="cuda")
    x = wide[..., 10:60]
    y = dr.layer_norm(ctx, x, w, b, activation="gelu")
    assert torch.equal(y.view(-1, 50), dr.layer_norm(ctx, x.reshape(-1, 50), w, b,
                                                     activation="gelu"))
    assert torch.equal(y[1, 2, 3], dr.layer_norm(ctx, x[1, 2, 3], w, b, activation="gelu"))
