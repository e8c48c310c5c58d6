"""Group norm (opendressi_amd.ops.group_norm, group_norm_bwd) where values or gradients are
unusual."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
# one pass; two passes; two passes whose vectors are cut by groups' edges; many items in one pass
# and in two
SHAPES = [((2, 8, 9, 32), 4), ((1, 90, 91, 64), 8), ((2, 70, 71, 66), 6), ((300, 4, 16), 2),
          ((700, 9, 520), 1)]


@pytest.fixture(scope="module")
def ctx():
    import opendressi_amd as od
    c = od.Context(0)
    yield c
    c.close()


def _inputs(shape, kind, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    c = shape[-1]
    return r(*shape).to(kind), r(*shape).to(kind), 1 + 0.2 * r(c), 0.3 * r(c)


@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_relu_masks_any_gradient(ctx, shape, groups, kind, bad):
    """Where relu's slope is zero, no gradient passes, whatever it is: the bits of a zero there."""
    from opendressi_amd import ops as K
    print(f"[group_norm relu] {shape} {groups} {kind} {bad}", flush=True)
    x, gy, w, b = _inputs(shape, kind, 1)
    z, mean, rstd = K.group_norm(ctx, x, groups, w, b)
    off = z < -0.1
    assert off.any()
    want = K.group_norm_bwd(ctx, gy.masked_fill(off, 0.0), x, mean, rstd, groups, w, b, "relu")
    got = K.group_norm_bwd(ctx, gy.masked_fill(off, bad), x, mean, rstd, groups, w, b, "relu")
    for p, q in zip(got, want):
        assert q.isfinite().all() and torch.equal(p, q)


@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
def test_relu_masks_what_it_gave_as_zero(ctx, shape, groups):
    """Each channel's bias puts one pixel of each item as near to relu's kink as float32 goes: the
    gradient passes where the output is above zero and nowhere else."""
    from opendressi_amd import ops as K
    print(f"[group_norm kink] {shape} {groups}", flush=True)
    x, _, w, _ = _inputs(shape, torch.float32, 2)
    n, c = shape[0], shape[-1]
    z, mean, rstd = K.group_norm(ctx, x, groups, w)
    # one pixel's z for each channel, with its sign turned
    at = torch.arange(c, device="cuda") % (x.numel() // (n * c))
    b = -z.view(n, -1, c)[0].gather(0, at[None])[0].contiguous()
    y = K.group_norm(ctx, x, groups, w, b, activation="relu")[0]
    _, _, gb = K.group_norm_bwd(ctx, torch.ones_like(x), x, mean, rstd, groups, w, b, "relu",
                                (False, False, True))
    assert torch.equal(gb.double(), (y > 0).view(-1, c).double().sum(0))


@pytest.mark.parametrize("hw", [32, 256, 1024])
@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("where", [0.0, 0.25, 0.5, 0.75, 1.0])
def test_one_pixel_far_from_the_rest(ctx, hw, kind, where):
    """One pixel 10^4 deviations off, wherever it is, costs the others nothing: the mean within 64
    roundings of a value's usual size (not of the far one's), the deviation and the outputs within
    64 of their own."""
    print(f"[group_norm far] {hw} {kind} {where}", flush=True)
    x, _, _, _ = _inputs((1, hw, hw, 8), kind, 3)
    x.view(-1, 8)[min(hw * hw - 1, int(hw * hw * where))] = 1e4
    _check_far(ctx, x)


@pytest.mark.parametrize("hw", [64, 256, 1024])
@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("side", ["left", "top", "frame", "corner"])
def test_a_border_far_from_the_rest(ctx, hw, kind, side):
    """The same for a column, a row, a frame or a patch."""
    print(f"[group_norm border] {hw} {kind} {side}", flush=True)
    x, _, _, _ = _inputs((1, hw, hw, 8), kind, 3)
    if side == "corner":
        x[:, :hw // 8, :hw // 8] = -1e4
    if side in ("left", "frame"):
        x[:, :, 0] = 1e4
    if side in ("top", "frame"):
        x[:, 0] = 1e4
    if side == "frame":
        x[:, -1] = x[:, :, -1] = 1e4
    _check_far(ctx, x)


def _check_far(ctx, x):
    from opendressi_amd import ops as K
    y, mean, rstd = K.group_norm(ctx, x, 2)
    xd = x.double().view(-1, 2, 4)
    exact = xd.mean((0, 2))
    dev = torch.sqrt((xd - exact[:, None]).square().mean((0, 2)) + 1e-5)
    u = 2.0 ** -24
    # E|x| of the rest is 0.8, and the far value adds its share
    tol = 64 * u * (0.8 + exact.abs())
    assert ((mean[0].double() - exact).abs() <= tol).all(), (mean[0].double() - exact).abs().max()
    assert ((rstd[0].double() * dev - 1).abs() <= 64 * u).all()
    want = (xd - exact[:, None]) / dev[:, None]
    half = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0
    err = (y.double().view(-1, 2, 4) - want).abs()
    assert (err <= (tol / dev)[:, None] + (72 * u + half) * want.abs() + 2.0 ** -25).all()
