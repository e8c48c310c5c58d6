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


def _rms(t):
    return float(t.double().square().mean().sqrt())


def test_gelu_is_as_good_as_its_formula_in_floats(ctx):
    """float32 images: the error of z Phi(z) and of its slope over normal z, against those of
    z 0.5 (1 + erf(z / sqrt 2)) and of its derivative in float32, whose roundings are as many (a
    quarter more for their other order)."""
    from opendressi_amd import ops as K
    x = _inputs((1, 512, 512, 8), torch.float32, 4)[0]
    z, mean, rstd = K.group_norm(ctx, x, 1)
    y = K.group_norm(ctx, x, 1, activation="gelu")[0]
    plain = z * (0.5 * (1 + torch.erf(z * 0.5 ** 0.5)))
    want = z.double() * torch.special.ndtr(z.double())
    assert _rms(y - want) <= 1.25 * _rms(plain - want)
    # z is the bias where x has no variance; two pixels' slopes add up to twice one's
    b = _inputs((1, 2 ** 16), torch.float32, 5)[0][0]
    x = torch.zeros((1, 2, 2 ** 16), device="cuda")
    _, mean, rstd = K.group_norm(ctx, x, 1, None, b, activation="gelu")
    slope = K.group_norm_bwd(ctx, torch.ones_like(x), x, mean, rstd, 1, None, b, "gelu")[2] / 2
    d, pdf = b.double(), 1 / math.sqrt(2 * math.pi)
    want = torch.special.ndtr(d) + d * torch.exp(-0.5 * d * d) * pdf
    plain = 0.5 * (1 + torch.erf(b * 0.5 ** 0.5)) + b * torch.exp(-0.5 * b * b) * pdf
    assert _rms(slope - want) <= 1.25 * _rms(plain - want)


def test_gelu_tail(ctx):
    """z Phi(z) of float32 images below zero, relative to itself: 2^-24 (z^2 + 6 |z| + 16), of the
    exponent's two roundings, of the tail's factor (0.4 / |z| as a difference from a half) and of
    the rest."""
    from opendressi_amd import ops as K
    b = torch.linspace(-12.0, -1e-3, 2 ** 16, device="cuda")
    x = torch.zeros((1, 2, 2 ** 16), device="cuda")
    y = K.group_norm(ctx, x, 1, None, b, activation="gelu")[0][0]
    d = b.double()
    want = d * 0.5 * torch.special.erfc(-d * math.sqrt(0.5))
    tol = 2.0 ** -24 * (d * d + 6 * d.abs() + 16)
    assert ((y.double() / want - 1).abs() <= tol).all()
    far = torch.tensor([-math.inf, -1e30, -40.0, 0.0, 40.0, 1e30, math.inf, math.nan],
                       device="cuda")
    y = K.group_norm(ctx, torch.zeros((1, 2, 8), device="cuda"), 1, None, far,
                     activation="gelu")[0][0, 0]
    assert y[0].isnan() and not y[1:4].any() and torch.equal(y[4:7], far[4:7]) and y[7].isnan()


@pytest.mark.parametrize("shape,groups", [((1, 64, 64, 131072), 131072),
                                          ((2, 48, 48, 69632), 69632)], ids=str)
def test_more_groups_than_a_launch_has_rows(ctx, shape, groups):
    """One channel a group, more of them than a launch's y dimension goes: statistics, outputs and
    gradients of a stretch of channels at each end and in the midst, against float64."""
    from opendressi_amd import ops as K
    print(f"[group_norm groups] {shape} {groups}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = torch.empty(shape, device="cuda").normal_(generator=gen)
    gy = torch.empty(shape, device="cuda").normal_(generator=gen)
    w = torch.rand(groups, generator=gen, device="cuda") + 0.5
    y, mean, rstd = K.group_norm(ctx, x, groups, w, None, 1e-5, "none")
    gx, gw, _ = K.group_norm_bwd(ctx, gy, x, mean, rstd, groups, w, None, "none",
                                 (True, True, False))
    u, n = 2.0 ** -24, shape[1] * shape[2]
    for a in (0, 65530, groups - 64):
        part = (slice(None),) * 3 + (slice(a, a + 64),)
        d, g = x[part].double(), gy[part].double()
        m, v = d.mean((1, 2)), d.var((1, 2), correction=0)
        r = 1 / torch.sqrt(v + 1e-5)
        assert ((mean[:, a:a + 64] - m).abs() <= 64 * u).all()
        assert ((rstd[:, a:a + 64] / r - 1).abs() <= 64 * u).all()
        at = lambda t: t[:, None, None]  # noqa: E731
        xh, ww = (d - at(m)) * at(r), w[a:a + 64].double()
        # 64 roundings of the mean and of the deviation, 8 of the arithmetic
        assert ((y[part] - xh * ww).abs() <= u * ww * (72 * xh.abs() + 72 * at(r))).all()
        # sums of n products in float32, in sequences of up to 2^11 and then by halves
        length = 2 * u * (math.sqrt(min(n * shape[0], 2 ** 11)) + 24)
        want = (g * xh).sum((0, 1, 2))
        assert ((gw[a:a + 64] - want).abs() <= (length + 144 * u) * (g.abs() * (xh.abs() + 1)).sum(
            (0, 1, 2))).all()
        mg, mgx = (at(t.mean((1, 2))) for t in (g, g * xh))
        want = at(r) * ww * (g - mg - xh * mgx)
        size = at(r) * ww * (g.abs() + at(g.abs().mean((1, 2))) +
                             xh.abs() * at((g * xh).abs().mean((1, 2))))
        assert ((gx[part] - want).abs() <= (length + 160 * u) * (size + at(r) * ww)).all()


def _check_sparse(x, gy, mean, rstd, groups, at, got):
    """Gradients where gy is zero but at the pixels `at` of x [N, P, C] (item, pixel), from the
    formula in float64 with the forward pass's statistics: what a call leaves out, or takes twice,
    is as large as the sums themselves."""
    gx, gw, gb = got
    n, px, c = x.shape
    per = c // groups
    i, p = (torch.tensor(t, device="cuda") for t in zip(*at))
    g, d = gy[i, p].double(), x[i, p].double()
    m, r = (t[i].double().repeat_interleave(per, 1) for t in (mean, rstd))
    xh = (d - m) * r
    u = 2.0 ** -24
    # a few terms each: a rounding of the sum, 4 of xh
    assert ((gb - g.sum(0)).abs() <= 8 * u * g.abs().sum(0)).all()
    assert ((gw - (g * xh).sum(0)).abs() <= 16 * u * (g * (xh.abs() + m.abs() * r)).abs().sum(0)).all()
    # gx = rstd (gy - A - xh B), A and B the item's sums over its values
    sums = torch.zeros((2, n, groups), dtype=torch.float64, device="cuda")
    sums[0].index_add_(0, i, g.view(-1, groups, per).sum(2))
    sums[1].index_add_(0, i, (g * xh).view(-1, groups, per).sum(2))
    a, b = (t[i].repeat_interleave(per, 1) / (px * per) for t in sums)
    want = r * (g - a - xh * b)
    half = torch.finfo(x.dtype).eps / 2
    assert ((gx[i, p] - want).abs() <= (half + 32 * u) * r * (g.abs() + a.abs() + (xh * b).abs())
            ).all()


def test_gradients_past_32_bits(ctx):
    """Gradients at a few pixels of an image of more than 2^32 values, before and behind the powers
    of two; everywhere else gx is the means' share alone."""
    from opendressi_amd import ops as K
    n_px, c = 2 ** 29 + 1031, 8
    gen = torch.Generator(device="cuda").manual_seed(15)
    x = torch.empty((1, n_px, c), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    mean, rstd = K.group_norm(ctx, x, 2)[1:]
    at = [(0, p) for p in (0, 5, 2 ** 28, 2 ** 29 - 1, 2 ** 29, 2 ** 29 + 517, n_px - 1)]
    gy = torch.zeros_like(x)
    for _, p in at:
        gy[0, p].normal_(generator=gen)
    gx, gw, gb = K.group_norm_bwd(ctx, gy, x, mean, rstd, 2)
    _check_sparse(x, gy, mean, rstd, 2, at, (gx, gw, gb))
    for _, p in at:
        gx[0, p] = 0
    # seven pixels' sums over 2^31 values, times |xh| of at most 10
    for part in gx[0].split(2 ** 27):
        assert part.isfinite().all() and float(part.abs().max()) <= 1e-6


@pytest.mark.parametrize("c", [8, 520])
def test_gradients_of_more_items_than_a_launch(ctx, c):
    """Gradients of a few rows, before and behind the first launch's last: gw and gb have each of
    them once, and gx is theirs."""
    from opendressi_amd import ops as K
    n = 2 ** 22 + 5
    gen = torch.Generator(device="cuda").manual_seed(16)
    x = torch.empty((n, 1, c), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    mean, rstd = K.group_norm(ctx, x, 2)[1:]
    at = [(i, 0) for i in (0, 7, 2 ** 21, 2 ** 22 - 1, 2 ** 22, 2 ** 22 + 2, n - 1)]
    gy = torch.zeros_like(x)
    for i, _ in at:
        gy[i].normal_(generator=gen)
    gx, gw, gb = K.group_norm_bwd(ctx, gy, x, mean, rstd, 2)
    _check_sparse(x, gy, mean, rstd, 2, at, (gx, gw, gb))
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[[i for i, _ in at]] = False
    assert not gx[rest].any()
