"""Group norm with an activation (opendressi_amd.ops.group_norm, group_norm_bwd, and
opendressi_amd.torch.group_norm) against float64, formula and differences."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = {"none": lambda z: z, "relu": torch.relu, "silu": lambda z: z * torch.sigmoid(z),
        "gelu": lambda z: z * torch.special.ndtr(z)}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in TYPES}


@pytest.fixture(scope="module")
def ctx():
    import opendressi_amd as od
    c = od.Context(0)
    yield c
    c.close()


def _inputs(shape, kind, seed, offset=0.0, affine=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    c = shape[-1]
    x = (r(*shape) * (0.5 + torch.rand(c, generator=gen, device="cuda")) + r(c) + offset).to(kind)
    return x, r(*shape).to(kind), (1 + 0.2 * r(c)).to(affine), (0.3 * r(c)).to(affine)


def _exact(x, gy, weight, bias, groups, eps, act):
    """y, its gradients, the groups' mean and 1 / deviation, all by the definition in float64;
    and, per value of y, what a relative error of rstd and an absolute one of the mean add to z."""
    n, c = x.shape[0], x.shape[-1]
    ws = [None if t is None else t.double().requires_grad_() for t in (weight, bias)]
    xd = x.double().requires_grad_()
    xg = xd.reshape(n, -1, groups, c // groups)
    mean = xg.mean((1, 3), keepdim=True)
    var = ((xg - mean) ** 2).mean((1, 3), keepdim=True)
    xh = ((xg - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    z = xh if ws[0] is None else xh * ws[0]
    z = z if ws[1] is None else z + ws[1]
    y = ACTS[act](z)
    wants = [xd] + [t for t in ws if t is not None]
    grads = list(torch.autograd.grad(y, wants, gy.double())) if y.numel() else \
        [torch.zeros_like(t) for t in wants]
    gx = grads.pop(0)
    gw, gb = (None if t is None else grads.pop(0) for t in ws)
    return (y.detach(), gx, gw, gb, mean.detach().reshape(n, groups),
            (1 / torch.sqrt(var + eps)).detach().reshape(n, groups), z.detach(), xh.detach())


def _spread(t, x, groups):
    """A group's value at each of its elements."""
    n, c = x.shape[0], x.shape[-1]
    return t.reshape(n, 1, groups, 1).expand(n, max(1, x.numel() // max(1, n * c)), groups,
                                             c // groups).reshape(x.shape)


# Statistics come from at most 2^11 values a thread in batches and about 20 levels of joining:
# 64 roundings of the mean (of the largest |x|) and of the relative deviation are allowed.
STAT = 64 * 2.0 ** -24


def _check(x, gy, weight, bias, groups, eps, act, got, kink=1e-5):
    """The outputs against float64 within what the roundings allow: the statistics' error as above
    carried through z, 8 roundings of the arithmetic, 2^-20 of the activation's exp or erf, and the
    output's own rounding."""
    y, mean, rstd, gx, gw, gb = got
    ey, egx, egw, egb, emean, erstd, z, xh = _exact(x, gy, weight, bias, groups, eps, act)
    big = x.double().abs().reshape(x.shape[0], -1).amax(1).reshape(-1, 1)
    d_mean = STAT * big
    # the deviation is that of values about the mean, so an offset leaves it as it is, but for the
    # mean's own error
    d_rstd = STAT + STAT * big * erstd * 2.0 ** -10
    assert ((mean.double() - emean).abs() <= d_mean + 1e-30).all()
    assert ((rstd.double() / erstd - 1).abs() <= d_rstd).all()
    w = 1.0 if weight is None else weight.double().abs()
    dz = w * (xh.abs() * _spread(d_rstd, x, groups) + _spread(d_mean * erstd, x, groups)) \
        + 8 * 2.0 ** -24 * (w * xh.abs() + z.abs()) + 8 * 2.0 ** -24 * w * _spread(
            big * erstd, x, groups)
    half = HALF_ULP[x.dtype]
    tol = 1.2 * dz + 2.0 ** -20 * z.abs() + half * ey.abs() + 2.0 ** -25
    assert ((y.double() - ey).abs() <= tol).all(), float(((y.double() - ey).abs() / tol).max())
    if gx is None:
        return
    # slopes change by at most 1.2 of dz, relu's by 1 where z is within dz of its kink
    g = gy.double().abs()
    ds = 1.2 * dz + 2.0 ** -19
    if act == "none":
        ds = torch.zeros_like(dz)
    if act == "relu":
        ds = (z.abs() <= dz).double()
    slope = 1.2
    gz = g * slope
    dgz = g * ds + 8 * 2.0 ** -24 * gz
    dxh = dz / w if weight is not None else dz
    n_sum = x.numel() // x.shape[-1]
    # sums in float32: sequences of up to 2^11 terms, then levels of halves
    length = 2.0 ** -24 * 2 * (math.sqrt(min(n_sum, 2 ** 11)) + 24)
    flat = lambda t: t.reshape(-1, x.shape[-1])  # noqa: E731
    if gb is not None:
        kind = HALF_ULP[bias.dtype if bias is not None else torch.float32]
        tb = flat(dgz).sum(0) + length * flat(gz).sum(0) + kind * egb.abs()
        assert ((gb.double() - egb).abs() <= tb).all()
    if gw is not None:
        kind = HALF_ULP[weight.dtype]
        tw = flat(dgz * xh.abs() + gz * dxh).sum(0) + length * flat(gz * xh.abs()).sum(0) \
            + kind * egw.abs()
        assert ((gw.double() - egw).abs() <= tw).all()
    # gx = rstd (w gz - A - xh B), A and B the group's means of w gz and w gz xh
    means = lambda t: _spread(t.reshape(x.shape[0], -1, groups, x.shape[-1] // groups).mean(  # noqa: E731
        (1, 3)), x, groups)
    wg = w * gz * torch.ones_like(z)
    d_a = means(w * dgz) + length * means(wg)
    d_b = means(w * (dgz * xh.abs() + gz * dxh)) + length * means(wg * xh.abs())
    size = wg + means(wg) + xh.abs() * means(wg * xh.abs())
    er = _spread(erstd, x, groups)
    tx = er * (w * dgz + d_a + xh.abs() * d_b + dxh * means(wg * xh.abs())
               + size * (_spread(d_rstd, x, groups) + 8 * 2.0 ** -24)) + half * egx.abs() + 2.0 ** -25
    assert ((gx.double() - egx).abs() <= tx).all(), float(((gx.double() - egx).abs() / tx).max())


def _run(ctx, x, gy, weight, bias, groups, eps, act):
    from opendressi_amd import ops as K
    y, mean, rstd = K.group_norm(ctx, x, groups, weight, bias, eps, act)
    need = (True, weight is not None, bias is not None)
    gx, gw, gb = K.group_norm_bwd(ctx, gy, x, mean, rstd, groups, weight, bias, act, need)
    torch.cuda.synchronize()
    return y, mean, rstd, gx, gw, gb


SHAPES = [((1, 1, 1, 8), 2), ((2, 1, 3, 4), 4), ((1, 7, 5, 3), 1), ((3, 16, 16, 32), 8),
          ((2, 33, 31, 33), 3), ((1, 61, 97, 66), 33), ((5, 8, 9, 24), 2), ((2, 40, 13, 96), 1),
          ((1, 64, 64, 129), 129), ((2, 6, 7, 1040), 2), ((1, 5, 5, 4100), 1),
          ((1, 3, 4, 2304), 3), ((70, 2, 2, 16), 4), ((1, 200, 201, 16), 4), ((1, 257, 64, 40), 5),
          ((2, 11, 520), 520)]


@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("act", list(ACTS))
def test_against_float64(ctx, shape, groups, kind, act):
    print(f"[group_norm] {shape} {groups} {kind} {act}", flush=True)
    x, gy, w, b = _inputs(shape, kind, 1)
    _check(x, gy, w, b, groups, 1e-5, act, _run(ctx, x, gy, w, b, groups, 1e-5, act))


@pytest.mark.parametrize("shape,groups", [((5000, 8), 2), ((2100, 5, 24), 3), ((2500, 1100), 1),
                                          ((600, 70, 33), 3), ((2300, 9, 520), 1)], ids=str)
@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_many_items(ctx, shape, groups, kind):
    """More items than workgroups whose channel sums are added: each takes several."""
    print(f"[group_norm items] {shape} {groups} {kind}", flush=True)
    x, gy, w, b = _inputs(shape, kind, 12)
    _check(x, gy, w, b, groups, 1e-5, "silu", _run(ctx, x, gy, w, b, groups, 1e-5, "silu"))


@pytest.mark.parametrize("shape,groups,kind", [((1, 1111, 1200, 64), 8, torch.bfloat16),
                                               ((2, 700, 1031, 66), 6, torch.float16),
                                               ((3, 401, 1031, 41), 41, torch.float32)], ids=str)
def test_larger_than_a_cache(ctx, shape, groups, kind):
    """Images of which the second pass finds only the last part where the first left it."""
    print(f"[group_norm large] {shape} {groups} {kind}", flush=True)
    x, gy, w, b = _inputs(shape, kind, 14)
    _check(x, gy, w, b, groups, 1e-5, "silu", _run(ctx, x, gy, w, b, groups, 1e-5, "silu"))


@pytest.mark.parametrize("offset", [0.0, 300.0, -3e4])
@pytest.mark.parametrize("shape,groups", [((2, 64, 65, 32), 4), ((1, 30, 30, 5), 1),
                                          ((1, 300, 300, 8), 1)], ids=str)
def test_far_from_zero(ctx, shape, groups, offset):
    """A mean many deviations from zero costs what float32 holds of the mean, no more."""
    print(f"[group_norm offset] {shape} {groups} {offset}", flush=True)
    x, gy, w, b = _inputs(shape, torch.float32, 2, offset)
    _check(x, gy, w, b, groups, 1e-5, "none", _run(ctx, x, gy, w, b, groups, 1e-5, "none"))


def test_one_value_far_from_the_rest(ctx):
    """The first pixel of the image 10^4 deviations off: as good as any other place for it."""
    for at in (0, 1777, 4095):
        x, gy, w, b = _inputs((1, 64, 64, 8), torch.float32, 3)
        x.view(-1, 8)[at] = 1e4
        _check(x, gy, w, b, 2, 1e-5, "none", _run(ctx, x, gy, w, b, 2, 1e-5, "none"))


@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("affine", TYPES, ids=str)
def test_affine_types(ctx, kind, affine):
    x, gy, w, b = _inputs((2, 20, 21, 48), kind, 4, affine=affine)
    for weight, bias in ((w, b), (w, None), (None, b), (None, None)):
        got = _run(ctx, x, gy, weight, bias, 6, 1e-3, "silu")
        assert got[0].dtype == kind and got[3].dtype == kind
        assert got[4] is None or got[4].dtype == affine
        _check(x, gy, weight, bias, 6, 1e-3, "silu", got)


def test_constant_groups(ctx):
    """A group without variance: xh = 0, y = act(b), no gradient but through b."""
    from opendressi_amd import ops as K
    x = torch.full((2, 16, 16, 8), 3.25, device="cuda")
    w, b = torch.ones(8, device="cuda"), torch.arange(8.0, device="cuda") - 4
    y, mean, rstd = K.group_norm(ctx, x, 2, w, b, 1e-5, "relu")
    assert torch.equal(y, torch.relu(b).expand_as(x)) and (mean == 3.25).all()
    assert torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5), rtol=1e-6)
    gx, gw, gb = K.group_norm_bwd(ctx, torch.ones_like(x), x, mean, rstd, 2, w, b, "none")
    assert not gw.any() and (gb == 512).all() and (gx.abs() <= 1e-3).all()


@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_strides(ctx, kind):
    """A channel slice of a wider image and an item slice are read where they lie; a crop, a
    transposed image and an expanded one too, packed first if need be: the packed image's bits."""
    from opendressi_amd import ops as K
    wide, gy, w, b = _inputs((4, 24, 20, 48), kind, 5)
    w, b = w[:16].contiguous(), b[:16].contiguous()
    for x in (wide[..., 16:32], wide[..., 3:19], wide[::2, :, :, 8:24], wide[:, 2:9, 4:17, :16],
              wide[..., :16].transpose(1, 2), wide[:1, ..., :16].expand(3, -1, -1, -1),
              wide[:, :1, :, 32:], wide.permute(0, 3, 1, 2)[..., 4:20]):
        g = gy[..., :16].expand_as(x) if x.shape == gy[..., :16].shape else \
            torch.ones_like(x, memory_format=torch.contiguous_format)
        packed = x.contiguous()
        want = K.group_norm(ctx, packed, 4, w, b, 1e-5, "silu")
        got = K.group_norm(ctx, x, 4, w, b, 1e-5, "silu")
        # a view that does not begin at 16 bytes takes narrower vectors, and another order of sums
        for p, q in zip(want, got):
            assert torch.allclose(p.float(), q.float(), rtol=4 * HALF_ULP[kind] + 1e-5, atol=1e-5)
        want = K.group_norm_bwd(ctx, g, packed, want[1], want[2], 4, w, b, "silu")
        got = K.group_norm_bwd(ctx, g, x, got[1], got[2], 4, w, b, "silu")
        assert torch.allclose(want[0].float(), got[0].float(), rtol=4 * HALF_ULP[kind] + 1e-4,
                              atol=1e-4)
        for p, q in zip(want[1:], got[1:]):
            assert torch.allclose(p, q, rtol=1e-4, atol=1e-3)


def test_empty_and_single(ctx):
    from opendressi_amd import ops as K
    w, b = torch.ones(8, device="cuda"), torch.zeros(8, device="cuda")
    for shape in ((0, 4, 4, 8), (2, 0, 4, 8), (0, 8)):
        x = torch.empty(shape, device="cuda")
        y, mean, rstd = K.group_norm(ctx, x, 2, w, b)
        assert y.shape == x.shape and mean.shape == (shape[0], 2)
        gx, gw, gb = K.group_norm_bwd(ctx, x, x, mean, rstd, 2, w, b)
        assert gx.shape == x.shape and not gw.any() and not gb.any()
    x, gy, w, b = _inputs((9, 8), torch.float32, 6)  # rows without pixels between
    _check(x, gy, w, b, 2, 1e-5, "gelu", _run(ctx, x, gy, w, b, 2, 1e-5, "gelu"))
    x, gy, w, b = _inputs((3, 1, 6), torch.float32, 6)  # one value a group
    y, mean, rstd = K.group_norm(ctx, x, 6, w, b)
    assert torch.equal(y, b.expand_as(y)) and torch.equal(mean, x[:, 0])


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_not_finite_stays_in_its_group(ctx, bad):
    from opendressi_amd import ops as K
    x, gy, w, b = _inputs((3, 20, 20, 16), torch.float32, 7)
    y0, mean, rstd = K.group_norm(ctx, x, 4, w, b, 1e-5, "silu")
    want = K.group_norm_bwd(ctx, gy, x, mean, rstd, 4, w, b, "silu")
    x[1, 3, 4, 5] = bad
    y, mean, rstd = K.group_norm(ctx, x, 4, w, b, 1e-5, "silu")
    gx, gw, gb = K.group_norm_bwd(ctx, gy, x, mean, rstd, 4, w, b, "silu")
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[1, :, :, 4:8] = True
    assert y[hit].isnan().all() and torch.equal(y[~hit], y0[~hit])
    assert gx[hit].isnan().all() and torch.equal(gx[~hit], want[0][~hit])
    ch = torch.arange(16, device="cuda") // 4 == 1
    assert gw[ch].isnan().all() and torch.equal(gw[~ch], want[1][~ch])


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_gradient_against_differences(ctx, act):
    """<gradient, d> against the operator's own central differences along random directions. The
    third derivative's term is below h^2, the forward's rounding adds 2^-22 of sqrt(values) / h."""
    import opendressi_amd.torch as dr
    vctx = dr.RasterizeHipContext(0)
    x, gy, w, b = _inputs((2, 9, 11, 12), torch.float32, 8)
    gy = gy.double()
    loss = lambda *t: float((dr.group_norm(vctx, t[0], 3, t[1], t[2], activation=act).double()  # noqa: E731
                             * gy).sum())
    args = [t.clone().requires_grad_() for t in (x, w, b)]
    out = dr.group_norm(vctx, *args[:1], 3, *args[1:], activation=act)
    out.backward(gy.float())
    h = 2.0 ** -7
    for i, t in enumerate(args):
        gen = torch.Generator(device="cuda").manual_seed(i)
        d = torch.randn(t.shape, generator=gen, device="cuda")
        ends = [[u.detach() + s * h * d if k == i else u.detach() for k, u in enumerate(args)]
                for s in (1, -1)]
        diff = (loss(*ends[0]) - loss(*ends[1])) / (2 * h)
        want = float((t.grad.double() * d.double()).sum())
        scale = float(gy.norm()) * (float(d.norm()) if i else math.sqrt(x.numel())) / 10
        assert abs(diff - want) <= scale * (h * h * 4) + 2.0 ** -22 * math.sqrt(x.numel()) * 4 / h


def test_torch_surface(ctx):
    """Through autograd, with and without the gradients that are not asked for, on a side stream,
    from host tensors; a second derivative is refused."""
    import opendressi_amd.torch as dr
    vctx = dr.RasterizeHipContext(0)
    x, gy, w, b = _inputs((2, 8, 8, 16), torch.float32, 9)
    got = _run(ctx, x, gy, w, b, 4, 1e-5, "silu")
    for need in ((True, True, True), (True, False, False), (False, True, False)):
        args = [t.clone().requires_grad_(n) for t, n in zip((x, w, b), need)]
        y = dr.group_norm(vctx, args[0], 4, args[1], args[2], activation="silu")
        y.backward(gy)
        assert torch.equal(y, got[0])
        for t, n, g in zip(args, need, got[3:]):
            assert (t.grad is None) != n and (not n or torch.equal(t.grad, g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = dr.group_norm(vctx, x * 1.0, 4, w, b, activation="silu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, got[0])
    xc = x.cpu().requires_grad_()
    y = dr.group_norm(vctx, xc, 4, w, b, activation="silu")
    assert y.device.type == "cpu" and torch.equal(y, got[0].cpu())
    y.backward(gy.cpu())
    assert torch.equal(xc.grad, got[3].cpu())
    xg = x.clone().requires_grad_()
    g, = torch.autograd.grad(dr.group_norm(vctx, xg, 4).square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_graph_replays(ctx):
    """Captured into a graph and replayed with other work between: the eager bits every time."""
    from opendressi_amd import ops as K
    x, gy, w, b = _inputs((2, 64, 48, 32), torch.bfloat16, 10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    run = lambda: (lambda f: f + K.group_norm_bwd(ctx, gy, x, f[1], f[2], 4, w, b, "silu"))(  # noqa: E731
        K.group_norm(ctx, x, 4, w, b, 1e-5, "silu"))
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(4):
        x.copy_(torch.randn(x.shape, device="cuda") * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = run()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), i


def test_same_bits_twice(ctx):
    x, gy, w, b = _inputs((3, 100, 100, 24), torch.bfloat16, 11)
    a, c = (_run(ctx, x, gy, w, b, 3, 1e-5, "gelu") for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_refusals(ctx):
    from opendressi_amd import ops as K
    x = torch.zeros((2, 4, 4, 8), device="cuda")
    w = torch.ones(8, device="cuda")
    for args, kw, err, what in (
            ((x, 3), {}, ValueError, "whole groups"), ((x, 0), {}, ValueError, "whole groups"),
            ((x, 2), dict(activation="tanh"), ValueError, "activation"),
            ((x.double(), 2), {}, TypeError, "float64"), ((x.cpu(), 2), {}, ValueError, "cpu"),
            ((x[0, 0, 0], 2), {}, ValueError, "N, ..., C"),
            ((x, 2, w[:7]), {}, ValueError, "weight"), ((x, 2, None, w.cpu()), {}, ValueError, "bias"),
            ((x, 2, w, w.half()), {}, TypeError, "one type"),
            ((x, 2, torch.ones(16, device="cuda")[::2]), {}, ValueError, "contiguous")):
        with pytest.raises(err, match=what):
            K.group_norm(ctx, *args, **kw)
    y, mean, rstd = K.group_norm(ctx, x, 2)
    for gy, m in ((x[:1], mean), (x.half(), mean), (x, mean[:1]), (x, mean.double())):
        with pytest.raises(ValueError):
            K.group_norm_bwd(ctx, gy, x, m, rstd, 2)


@pytest.mark.parametrize("c", [8, 520])
def test_more_items_than_a_launch(ctx, c):
    """Rows past the first launch's last are those of a call on them alone, and count in the
    weight's gradients."""
    from opendressi_amd import ops as K
    n = 2 ** 22 + 5
    gen = torch.Generator(device="cuda").manual_seed(13)
    x = torch.empty((n, c), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    w, b = torch.full((c,), 1.5, device="cuda"), torch.full((c,), 0.5, device="cuda")
    at = torch.tensor([0, 2 ** 22 - 1, 2 ** 22, n - 1], device="cuda")
    y, mean, rstd = K.group_norm(ctx, x, 2, w, b, 1e-5, "silu")
    few = K.group_norm(ctx, x[at], 2, w, b, 1e-5, "silu")
    for p, q in zip((y, mean, rstd), few):
        assert torch.equal(p[at], q)
    del y
    gx, gw, gb = K.group_norm_bwd(ctx, x, x, mean, rstd, 2, w, b, "none")
    want = K.group_norm_bwd(ctx, x[at], x[at], *few[1:], 2, w, b, "none")
    assert torch.equal(gx[at], want[0])
    # sums of gy, of unit variance: 2^22 roundings of sums of a few thousand in float32
    col = sum(p.double().sum(0) for p in x.split(2 ** 19))
    assert ((gb.double() - col).abs() <= 2.0 ** -24 * 2 ** 22).all()


def test_past_32_bits(ctx):
    """An image of more than 2^32 values: its ends and the places around the powers of two, and
    the sums over all of it."""
    from opendressi_amd import ops as K
    n_px, c = 2 ** 29 + 1031, 8
    x = torch.empty((1, n_px, c), dtype=torch.bfloat16, device="cuda")
    step = 2 ** 26
    for i in range(0, n_px, step):
        gen = torch.Generator(device="cuda").manual_seed(i)
        m = min(step, n_px - i)
        x[0, i:i + m] = torch.randn((m, c), generator=gen, device="cuda") + 1
    y, mean, rstd = K.group_norm(ctx, x, 2)
    parts = x[0].view(-1, c).split(step)
    total = sum(p.double().view(-1, 2, 4).sum((0, 2)) for p in parts) / (n_px * 4)
    var = sum((p.double().view(-1, 2, 4) - total[:, None]).square().sum((0, 2))
              for p in parts) / (n_px * 4)
    assert ((mean[0].double() - total).abs() <= 16 * STAT).all()
    assert ((rstd[0].double() * torch.sqrt(var + 1e-5) - 1).abs() <= STAT).all()
    at = torch.tensor([0, 2 ** 28, 2 ** 29 - 1, 2 ** 29, n_px - 1], device="cuda")
    want = (x[0, at].double().view(-1, 2, 4) - total[:, None]) / torch.sqrt(var + 1e-5)[:, None]
    assert torch.allclose(y[0, at].double().view(-1, 2, 4), want, rtol=2.0 ** -8, atol=1e-4)
    del y
    gx, gw, gb = K.group_norm_bwd(ctx, x, x, mean, rstd, 2)  # gy = x: gx is eps' share of x
    assert gx[0, at].isfinite().all() and (gx[0, at].abs() <= 1e-3).all()
    # sum of x, and of x xh = sum of xh^2 / rstd + mean xh
    col = sum(p.double().sum(0) for p in parts)
    assert ((gb.double() - col).abs() <= 2.0 ** -17 * n_px).all()
