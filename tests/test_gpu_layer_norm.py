"""Layer norm with an activation (opendressi_amd.ops.layer_norm, layer_norm_bwd, and
opendressi_amd.torch.layer_norm) against float64, formula and differences."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = {"none": lambda z: z, "relu": torch.relu, "silu": lambda z: z * torch.sigmoid(z),
        "gelu": lambda z: z * torch.special.ndtr(z)}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in TYPES}
U = 2.0 ** -24  # half a step of float32


@pytest.fixture(scope="module")
def ctx():
    import opendressi_amd as od
    c = od.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def vctx():
    import opendressi_amd.torch as dr
    return dr.RasterizeHipContext(0)


def _inputs(shape, kind, seed, offset=0.0, affine=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    c = shape[-1]
    x = (r(*shape) * (0.5 + torch.rand(c, generator=gen, device="cuda")) + r(c) + offset).to(kind)
    return x, r(*shape).to(kind), (1 + 0.2 * r(c)).to(affine), (0.3 * r(c)).to(affine)


def _run(ctx, x, gy, weight, bias, eps, act):
    from opendressi_amd import ops as K
    y, mean, rstd = K.layer_norm(ctx, x, weight, bias, eps, act)
    need = (True, weight is not None, bias is not None)
    gx, gw, gb = K.layer_norm_bwd(ctx, gy, x, mean, rstd, weight, bias, act, need)
    torch.cuda.synchronize()
    return y, mean, rstd, gx, gw, gb


def _check(x, gy, weight, bias, eps, act, got):
    """Outputs against float64 within what the roundings allow.

    Row sums are added by up to 64 terms in a lane, then in halves: 96 roundings of the row's
    largest |x| for the mean (64 of the sum, the rest for the second sum and the mean itself), as
    many of the relative deviation, to which the mean's error adds its square. 8 roundings of the
    arithmetic of z, 2^-20 of the activation's exp or erf, and the output's own half step follow.
    Sums over n rows: sequences of up to 2^11 rows and levels above them, whose roundings add up as
    a random walk does, twice over."""
    y, mean, rstd, gx, gw, gb = got
    c = x.shape[-1]
    xd, g = x.reshape(-1, c).double(), gy.reshape(-1, c).double()
    w = torch.ones(c, device="cuda", dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    em = xd.mean(1, keepdim=True)
    er = (((xd - em) ** 2).mean(1, keepdim=True) + eps) ** -0.5
    xh = (xd - em) * er
    z = (xh * w + b).requires_grad_()
    ey = ACTS[act](z)
    gz = torch.autograd.grad(ey, z, g)[0]
    z, ey = z.detach(), ey.detach()
    big = xd.abs().amax(1, keepdim=True)
    d_mean = 96 * U * big
    d_rstd = 96 * U + (d_mean * er) ** 2
    flat = lambda t: t.reshape(-1, 1).double()  # noqa: E731
    assert mean.shape == x.shape[:-1] and rstd.shape == x.shape[:-1]
    assert ((flat(mean) - em).abs() <= d_mean + 1e-30).all()
    assert ((flat(rstd) / er - 1).abs() <= d_rstd).all()
    d_xh = xh.abs() * d_rstd + d_mean * er + 4 * U * (xh.abs() + big * er)
    dz = w.abs() * d_xh + 8 * U * ((w * xh).abs() + z.abs())
    half = HALF_ULP[x.dtype]
    tol = 1.2 * dz + 2.0 ** -20 * z.abs() + half * ey.abs() + 2.0 ** -25
    err = (y.reshape(-1, c).double() - ey).abs()
    assert y.dtype == x.dtype and (err <= tol).all(), float((err / tol).max())
    if gx is None:
        return
    # slopes change by at most 1.2 of dz, relu's by 1 where z is within dz of its kink
    ds = {"none": torch.zeros_like(dz), "relu": (z.abs() <= dz).double()}.get(
        act, 1.2 * dz + 2.0 ** -19)
    size = 1.2 * g.abs()
    dgz = g.abs() * ds + 8 * U * size
    length = U * 2 * (math.sqrt(min(len(xd), 2 ** 11)) + 24)
    for got_p, p, term, d_term in ((gb, bias, gz, dgz),
                                   (gw, weight, gz * xh, dgz * xh.abs() + size * d_xh)):
        if p is None:
            assert got_p is None
            continue
        want = term.sum(0)
        tp = d_term.sum(0) + length * term.abs().sum(0) + HALF_ULP[p.dtype] * want.abs() + 1e-30
        err = (got_p.double() - want).abs()
        assert got_p.dtype == p.dtype and (err <= tp).all(), float((err / tp).max())
    # gx = rstd (w gz - A - xh B), A and B the row's means of w gz and w gz xh
    mean1 = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    egx = er * (w * gz - mean1(w * gz) - xh * mean1(w * gz * xh))
    wa, wsize = w.abs(), w.abs() * size
    d_a = mean1(wa * dgz) + 96 * U * mean1(wsize)
    d_b = mean1(wa * (dgz * xh.abs() + size * d_xh)) + 96 * U * mean1(wsize * xh.abs())
    parts = wsize + mean1(wsize) + xh.abs() * mean1(wsize * xh.abs())
    tx = er * (wa * dgz + d_a + xh.abs() * d_b + d_xh * mean1(wsize * xh.abs())
               + parts * (d_rstd + 8 * U)) + half * egx.abs() + 2.0 ** -25
    err = (gx.reshape(-1, c).double() - egx).abs()
    assert gx.dtype == x.dtype and (err <= tx).all(), float((err / tx).max())


# widths about every size at which a row's lanes, vectors or workgroups change, and few or many rows
SHAPES = [(5, 1), (300, 1), (4, 2), (1001, 3), (7, 4), (2, 5), (333, 7), (1, 8), (40, 9), (3, 12),
          (17, 16), (5000, 17), (2, 24), (61, 97, 33), (129, 63), (3, 7, 5, 64), (1, 65), (700, 66),
          (12, 100), (9, 127), (64, 128), (5, 129), (77, 250), (1, 256), (31, 257), (6, 511),
          (2000, 512), (4, 513), (3, 1000), (10, 1023), (257, 1024), (2, 1025), (5, 1032),
          (3, 2047), (33, 2048), (2, 2049), (1021, 2056), (4, 4095), (19, 4096), (1, 4097),
          (3, 5001), (2, 8192), (300, 8193), (5, 12288), (1, 16384), (3, 16385), (2, 20000),
          (1, 32768), (4, 32769), (2, 50001), (3, 65536), (1, 262147)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_against_float64(ctx, shape, kind):
    for act in ("silu", "none"):
        print(f"[layer_norm] {shape} {kind} {act}", flush=True)
        x, gy, w, b = _inputs(shape, kind, 1)
        _check(x, gy, w, b, 1e-5, act, _run(ctx, x, gy, w, b, 1e-5, act))


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(50, 41), (3, 30, 31, 64), (77, 600), (5, 3001), (3, 40000)],
                         ids=str)
def test_activations(ctx, shape, kind, act):
    print(f"[layer_norm act] {shape} {kind} {act}", flush=True)
    x, gy, w, b = _inputs(shape, kind, 2)
    _check(x, gy, w, b, 1e-5, act, _run(ctx, x, gy, w, b, 1e-5, act))


@pytest.mark.parametrize("shape", [(150001, 8), (70001, 33), (100003, 64), (30011, 200),
                                   (20011, 520), (9001, 1500), (3001, 4100), (520, 20001)], ids=str)
@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_many_rows(ctx, shape, kind):
    """More rows than workgroups take at once: each goes round several times."""
    print(f"[layer_norm rows] {shape} {kind}", flush=True)
    x, gy, w, b = _inputs(shape, kind, 3)
    _check(x, gy, w, b, 1e-5, "silu", _run(ctx, x, gy, w, b, 1e-5, "silu"))


@pytest.mark.parametrize("offset", [0.0, 300.0, -3e4])
@pytest.mark.parametrize("shape", [(64, 65, 32), (30, 5), (7, 3000), (2, 40000)], ids=str)
def test_far_from_zero(ctx, shape, offset):
    """A mean many deviations from zero costs what float32 holds of the mean, no more."""
    x, gy, w, b = _inputs(shape, torch.float32, 4, offset)
    _check(x, gy, w, b, 1e-5, "none", _run(ctx, x, gy, w, b, 1e-5, "none"))


@pytest.mark.parametrize("c", [64, 1000, 40000])
def test_one_value_far_from_the_rest(ctx, c):
    for at in (0, c // 3, c - 1):
        x, gy, w, b = _inputs((9, c), torch.float32, 5)
        x[:, at] = 1e4
        _check(x, gy, w, b, 1e-5, "none", _run(ctx, x, gy, w, b, 1e-5, "none"))


@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("affine", TYPES, ids=str)
def test_affine_types(ctx, kind, affine):
    for shape in ((20, 21, 48), (40, 2051), (3, 33000)):
        x, gy, w, b = _inputs(shape, kind, 6, affine=affine)
        for weight, bias in ((w, b), (w, None), (None, b), (None, None)):
            _check(x, gy, weight, bias, 1e-3, "silu", _run(ctx, x, gy, weight, bias, 1e-3, "silu"))


def test_weight_and_bias_at_any_address(ctx):
    """Weight, bias and rows that begin anywhere their type may."""
    for kind in TYPES:
        for c in (33, 64, 1031, 8192):
            buf, gbuf, w, b = _inputs((40, c + 3), kind, 7, affine=kind)
            w, b = w[1:c + 1], b[3:c + 3]
            flat, gflat = buf.view(-1), gbuf.view(-1)
            for first in (1, 3):
                x, gy = (t[first:first + 39 * c].view(39, c) for t in (flat, gflat))
                _check(x, gy, w, b, 1e-5, "gelu", _run(ctx, x, gy, w, b, 1e-5, "gelu"))


def test_constant_rows(ctx):
    """A row without variance: xh = 0, y = act(b), no gradient but through b."""
    from opendressi_amd import ops as K
    x = torch.full((2, 16, 16, 8), 3.25, device="cuda")
    w, b = torch.ones(8, device="cuda"), torch.arange(8.0, device="cuda") - 4
    y, mean, rstd = K.layer_norm(ctx, x, w, b, 1e-5, "relu")
    assert torch.equal(y, torch.relu(b).expand_as(x)) and (mean == 3.25).all()
    assert torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5), rtol=1e-6)
    gx, gw, gb = K.layer_norm_bwd(ctx, torch.ones_like(x), x, mean, rstd, w, b, "none")
    assert not gw.any() and (gb == 512).all() and (gx.abs() <= 1e-3).all()


def test_single_channels(ctx):
    """Rows of one value: y = act(b), gx zero."""
    from opendressi_amd import ops as K
    for kind in TYPES:
        x, gy, w, b = _inputs((1000, 1), kind, 8, affine=kind)
        y, mean, rstd = K.layer_norm(ctx, x, w, b)
        assert torch.equal(y, b.expand_as(y)) and torch.equal(mean, x[:, 0].float())
        gx, gw, gb = K.layer_norm_bwd(ctx, gy, x, mean, rstd, w, b)
        assert not gx.any() and not gw.any()


@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_strides(ctx, kind):
    """Channel, item and pixel slices of wider images, crops, transposed and expanded ones: the
    bits of the packed image."""
    from opendressi_amd import ops as K
    wide, gy, w, b = _inputs((4, 24, 20, 48), kind, 9)
    w, b = w[:16].contiguous(), b[:16].contiguous()
    for x in (wide[..., 16:32], wide[..., 3:19], wide[::2, :, :, 8:24], wide[:, 2:9, 4:17, :16],
              wide[..., :16].transpose(1, 2), wide[:1, ..., :16].expand(3, -1, -1, -1),
              wide[:, :1, :, 32:], wide.permute(0, 3, 1, 2)[..., 4:20], wide[:, 3, 5, 7:23],
              wide[0, 0, 0, :16], wide[..., 0, :16].expand(2, 4, 24, 16), wide[:, :, ::3, 1:17]):
        g = torch.randn(x.shape, device="cuda").to(kind)
        packed = x.contiguous()
        want = K.layer_norm(ctx, packed, w, b, 1e-5, "silu")
        got = K.layer_norm(ctx, x, w, b, 1e-5, "silu")
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        assert torch.equal(got[0], K.layer_norm(ctx, x, w, b, 1e-5, "silu", stats=False)[0])
        want = K.layer_norm_bwd(ctx, g, packed, *want[1:], w, b, "silu")
        got = K.layer_norm_bwd(ctx, g, x, *got[1:], w, b, "silu")
        assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_crops_and_far_pixels(ctx, kind):
    """Many rows that are not evenly spaced, and rows more than 2^22 elements apart: the packed
    rows' bits."""
    from opendressi_amd import ops as K
    wide, _, w, b = _inputs((3, 301, 203, 40), kind, 31)
    far = torch.randn(2 ** 23 + 5000, device="cuda").to(kind)
    for x in (wide[:, 5:300, 7:200, 3:36], wide[1:, ::2, :, :33],
              far.as_strided((2, 33), (2 ** 22 + 77, 1)),
              far.as_strided((2, 4, 33), (50, 2 ** 21 + 3, 1))):
        g = torch.randn(x.shape, device="cuda").to(kind)
        packed, args = x.contiguous(), (w[:33].contiguous(), b[:33].contiguous())
        want = K.layer_norm(ctx, packed, *args, 1e-5, "gelu")
        got = K.layer_norm(ctx, x, *args, 1e-5, "gelu")
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        want = K.layer_norm_bwd(ctx, g, packed, *want[1:], *args, "gelu")
        got = K.layer_norm_bwd(ctx, g, x, *got[1:], *args, "gelu")
        assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.parametrize("shape", [(7, 256), (5, 512), (9, 768), (300, 1536), (600, 3000),
                                   (513, 640), (2, 10240)], ids=str)
@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_whole_waves(ctx, shape, kind):
    print(f"[layer_norm whole] {shape} {kind}", flush=True)
    x, gy, w, b = _inputs(shape, kind, 32)
    _check(x, gy, w, b, 1e-5, "gelu", _run(ctx, x, gy, w, b, 1e-5, "gelu"))


@pytest.mark.parametrize("c", [16, 33, 1100, 20000, 40000])
def test_only_what_is_wanted(ctx, c):
    """Each gradient alone has the bits that it has beside the others; two runs have the same."""
    from opendressi_amd import ops as K
    x, gy, w, b = _inputs((1500 if c < 20000 else 30, c), torch.bfloat16, 10)
    _, mean, rstd = K.layer_norm(ctx, x, w, b, 1e-5, "gelu")
    both = K.layer_norm_bwd(ctx, gy, x, mean, rstd, w, b, "gelu")
    for k in range(8):
        need = tuple(bool(k >> i & 1) for i in range(3))
        got = K.layer_norm_bwd(ctx, gy, x, mean, rstd, w, b, "gelu", need)
        for wanted, p, q in zip(need, both, got):
            assert (q is None) if not wanted else torch.equal(p, q)


def test_empty(ctx):
    from opendressi_amd import ops as K
    w, b = torch.ones(8, device="cuda"), torch.zeros(8, device="cuda")
    for shape in ((0, 4, 4, 8), (2, 0, 4, 8), (0, 8)):
        x = torch.empty(shape, device="cuda")
        y, mean, rstd = K.layer_norm(ctx, x, w, b)
        assert y.shape == x.shape and mean.shape == rstd.shape == shape[:-1]
        gx, gw, gb = K.layer_norm_bwd(ctx, x, x, mean, rstd, w, b)
        assert gx.shape == x.shape and not gw.any() and not gb.any()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("c", [16, 33, 700, 3000, 40000])
def test_not_finite_stays_in_its_row(ctx, bad, c):
    from opendressi_amd import ops as K
    x, gy, w, b = _inputs((300 if c < 40000 else 4, c), torch.float32, 11)
    y0, mean, rstd = K.layer_norm(ctx, x, w, b, 1e-5, "silu")
    want = K.layer_norm_bwd(ctx, gy, x, mean, rstd, w, b, "silu")
    x[2, c // 2] = bad
    y, mean, rstd = K.layer_norm(ctx, x, w, b, 1e-5, "silu")
    gx, gw, _ = K.layer_norm_bwd(ctx, gy, x, mean, rstd, w, b, "silu")
    rest = torch.arange(len(x), device="cuda") != 2
    assert y[2].isnan().all() and torch.equal(y[rest], y0[rest])
    assert gx[2].isnan().all() and torch.equal(gx[rest], want[0][rest])
    assert gw.isnan().all()


@pytest.mark.parametrize("c", [64, 33, 3000])
def test_masked_gradients_stay_out(ctx, c):
    """relu's mask takes an infinite or NaN gradient out, by the sign that the forward pass gave."""
    from opendressi_amd import ops as K
    x, gy, w, b = _inputs((200, c), torch.float32, 12)
    y, mean, rstd = K.layer_norm(ctx, x, w, b, 1e-5, "relu")
    want = K.layer_norm_bwd(ctx, gy * (y > 0), x, mean, rstd, w, b, "relu")
    gy[y <= 0] = math.nan
    got = K.layer_norm_bwd(ctx, gy, x, mean, rstd, w, b, "relu")
    assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
@pytest.mark.parametrize("shape", [(9, 11, 12), (5, 700)], ids=str)
def test_gradient_against_differences(vctx, act, shape):
    """<gradient, d> against the operator's own central differences along random directions. The
    third derivative's term is below h^2, the forward's rounding adds 2^-22 of sqrt(values) / h."""
    import opendressi_amd.torch as dr
    x, gy, w, b = _inputs(shape, torch.float32, 13)
    gy = gy.double()
    loss = lambda *t: float((dr.layer_norm(vctx, *t, activation=act).double() * gy).sum())  # noqa: E731
    args = [t.clone().requires_grad_() for t in (x, w, b)]
    dr.layer_norm(vctx, *args, activation=act).backward(gy.float())
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


def test_torch_surface(ctx, vctx):
    """Through autograd, with and without the gradients that are not asked for, without any, from
    host tensors; a second derivative is refused."""
    import opendressi_amd.torch as dr
    x, gy, w, b = _inputs((8, 8, 16), torch.float32, 14)
    want = _run(ctx, x, gy, w, b, 1e-5, "silu")
    for k in range(8):
        t = [v.clone().requires_grad_(bool(k >> i & 1)) for i, v in enumerate((x, w, b))]
        y = dr.layer_norm(vctx, *t, activation="silu")
        assert torch.equal(y, want[0]) and y.requires_grad == (k > 0)
        if k:
            y.backward(gy)
        for v, g in zip(t, want[3:]):
            assert torch.equal(v.grad, g) if v.requires_grad else v.grad is None
    with torch.no_grad():
        y = dr.layer_norm(vctx, x.requires_grad_(), w, b, activation="silu")
    assert torch.equal(y, want[0]) and not y.requires_grad
    host = [v.detach().cpu().requires_grad_() for v in (x, w, b)]
    y = dr.layer_norm(vctx, *host, activation="silu")
    assert y.device.type == "cpu" and torch.equal(y, want[0].cpu())
    y.backward(gy.cpu())
    assert all(torch.equal(v.grad, g.cpu()) for v, g in zip(host, want[3:]))
    assert torch.equal(dr.layer_norm(vctx, host[0].detach()).cpu(),
                       dr.layer_norm(vctx, x.detach()).cpu())
    # an expanded gradient, a weight that is a slice of a table
    table = torch.randn(16, 3, device="cuda")
    dr.layer_norm(vctx, x, table[:, 1], None).sum().backward()
    y = dr.layer_norm(vctx, x, w, b, activation="silu")
    g, = torch.autograd.grad(y, x, gy, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_streams_and_threads(vctx):
    """Calls on two streams, from two threads: each has the result that it has alone."""
    import threading

    import opendressi_amd.torch as dr
    cases = [_inputs((20000, c), torch.float32, c) for c in (64, 100)]
    want = []
    for x, gy, w, b in cases:
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = dr.layer_norm(vctx, *leaves, activation="gelu")
        want.append((y.detach(), *torch.autograd.grad(y, leaves, gy)))
    torch.cuda.synchronize()
    out, streams = [None, None], [torch.cuda.Stream(), torch.cuda.Stream()]

    def work(k):
        x, gy, w, b = cases[k]
        with torch.cuda.stream(streams[k]):
            for _ in range(5):
                leaves = [t.clone().requires_grad_() for t in (x, w, b)]
                y = dr.layer_norm(vctx, *leaves, activation="gelu")
                out[k] = (y.detach(), *torch.autograd.grad(y, leaves, gy))

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for a, e in zip(out, want):
        assert all(torch.equal(p, q) for p, q in zip(a, e))


@pytest.mark.parametrize("c", [64, 33, 4096, 40000])
def test_captured(ctx, c):
    """Two graphs of forward and backward, replayed in turn over new inputs with eager work
    between them: the eager bits each time."""
    from opendressi_amd import ops as K
    rows = 3000 if c < 100 else 40
    sets, graphs, outs = [], [], []
    s = torch.cuda.Stream()
    for k in range(2):
        x, gy, w, b = _inputs((rows, c), torch.bfloat16, 20 + k)
        sets.append((x, gy, w, b))
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _run(ctx, x, gy, w, b, 1e-5, "silu")
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y, mean, rstd = K.layer_norm(ctx, x, w, b, 1e-5, "silu")
            outs.append((y, *K.layer_norm_bwd(ctx, gy, x, mean, rstd, w, b, "silu")))
        graphs.append(g)
    for r in range(4):
        for k in range(2):
            x, gy, w, b = sets[k]
            new = _inputs((rows, c), torch.bfloat16, 100 + 10 * r + k)
            for t, v in zip((x, gy), new):
                t.copy_(v)
            graphs[k].replay()
            eager = _run(ctx, new[0], new[1], w, b, 1e-5, "silu")
            torch.cuda.synchronize()
            for p, q in zip(outs[k], (eager[0], *eager[3:])):
                assert torch.equal(p, q)


def test_captured_through_autograd(vctx):
    """Forward and gradients of the torch surface in one graph, replayed over new values with eager
    calls on other leaves between them."""
    import opendressi_amd.torch as dr

    def step(leaves, gy):
        return torch.autograd.grad(dr.layer_norm(vctx, *leaves, activation="silu"), leaves, gy)

    x, gy, w, b = _inputs((4000, 48), torch.float32, 40)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(leaves, gy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step(leaves, gy)
    for r in range(3):
        new = _inputs((4000, 48), torch.float32, 41 + r)
        with torch.no_grad():
            for t, v in zip((x, gy, w, b), new):
                t.copy_(v)
        graph.replay()
        eager = step([t.clone().requires_grad_() for t in (new[0], *new[2:])], new[1])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager))


def test_past_32_bits(ctx):
    """Rows whose elements lie past 2^32: those there are as good as the first, and the sums of
    the last rows are in the gradients of weight and bias."""
    from opendressi_amd import ops as K
    rows, c = 2 ** 27 + 37, 33
    x = torch.zeros((rows, c), dtype=torch.float16, device="cuda")
    gy = torch.zeros_like(x)
    tail, gtail, w, b = _inputs((41, c), torch.float16, 30)
    at = torch.tensor([*range(20), *range(rows - 21, rows)], device="cuda")
    x[at], gy[at] = tail, gtail
    y, mean, rstd = K.layer_norm(ctx, x, w, b, 1e-5, "silu")
    gx, gw, gb = K.layer_norm_bwd(ctx, gy, x, mean, rstd, w, b, "silu")
    torch.cuda.synchronize()
    _check(tail, gtail, w, b, 1e-5, "silu", (y[at], mean[at], rstd[at], gx[at], gw, gb))
    assert not gx[20:rows - 21].any()


@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1001, 1), (777, 3), (5000, 33), (1301, 64), (700, 1000),
                                   (300, 2051), (41, 8193), (30, 16384), (5, 16392), (9, 20001),
                                   (7, 32768), (5, 40000)], ids=str)
def test_in_place(ctx, kind, shape):
    """Through the C interface, y over x and gx over gy or x: the bits that they have apart, or
    refused where another lane may have written what one reads."""
    import opendressi_amd as od
    from opendressi_amd import _lib as L
    from opendressi_amd import ops as K
    x, gy, w, b = _inputs(shape, kind, 50)
    rows, c = shape
    code, vec = TYPES.index(kind), 4 if kind == torch.float32 else 8
    y, mean, rstd = K.layer_norm(ctx, x, w, b, 1e-5, "silu")
    gx, gw, gb = K.layer_norm_bwd(ctx, gy, x, mean, rstd, w, b, "silu")
    scratch = torch.empty(max(L.lib.dressi_layer_norm_scratch(code, 1, rows, c, k) for k in (0, 1)),
                          dtype=torch.uint8, device="cuda")
    size = scratch.numel()
    ctx.use_torch_stream()

    def forward(x):
        L.check(L.lib.dressi_layer_norm(
            ctx.handle, x.data_ptr(), code, 1, rows, c, 0, c, w.data_ptr(), b.data_ptr(), 0, 1e-5,
            L.ACT_SILU, scratch.data_ptr(), size, x.data_ptr(), None, None))
        return x

    def backward(gy, x, gx):
        L.check(L.lib.dressi_layer_norm_bwd(
            ctx.handle, gy.data_ptr(), x.data_ptr(), code, 1, rows, c, 0, c, w.data_ptr(),
            b.data_ptr(), 0, L.ACT_SILU, mean.data_ptr(), rstd.data_ptr(), scratch.data_ptr(), size,
            gx.data_ptr(), got_w.data_ptr(), got_b.data_ptr()))
        return gx

    if c <= 32768 or c % vec == 0:
        assert torch.equal(forward(x.clone()), y)
    else:
        with pytest.raises(od.DressiError, match="overlap"):
            forward(x.clone())
    for over in (0, 1):
        args, (got_w, got_b) = [gy.clone(), x.clone()], (torch.empty_like(w) for _ in range(2))
        if c <= 16384 or c % vec == 0:
            assert torch.equal(backward(*args, args[over]), gx)
            assert torch.equal(got_w, gw) and torch.equal(got_b, gb)
        else:
            with pytest.raises(od.DressiError, match="overlap"):
                backward(*args, args[over])


def test_refusals(ctx, vctx):
    import opendressi_amd as od
    import opendressi_amd.torch as dr
    from opendressi_amd import ops as K
    x, gy, w, b = _inputs((4, 16), torch.float32, 15)
    y, mean, rstd = K.layer_norm(ctx, x, w, b)
    for bad, error in ((lambda: K.layer_norm(ctx, x.double(), w, b), TypeError),
                       (lambda: K.layer_norm(ctx, x, w.half(), b), TypeError),
                       (lambda: K.layer_norm(ctx, x, w[:8], b), ValueError),
                       (lambda: K.layer_norm(ctx, x.cpu(), w, b), ValueError),
                       (lambda: K.layer_norm(ctx, x, w, b, activation="tanh"), ValueError),
                       (lambda: K.layer_norm(ctx, x, w, b, eps=-1.0), od.DressiError),
                       (lambda: K.layer_norm(ctx, x, w, b, eps=math.nan), od.DressiError),
                       (lambda: K.layer_norm(ctx, x[0, 0], None, None), ValueError),
                       (lambda: K.layer_norm(ctx, x[:, :0], None, None), ValueError),
                       (lambda: K.layer_norm_bwd(ctx, gy[:2], x, mean, rstd, w, b), ValueError),
                       (lambda: K.layer_norm_bwd(ctx, gy.half(), x, mean, rstd, w, b), ValueError),
                       (lambda: K.layer_norm_bwd(ctx, gy, x, mean[:2], rstd, w, b), ValueError),
                       (lambda: K.layer_norm_bwd(ctx, gy, x, mean, rstd.double(), w, b), ValueError),
                       (lambda: dr.layer_norm(vctx, [1.0, 2.0], w, b), TypeError),
                       (lambda: dr.layer_norm(vctx, x, 1.0), TypeError)):
        with pytest.raises(error):
            bad()
