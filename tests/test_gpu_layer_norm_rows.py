"""Layer norm over many rows: that each row is in the sums of weight's and bias's gradients once,
rounds of every kernel's loop, and rows past the caches."""
import pytest
import torch

from test_gpu_layer_norm import HALF_ULP, TYPES, U, _check, _inputs, ctx  # noqa: F401

pytestmark = pytest.mark.gpu


def _whole(shape, kind, seed):
    """x and gy of small whole numbers, a weight of powers of two, mean 0 and rstd 1."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda m, *s: torch.randint(-m, m + 1, s, generator=gen, device="cuda",  # noqa: E731
                                       dtype=torch.int8)
    rows, c = shape
    x, gy = draw(3, *shape).to(kind), draw(2, *shape).to(kind)
    w = torch.tensor([0.5, 1.0, 2.0], device="cuda")[draw(1, c).long() + 1]
    return (x, gy, w, torch.zeros(rows, device="cuda"),
            torch.ones(rows, device="cuda"))


def _sums(x, gy):
    """Sums over rows of gy x and gy, in float64, some rows at a time."""
    gw = gb = 0
    for a, b in zip(x.split(1 << 20), gy.split(1 << 20)):
        a, b = a.double(), b.double()
        gw, gb = gw + (a * b).sum(0), gb + b.sum(0)
    return gw, gb


# every backward kernel, each workgroup going round at least twice
@pytest.mark.parametrize("shape", [(1200001, 1), (1200001, 3), (1200003, 5), (700001, 8),
                                   (400001, 12), (300003, 33), (150001, 64), (100003, 130),
                                   (100003, 200), (70001, 264), (70001, 300), (40001, 512),
                                   (40001, 520), (20001, 1030), (9001, 1500), (9001, 2056),
                                   (3001, 4100), (2001, 9000), (1101, 16384), (1501, 20001),
                                   (701, 50001)], ids=str)
@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_each_row_counts_once(ctx, shape, kind):  # noqa: F811
    """With the mean 0, the deviation 1 and no activation, gb and gw are sums of whole numbers, of
    which float32 holds every partial one (2^21 rows of at most 6): equal, or a row is missing or
    there twice. gx = w gy - A - x B, A and B the row's means of w gy and w gy x: their sums are
    whole halves (32 bits hold them too), and each is rounded twice, by 1 / C and as a product; so
    are the differences."""
    from opendressi_amd import ops as K
    print(f"[layer_norm sums] {shape} {kind}", flush=True)
    x, gy, w, mean, rstd = _whole(shape, kind, 60)
    gx, gw, gb = K.layer_norm_bwd(ctx, gy, x, mean, rstd, w)
    torch.cuda.synchronize()
    want_w, want_b = _sums(x, gy)
    assert torch.equal(gb.double(), want_b) and torch.equal(gw.double(), want_w)
    for got, a, b in zip(gx.split(1 << 18), x.split(1 << 18), gy.split(1 << 18)):
        a, t = a.double(), b.double() * w.double()
        ma, mb = t.mean(1, keepdim=True), (t * a).mean(1, keepdim=True)
        want = t - ma - a * mb
        tol = 4 * U * (t.abs() + ma.abs() + (a * mb).abs()) + HALF_ULP[kind] * want.abs() + 2.0 ** -25
        assert ((got.double() - want).abs() <= tol).all()


# rows past a wave: more of them than workgroups in a launch
@pytest.mark.parametrize("shape", [(6001, 2056), (6001, 4100), (1301, 8193), (1101, 16384),
                                   (1101, 20001), (1101, 32768), (1001, 40000), (701, 50001)],
                         ids=str)
@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_rounds_of_long_rows(ctx, shape, kind):  # noqa: F811
    from opendressi_amd import ops as K
    print(f"[layer_norm rounds] {shape} {kind}", flush=True)
    x, gy, w, b = _inputs(shape, kind, 61)
    y, mean, rstd = K.layer_norm(ctx, x, w, b, 1e-5, "silu")
    grads = K.layer_norm_bwd(ctx, gy, x, mean, rstd, w, b, "silu")
    torch.cuda.synchronize()
    for part in torch.arange(shape[0], device="cuda").split(512):
        part = slice(int(part[0]), int(part[-1]) + 1)
        _check(x[part], gy[part], w, b, 1e-5, "silu", (y[part], mean[part], rstd[part],
                                                       None, None, None))
    _check(x, gy, w, b, 1e-5, "silu", (y, mean, rstd, *grads))


# x past 256 MB in 16 bits, and more rows than a launch's workgroups take at once
LARGE = [(134300003, 1), (45000001, 3), (16800009, 8), (4200003, 33), (2100005, 64), (1050001, 130),
         (700001, 200), (600001, 264), (270001, 512), (260001, 520), (135001, 1030), (95001, 1500),
         (70001, 2056), (30001, 5001), (9001, 16384), (5001, 32768), (3501, 40000)]
PIECE = 1 << 22  # elements: 16 MB at most, well within the caches


@pytest.mark.parametrize("shape", LARGE, ids=str)
@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_past_the_caches(ctx, shape, kind):  # noqa: F811
    """Reads and writes of large calls go past the caches: the bits of the same rows in pieces
    that go through them, and exact sums of all rows (sums of n whole numbers of either sign up to
    6 stay below 6 sqrt(40 n) < 2^19, but for a chance of exp(-20))."""
    from opendressi_amd import ops as K
    print(f"[layer_norm large] {shape} {kind}", flush=True)
    rows, c = shape
    gen = torch.Generator(device="cuda").manual_seed(62)
    x = torch.empty(shape, dtype=kind, device="cuda").normal_(generator=gen)
    w = 1 + 0.2 * torch.randn(c, generator=gen, device="cuda")
    b = 0.3 * torch.randn(c, generator=gen, device="cuda")
    step = max(1, PIECE // c)
    y, mean, rstd = K.layer_norm(ctx, x, w, b, 1e-5, "gelu")
    short = K.layer_norm(ctx, x, w, b, 1e-5, "gelu", stats=False)[0]
    torch.cuda.synchronize()
    assert torch.equal(y, short)
    del short
    for i in range(0, rows, step):
        part = slice(i, min(i + step, rows))
        for p, q in zip((y, mean, rstd), K.layer_norm(ctx, x[part], w, b, 1e-5, "gelu")):
            assert torch.equal(p[part], q), i
    del x, y
    x, gy, w, mean, rstd = _whole(shape, kind, 63)
    gx, gw, gb = K.layer_norm_bwd(ctx, gy, x, mean, rstd, w)
    torch.cuda.synchronize()
    want_w, want_b = _sums(x, gy)
    assert torch.equal(gb.double(), want_b) and torch.equal(gw.double(), want_w)
    for i in range(0, rows, step):
        part = slice(i, min(i + step, rows))
        got = K.layer_norm_bwd(ctx, gy[part], x[part], mean[part], rstd[part], w,
                               need=(True, False, False))[0]
        assert torch.equal(gx[part], got), i
