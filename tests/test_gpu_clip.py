"""The norm of many gradients and clipping to it (opendressi_amd.torch.grad_norm, clip_grad_norm_)
against float64."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # half a step of float32


@pytest.fixture(scope="module")
def vctx():
    import opendressi_amd.torch as dr
    return dr.RasterizeHipContext(0)


def _params(sizes, kinds, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, s in enumerate(sizes):
        s = s if isinstance(s, tuple) else (s,)
        kind = kinds[i % len(kinds)]
        p = torch.zeros(s, dtype=kind, device="cuda")
        p.grad = (scale * torch.randn(s, generator=gen, device="cuda")).to(kind)
        out.append(p)
    return out


def _norm(grads, norm_type):
    flat = torch.cat([g.double().reshape(-1) for g in grads]) if grads else torch.zeros(1)
    if flat.numel() == 0:
        return 0.0
    return float(flat.abs().max()) if norm_type == math.inf else float(flat.square().sum().sqrt())


def _check(before, after, norm, max_norm, norm_type):
    """The norm is float64's, rounded once (the float64 sums err by 2^-53 a term at most); the
    factor is rounded once and so is its product: two half steps of float32, then the half step of
    the gradient's type (below a type's normal values, of its smallest)."""
    want = _norm(before, norm_type)
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(float(norm) - want) <= want * U * (1 + 2.0 ** -10)
    factor = min(1.0, max_norm / (want + 1e-6))
    for g, q in zip(before, after):
        exact = g.double() * factor
        if factor == 1.0:
            assert torch.equal(g, q)
            continue
        f = torch.finfo(g.dtype)
        tol = exact.abs() * (2.01 * U + (f.eps / 2 if g.dtype != torch.float32 else 0.0)) \
            + f.tiny * f.eps
        assert ((q.double() - exact).abs() <= tol).all()


SIZES = [[1], [3], [0], [1, 0, 5], [255], [1024, 1], [4095, 4096, 4097], [16383], [16384], [16385],
         [(642, 3), 1, 3], [(97, 61), 97, 33, 1, 31, (65, 33), (3, 65), 3, 12289], [1] * 63,
         [7] * 64, [5] * 65, [1000] * 127, [3] * 128, [9] * 129, list(range(1, 300)),
         [300001, 5, 70000], [2 ** 20 + 1], [1 << 22, 3, 1 << 21]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("kinds", [[t] for t in TYPES] + [TYPES], ids=str)
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_against_float64(vctx, sizes, kinds, norm_type):
    import opendressi_amd.torch as dr
    print(f"[clip] {len(sizes)} x {sizes[0]} {kinds} {norm_type}", flush=True)
    for share in (0.3, 0.99, 1.5):
        params = _params(sizes, kinds, 1)
        before = [p.grad.clone() for p in params]
        limit = share * _norm(before, norm_type)
        only = dr.grad_norm(vctx, params, norm_type)
        assert all(torch.equal(p.grad, g) for p, g in zip(params, before))
        norm = dr.clip_grad_norm_(vctx, params, limit, norm_type)
        torch.cuda.synchronize()
        assert torch.equal(only, norm)
        _check(before, [p.grad for p in params], norm, limit, norm_type)


@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_large(vctx, kind):
    """Tensors of which a cache holds a part, with odd tails."""
    import opendressi_amd.torch as dr
    params = _params([2 ** 27 + 3, 77, 2 ** 25 + 1], [kind], 2)
    before = [p.grad.clone() for p in params]
    norm = dr.clip_grad_norm_(vctx, params, 100.0)
    torch.cuda.synchronize()
    _check(before, [p.grad for p in params], norm, 100.0, 2.0)


def test_past_32_bits(vctx):
    """A tensor of more than 2^32 elements: its last ones count and are scaled."""
    import opendressi_amd.torch as dr
    n = 2 ** 32 + 5001
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros_like(p)
    at = torch.tensor([0, 2 ** 31, 2 ** 32 - 1, 2 ** 32, n - 1], device="cuda")
    g[at] = torch.tensor([3.0, 4.0, 12.0, 84.0, 132.0], dtype=torch.bfloat16, device="cuda")
    p.grad = g
    norm = dr.clip_grad_norm_(vctx, [p], 157.0 / 2)  # 3, 4, 12, 84 and 132 make 157
    assert float(norm) == 157.0
    # 157 / 2 / (157 + 1e-6) is a half but for 3e-9 of it, which bfloat16 does not see
    assert g[at].tolist() == [1.5, 2.0, 6.0, 42.0, 66.0]
    assert float(dr.clip_grad_norm_(vctx, [p], 1.0, math.inf)) == 66.0
    assert float(g[n - 1]) == 1.0 and int((g != 0).sum()) == 5


def test_any_address(vctx):
    """Gradients that begin anywhere their type may; what lies about them stays."""
    import opendressi_amd.torch as dr
    for kind in TYPES:
        for n in (1, 7, 8, 61, 5000, 40001):
            for first in range(9):
                buf = torch.randn(n + 20, device="cuda").to(kind)
                p = torch.zeros(n, dtype=kind, device="cuda")
                p.grad = buf[first:first + n]
                kept, before = buf.clone(), p.grad.clone()
                norm = dr.clip_grad_norm_(vctx, [p], 0.5 * _norm([before], 2.0))
                _check([before], [p.grad], norm, 0.5 * _norm([before], 2.0), 2.0)
                kept[first:first + n] = p.grad
                assert torch.equal(kept, buf)


def test_layouts(vctx):
    """Transposed, channels-last and sliced gradients, a scalar, None, one tensor, a generator."""
    import opendressi_amd.torch as dr
    shapes = [(8, 5), (4, 6, 3, 7), (9, 10), ()]
    params = [torch.zeros(s, device="cuda") for s in shapes] + [torch.zeros(3, device="cuda")]
    gen = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    wide = r(20, 30)
    params[0].grad = r(5, 8).t()
    params[1].grad = r(4, 6, 3, 7).to(memory_format=torch.channels_last)
    params[2].grad = wide[1:19:2, 3:13]
    params[3].grad = r()
    before = [p.grad.clone() for p in params[:4]]
    kept = wide.clone()
    norm = dr.clip_grad_norm_(vctx, (p for p in params), 2.0)
    _check(before, [p.grad for p in params[:4]], norm, 2.0, 2.0)
    assert params[4].grad is None
    kept[1:19:2, 3:13] = params[2].grad
    assert torch.equal(kept, wide)
    before = [params[0].grad.clone()]
    norm = dr.clip_grad_norm_(vctx, params[0], 0.5)
    _check(before, [params[0].grad], norm, 0.5, 2.0)
    assert float(dr.clip_grad_norm_(vctx, [], 1.0)) == 0.0
    assert float(dr.grad_norm(vctx, [params[4]])) == 0.0


@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("n", [100, 70000])
def test_not_finite(vctx, kind, n):
    import opendressi_amd.torch as dr
    for bad in (math.nan, math.inf, -math.inf):
        for norm_type in (2.0, math.inf):
            params = _params([n, 5], [kind], 4)
            params[0].grad[n // 2] = bad
            before = [p.grad.clone() for p in params]
            same = lambda: all(torch.equal(p.grad.nan_to_num(9.0), b.nan_to_num(9.0))  # noqa: E731
                               for p, b in zip(params, before))
            with pytest.raises(RuntimeError):
                dr.clip_grad_norm_(vctx, params, 1.0, norm_type, error_if_nonfinite=True)
            assert same()
            norm = dr.clip_grad_norm_(vctx, params, math.inf, norm_type)
            assert same() and not math.isfinite(float(norm))
            norm = dr.clip_grad_norm_(vctx, params, 1.0, norm_type)
            if math.isnan(bad):
                assert math.isnan(float(norm)) and all(p.grad.isnan().all() for p in params)
            else:
                assert float(norm) == math.inf and params[0].grad[n // 2].isnan()
                assert not params[1].grad.any() and int(params[0].grad.isnan().sum()) == 1


def test_refused(vctx):
    """A parameter that is there twice, gradients that share memory: nothing is written."""
    import opendressi_amd as od
    import opendressi_amd.torch as dr
    for n in (10, 100000):
        a, b = _params([n, n], [torch.float32], 10)
        before = a.grad.clone()
        with pytest.raises(od.DressiError, match="share memory"):
            dr.clip_grad_norm_(vctx, [a, b, a], 1.0)
        parts = a.grad[n // 2:], a.grad[:n // 2 + 1]
        p = [torch.zeros(len(t), device="cuda") for t in parts]
        p[0].grad, p[1].grad = parts
        with pytest.raises(od.DressiError, match="share memory"):
            dr.clip_grad_norm_(vctx, p, 1.0)
        dr.grad_norm(vctx, p)
        assert torch.equal(a.grad, before)
    p = torch.zeros(4, 6, device="cuda")
    p.grad = torch.ones(1, 6, device="cuda").expand(4, 6)
    with pytest.raises(ValueError):
        dr.clip_grad_norm_(vctx, [p], 1.0)
    assert abs(float(dr.grad_norm(vctx, [p])) - 24 ** 0.5) < 1e-6
    wide = torch.ones(4, 12, device="cuda")
    p, q = torch.zeros(4, 6, device="cuda"), torch.zeros(4, 6, device="cuda")
    p.grad = q.grad = wide[:, :6]
    with pytest.raises(ValueError):
        dr.clip_grad_norm_(vctx, [p, q], 1.0)
    assert (wide == 1).all()
    with pytest.raises(ValueError):
        dr.clip_grad_norm_(vctx, [torch.zeros(3)], -1.0)
    host = torch.zeros(3)
    host.grad = torch.ones(3)
    with pytest.raises(ValueError):
        dr.clip_grad_norm_(vctx, [p, host], 1.0)


def test_extreme_sizes(vctx):
    """Squares that are no float32: the sum is taken in float64. A norm of zero scales nothing."""
    import opendressi_amd.torch as dr
    for scale in (1e-30, 1e30):
        params = _params([1000, 70001], [torch.float32], 5, scale)
        before = [p.grad.clone() for p in params]
        want = _norm(before, 2.0)
        norm = dr.clip_grad_norm_(vctx, params, 1.0)
        _check(before, [p.grad for p in params], norm, 1.0, 2.0)
        assert abs(float(norm) / want - 1) < 1e-6
    p = torch.zeros(50, device="cuda")
    p.grad = torch.zeros(50, device="cuda")
    assert float(dr.clip_grad_norm_(vctx, [p], 1.0)) == 0.0 and not p.grad.any()
    p.grad.fill_(2.0)
    dr.clip_grad_norm_(vctx, [p], 0.0)
    assert not p.grad.any()


def test_written_in_place(vctx):
    """A backward pass over gradients from before the call is refused."""
    import opendressi_amd.torch as dr
    p = torch.zeros(10, device="cuda")
    p.grad = torch.ones(10, device="cuda")
    a = torch.ones(10, device="cuda", requires_grad=True)
    y = (a * p.grad).sum()
    dr.grad_norm(vctx, [p])
    dr.clip_grad_norm_(vctx, [p], math.inf)
    y.backward(retain_graph=True)
    dr.clip_grad_norm_(vctx, [p], 1.0)
    with pytest.raises(RuntimeError):
        y.backward()


@pytest.mark.parametrize("sizes", [[100, 7], [200000, 3, 5000], [11] * 150], ids=len)
def test_captured(vctx, sizes):
    """Two graphs, replayed in turn over new gradients with eager calls between them."""
    import opendressi_amd.torch as dr
    sets = [_params(sizes, TYPES, 6 + k) for k in range(2)]
    graphs, norms, s = [], [], torch.cuda.Stream()
    for params in sets:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            dr.clip_grad_norm_(vctx, params, 1e9)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            norms.append(dr.clip_grad_norm_(vctx, params, 2.0))
            with pytest.raises(RuntimeError):
                dr.clip_grad_norm_(vctx, params, 2.0, error_if_nonfinite=True)
        graphs.append(g)
    for r in range(4):
        for k in range(2):
            new = _params(sizes, TYPES, 50 + 10 * r + k)
            for p, q in zip(sets[k], new):
                p.grad.copy_(q.grad)
            graphs[k].replay()
            want = dr.clip_grad_norm_(vctx, new, 2.0)
            torch.cuda.synchronize()
            assert torch.equal(norms[k], want)
            assert all(torch.equal(p.grad, q.grad) for p, q in zip(sets[k], new))


def test_streams(vctx):
    """Calls on two streams at once: each has its own norm."""
    import opendressi_amd.torch as dr
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    sets = [_params([300000, 5], [torch.float32], 7 + k, 1.0 + k) for k in range(2)]
    before = [[p.grad.clone() for p in s] for s in sets]
    torch.cuda.synchronize()
    norms = []
    for s, params in zip(streams, sets):
        with torch.cuda.stream(s):
            norms.append(dr.clip_grad_norm_(vctx, params, 3.0))
    torch.cuda.synchronize()
    for norm, b, params in zip(norms, before, sets):
        _check(b, [p.grad for p in params], norm, 3.0, 2.0)


def test_same_bits_each_time(vctx):
    import opendressi_amd.torch as dr
    got = []
    for _ in range(3):
        params = _params([3000001, 70, 12345], TYPES, 8)
        got.append([dr.clip_grad_norm_(vctx, params, 1.0)] + [p.grad for p in params])
    assert all(torch.equal(a, b) for other in got[1:] for a, b in zip(got[0], other))


def test_beside_an_optimizer(vctx):
    """Clipped and stepped by torch's SGD: the step of gradients clipped by the formula."""
    import opendressi_amd.torch as dr
    params = _params([(40, 30), 7], [torch.float32], 9)
    opt = torch.optim.SGD(params, lr=0.5)
    grads = [p.grad.double() for p in params]
    factor = 1.0 / (_norm(grads, 2.0) + 1e-6)
    dr.clip_grad_norm_(vctx, params, 1.0)
    opt.step()
    for p, g in zip(params, grads):
        assert torch.allclose(p.double(), -0.5 * factor * g, rtol=4 * U, atol=0.0)
