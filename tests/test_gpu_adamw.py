"""AdamW over many tensors (opendressi_amd.torch.AdamW) against the formula: 32-bit moments in
float64 with bounds from the count of roundings, 8-bit moments code for code."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F64, F32 = np.float64, np.float32
U = 2.0 ** -24  # a float32 operation's relative error at most


@pytest.fixture(scope="module")
def ctx():
    import opendressi_amd.torch as dr
    return dr.RasterizeHipContext()


def _np(t):
    return t.detach().float().cpu().numpy()


def _padded(n):
    return -(-n // 32) * 32


def _values(rng, n, size=1.0):
    """Gradients of mixed magnitude, some exactly zero."""
    g = rng.standard_normal(n) * size * 10.0 ** rng.uniform(-3, 0, n)
    return np.where(rng.random(n) < 0.2, 0.0, g).astype(F32)


def _shares(opt, flat):
    """Each parameter's elements of a flat state buffer, and the paddings."""
    flat, out, pads, at = _np(flat), [], [], 0
    for p in opt._params:
        n = p.numel()
        out.append(flat[at:at + n])
        pads.append(flat[at + n:at + _padded(n)])
        at += _padded(n)
    assert at == flat.size
    return out, pads


SIZES = [[1], [31, 32, 33], [4, 4095, 4096, 4097], [1023, 1024, 1025, 7], [2 ** 20 + 5, 3]]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("clip", [None, 0.5])
@pytest.mark.parametrize("master", [True, False])
def test_steps_32(ctx, sizes, kind, clip, master):
    """Three steps against float64. The bounds add up the roundings of one step: 3 of a moment's
    update and the rounding of its two coefficients; 6 of the quotient; and the norm's."""
    import opendressi_amd.torch as dr
    print(f"[adamw 32] {sizes} {kind} clip {clip} master {master}", flush=True)
    rng = np.random.default_rng(sum(sizes))
    lr, b1, b2, eps, wd = 0.01, 0.9, 0.99, 1e-8, 0.1
    ps = [torch.tensor(_values(rng, n)).to(kind).cuda() for n in sizes]
    opt = dr.AdamW(ctx, ps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, max_grad_norm=clip,
                   master_weights=master)
    keeps = kind != torch.float32 and master
    m, v = [[np.zeros(n) for n in sizes] for _ in range(2)]
    for t in (1, 2, 3):
        g = [torch.tensor(_values(rng, n)).to(kind).cuda() for n in sizes]
        for p, x in zip(ps, g):
            p.grad = x
        g = [_np(x).astype(F64) for x in g]
        before = _shares(opt, opt.master)[0] if keeps else [_np(p) for p in ps]
        opt.step()
        c = 1.0
        if clip:
            norm = math.sqrt(sum(float((x * x).sum()) for x in g))
            # a double sum, its root rounded once
            assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
            c = min(1.0, clip / (norm + 1e-6))
        (gm, pad_m), (gv, pad_v) = (_shares(opt, x) for x in opt.moments())
        assert not any(x.any() for x in pad_m + pad_v)
        after = _shares(opt, opt.master)[0] if keeps else [_np(p) for p in ps]
        for i, x in enumerate(g):
            x = x * c
            em = 8 * U * (np.abs(m[i]) + np.abs(x))
            ev = 12 * U * (v[i] + x * x) + 2.0 ** -148
            m[i] = b1 * m[i] + (1 - b1) * x
            v[i] = b2 * v[i] + (1 - b2) * x * x
            assert (np.abs(gm[i] - m[i]) <= em).all(), (t, i)
            assert (np.abs(gv[i] - v[i]) <= ev).all(), (t, i)
            # go on from what is there, so that a step's bounds do not add up
            m[i], v[i] = gm[i].astype(F64), gv[i].astype(F64)
            den = np.sqrt(v[i]) / math.sqrt(1 - b2 ** t) + eps
            u = lr / (1 - b1 ** t) * m[i] / den
            p = before[i].astype(F64) * (1 - lr * wd) - u
            tol = 16 * U * (np.abs(u) + np.abs(before[i]))
            if kind != torch.float32 and not keeps:  # rounded to the parameter's type
                ulp = 2.0 ** -8 if kind == torch.bfloat16 else 2.0 ** -11
                tol = tol + ulp * np.abs(p) + 2.0 ** -25
            assert (np.abs(after[i] - p) <= tol).all(), (t, i)
            if keeps:  # the parameter is its master's rounding
                want = torch.tensor(after[i]).to(kind)
                assert torch.equal(ps[i].cpu(), want)


def _mix(i, t, seed=0):
    """The step's 32 random bits of elements i."""
    mask = 0xffffffff
    key = (t * 0x9e3779b9 + seed * 0x632be5ab + 0x7f4a7c15) & mask
    x = [(int(a) & mask) ^ key ^ (((int(a) >> 32) * 0x85ebca6b) & mask) for a in i]
    x = [((a ^ (a >> 16)) * 0x7feb352d) & mask for a in x]
    x = [((a ^ (a >> 15)) * 0x846ca68b) & mask for a in x]
    return np.array([a ^ (a >> 16) for a in x], np.int64)


def _round_block(x, top, r):
    """The value that x (float32, 32 of them) is stored as, in float64 from the definition: a
    multiple of its step, rounded down after r 2^-20 steps were added."""
    x = x.astype(F64)
    mag = np.abs(x)
    e = max(math.frexp(mag.max())[1] - 1 if mag.max() else -127, top - 127)
    low = e - (top - 1)
    own = np.maximum(np.where(mag > 0, np.frexp(mag)[1] - 1, low), low)
    step = 2.0 ** (own - 3.0)
    q = np.floor(mag / step + r * 2.0 ** -20) * step
    if top == 30:
        q = np.where(mag > 0, np.maximum(q, 2.0 ** (low - 3.0)), q)
    return q * np.sign(x)


def _rounded(x, top, r):
    x = np.concatenate([x, np.zeros(_padded(x.size) - x.size, F32)])
    r = np.concatenate([r, np.zeros(x.size - r.size, np.int64)])
    return np.concatenate([_round_block(a, top, b) for a, b in
                           zip(x.reshape(-1, 32), r.reshape(-1, 32))])


@pytest.mark.parametrize("sizes", [[1], [31, 32, 33], [5, 1000, 1027]], ids=str)
@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("size", [1.0, 1e-4, 3e-12, 1e8])
def test_steps_8(ctx, sizes, kind, size):
    """Four steps, every code's value as the definition gives it from the float32 moments."""
    import opendressi_amd.torch as dr
    if kind == torch.float16 and size not in (1.0, 1e-4):
        pytest.skip("beyond float16")
    print(f"[adamw 8] {sizes} {kind} size {size}", flush=True)
    rng = np.random.default_rng(sum(sizes))
    b1, b2 = F32(0.9), F32(0.999)
    ps = [torch.tensor(_values(rng, n)).to(kind).cuda() for n in sizes]
    opt = dr.AdamW(ctx, ps, lr=1e-3, state_bits=8, seed=7)
    start = [p.detach().clone() for p in ps]
    m, v = [[np.zeros(n, F32) for n in sizes] for _ in range(2)]
    for t in (1, 2, 3, 4):
        at = 0
        for p, n in zip(ps, sizes):
            p.grad = torch.tensor(_values(rng, n, size)).to(kind).cuda()
        opt.step()
        (gm, pad_m), (gv, pad_v) = (_shares(opt, x) for x in opt.moments())
        assert not any(x.any() for x in pad_m + pad_v)
        for i, n in enumerate(sizes):
            g = _np(ps[i].grad)
            m[i] = m[i] * b1 + g * F32(1 - 0.9)
            v[i] = v[i] * b2 + (g * g) * F32(1 - 0.999)
            r = _mix(range(at, at + n), t, 7)
            m[i] = _rounded(m[i], 14, ((r & 0xffff) << 4) + 8)[:n].astype(F32)
            v[i] = _rounded(v[i], 30, ((r >> 16) << 4) + 8)[:n].astype(F32)
            assert np.array_equal(gm[i], m[i]), (t, i)
            assert np.array_equal(gv[i], v[i]), (t, i)
            at += _padded(n)
    assert all(torch.isfinite(p).all() for p in ps)
    assert any(not torch.equal(p, q) for p, q in zip(ps, start))


@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_large_8_bit(ctx, kind):
    """Enough elements for the larger share of a workgroup: the codes of a stretch in their midst
    and of the ragged end, and the norm over all."""
    import opendressi_amd.torch as dr
    n, b1, b2 = 2 ** 23 + 4099, F32(0.9), F32(0.999)
    gen = torch.Generator(device="cuda").manual_seed(2)
    p = torch.randn(n, generator=gen, device="cuda").to(kind)
    p.grad = torch.randn(n, generator=gen, device="cuda").to(kind)
    opt = dr.AdamW(ctx, [p], lr=1e-2, state_bits=8, max_grad_norm=1e9)
    opt.step()
    norm = math.sqrt(float(p.grad.double().square().sum()))
    assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    m, v = opt.moments()
    for a, b in ((0, 320), (2 ** 22 - 64, 2 ** 22 + 64), (2 ** 23 - 32, n)):
        g = _np(p.grad[a:b])
        r = _mix(range(a, b), 1)
        want_m = _rounded(F32(0) * b1 + g * F32(1 - 0.9), 14, ((r & 0xffff) << 4) + 8)
        want_v = _rounded(F32(0) * b2 + (g * g) * F32(1 - 0.999), 30, ((r >> 16) << 4) + 8)
        assert np.array_equal(_np(m[a:b]), want_m[:b - a].astype(F32))
        assert np.array_equal(_np(v[a:b]), want_v[:b - a].astype(F32))


@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_larger_than_a_cache(ctx, kind):
    """A step of several hundred MB does to each stretch what a step on that stretch alone does."""
    import opendressi_amd.torch as dr
    n, cut = 12 * 2 ** 20 + 1029, 3 * 2 ** 20
    gen = torch.Generator(device="cuda").manual_seed(3)
    p = torch.randn(n, generator=gen, device="cuda").to(kind)
    parts = [torch.nn.Parameter(q.clone()) for q in p.split(cut)]
    opt = dr.AdamW(ctx, [p], lr=1e-2)
    opts = [dr.AdamW(ctx, [q], lr=1e-2) for q in parts]
    for _ in range(2):
        g = torch.randn(n, generator=gen, device="cuda").to(kind)
        p.grad = g
        opt.step()
        for q, h, o in zip(parts, g.split(cut), opts):
            q.grad = h.clone()
            o.step()
    assert torch.equal(p, torch.cat([q.detach() for q in parts]))
    for i, m in enumerate(opt.moments()):
        assert torch.equal(m, torch.cat([o.moments()[i] for o in opts]))


def test_larger_than_a_cache_8_bit(ctx):
    """The codes of a second step over several hundred MB, against the rounding in numpy."""
    import opendressi_amd.torch as dr
    n, b1, b2 = 12 * 2 ** 20 + 1029, F32(0.9), F32(0.999)
    gen = torch.Generator(device="cuda").manual_seed(4)
    p = torch.randn(n, generator=gen, device="cuda")
    opt = dr.AdamW(ctx, [p], lr=1e-2, state_bits=8)
    was = [torch.zeros(n, device="cuda")] * 2
    for t in (1, 2):
        p.grad = torch.randn(n, generator=gen, device="cuda")
        opt.step()
        m, v = opt.moments()
        for a, b in ((0, 320), (2 ** 23 - 64, 2 ** 23 + 64), (n - 1029, n)):
            g = _np(p.grad[a:b])
            r = _mix(range(a, b), t)
            want_m = _rounded(_np(was[0][a:b]) * b1 + g * F32(1 - 0.9), 14, ((r & 0xffff) << 4) + 8)
            want_v = _rounded(_np(was[1][a:b]) * b2 + (g * g) * F32(1 - 0.999), 30,
                              ((r >> 16) << 4) + 8)
            assert np.array_equal(_np(m[a:b]), want_m[:b - a].astype(F32))
            assert np.array_equal(_np(v[a:b]), want_v[:b - a].astype(F32))
        was = [m.clone(), v.clone()]


def test_values_larger_than_a_cache(ctx):
    """The values of more codes than a cache holds: each stretch's as numpy rounds them."""
    import opendressi_amd.torch as dr
    n, b1, b2 = 84 * 2 ** 20 + 1029, F32(0.9), F32(0.999)
    gen = torch.Generator(device="cuda").manual_seed(5)
    p = torch.zeros(n, device="cuda")
    p.grad = torch.randn(n, generator=gen, device="cuda")
    opt = dr.AdamW(ctx, [p], state_bits=8)
    opt.step()
    m, v = opt.moments()
    assert m.isfinite().all() and v.isfinite().all()
    for a, b in ((0, 2080), (2 ** 26 - 64, 2 ** 26 + 2048), (n - 1029, n)):
        g = _np(p.grad[a:b])
        r = _mix(range(a, b), 1)
        want_m = _rounded(F32(0) * b1 + g * F32(1 - 0.9), 14, ((r & 0xffff) << 4) + 8)
        want_v = _rounded(F32(0) * b2 + (g * g) * F32(1 - 0.999), 30, ((r >> 16) << 4) + 8)
        assert np.array_equal(_np(m[a:b]), want_m[:b - a].astype(F32))
        assert np.array_equal(_np(v[a:b]), want_v[:b - a].astype(F32))


def test_8_bit_moments_follow(ctx):
    """The slow moment moves by 0.1 % a step, a fraction of its code's step. Under a constant
    gradient v = g^2 (1 - b2^t); the rounding being unbiased, the mean over 2^16 elements follows.
    One rounding is off by a standard deviation of at most a step's half, 2^-4 of the value, and
    the errors of the t steps decay with b2: their sum's deviation is at most
    2^-4 sqrt(sum b2^2k) < 1.4 of the value for one element, 1.4 / 2^8 for the mean: five times
    that is the bound."""
    import opendressi_amd.torch as dr
    n, steps = 2 ** 16, 2000
    p = torch.zeros(n, device="cuda")
    opt = dr.AdamW(ctx, [p], lr=0.0, state_bits=8)
    p.grad = torch.full((n,), 0.37, device="cuda")
    for t in range(steps):
        opt.step()
    m, v = (x.double().mean().item() for x in opt.moments())
    assert abs(v / (0.37 ** 2 * (1 - 0.999 ** steps)) - 1) < 5 * 1.4 / 2 ** 8
    assert abs(m / 0.37 - 1) < 5 * 1.4 / 2 ** 8
    # and decays where the gradient ends
    p.grad.zero_()
    for t in range(1000):
        opt.step()
    left = opt.moments()[1].double().mean().item() / v
    assert abs(left / 0.999 ** 1000 - 1) < 5 * 1.4 / 2 ** 8


def test_8_bit_second_moment_is_never_zero(ctx):
    """Beside a neighbour 2^40 times as large in its square, v keeps its smallest code: the update
    stays small when the gradient ends."""
    import opendressi_amd.torch as dr
    p = torch.zeros(32, device="cuda")
    p.grad = torch.full((32,), 1e-6, device="cuda")
    p.grad[5] = 1.0
    opt = dr.AdamW(ctx, [p], lr=1e-3, weight_decay=0.0, state_bits=8)
    opt.step()
    assert (opt.moments()[1] > 0).all()
    p.grad.zero_()
    before = p.clone()
    opt.step()
    # |m| <= |g| (1 - b1) and v >= its smallest code, so an update is at most lr's size
    assert ((p - before).abs() <= 1.01e-3).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("bits", [8, 32])
def test_not_finite(ctx, bad, bits):
    """What is not finite stays in its element (32 bits) or its block of 32 (8 bits)."""
    import opendressi_amd.torch as dr
    p = torch.zeros(100, device="cuda")
    p.grad = torch.ones(100, device="cuda")
    p.grad[40] = bad
    opt = dr.AdamW(ctx, [p], state_bits=bits)
    opt.step()
    m, v = opt.moments()
    hit = torch.zeros(100, dtype=torch.bool, device="cuda")
    if bits == 8:
        hit[32:64] = True
        assert m[:100][hit].isnan().all() and v[:100][hit].isnan().all()
    hit[40] = True
    assert torch.isfinite(m[:100][~hit]).all() and torch.isfinite(v[:100][~hit]).all()
    assert p[40].isnan() and torch.isfinite(p[torch.arange(100, device="cuda") != 40]).all()
    p.grad = torch.ones(100, device="cuda")
    opt.step()
    assert not torch.isfinite(p[hit]).any() and torch.isfinite(p[~hit]).all()


def test_clip_not_finite(ctx):
    """A norm that is not a number makes every update so; an infinite one leaves no gradient but
    where it came from."""
    import opendressi_amd.torch as dr
    for bad in (math.nan, math.inf):
        p = torch.ones(64, device="cuda")
        p.grad = torch.ones(64, device="cuda")
        p.grad[3] = bad
        opt = dr.AdamW(ctx, [p], lr=0.1, weight_decay=0.0, max_grad_norm=1.0)
        opt.step()
        if math.isnan(bad):
            assert opt.grad_norm.isnan() and p.isnan().all()
        else:
            assert opt.grad_norm == math.inf and p[3].isnan()
            assert (p[torch.arange(64, device="cuda") != 3] == 1).all()


def _plain(opts, ps, gs, steps=2):
    for _ in range(steps):
        for p, g in zip(ps, gs):
            p.grad = g
        opts.step()
    return [p.detach().clone() for p in ps]


@pytest.mark.parametrize("clip", [None, 1e-3])
def test_many_tensors_and_groups(ctx, clip):
    """More tensors and more hyperparameter sets than one launch holds, empty ones among them and
    gradients missing at times: each tensor as if it were alone, with its share of the norm."""
    import opendressi_amd.torch as dr
    rng = np.random.default_rng(3)
    n = [int(x) for x in rng.integers(0, 300, 200)]
    ps = [torch.tensor(_values(rng, k)).cuda() for k in n]
    qs = [p.clone() for p in ps]
    hyper = [dict(lr=1e-3 * (i + 1), weight_decay=0.01 * i) for i in range(20)]
    opt = dr.AdamW(ctx, [dict(params=ps[i::20], **h) for i, h in enumerate(hyper)],
                   max_grad_norm=clip)
    alone = [dr.AdamW(ctx, [q], **hyper[i % 20]) for i, q in enumerate(qs)]
    for t in range(3):
        gs = [torch.tensor(_values(rng, k)).cuda() if rng.random() < 0.8 else None for k in n]
        for p, g in zip(ps, gs):
            p.grad = g
        opt.step()
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs if g is not None))
        if clip:
            assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
        for o, q, g in zip(alone, qs, gs):
            q.grad = g * (clip / (norm + 1e-6)) if clip and g is not None else g
            o.step()
    for i, (p, q) in enumerate(zip(ps, qs)):
        if clip:
            # the factor is off by 4 roundings: so is a gradient; each of three updates, of lr's
            # size at most 3 times over, moves by twice that at most
            tol = 3 * 3 * hyper[i % 20]["lr"] * 16 * U + 4 * U * p.abs()
            assert ((p - q).abs() <= tol).all(), i
        else:
            assert torch.equal(p, q), i


def test_8_bit_first_step_is_the_32_bit_one(ctx):
    """The update takes the moments as computed, before they are rounded."""
    import opendressi_amd.torch as dr
    rng = np.random.default_rng(4)
    ps = [torch.tensor(_values(rng, k)).cuda() for k in rng.integers(0, 3000, 100)]
    qs = [p.clone() for p in ps]
    gs = [torch.tensor(_values(rng, p.numel())).cuda() for p in ps]
    a = _plain(dr.AdamW(ctx, ps, max_grad_norm=1.0), ps, gs, 1)
    b = _plain(dr.AdamW(ctx, qs, max_grad_norm=1.0, state_bits=8), qs, gs, 1)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("kind", TYPES, ids=str)
def test_unaligned_views_and_orders(ctx, bits, kind):
    """Parameters that begin anywhere in a buffer, gradients in another order, channels-last
    weights: the same bits as packed ones, and nothing written beside them."""
    import opendressi_amd.torch as dr
    rng = np.random.default_rng(5)
    shapes = [(1003,), (5, 3, 3, 7), (33, 65)]
    vals = [torch.tensor(_values(rng, math.prod(s))).to(kind).view(s).cuda() for s in shapes]
    grads = [torch.tensor(_values(rng, math.prod(s))).to(kind).view(s).cuda() for s in shapes]
    plain = [v.clone() for v in vals]
    want = _plain(dr.AdamW(ctx, plain, state_bits=bits), plain, grads)
    buf = torch.full((1003 + 5,), 9.0, dtype=kind, device="cuda")
    odd = buf[3:3 + 1003]
    odd.copy_(vals[0])
    other = torch.empty((65, 33), dtype=kind, device="cuda").t().copy_(grads[2])
    views = [odd, vals[1].clone(), vals[2].clone()]
    got = _plain(dr.AdamW(ctx, views, state_bits=bits), views,
                 [grads[0], grads[1].permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2), other])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert (buf[:3] == 9).all() and (buf[1006:] == 9).all()
    # in its own order: a channels-last weight is updated where it lies
    cl = vals[1].permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    assert not cl.is_contiguous()
    got = _plain(dr.AdamW(ctx, [cl]), [cl], [grads[1]])
    again = vals[1].clone()
    assert torch.equal(got[0], _plain(dr.AdamW(ctx, [again]), [again], [grads[1]])[0])


def test_another_stream(ctx):
    """On a side stream: ordered with what torch queues there."""
    import opendressi_amd.torch as dr
    p = torch.zeros(1 << 20, device="cuda")
    opt = dr.AdamW(ctx, [p], lr=1e-2, max_grad_norm=1.0, weight_decay=0.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            p.grad = torch.ones_like(p)
            opt.step()
        norm = opt.grad_norm.clone()
        q = p.clone()
    torch.cuda.current_stream().wait_stream(side)
    assert abs(float(norm) - 1024) < 1e-3
    assert abs(float(q[0]) + 0.05) < 1e-5 and (q == q[0]).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_resume(ctx, bits):
    """From a state dict the run goes on with the same bits."""
    import opendressi_amd.torch as dr
    rng = np.random.default_rng(1)
    ps = [torch.tensor(_values(rng, n)).bfloat16().cuda() for n in (100, 37)]
    gs = [torch.tensor(_values(rng, n)).bfloat16().cuda() for n in (100, 37)]
    opt = dr.AdamW(ctx, ps, state_bits=bits, lr=0.1, seed=3)
    _plain(opt, ps, gs, 3)
    kept = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in
            opt.state_dict().items()}
    qs = [p.detach().clone() for p in ps]
    other = dr.AdamW(ctx, qs, state_bits=bits)
    other.load_state_dict(kept)
    for a, b in zip(_plain(opt, ps, gs, 2), _plain(other, qs, gs, 2)):
        assert torch.equal(a, b)
    bad = dict(kept, exp_avg=kept["exp_avg"][:-32])
    with pytest.raises(ValueError, match="exp_avg"):
        other.load_state_dict(bad)
    with pytest.raises(ValueError, match="parameters"):
        other.load_state_dict(dict(kept, step=[1]))


def test_group_added_later(ctx):
    import opendressi_amd.torch as dr
    a, b = torch.zeros(40, device="cuda"), torch.zeros(50, device="cuda")
    opt = dr.AdamW(ctx, [a], lr=0.1, weight_decay=0.0)
    a.grad = torch.ones_like(a)
    opt.step()
    m = opt.moments()[0][:40].clone()
    opt.add_param_group({"params": b, "lr": 0.5})
    assert torch.equal(opt.moments()[0][:40], m)
    b.grad = torch.ones_like(b)
    opt.step()
    assert opt.state_dict()["step"] == [2, 1]
    assert torch.allclose(b, torch.full_like(b, -0.5)) and torch.allclose(a, torch.full_like(a, -0.2))


@pytest.mark.parametrize("kind", TYPES[1:], ids=str)
def test_parameters_written_between_steps(ctx, kind):
    """A 16-bit parameter that is clamped or replaced between steps keeps what was written: the
    next step starts from it, not from the old master copy."""
    import opendressi_amd.torch as dr
    rng = np.random.default_rng(8)
    p = torch.tensor(_values(rng, 3001)).to(kind).cuda()
    opt = dr.AdamW(ctx, [p], lr=1e-2, weight_decay=0.0)
    for t in range(4):
        p.grad = torch.tensor(_values(rng, 3001)).to(kind).cuda()
        if t == 1:
            p.data.clamp_(-0.5, 0.5)
        if t == 2:
            p.data = torch.tensor(_values(rng, 3001)).to(kind).cuda()
        before = torch.where(opt.master[:3001].to(kind) == p, opt.master[:3001], p.float()).clone()
        opt.step()
        # no update is larger than lr times (1 - b1) / sqrt(1 - b2), about 3.2
        assert ((opt.master[:3001] - before).abs() <= 3.3e-2).all(), t
        assert torch.equal(opt.master[:3001].to(kind), p)


def test_mixed_types(ctx):
    """Master copies for the 16-bit parameters alone, each at its place."""
    import opendressi_amd.torch as dr
    rng = np.random.default_rng(9)
    sizes, kinds = (100, 33, 64, 7), (torch.float32, torch.bfloat16, torch.float32, torch.float16)
    ps = [torch.tensor(_values(rng, n)).to(k).cuda() for n, k in zip(sizes, kinds)]
    alone = [p.clone() for p in ps]
    opts = [dr.AdamW(ctx, [p], lr=1e-2) for p in alone]
    opt = dr.AdamW(ctx, ps[:2], lr=1e-2)
    opt.add_param_group({"params": ps[2:]})
    assert opt.master.numel() == 64 + 32
    for _ in range(3):
        for p, q, o in zip(ps, alone, opts):
            p.grad = torch.tensor(_values(rng, p.numel())).to(p.dtype).cuda()
            q.grad = p.grad.clone()
            o.step()
        opt.step()
    for p, q in zip(ps, alone):
        assert torch.equal(p, q)
    assert torch.equal(opt.master[64:71], opts[3].master[:7])


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps(ctx, bits):
    """A step in a graph goes on counting: replays, with other work between, are the eager steps.
    The rates' powers come from the device's pow there, a rounding of a double apart."""
    import opendressi_amd.torch as dr
    rng = np.random.default_rng(10)
    sizes = (5000, 77)
    ps = [torch.tensor(_values(rng, n)).cuda() for n in sizes]
    qs = [p.clone() for p in ps]
    kw = dict(lr=1e-2, state_bits=bits, max_grad_norm=1.0)
    groups = lambda t: [dict(params=t[:1]), dict(params=t[1:], lr=3e-2)]  # noqa: E731
    opt, ref = dr.AdamW(ctx, groups(ps), capturable=True, **kw), dr.AdamW(ctx, groups(qs), **kw)
    for p, q in zip(ps, qs):
        p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    ref.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for t in range(5):
        for p, q in zip(ps, qs):
            g = torch.tensor(_values(rng, p.numel())).cuda()
            p.grad.copy_(g)
            q.grad.copy_(g)
        graph.replay()
        torch.cuda.synchronize()
        ref.step()
        for p, q in zip(ps, qs):
            assert torch.allclose(p, q, rtol=4 * U, atol=1e-2 * 16 * U), t
    assert opt.state_dict()["step"] == ref.state_dict()["step"] == [6, 6]
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ref.step()
    torch.cuda.synchronize()
    ps[0].grad = None
    with pytest.raises(RuntimeError, match="every"):
        opt.step()
    # the state goes from one to the other
    ref.load_state_dict(opt.state_dict())
    opt.load_state_dict(ref.state_dict())
    assert opt._counts.tolist() == [6, 6]


def test_hooks_closures_and_schedulers(ctx):
    import opendressi_amd.torch as dr
    p = torch.zeros(8, device="cuda", requires_grad=True)
    opt = dr.AdamW(ctx, [p], lr=0.5, weight_decay=0.0)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)
    seen = []
    pre = opt.register_step_pre_hook(lambda o, a, k: seen.append("pre"))
    opt.register_step_post_hook(lambda o, a, k: seen.append("post"))

    def closure():
        opt.zero_grad()
        loss = p.sum()
        loss.backward()
        seen.append("loss")
        return loss

    assert float(opt.step(closure)) == 0.0
    sched.step()
    pre.remove()
    opt.step()
    assert seen == ["pre", "loss", "post", "post"]
    assert torch.allclose(p.detach(), torch.full_like(p, -0.75))


def test_marks_what_it_writes(ctx):
    """A backward pass that needs a parameter's values of before the step is refused, as after
    any write in place; one that needs no written parameter's is not."""
    import opendressi_amd.torch as dr
    p, q = (torch.nn.Parameter(torch.full((40,), x, device="cuda")) for x in (2.0, 3.0))
    opt = dr.AdamW(ctx, [p, q], lr=0.1)
    p.grad = torch.ones(40, device="cuda")  # q has none
    one, other = (p * p).sum(), (q * q).sum()
    opt.step()
    assert (p._version, q._version) == (1, 0)
    other.backward()
    assert (q.grad == 6.0).all()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        one.backward()
    opt.step()
    assert (p._version, q._version) == (2, 1)


def test_state_is_freed(ctx):
    """Nothing but the optimizer holds its state."""
    import gc

    import opendressi_amd.torch as dr
    p = torch.zeros(1 << 22, device="cuda")
    gc.disable()
    try:
        before = torch.cuda.memory_allocated()
        opt = dr.AdamW(ctx, [p])
        assert torch.cuda.memory_allocated() >= before + 8 * p.numel()
        del opt
        assert torch.cuda.memory_allocated() == before
    finally:
        gc.enable()


def test_refusals(ctx):
    import opendressi_amd.torch as dr
    p = torch.zeros(8, device="cuda")
    for kw, what in ((dict(state_bits=16), "state_bits"), (dict(lr=-1.0), "lr"),
                     (dict(betas=(1.0, 0.9)), "betas"), (dict(eps=-1e-8), "eps"),
                     (dict(weight_decay=math.nan), "weight_decay"),
                     (dict(max_grad_norm=0.0), "max_grad_norm")):
        with pytest.raises(ValueError, match=what):
            dr.AdamW(ctx, [p], **kw)
    with pytest.raises(TypeError, match="float64"):
        dr.AdamW(ctx, [p.double()])
    with pytest.raises(ValueError, match="cpu"):
        dr.AdamW(ctx, [p.cpu()])
    with pytest.raises(ValueError, match="densely"):
        dr.AdamW(ctx, [torch.zeros(8, 8, device="cuda")[:, ::2]])
    with pytest.raises(ValueError, match="densely"):
        dr.AdamW(ctx, [torch.zeros(1, device="cuda").expand(4)])
    opt = dr.AdamW(ctx, [p])
    opt.step()  # no gradient: nothing happens
    assert opt.state_dict()["step"] == [0] and not p.any()
    p.grad = torch.sparse_coo_tensor([[1]], [1.0], (8,), device="cuda")
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    p.grad = None
    p.data = torch.zeros(9, device="cuda")
    p.grad = torch.zeros(9, device="cuda")
    with pytest.raises(ValueError, match="changed"):
        opt.step()
    assert opt.state_dict()["step"] == [0]


def test_past_32_bits(ctx):
    """A parameter of more than 2^32 elements: its ends are updated, and every state's place."""
    import opendressi_amd.torch as dr
    n = 2 ** 32 + 4129
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    spots = [0, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 4096, n - 1]
    idx = torch.tensor(spots, device="cuda")
    p.grad[idx] = 1.0
    opt = dr.AdamW(ctx, [p], lr=0.5, weight_decay=0.0, state_bits=8, master_weights=False,
                   max_grad_norm=1e4)
    opt.step()
    assert abs(float(opt.grad_norm) - math.sqrt(len(spots))) < 1e-6
    assert (p[idx] == -0.5).all()
    assert int((p != 0).count_nonzero()) == len(spots)
    m = opt._moments[0]
    assert int(m.count_nonzero()) == len(spots) and (m[idx] != 0).all()
