"""What AdamW keeps between steps (opendressi_amd.torch.AdamW): its order, its counts, and the
codes of clipped steps."""
import math

import numpy as np
import pytest
import torch
from test_gpu_adamw import F32, U, _mix, _np, _rounded
from test_gpu_adamw import _values as _mixed

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ctx():
    import opendressi_amd.torch as dr
    return dr.RasterizeHipContext()


def _values(shapes, seed, kind=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(s, generator=gen, device="cuda").to(kind) for s in shapes]


def _steps(opt, params, shapes, seeds):
    for s in seeds:
        for p, g in zip(params, _values(shapes, s, params[0].dtype)):
            p.grad = g
        opt.step()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("resumed", [False, True])
def test_channels_last_after_some_steps(ctx, bits, kind, resumed):
    """Weights that become channels-last after two steps, in the same run or in one that goes on
    from its state, take the steps of weights that stay as they are, bit for bit."""
    import opendressi_amd.torch as dr
    shapes = [(20, 12, 3, 3), (33,), (7, 5, 2, 4)]
    kw = dict(lr=0.05, state_bits=bits, seed=5, max_grad_norm=1.0)
    print(f"[adamw order] {bits} {kind} resumed {resumed}", flush=True)
    want = _values(shapes, 0, kind)
    ref = dr.AdamW(ctx, want, **kw)
    _steps(ref, want, shapes, range(1, 6))
    got = _values(shapes, 0, kind)
    opt = dr.AdamW(ctx, got, **kw)
    _steps(opt, got, shapes, (1, 2))
    if resumed:
        kept = opt.state_dict()
        got = [p.clone(memory_format=torch.channels_last) if p.dim() == 4 else p.clone()
               for p in got]
        opt = dr.AdamW(ctx, got, **kw)
        opt.load_state_dict(kept)
    else:
        for p in got:
            if p.dim() == 4:
                p.data = p.data.to(memory_format=torch.channels_last)
    _steps(opt, got, shapes, (3, 4))
    assert not got[0].is_contiguous()
    got[0].data = got[0].data.contiguous()
    _steps(opt, got, shapes, (5,))
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    for a, b in zip(opt.moments(), ref.moments()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [8, 32])
def test_after_a_capture(ctx, bits):
    """Once a graph holds the state, a group is refused, and the graph goes on as the eager steps
    do."""
    import opendressi_amd.torch as dr
    shapes = [(40, 3), (65,)]
    ps, qs = _values(shapes, 0), _values(shapes, 0)
    opt = dr.AdamW(ctx, ps, lr=0.05, state_bits=bits, capturable=True)
    ref = dr.AdamW(ctx, qs, lr=0.05, state_bits=bits, capturable=True)
    _steps(ref, qs, shapes, (1, 2, 3))
    for p, g in zip(ps, _values(shapes, 1)):
        p.grad = g
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for t in (2, 3):
        with pytest.raises(RuntimeError, match="captured"):
            opt.add_param_group({"params": torch.zeros(9, device="cuda")})
        for p, g in zip(ps, _values(shapes, t)):
            p.grad.copy_(g)
        graph.replay()
        torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    assert all(torch.equal(a, b) for a, b in zip(opt.moments(), ref.moments()))


def test_a_refused_step_does_not_count(ctx):
    """More tensors than a clipped step takes: refused before its counts on the device move."""
    from opendressi_amd._lib import AdamwSet, AdamwTensor, lib
    n = 1024 * 64 + 1
    p, state = torch.zeros(32, device="cuda"), torch.zeros(2, 32, device="cuda")
    table = (AdamwTensor * n)(*[(p.data_ptr(), p.data_ptr(), None, 1, 0, 0, 0)] * n)
    sets = (AdamwSet * 1)((1e-3, 0.9, 0.999, 1e-8, 0.0, 0))
    scratch = torch.empty(lib.dressi_adamw_scratch(), dtype=torch.uint8, device="cuda")
    norm, steps = torch.zeros((), device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    rates = torch.empty(lib.dressi_adamw_set_bytes(), dtype=torch.uint8, device="cuda")
    ctx._ctx.use_torch_stream()
    rc = lib.dressi_adamw_step(ctx._ctx.handle, table, n, sets, 1, 32, 32, state[0].data_ptr(),
                               state[1].data_ptr(), None, None, 0, 1.0, scratch.data_ptr(),
                               norm.data_ptr(), steps.data_ptr(), rates.data_ptr())
    assert rc == -1 and b"too many tensors" in lib.dressi_last_error()
    assert int(steps) == 0 and not p.any() and not state.any()


@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [[33, 1000], [2 ** 23 + 4099]], ids=str)
def test_clipped_8_bit_codes(ctx, sizes, kind):
    """Three steps whose clip is active, from the norm on the device (a double sum, its root
    rounded once): the factor in float32, and every code as the definition gives it."""
    import opendressi_amd.torch as dr
    print(f"[adamw clipped 8] {sizes} {kind}", flush=True)
    rng = np.random.default_rng(11)
    b1, b2 = F32(0.9), F32(0.999)
    ps = [torch.tensor(_mixed(rng, n)).to(kind).cuda() for n in sizes]
    opt = dr.AdamW(ctx, ps, state_bits=8, max_grad_norm=0.25, seed=2)
    # of a large tensor its first elements, those around a workgroup's share, and the ragged end
    spans = [[(0, n)] if n < 5000 else [(0, 96), (2 ** 22 - 32, 2 ** 22 + 32), (2 ** 23 - 32, n)]
             for n in sizes]
    m, v = [[[np.zeros(b - a, F32) for a, b in s] for s in spans] for _ in range(2)]
    for t in (1, 2, 3):
        for p, n in zip(ps, sizes):
            p.grad = torch.tensor(_mixed(rng, n)).to(kind).cuda()
        opt.step()
        norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in ps))
        assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
        c = F32(0.25) / (F32(float(opt.grad_norm)) + F32(1e-6))
        assert c < 1
        gm, gv = opt.moments()
        at = 0
        for i, n in enumerate(sizes):
            for k, (a, b) in enumerate(spans[i]):
                g = _np(ps[i].grad[a:b]) * c
                r = _mix(range(at + a, at + b), t, 2)
                x = m[i][k] * b1 + g * F32(1 - 0.9)
                y = v[i][k] * b2 + (g * g) * F32(1 - 0.999)
                m[i][k] = _rounded(x, 14, ((r & 0xffff) << 4) + 8)[:b - a].astype(F32)
                v[i][k] = _rounded(y, 30, ((r >> 16) << 4) + 8)[:b - a].astype(F32)
                assert np.array_equal(_np(gm[at + a:at + b]), m[i][k]), (t, i, k)
                assert np.array_equal(_np(gv[at + a:at + b]), v[i][k]), (t, i, k)
            at += -(-n // 32) * 32
