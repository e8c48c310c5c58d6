"""AdamW's bookkeeping (opendressi_amd.torch.AdamW) without a GPU: parameters on the host, the
step's entry point replaced by the formula in numpy."""
import copy
import ctypes as C
import pickle
import threading
import types

import numpy as np
import pytest
import torch

from opendressi_amd.torch import optim


def _array(address, n):
    return np.ctypeslib.as_array((C.c_float * n).from_address(address))


class _Lib:
    """dressi_adamw_step over host memory, float32 with 32-bit moments."""

    def __init__(self, real):
        self.dressi_adamw_scratch = real.dressi_adamw_scratch
        self.dressi_adamw_set_bytes = real.dressi_adamw_set_bytes
        self.calls = 0

    def dressi_adamw_step(self, handle, table, n, sets, n_sets, bits, total, m, v, m_scale, v_scale,
                          seed, max_norm, scratch, norm, counts, device_sets):
        self.calls += 1
        if bits != 32:
            return 0
        for e in table[:n]:
            s = sets[e.set]
            g, p = _array(e.grad, e.n), _array(e.param, e.n)
            em, ev = (_array(a + 4 * e.state, e.n) for a in (m, v))
            em[:] = em * s.beta1 + g * (1 - s.beta1)
            ev[:] = ev * s.beta2 + g * g * (1 - s.beta2)
            den = np.sqrt(ev / (1 - s.beta2 ** s.step)) + s.eps
            p[:] = p * (1 - s.lr * s.weight_decay) - em / den * (s.lr / (1 - s.beta1 ** s.step))
        return 0


@pytest.fixture
def lib(monkeypatch):
    fake = _Lib(optim.lib)
    monkeypatch.setattr(optim, "lib", fake)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return fake


CTX = types.SimpleNamespace(device=torch.device("cpu"), lock=threading.RLock(),
                            _ctx=types.SimpleNamespace(use_torch_stream=lambda: None, handle=None))
SHAPES = [(4, 3, 2, 5), (7,), (6, 5)]


def _values(seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=gen) for s in SHAPES]


def _another_order(t):
    """t's values in another order of memory (channels last, or columns first)."""
    if t.dim() == 4:
        return t.contiguous(memory_format=torch.channels_last)
    return t.t().contiguous().t() if t.dim() == 2 else t


def _steps(opt, params, seeds):
    for s in seeds:
        for p, g in zip(params, _values(s)):
            p.grad = g
        opt.step()


@pytest.mark.parametrize("when", [0, 2])
@pytest.mark.parametrize("back", [False, True])
def test_another_order_between_steps(lib, when, back):
    """A parameter that is laid out anew before or after its first step, and back, takes the steps
    of one that is not: the same values at the same indices."""
    want = _values(0)
    _steps(optim.AdamW(CTX, want, lr=0.1), want, range(1, 7))
    got = _values(0)
    opt = optim.AdamW(CTX, got, lr=0.1)
    _steps(opt, got, range(1, 1 + when))
    for p in got:
        p.data = _another_order(p.data)
    assert not got[0].is_contiguous() and not got[2].is_contiguous()
    _steps(opt, got, range(1 + when, 5))
    if back:
        for p in got:
            p.data = p.data.contiguous()
    _steps(opt, got, range(5, 7))
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    assert got[0].is_contiguous() == got[2].is_contiguous() == back


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("then", [False, True])
def test_resume_in_another_order(lib, first, then):
    """State goes from parameters in one order to ones in another."""
    want = _values(0)
    _steps(optim.AdamW(CTX, want, lr=0.1), want, range(1, 6))
    a = [_another_order(t) if first else t for t in _values(0)]
    opt = optim.AdamW(CTX, a, lr=0.1)
    _steps(opt, a, range(1, 4))
    kept = opt.state_dict()
    b = [_another_order(t) if then else t.contiguous() for t in a]
    b = [t.clone(memory_format=torch.preserve_format) for t in b]
    other = optim.AdamW(CTX, b)
    other.load_state_dict(kept)
    _steps(other, b, range(4, 6))
    for p, q in zip(b, want):
        assert torch.equal(p, q)
    assert [s for s, _ in other.state_dict()["layout"]] == SHAPES


def test_resume_without_a_layout(lib):
    """A dict that does not say so is in the order that the parameters have when it is loaded."""
    want = [_another_order(t) for t in _values(0)]
    opt = optim.AdamW(CTX, want, lr=0.1)
    _steps(opt, want, range(1, 3))
    kept = {k: v for k, v in opt.state_dict().items() if k != "layout"}
    got = [t.contiguous() for t in want]
    other = optim.AdamW(CTX, got)
    for p in got:
        p.data = _another_order(p.data).clone(memory_format=torch.preserve_format)
    other.load_state_dict(dict(kept, exp_avg=kept["exp_avg"].clone(),
                               exp_avg_sq=kept["exp_avg_sq"].clone()))
    _steps(opt, want, range(3, 5))
    _steps(other, got, range(3, 5))
    for p, q in zip(got, want):
        assert torch.equal(p, q)


def test_state_of_other_shapes_is_refused(lib):
    """Shapes of the same padded sizes, or transposed, are not the same parameters."""
    opt = optim.AdamW(CTX, _values(0))
    kept = opt.state_dict()
    for shapes in ([(4, 3, 2, 5), (9,), (6, 5)], [(4, 3, 2, 5), (7,), (5, 6)]):
        other = optim.AdamW(CTX, [torch.zeros(s) for s in shapes])
        with pytest.raises(ValueError, match="shape"):
            other.load_state_dict(kept)
    for bad in (kept["layout"][:2], [((4, 3, 2, 5), (30, 10, 5, 2))] + kept["layout"][1:],
                [((4, 3, 2, 5), (30, 10, 5))] + kept["layout"][1:]):
        with pytest.raises(ValueError, match="layouts|strides"):
            opt.load_state_dict(dict(kept, layout=bad))
    assert opt.state_dict()["layout"] == kept["layout"]


def test_another_shape_between_steps(lib):
    """The same elements in the same order under another shape go on; in another order they are
    refused, for which of the old ones is which nobody says."""
    p, q = torch.zeros(6), torch.zeros(6)
    opt, ref = optim.AdamW(CTX, [p], lr=0.1), optim.AdamW(CTX, [q], lr=0.1)
    g = torch.arange(6.0) - 2
    for o, t in ((opt, p), (ref, q)):
        t.grad = g
        o.step()
    p.grad = None
    p.data = p.data.view(2, 3)
    p.grad, q.grad = g.view(2, 3), g
    opt.step(), ref.step()
    assert torch.equal(p.flatten(), q)
    assert opt.state_dict()["layout"] == [((2, 3), (3, 1))]
    p.grad = None
    p.data = p.data.reshape(3, 2).t().contiguous().t()
    p.grad = torch.ones(3, 2)
    before, calls = p.clone(), lib.calls
    with pytest.raises(ValueError, match="shape"):
        opt.step()
    assert torch.equal(p, before) and lib.calls == calls


def test_parameters_that_share_memory_are_refused(lib):
    """All tensors are stepped at once: one of them twice, or two over the same elements, would be
    read and written by two workgroups."""
    p, flat, none = torch.zeros(8), torch.zeros(20), torch.zeros(0)
    for params in ([p, p], [p, torch.ones(3), p.view(2, 4)], [flat[:11], flat[10:]],
                   [flat[4:6], flat], [none, none],
                   [dict(params=[p, p])], [dict(params=p), dict(params=p)]):
        with pytest.raises(ValueError, match="share|twice|more than one"):
            optim.AdamW(CTX, params)
    opt = optim.AdamW(CTX, [flat[:10], flat[10:], none, torch.zeros(0)])
    with pytest.raises(ValueError, match="share"):
        opt.add_param_group({"params": [flat[9:11]]})
    assert len(opt.param_groups) == 1 and len(opt.state_dict()["step"]) == 4


def test_state_stays_where_a_graph_has_it(lib, monkeypatch):
    """Replays write the state that the capture saw: after one, no call replaces it or changes
    its order."""
    params = _values(0)
    opt = optim.AdamW(CTX, params, capturable=True)
    _steps(opt, params, (1,))
    opt.add_param_group({"params": torch.zeros(3)})
    opt.param_groups[1]["params"][0].grad = torch.ones(3)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    _steps(opt, params, (2,))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    held = [t.data_ptr() for t in (*opt.moments(), opt._counts, opt._device_sets)]
    with pytest.raises(RuntimeError, match="captured"):
        opt.add_param_group({"params": torch.zeros(4)})
    kept = opt.state_dict()
    other = [(s, tuple(torch.zeros(s).t().contiguous().t().stride())) if len(s) == 2 else (s, t)
             for s, t in kept["layout"]]
    with pytest.raises(ValueError, match="captured"):
        opt.load_state_dict(dict(kept, layout=other))
    opt.load_state_dict(kept)
    assert len(opt.param_groups) == 2 and opt.state_dict()["layout"] == kept["layout"]
    assert held == [t.data_ptr() for t in (*opt.moments(), opt._counts, opt._device_sets)]


def test_copies_are_refused(lib):
    """A copy would have had no parameters and no state."""
    opt = optim.AdamW(CTX, _values(0))
    for make in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="state_dict"):
            make(opt)


def test_state_dict_hooks(lib):
    """Before and after, in their order, with the dict they are given or give back."""
    opt, seen = optim.AdamW(CTX, _values(0), seed=3), []
    opt.register_state_dict_pre_hook(lambda o: seen.append("save"))
    opt.register_state_dict_post_hook(lambda o, d: d.update(mark=1))
    opt.register_state_dict_post_hook(lambda o, d: dict(d, more=o is opt))
    first = opt.register_state_dict_pre_hook(lambda o: seen.append("first"), prepend=True)
    kept = opt.state_dict()
    assert kept["mark"] == 1 and kept["more"] is True and seen == ["first", "save"]
    first.remove()
    opt = optim.AdamW(CTX, _values(0))
    opt.register_load_state_dict_pre_hook(lambda o, d: seen.append(d.pop("mark")))
    opt.register_load_state_dict_pre_hook(lambda o, d: dict(d, seed=9))
    opt.register_load_state_dict_post_hook(lambda o: seen.append(o.seed))
    opt.load_state_dict(kept)
    assert opt.seed == 9 and seen[-2:] == [1, 9]
    assert kept["seed"] == 3 and kept["mark"] == 1


def test_a_refused_state_changes_nothing(lib):
    """Whatever a state dict is refused for, the optimizer is as it was, its rates too."""
    params = _values(0)
    opt = optim.AdamW(CTX, params, lr=0.25, capturable=True, seed=4)
    _steps(opt, params, (1, 2))
    moments = [t.clone() for t in opt.moments()]
    good = dict(opt.state_dict(), seed=5, exp_avg=torch.ones_like(moments[0]))
    good["param_groups"] = [dict(good["param_groups"][0], lr=0.5)]
    bad = [dict(good, step=[1, 2, 3]), dict(good, step=[1, 1]), dict(good, step=["x", 1, 1]),
           dict(good, exp_avg_sq=torch.zeros(3)), dict(good, param_groups=[]),
           dict(good, param_groups=[dict(lr=-1.0)]), dict(good, layout=[]), dict(good, seed="x"),
           dict(good, param_groups=[dict(lr=0.5)]),
           {k: v for k, v in good.items() if k != "exp_avg"}]
    for state in bad:
        with pytest.raises((ValueError, KeyError, TypeError)):
            opt.load_state_dict(state)
        assert opt.param_groups[0]["lr"] == 0.25 and opt.seed == 4
        assert all(torch.equal(a, b) for a, b in zip(opt.moments(), moments))
    opt.load_state_dict(good)
    assert opt.param_groups[0]["lr"] == 0.5 and opt.seed == 5 and (opt.moments()[0] == 1).all()


def test_the_norm_of_no_gradients(lib):
    """A step without gradients leaves no older step's norm behind."""
    opt = optim.AdamW(CTX, _values(0), max_grad_norm=1.0)
    opt.grad_norm.fill_(7.0)
    opt.step()
    assert float(opt.grad_norm) == 0.0 and lib.calls == 0


def test_a_norm_that_is_zero_in_32_bits_is_refused(lib):
    for bad in (0.0, -1.0, float("nan"), float("inf"), 1e-46, 1e-300):
        with pytest.raises(ValueError, match="max_grad_norm"):
            optim.AdamW(CTX, _values(0), max_grad_norm=bad)
    for good in (1e-40, 1e-6, 1e30, 1e39):
        optim.AdamW(CTX, _values(0), max_grad_norm=good)


def test_sets_of_parameters_are_refused(lib):
    """Their order is another in every run, and state lies in it."""
    for params in (set(_values(0)), [dict(params=set(_values(0)))],
                   [dict(params=frozenset(_values(0)))]):
        with pytest.raises(TypeError, match="order"):
            optim.AdamW(CTX, params)
    assert len(optim.AdamW(CTX, (t for t in _values(0))).state_dict()["step"]) == 3
