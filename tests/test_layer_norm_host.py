"""Layer norm's and clipping's refusals, without a GPU."""
import contextlib
import ctypes as C
import math
import random
import threading
import types

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from opendressi_amd import _lib as L
from opendressi_amd.torch import clip, norm, strides

# never read: every call here is refused before the context is used
CTX = C.cast(C.create_string_buffer(4096), C.c_void_p)
X, Y, W = (0x1000 * k for k in (1, 2, 3))  # addresses, not memory


def _refused(rc, *words):
    text = L.lib.dressi_last_error().decode()
    assert rc != 0 and all(w in text for w in words), text


def _forward(ctx=CTX, x=X, type=0, items=2, px=3, c=8, item=24, step=8, aff=0, eps=1e-5, act=0,
             scratch=None, size=0, y=Y, mean=X, rstd=X):
    return L.lib.dressi_layer_norm(ctx, x, type, items, px, c, item, step, W, W, aff, eps, act,
                                   scratch, size, y, mean, rstd)


def _backward(ctx=CTX, gy=X, x=X, type=0, items=2, px=3, c=8, step=8, aff=0, act=0, mean=X, rstd=X,
              scratch=X, size=1 << 30, gx=Y, gw=W, gb=W):
    return L.lib.dressi_layer_norm_bwd(ctx, gy, x, type, items, px, c, 24, step, W, W, aff, act,
                                       mean, rstd, scratch, size, gx, gw, gb)


def test_layer_norm_refuses():
    for bad, word in ((dict(ctx=None), "context"), (dict(type=3), "type"), (dict(aff=9), "type"),
                      (dict(act=4), "activation"), (dict(c=0), "channels"),
                      (dict(c=(1 << 24) + 1, step=1 << 25), "channels"),
                      (dict(items=1 << 30, px=1 << 30), "rows"), (dict(step=7), "overlap"),
                      (dict(x=X + 2), "aligned"), (dict(x=None), "arguments")):
        _refused(_forward(**bad), word)
        _refused(_backward(**bad), word)
    for bad, word in ((dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"),
                      (dict(eps=math.inf), "eps"), (dict(y=None), "arguments"),
                      (dict(mean=None), "arguments"), (dict(rstd=None), "arguments"),
                      (dict(y=Y + 1), "aligned")):
        _refused(_forward(**bad), word)
    for bad, word in ((dict(gy=None), "arguments"), (dict(mean=None), "arguments"),
                      (dict(rstd=None), "arguments"), (dict(gx=Y + 2), "aligned"),
                      (dict(px=5000, size=16), "scratch"), (dict(px=5000, scratch=None), "scratch"),
                      (dict(px=5000, scratch=X + 8), "scratch")):
        _refused(_backward(**bad), word)


def _at(w=W, b=W, aff=0, mean=X, rstd=X, gw=W, gb=W, items=2, y=Y):
    """Both calls' results with these addresses, and texts."""
    out = []
    for call in (lambda: L.lib.dressi_layer_norm(CTX, X, 0, items, 3, 8, 24, 8, w, b, aff, 1e-5, 0,
                                                 None, 0, y, mean, rstd),
                 lambda: L.lib.dressi_layer_norm_bwd(CTX, X, X, 0, items, 5000, 8, 40000, 8, w, b,
                                                     aff, 0, mean, rstd, None, 0, Y, gw, gb)):
        out += [call(), L.lib.dressi_last_error().decode()]
    return out


def test_layer_norm_refuses_what_is_not_aligned():
    """Weight, bias and their gradients to their type, statistics to float32; the weight's type is
    not the rows'."""
    for bad in (dict(w=W + 1, aff=1), dict(b=W + 1, aff=2), dict(w=W + 2), dict(b=W + 2),
                dict(mean=X + 2), dict(rstd=X + 1)):
        forward, text, backward, other = _at(**bad)
        assert forward != 0 and backward != 0 and "aligned" in text and "aligned" in other
    for bad in (dict(gw=W + 1, aff=2), dict(gb=W + 1, aff=1), dict(gw=W + 2), dict(gb=W + 2)):
        for items in (2, 0):
            _, _, backward, text = _at(items=items, **bad)
            assert backward != 0 and "not aligned to its type" in text
    for fine in (dict(w=W + 2, b=W + 2, aff=1), dict(mean=X + 4, rstd=X + 8)):
        forward, text, backward, other = _at(y=None, **fine)  # refused, but not for their addresses
        assert "arguments" in text and "scratch" in other


def test_layer_norm_refuses_results_over_what_is_read():
    """Over part of the rows, over rows with gaps, and in place where a row's last vector is read
    by others than those that write it."""
    far = 1 << 40
    for bad in (dict(y=X + 4), dict(y=X + 188), dict(x=Y + 188), dict(y=X, step=9, item=27),
                dict(y=X, item=25)):
        _refused(_forward(**bad), "overlap")
    for bad in (dict(gx=X + 4), dict(gx=X + 188), dict(gy=far, gx=X + 64), dict(gx=X - 64),
                dict(gy=far, gx=X, step=9)):
        _refused(_backward(**bad), "overlap")
    for type, c in ((0, 32769), (1, 32772), (2, 50001)):
        rows = dict(type=type, c=c, step=c, items=1, scratch=far, size=1 << 30)
        _refused(_forward(y=X, item=3 * c, **rows), "overlap")
        _refused(_backward(gx=X, **rows), "overlap")
        _refused(_backward(gy=far, gx=X, **rows), "overlap")
    _refused(_backward(gx=X, type=1, c=16387, step=16387, items=1), "overlap")


def test_nothing_to_do():
    assert _forward(items=0) == 0 and _forward(px=0) == 0
    assert _backward(gx=None, gw=None, gb=None) == 0
    assert L.lib.dressi_layer_norm_scratch(0, 0, 5, 8, 1) == 0


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="for hosts without a device")
def test_a_device_that_cannot_be_made_current_is_reported():
    """Before anything is launched, without rows too, whose gradients of weight and bias are zero."""
    ctx = C.cast(C.create_string_buffer(C.string_at(C.byref(C.c_int(99)), 4) + bytes(4092), 4096),
                 C.c_void_p)
    for call in (lambda: _forward(ctx=ctx), lambda: _backward(ctx=ctx),
                 lambda: _backward(ctx=ctx, items=0), lambda: _backward(ctx=ctx, px=0, gx=None)):
        _refused(call(), "scope")


def test_layer_norm_scratch():
    """Forward for rows beyond a workgroup alone, backward where several workgroups add to the
    weight's gradient; by the number of rows, however they are given."""
    scratch = L.lib.dressi_layer_norm_scratch
    assert scratch(0, 5, 1000, 32768, 0) == 0 and scratch(1, 5, 1000, 32769, 0) > 0
    assert scratch(0, 1, 1, 64, 1) == 0 and scratch(0, 1, 10000, 64, 1) > 0
    assert scratch(1, 1, 6000, 24, 1) == scratch(1, 6000, 1, 24, 1) == scratch(1, 20, 300, 24, 1)


def _table(*rows):
    t = np.zeros(len(rows), [("data", "<u8"), ("n", "<u8"), ("type", "<u4"), ("unused", "<u4")])
    for e, (data, n, kind) in zip(t, rows):
        e["data"], e["n"], e["type"] = data, n, kind
    return t


def _clip(table, kind=0, max_norm=1.0, ctx=CTX, scratch=X, norm=X):
    return L.lib.dressi_clip_norm(ctx, table.ctypes.data, len(table), kind, max_norm, scratch, norm)


def test_clip_norm_scratch():
    """None where one workgroup holds all vectors of 16 bytes (8192) of at most 128 tensors."""
    def bytes_of(*sizes, kind=0):
        t = _table(*((0x1000, n, kind) for n in sizes))
        return L.lib.dressi_clip_norm_scratch(t.ctypes.data, len(t))
    assert bytes_of() == bytes_of(1, 0, 5) == bytes_of(32768) == bytes_of(65536, kind=1) == 0
    assert bytes_of(*[1] * 128) == bytes_of(*[1] * 128 + [0] * 50) == 0
    assert bytes_of(32769) > 0 and bytes_of(65537, kind=2) > 0 and bytes_of(*[1] * 129) > 0


def test_clip_norm_refuses():
    good = _table((0x10000, 100, 0), (0x100000, 100000, 1))
    for bad, word in ((dict(ctx=None), "context"), (dict(norm=None), "arguments"),
                      (dict(kind=2), "norm"), (dict(max_norm=-1.0), "max_norm"),
                      (dict(max_norm=math.nan), "max_norm"), (dict(scratch=X + 4), "scratch"),
                      (dict(scratch=None), "scratch")):
        _refused(_clip(good, **bad), word)
    for rows, word in (([(0x10000, 100, 3)], "type"), ([(0, 100, 0)], "NULL"),
                       ([(0x10002, 100, 0)], "aligned"), ([(0x10001, 100, 1)], "aligned"),
                       ([(0x10000, (1 << 40) + 1, 0)], "large"),
                       ([(0x10000, 100, 0), (0x10000, 100, 0)], "share"),
                       ([(0x10000, 100, 0), (0x20000, 1, 0), (0x10000 + 396, 2, 1)], "0 and 2"),
                       ([(0x10000 + 198, 1, 2), (0x10000, 100, 1)], "0 and 1")):
        _refused(_clip(_table(*rows)), word)


HOST = types.SimpleNamespace(device=torch.device("cuda", 0), lock=threading.RLock())


def _param(grad, shape=(3,)):
    p = torch.zeros(shape, dtype=grad.dtype)
    p.grad = grad
    return p


def test_clip_grad_norm_refuses():
    p = _param(torch.ones(3))
    for args, error in (((-1.0,), ValueError), ((math.nan,), ValueError), ((1.0, 1.0), ValueError),
                        ((1.0, 0.0), ValueError), ((1.0, 2.0), ValueError)):
        with pytest.raises(error):  # the last for its device
            clip.clip_grad_norm_(HOST, [p], *args)
    with pytest.raises(TypeError):
        clip.clip_grad_norm_(HOST, [_param(torch.ones(3, dtype=torch.float64))], 1.0)
    for sparse in (torch.eye(3).to_sparse(), torch.eye(3).to_sparse_csr()):
        with pytest.raises(RuntimeError, match="sparse"):
            clip.grad_norm(HOST, [types.SimpleNamespace(grad=sparse)])
    with pytest.raises(ValueError):
        clip.grad_norm(HOST, [p], 3.0)


@pytest.fixture
def host(monkeypatch):
    """A context for gradients on the host, whose calls pass for the library's: the norms of packed
    gradients of float32, and nothing scaled."""
    def call(self, ctx, kind, max_norm):
        copies = {id(v): packed for v, packed in self.views}
        return torch.cat([copies.get(id(g), g).reshape(-1) for g in self.grads]).norm()

    monkeypatch.setattr(clip._Gradients, "clip", call)
    return types.SimpleNamespace(device=types.SimpleNamespace(index=-1), lock=threading.RLock())


def test_without_a_limit_any_gradients_are_taken(host):
    """Nothing is written then: expanded gradients and the same twice count as they come."""
    wide = torch.ones(4, 12)
    p = _param(torch.ones(1, 6).expand(4, 6), (4, 6))
    q = _param(wide[:, :6], (4, 6))
    for params, n in (([p], 24), ([q, q], 48), ([p, q], 48)):
        norm = clip.clip_grad_norm_(host, params, math.inf)
        assert torch.equal(norm, clip.grad_norm(host, params)) and abs(float(norm) ** 2 - n) < 1e-3
        with pytest.raises(ValueError):
            clip.clip_grad_norm_(host, params, 1.0)


def _some(rng, base):
    """A strided tensor in the bytes of base, and the bytes of each of its elements."""
    kind = rng.choice([torch.float32, torch.bfloat16])
    flat = base.view(kind)
    shape = [rng.choice([1, 1, 2, 3, 5]) for _ in range(rng.randint(1, 3))]
    steps = [rng.choice([1, 2, 3, 4, 6, 7, 12, 24, 25]) for _ in shape]
    room = len(flat) - 1 - sum(s * (n - 1) for s, n in zip(steps, shape))
    t = flat.as_strided(shape, steps, rng.randint(0, min(room, 30)))
    at = t.storage_offset() + sum((torch.arange(n) * s).view([-1] + [1] * (len(shape) - 1 - i))
                                  for i, (n, s) in enumerate(zip(shape, steps)))
    size = t.element_size()
    return t, [int(a) * size + k for a in at.reshape(-1) for k in range(size)]


def test_shared_elements_are_found():
    """Against the elements' bytes counted out, as below."""
    rng, base, seen = random.Random(6), torch.zeros(2400, dtype=torch.uint8), [0, 0]
    for _ in range(5000):
        t, at = _some(rng, base)
        assert clip._apart(t) == (len(at) == len(set(at))), (t.shape, t.stride())
        seen[clip._apart(t)] += 1
    assert min(seen) > 500
    assert clip._apart(base.as_strided((2, 4), (3, 2))) and not clip._apart(base[:1].expand(2))
    assert not clip._apart(base.as_strided((3, 4), (3, 2)))
    assert clip._apart(base.as_strided((3, 0), (0, 1))) and clip._apart(base.as_strided((), ()))


def test_strides_that_cross_are_taken(host):
    """Elements that lie apart by strides of which none reaches past the others' span."""
    g = torch.arange(12.0).as_strided((2, 4), (3, 2))  # 0 2 4 6, 3 5 7 9
    clip.clip_grad_norm_(host, [_param(g, (2, 4))], 1.0)


def test_shared_memory_is_found():
    """Against the elements' bytes counted out: nothing that shares is passed, nothing else is
    refused."""
    rng, base, seen = random.Random(5), torch.zeros(2400, dtype=torch.uint8), set()
    while len(seen) < 2 or rng.random() > 2e-4:
        made = [_some(rng, base) for _ in range(rng.randint(2, 4))]
        made = [(t, b) for t, b in made if len(b) == len(set(b))]
        every = [x for _, b in made for x in b]
        want = len(every) != len(set(every))
        dense = [clip._dense(t) for t, _ in made]
        assert strides.shared([t for t, _ in made], dense) == want, made
        seen.add(want)


def test_shared_memory_of_large_tables():
    """By addresses alone, whatever the sizes; columns of one table lie apart."""
    wide = torch.empty(50000, 600, dtype=torch.bfloat16)
    columns = [wide[:, 3 * i:3 * i + 3] for i in range(200)]
    assert not strides.shared(columns, [False] * 200)
    assert strides.shared(columns + [wide[49999, 599:]], [False] * 200 + [True])
    assert not strides.shared([wide[::2, 1::2], wide[1::2, 1::2], wide[:, ::2]], [False] * 3)
    assert strides.shared([wide[::2, 1::2], wide[1::2], wide[:, :1]], [False] * 3)


def test_clip_grad_norm_refuses_shared_memory(host):
    wide = torch.ones(4, 12)
    flat = wide.view(-1)
    for a, b in ((wide[:, :6], wide[:, 3:9]), (wide[:, :6], flat[13:20]), (flat[5:15], wide[:, 2:4]),
                 (wide[:, :6], flat[36:37]), (wide[:, :6], wide[:, :6]), (wide.t()[:5], wide[2])):
        params = [_param(a, a.shape), _param(torch.ones(7), (7,)), _param(b, b.shape)]
        for some in (params, params[::-1]):
            with pytest.raises(ValueError, match="share memory"):
                clip.clip_grad_norm_(host, some, 1.0)
    for a, b in ((wide[:, :6], wide[:, 6:]), (wide[:, :6], flat[18:24]), (wide[::2, ::2], wide[1::2]),
                 (wide[:, ::2], wide[:, 1::2]), (wide.t()[:5], wide.t()[5:])):
        clip.clip_grad_norm_(host, [_param(a, a.shape), _param(b, b.shape)], 1.0)


def test_elements_that_share_memory():
    base = torch.zeros(40)
    assert clip._apart(base[::2]) and clip._apart(base.view(4, 10)[:, 3:7].t())
    assert not clip._apart(base[:1].expand(5)) and not clip._apart(base.as_strided((5, 5), (2, 1)))


@pytest.mark.parametrize("op", [norm.layer_norm, lambda *t: norm.group_norm(*t[:2], 1, *t[2:])],
                         ids=["layer_norm", "group_norm"])
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("dual", range(3))
def test_forward_mode_is_refused(monkeypatch, op, grad, dual):
    """A dual tensor's derivative is refused, not lost; beside ordinary ones nothing changes."""
    def kernel(ctx, x, *args, **kwargs):
        return 2 * x, x.mean(-1), x.mean(-1)

    monkeypatch.setattr(norm.K, "layer_norm", kernel)
    monkeypatch.setattr(norm.K, "group_norm", kernel)
    host = types.SimpleNamespace(device=torch.device("cpu"), lock=threading.RLock(), _ctx=None)
    args = [torch.randn(4, 8), torch.ones(8), torch.zeros(8)]
    with forward_ad.dual_level(), contextlib.nullcontext() if grad else torch.no_grad():
        assert torch.equal(op(host, *args), 2 * args[0])
        args[dual] = forward_ad.make_dual(args[dual], torch.ones_like(args[dual]))
        with pytest.raises(NotImplementedError):
            op(host, *args)
