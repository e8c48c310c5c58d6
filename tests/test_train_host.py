"""Host side of group norm and AdamW, without a GPU: layouts that Python and the library share,
sizes, and refusals that come before any work."""
import ctypes as C
import types

import pytest
import torch


def test_table_layout():
    """The array that the optimizer fills is the library's struct, field for field."""
    from opendressi_amd._lib import AdamwSet, AdamwTensor
    from opendressi_amd.torch.optim import _ENTRY
    assert _ENTRY.itemsize == C.sizeof(AdamwTensor) == 48 and C.sizeof(AdamwSet) == 48
    for name, _ in AdamwTensor._fields_:
        field = getattr(AdamwTensor, name)
        kind, offset = _ENTRY.fields[name]
        assert (offset, kind.itemsize) == (field.offset, field.size), name


def test_entry_points_refuse():
    from opendressi_amd._lib import lib
    assert lib.dressi_group_norm(None, None, 0, 1, 1, 8, 8, 8, 1, None, None, 0, 1e-5, 0, None, 0,
                                 None, None, None) == -1
    assert b"context" in lib.dressi_last_error()
    assert lib.dressi_group_norm_bwd(None, None, None, 0, 1, 1, 8, 8, 8, 1, None, None, 0, 0, None,
                                     None, None, 0, None, None, None) == -1
    assert lib.dressi_adamw_step(None, None, 0, None, 0, 32, 0, None, None, None, None, 0, 0.0,
                                 None, None, None, None) == -1
    assert lib.dressi_adamw_values(None, 0, None, None, None, None, None, None) == -1


def test_scratch_sizes():
    from opendressi_amd._lib import lib
    size = lambda n, px, c, g, bwd, kind=0, at=0: lib.dressi_group_norm_scratch(  # noqa: E731
        kind, n, px, c, px * c, c, g, at, bwd)
    assert size(1, 64, 32, 8, 0) == 0  # one launch, nothing between
    assert size(1, 64, 32, 8, 1) == 8 * 32
    assert size(4, 64, 32, 8, 1) == 4 * 8 * 32
    assert size(1, 512 * 512, 64, 8, 0, 1) > 0
    for bad in ((0, 64, 32, 8), (1, 0, 32, 8), (1, 64, 0, 8), (1, 64, 32, 0), (1, 64, 32, 5)):
        assert size(*bad, 1) == 0
    assert size(1, 64, 32, 8, 1, 3) == 0
    # sums for the weight's gradient do not grow with the items without end
    assert size(10 ** 6, 1, 64, 4, 1) <= 2048 * 64 * 8
    assert size(10 ** 6, 1, 4096, 1, 1) <= 2048 * 4096 * 8 + 10 ** 6 * 8 * 4
    # addresses that are not aligned take narrower vectors, whose cut may be another
    assert size(3, 61 * 97, 32, 8, 1, 1, 0) > 0 and size(3, 61 * 97, 32, 8, 1, 1, 2) > 0


def test_pixel_strides():
    from opendressi_amd.ops import _pixel_strides
    x = torch.zeros(4, 6, 5, 16)
    assert _pixel_strides(x) == (30, 480, 16)
    assert _pixel_strides(x[..., 4:8]) == (30, 480, 16)
    assert _pixel_strides(x[::2]) == (30, 960, 16)
    assert _pixel_strides(x[:, :1]) == (5, 480, 16)
    assert _pixel_strides(x[:, :, 1:2]) == (6, 480, 80)
    assert _pixel_strides(x[:, 0, 0]) == (1, 480, 16)
    assert _pixel_strides(x.expand(4, 6, 5, 16)[:1].expand(7, -1, -1, -1)) == (30, 0, 16)
    for other in (x[:, 1:4, 1:3], x.transpose(1, 2), x[..., ::2], x.permute(0, 3, 1, 2),
                  x[:, :1, :1].expand(-1, 6, 5, -1)):
        assert _pixel_strides(other) is None
    # pixels of one channel each, apart
    assert _pixel_strides(x[..., 3:4]) == (30, 480, 16)


def test_dense():
    from opendressi_amd.torch.optim import _dense, _flat
    x = torch.arange(24.0).view(2, 3, 4)
    for t in (x, x.transpose(0, 2), x[1], x.permute(2, 0, 1), torch.zeros(0, 3), torch.tensor(1.0),
              torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last)):
        assert _dense(t)
    for t in (x[:, ::2], x[..., 1:], x[:1].expand(2, 3, 4), x[:, :2]):
        assert not _dense(t)
    assert torch.equal(_flat(x.transpose(0, 2)), torch.arange(24.0))


def test_arguments_before_any_work():
    from opendressi_amd import ops as K
    ctx = types.SimpleNamespace(device=0)
    x = torch.zeros(2, 4, 4, 8)
    for args, err, what in (((x, 2), ValueError, "cuda:0"), ((x.double(), 2), TypeError, "float64"),
                            ((x, 3), ValueError, "whole groups"), ((x, 0), ValueError, "whole"),
                            ((x[0, 0, 0], 1), ValueError, "N, ..., C")):
        with pytest.raises(err, match=what):
            K.group_norm(ctx, *args)
    with pytest.raises(ValueError, match="activation"):
        K.group_norm(ctx, x, 2, activation="tanh")
