"""The layer's operators without a GPU: the generator, schemas, fake kernels, refusals, workspaces."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from layers_oracle import philox
from torchmatch_amd import _native, attention


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_the_generator_is_the_published_one(counter, key, want):
    """The known answers that its authors published with it."""
    assert tuple(philox(np.array([counter], dtype=np.uint64), key)[0]) == want


def _normed(**changes):
    sections, heads = changes.pop("sections", (16, 16)), changes.pop("heads", (2, 1))
    rotation = {"x": 4096, "positions": 4096, "freqs": 4096, "B": 1, "L": 4, "H": 3, "D": 64,
                "axes": len(sections), "dtype": _native.TM_BF16, "x_l": 192, "x_h": 64}
    fields = {"weight": 4096, "weight_type": _native.TM_BF16, "groups": len(heads), "eps": 1e-6}
    for name, value in changes.items():
        (rotation if name in dict(_native.Rotation._fields_) else fields)[name] = value
    r = _native.Rotation(**rotation)
    for i, n in enumerate(sections):
        r.sections[i] = n
    a = _native.NormRotation(rotation=r, **fields)
    for i, n in enumerate(heads):
        a.heads[i] = n
    return a


@pytest.mark.parametrize("changes,code", [
    ({"B": 0}, _native.TM_OK),
    ({"L": 0}, _native.TM_OK),
    ({"B": -1}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"H": 2}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"H": 4}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"heads": (3, 0)}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"heads": (2**31 - 1, 2**31 - 1)}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"groups": 0}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"groups": 9}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"eps": -1.0}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"eps": float("nan")}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"eps": float("inf")}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"inverse": 1}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"weight_type": _native.TM_F16}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"sections": (16, 17)}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"axes": 5}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"pos_type": 3}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"x": None}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"D": 513}, _native.TM_ERR_UNSUPPORTED_SHAPE),
    ({"H": 65537, "D": 1, "sections": (0,), "heads": (65537,)}, _native.TM_ERR_UNSUPPORTED_SHAPE),
])
def test_norm_rotate_refusals(changes, code):
    a = _normed(**changes)
    assert _native.lib().tm_norm_rotate(ctypes.byref(a), 4096, None) == code


def test_norm_rotate_backward_refusals():
    lib = _native.lib()
    size = lib.tm_norm_rotate_backward_workspace_bytes(ctypes.byref(_normed()))
    assert size >= 2 * 64 * 4

    def back(dx=4096, dw=4096, ws=4096, bytes_=size, dout=4096, **changes):
        a = _normed(**changes)
        return lib.tm_norm_rotate_backward(ctypes.byref(a), dout, 768, 192, 64, dx, dw, ws,
                                           bytes_, None)

    assert back(bytes_=size - 1) == _native.TM_ERR_WORKSPACE
    assert back(ws=None) == _native.TM_ERR_WORKSPACE
    assert back(ws=4098) == _native.TM_ERR_WORKSPACE
    assert back(dout=None) == _native.TM_ERR_INVALID_ARGUMENT
    assert back(weight=None) == _native.TM_ERR_INVALID_ARGUMENT
    assert back(dx=None, dw=None) == _native.TM_OK
    assert back(dw=None, B=0) == _native.TM_OK


def _block(**changes):
    fields = {"x": 4096, "gate": 4096, "up": 4096, "down": 4096, "x_l": 64, "w_l": 64,
              "down_l": 96, "dtype": _native.TM_BF16, "activation": _native.TM_SILU, "T": 10,
              "C": 64, "F": 96, "O": 32}
    fields.update(changes)
    return _native.FeedForward(**fields)


@pytest.mark.parametrize("changes,code", [
    ({"T": 0}, _native.TM_OK),
    ({"T": -1}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"C": 0}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"F": 0}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"O": -5}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"dtype": 3}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"activation": 4}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"x": 4098}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"gate": None}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"x_l": 68}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"w_l": 56}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"down_l": -96}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"x_l": 1 << 22}, _native.TM_ERR_UNSUPPORTED_SHAPE),
    ({"T": 2**31 - 1}, _native.TM_ERR_UNSUPPORTED_SHAPE),
    ({"T": 1 << 30, "O": 1 << 20}, _native.TM_ERR_UNSUPPORTED_SHAPE),
    ({}, _native.TM_ERR_WORKSPACE),
])
def test_feed_forward_refusals(changes, code):
    f = _block(**changes)
    assert _native.lib().tm_feed_forward_forward(ctypes.byref(f), 4096, None, None, 0,
                                                 None) == code


def test_feed_forward_backward_refusals():
    lib = _native.lib()
    size = lib.tm_feed_forward_backward_workspace_bytes(ctypes.byref(_block()))
    assert size >= 2 * 10 * 96 * 2

    def back(saved=4096, dout=4096, do_l=32, dx=4096, dgate=4096, dup=4096, ddown=4096, ws=4096,
             bytes_=size, **changes):
        f = _block(**changes)
        return lib.tm_feed_forward_backward(ctypes.byref(f), saved, dout, do_l, dx, dgate, dup,
                                            ddown, ws, bytes_, None)

    assert back(bytes_=size - 1) == _native.TM_ERR_WORKSPACE
    assert back(ws=None) == _native.TM_ERR_WORKSPACE
    assert back(ws=4098) == _native.TM_ERR_WORKSPACE
    assert back(dgate=None) == _native.TM_ERR_INVALID_ARGUMENT
    assert back(do_l=31) == _native.TM_ERR_INVALID_ARGUMENT
    assert back(do_l=24) == _native.TM_ERR_INVALID_ARGUMENT
    assert back(saved=None) == _native.TM_ERR_INVALID_ARGUMENT
    assert back(dout=None) == _native.TM_ERR_INVALID_ARGUMENT
    assert back(do_l=1 << 22) == _native.TM_ERR_UNSUPPORTED_SHAPE
    assert back(dx=None, dgate=None, dup=None, ddown=None) == _native.TM_OK
    assert back(dgate=None, dup=None, ddown=None, T=0) == _native.TM_OK


def test_pad_rows_refusals():
    pad = lambda x=4096, l=5, rows=3, n=5, dtype=0, out=4096: _native.lib().tm_pad_rows(  # noqa: E731
        x, l, rows, n, dtype, out, None)
    assert pad(rows=0) == _native.TM_OK
    for bad in ({"rows": -1}, {"n": 0}, {"dtype": 3}, {"out": 4098}, {"x": None}, {"out": None}):
        assert pad(**bad) == _native.TM_ERR_INVALID_ARGUMENT
    assert pad(rows=1 << 40) == _native.TM_ERR_UNSUPPORTED_SHAPE


def test_feed_forward_sizes():
    lib = _native.lib()
    saved = lambda **c: lib.tm_feed_forward_saved_bytes(ctypes.byref(_block(**c)))  # noqa: E731
    assert saved() == 10 * 96 * 8 and saved(dtype=_native.TM_F32) == 10 * 96 * 12
    assert saved(F=90, down_l=96) == 10 * 96 * 8
    assert saved(T=0) == 0
    size = lib.tm_feed_forward_workspace_bytes(ctypes.byref(_block()))
    assert size >= 10 * 96 * 2
    assert lib.tm_feed_forward_workspace_bytes(ctypes.byref(_block(T=0))) == 0


def test_dropout_refusals():
    drop = lambda x=4096, out=4096, n=8, dtype=0, p=0.5: _native.lib().tm_dropout(  # noqa: E731
        x, None, out, n, dtype, p, 0, None, 0, None)
    assert drop(n=0) == _native.TM_OK
    assert drop(n=-1) == _native.TM_ERR_INVALID_ARGUMENT
    assert drop(x=None) == _native.TM_ERR_INVALID_ARGUMENT
    assert drop(out=None) == _native.TM_ERR_INVALID_ARGUMENT
    assert drop(dtype=3) == _native.TM_ERR_INVALID_ARGUMENT
    for p in (-0.1, 1.5, float("nan")):
        assert drop(p=p) == _native.TM_ERR_INVALID_ARGUMENT


def test_no_host_fallback():
    x = torch.rand(1, 3, 2, 16)
    with pytest.raises(ValueError, match="ROCm"):
        attention.norm_rotate(x, None, torch.rand(1, 3, 1), torch.rand(8), (8,))
    with pytest.raises(ValueError, match="ROCm"):
        attention.dropout(x, 0.1, 0)
    with pytest.raises(TypeError, match="tensor"):
        attention.dropout([1.0], 0.1, 0)
    with pytest.raises(NotImplementedError):
        torch.ops.attention.dropout(x, 0.1)


def test_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(2, 7, 4, 16, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(2, 16, device="cuda")
        pos, f = torch.empty(2, 7, 1, device="cuda"), torch.empty(8, device="cuda")
        y = torch.ops.attention.norm_rotate(x, w, pos, f, [8], [3, 1], 1e-6)
        assert y.shape == x.shape and y.dtype == x.dtype
        dx, dw = torch.ops.attention.norm_rotate_backward(y, x, w, pos, f, [8], [3, 1], 1e-6)
        assert dx.shape == x.shape and dw.shape == w.shape and dw.dtype == torch.float32
        assert torch.ops.attention.dropout(x, 0.1, residual=x).shape == x.shape
        w, d = (torch.empty(n, m, dtype=torch.bfloat16, device="cuda")
                for n, m in ((20, 16), (5, 20)))
        y = torch.ops.attention.feed_forward(x, w, w, d, "silu")
        assert y.shape == (2, 7, 4, 5) and y.dtype == x.dtype
        _, saved = torch.ops.attention.feed_forward_save(x, w, w, d, "silu")
        assert saved.shape == (56 * 24 * 8,) and saved.dtype == torch.uint8
        grads = torch.ops.attention.feed_forward_backward(y, x, w, w, d, saved, "silu",
                                                          need_up=False)
        assert [g.shape for g in grads] == [x.shape, w.shape, (0,), d.shape]


def test_tangents_without_a_device():
    """Where a tangent goes is seen on meta tensors."""
    import torch.autograd.forward_ad as fw

    meta = lambda *s: torch.randn(*s, device="meta")  # noqa: E731
    x, pos, f = meta(1, 4, 2, 16), meta(1, 4, 1), meta(8)
    drop, norm = torch.ops.attention.dropout, torch.ops.attention.norm_rotate
    with fw.dual_level():
        dual = fw.make_dual(x, meta(1, 4, 2, 16))
        assert fw.unpack_dual(drop(dual, 0.1)).tangent.shape == x.shape
        assert fw.unpack_dual(drop(x, 0.1, residual=dual)).tangent.shape == x.shape
        assert fw.unpack_dual(drop(x, 0.1, residual=x)).tangent is None
        with pytest.raises(NotImplementedError, match="forward"):
            norm(dual, None, pos, f, [8], [2], 1e-6)
        with pytest.raises(NotImplementedError, match="forward"):
            norm(x, fw.make_dual(meta(1, 16), meta(1, 16)), pos, f, [8], [2], 1e-6)
        with pytest.raises(NotImplementedError, match="positions"):
            norm(x, None, fw.make_dual(pos, meta(1, 4, 1)), f, [8], [2], 1e-6)
