"""The attention entries without a GPU: schemas, fake kernels, refusals, workspaces."""

from __future__ import annotations

import ctypes

import pytest
import torch

from torchmatch_amd import _native, attention


def _problem(**changes):
    fields = {"B": 2, "Lq": 300, "Lk": 500, "H": 8, "Hkv": 2, "D": 64, "dtype": _native.TM_BF16,
              "scale": 0.125, "q": 4096, "k": 4096, "v": 4096, "q_b": 64 * 8 * 300,
              "q_l": 64 * 8, "q_h": 64, "k_b": 64 * 2 * 500, "k_l": 64 * 2, "k_h": 64,
              "v_b": 64 * 2 * 500, "v_l": 64 * 2, "v_h": 64}
    fields.update(changes)
    return _native.Attention(**fields)


def _forward(**changes):
    a = _problem(**changes)
    return _native.lib().tm_attention_forward(ctypes.byref(a), 4096, None, None, None, 0, None)


@pytest.mark.parametrize("changes,code", [
    ({"B": -1}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"H": 7}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"H": 0}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"dtype": 3}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"D": 63}, _native.TM_ERR_UNSUPPORTED_SHAPE),
    ({"D": 264}, _native.TM_ERR_UNSUPPORTED_SHAPE),
    ({"scale": float("nan")}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"cap": -1.0}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"cap": 2000.0}, _native.TM_ERR_UNSUPPORTED_SHAPE),
    ({"q_docs": 4096}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"slopes": 4096, "q_positions": 4096, "axes": 1}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"q_positions": 4096, "k_positions": 4096, "axes": 1}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"slopes": 4096, "q_positions": 4096, "k_positions": 4096, "axes": 4},
     _native.TM_ERR_UNSUPPORTED_SHAPE),
    ({"k_l": 129}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"q": 4098}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"q": None}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"v_l": 1 << 26}, _native.TM_ERR_UNSUPPORTED_SHAPE),
    ({"Lq": 2, "B": 1, "Lk": 1 << 20}, _native.TM_ERR_WORKSPACE),
    ({"B": 1 << 20}, _native.TM_ERR_UNSUPPORTED_SHAPE),
    ({"Lk": (1 << 31) - 1}, _native.TM_ERR_UNSUPPORTED_SHAPE),
    ({"B": 0}, _native.TM_OK),
    ({"Lq": 0}, _native.TM_OK),
])
def test_refusals(changes, code):
    assert _forward(**changes) == code


@pytest.mark.parametrize("changes", [{"B": 0}, {"Lq": 0}, {"Lk": 0}, {"B": 0, "Lq": 1},
                                     {"Lq": 0, "Lk": 0}, {"B": 0, "q_docs": 4096, "k_docs": 4096}])
def test_workspaces_of_nothing(changes):
    """Sizes of zero have a workspace of their own size, not a division by zero blocks."""
    lib, a = _native.lib(), _problem(**changes)
    assert lib.tm_attention_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.tm_attention_backward_workspace_bytes(ctypes.byref(a)) <= 2 * 256 * 75


def test_workspaces_of_split_key_gradients():
    """Few key blocks: float32 parts of dk and dv; many: none."""
    size = lambda **c: _native.lib().tm_attention_backward_workspace_bytes(  # noqa: E731
        ctypes.byref(_problem(**c)))
    sums = lambda b, lq: 2 * ((b * 8 * lq * 4 + 255) // 256 * 256)  # noqa: E731
    part = 2 * 500 * 2 * 64 * 4  # of one split
    assert (size() - sums(2, 300)) % (2 * part) == 0 and size() - sums(2, 300) >= 2 * 2 * part
    assert size(B=64) == sums(64, 300)
    assert size(Lk=0) == sums(2, 300)


def test_workspaces():
    lib = _native.lib()
    size = lambda **c: lib.tm_attention_workspace_bytes(ctypes.byref(_problem(**c)))  # noqa: E731
    assert size(B=64) == 0  # enough rows: nothing is split
    assert size(B=64, q_docs=4096, k_docs=4096) >= 64 * (5 + 8) * 16
    one = size(B=1, Lq=1, Lk=1 << 20)
    assert one >= 2 * 8 * 64 * 4  # partial results of a split over keys
    back = lib.tm_attention_backward_workspace_bytes(ctypes.byref(_problem()))
    assert back >= 2 * 2 * 8 * 300 * 4
    assert lib.tm_attention_max_head_dim() == 256


def test_rotation_refusals():
    lib = _native.lib()

    def rotate(sections=(16, 16), **changes):
        fields = {"x": 4096, "positions": 4096, "freqs": 4096, "B": 1, "L": 4, "H": 2, "D": 64,
                  "axes": len(sections), "dtype": _native.TM_F32, "x_l": 128, "x_h": 64}
        fields.update(changes)
        r = _native.Rotation(**fields)
        for i, n in enumerate(sections):
            r.sections[i] = n
        return lib.tm_rotate(ctypes.byref(r), 4096, None)

    assert rotate(B=0) == _native.TM_OK
    assert rotate((16, 17)) == _native.TM_ERR_INVALID_ARGUMENT
    assert rotate((-1, 8)) == _native.TM_ERR_INVALID_ARGUMENT
    assert rotate(axes=0) == _native.TM_ERR_INVALID_ARGUMENT
    assert rotate(axes=5) == _native.TM_ERR_INVALID_ARGUMENT
    assert rotate(pos_type=3) == _native.TM_ERR_INVALID_ARGUMENT
    assert rotate(freqs=None) == _native.TM_ERR_INVALID_ARGUMENT
    assert rotate(H=1 << 20) == _native.TM_ERR_UNSUPPORTED_SHAPE


def test_no_host_fallback():
    x = torch.rand(1, 3, 2, 16)
    with pytest.raises(ValueError, match="ROCm"):
        attention.attend(x, x, x)
    with pytest.raises(NotImplementedError):
        torch.ops.attention.attend(x, x, x, scale=1.0)
    with pytest.raises(NotImplementedError):
        torch.ops.attention.rotate(x, torch.rand(1, 3, 1), torch.rand(8), [8])
    with pytest.raises(TypeError, match="tensor"):
        attention.attend([1.0], x, x)
    with pytest.raises(ValueError, match="theta"):
        attention.rotary_frequencies((4,), theta=0.0, device="cpu")


def test_ops_are_the_registered_ones():
    for name in attention.ops.__all__:
        assert getattr(attention.ops, name) is getattr(torch.ops.attention, name)
    f = attention.rotary_frequencies((2, 3), theta=100.0, device="cpu")
    want = torch.tensor([1.0, 0.1, 1.0, 100 ** (-1 / 3), 100 ** (-2 / 3)])
    torch.testing.assert_close(f, want)


def test_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q = torch.empty(2, 7, 4, 16, dtype=torch.bfloat16, device="cuda")
        k = torch.empty(2, 9, 2, 16, dtype=torch.bfloat16, device="cuda")
        out, lse = torch.ops.attention.attend(q, k, k, scale=1.0)
        assert out.shape == q.shape and out.dtype == q.dtype
        assert lse.shape == (2, 4, 7) and lse.dtype == torch.float32
        out, low, lse = torch.ops.attention.attend_forward(q, k, k, scale=1.0)
        assert low.shape == q.shape
        grads = torch.ops.attention.attend_backward(out, q, k, k, out, low, lse, scale=1.0)
        assert [g.shape for g in grads] == [q.shape, k.shape, k.shape]
        y = torch.ops.attention.rotate(q, torch.empty(2, 7, 1, device="cuda"),
                                       torch.empty(8, device="cuda"), [8])
        assert y.shape == q.shape
