"""Forward-mode differentiation: rotate has it (it is linear), attend refuses it, and no tangent
is dropped.  Fake kernels on meta tensors are enough to see where a tangent goes."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

from attention_oracle import UNIT, assert_within, rotation
from torchmatch_amd import attention as att

ATTEND, ROTATE = torch.ops.attention.attend, torch.ops.attention.rotate


def _meta(*shape):
    return torch.randn(*shape, device="meta")


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [False, True])
def test_attend_refuses_tangents(which, grad):
    with fw.dual_level():
        t = [_meta(1, 4, 2, 16).requires_grad_(grad) for _ in range(3)]
        t[which] = fw.make_dual(t[which], _meta(1, 4, 2, 16))
        with pytest.raises(NotImplementedError, match="forward"):
            ATTEND(*t, scale=1.0)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
            ATTEND(*t, scale=1.0)


def test_attend_refuses_tangents_of_constants():
    q = _meta(1, 4, 2, 16)
    with fw.dual_level():
        slopes = fw.make_dual(_meta(2), _meta(2))
        with pytest.raises(NotImplementedError, match="slopes"):
            ATTEND(q, q, q, slopes, scale=1.0)
    pos = _meta(1, 4, 1)
    with fw.dual_level():
        dual = fw.make_dual(pos, _meta(1, 4, 1))
        with pytest.raises(NotImplementedError, match="q_positions"):
            ATTEND(q, q, q, _meta(2), dual, pos, scale=1.0)
        with pytest.raises(NotImplementedError, match="k_positions"):
            ATTEND(q, q, q, _meta(2), pos, dual, scale=1.0)


def test_jvp_of_attend_is_refused():
    q = _meta(1, 4, 2, 16)
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(lambda x: ATTEND(x, q, q, scale=1.0)[0], (q,), (q,))


@pytest.mark.parametrize("grad", [False, True])
def test_rotate_keeps_tangents(grad):
    x, pos, freqs = _meta(1, 4, 2, 16), _meta(1, 4, 1), _meta(8)
    with fw.dual_level():
        y = ROTATE(fw.make_dual(x.requires_grad_(grad), _meta(1, 4, 2, 16)), pos, freqs, [8])
        tangent = fw.unpack_dual(y).tangent
        assert tangent is not None and tangent.shape == x.shape
        assert y.requires_grad == grad
        plain = ROTATE(x, pos, freqs, [8])
        assert fw.unpack_dual(plain).tangent is None
    with fw.dual_level(), pytest.raises(NotImplementedError, match="positions"):
        ROTATE(x, fw.make_dual(pos, _meta(1, 4, 1)), freqs, [8])
    with fw.dual_level(), pytest.raises(NotImplementedError, match="freqs"):
        ROTATE(x, pos, fw.make_dual(freqs, _meta(8)), [8])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_tangents_of_rotate(device, dtype, interleaved):
    x, t = (torch.randn(2, 30, 3, 80, device=device).to(dtype) for _ in range(2))
    pos = 30 * torch.rand(2, 30, 2, device=device)
    freqs = att.rotary_frequencies((8, 16))

    def turn(x):
        return att.rotate(x, pos, freqs, (8, 16), interleaved=interleaved)

    want = rotation(t, pos, freqs, (8, 16), interleaved=interleaved)
    # the result's rounding, and 2^-18 (hardware sines) or 2^-21 of the pair's size
    bound = UNIT[dtype] * want.abs() + (2.0**-21 if dtype == torch.float32 else 2.0**-18) * \
        2 * t.double().cpu().abs().amax(-1, keepdim=True)
    y, tangent = torch.func.jvp(turn, (x,), (t,))
    assert torch.equal(y, turn(x))
    assert_within(tangent, want, bound, "tangent")
    with fw.dual_level():
        dual = fw.unpack_dual(turn(fw.make_dual(x, t)))
    assert torch.equal(dual.tangent, tangent) and torch.equal(dual.primal, y)


@pytest.mark.gpu
def test_attend_refuses_tangents_on_the_device(device):
    q, k, v = (torch.randn(1, 8, 2, 32, device=device) for _ in range(3))
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(lambda x: att.attend(x, k, v), (q,), (q,))
