"""attention.rotate on the GPU against the 64-bit oracle."""

from __future__ import annotations

import pytest
import torch

from attention_oracle import UNIT, assert_within, rotation
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _bound(x, y, dtype):
    """The result's rounding, and 2^-18 (16-bit types: hardware sines) or 2^-21 of the
    pair's size for the sines and products."""
    size = x.double().cpu().abs().amax(-1, keepdim=True) * 2
    return UNIT[dtype] * y.abs() + (2.0**-21 if dtype == torch.float32 else 2.0**-18) * size


def _check(x, pos, sections, **kw):
    freqs = att.rotary_frequencies(sections)
    y = att.rotate(x, pos, freqs, sections, **kw)
    want = rotation(x, pos if pos.ndim == 3 else pos.expand(x.shape[0], *pos.shape), freqs,
                    sections, **kw)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    assert_within(y, want, _bound(x, want, x.dtype), "y")
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,sections", [(64, (32,)), (128, (16, 24, 24)), (64, (16, 16)),
                                        (96, (8, 8)), (128, (8, 0, 24)), (32, (3, 5, 2)),
                                        (10, (5,)), (6, (1,)), (7, (3,)), (256, (30, 32, 33, 33))])
def test_sections(device, dtype, interleaved, d, sections):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 37, 3, d, generator=g).to(dtype).to(device)
    pos = (100 * torch.rand(2, 37, len(sections), generator=g)).to(device)
    _check(x, pos, sections, interleaved=interleaved)
    _check(x, pos, sections, interleaved=interleaved, inverse=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,n,h", [(1, 1, 1), (1, 1, 40), (8, 1, 40), (1, 4097, 1), (3, 700, 5),
                                   (2, 5000, 8)])
def test_shapes(device, dtype, b, n, h):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(b, n, h, 64, generator=g).to(dtype).to(device)
    pos = torch.randint(0, 50, (b, n, 2), generator=g).to(device)
    _check(x, pos, (16, 16))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_position_types_and_far_positions(device, dtype, kind):
    x = torch.randn(1, 64, 2, 64, device=device).to(dtype)
    pos = torch.arange(64, device=device).view(1, 64, 1) * 16381 + 1_000_000
    _check(x, pos.to(kind), (32,))
    _check(x, -pos.to(kind), (32,))
    _check(x, pos.to(kind)[0], (32,))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(device, dtype):
    x = torch.randn(2, 50, 8, 64, device=device).to(dtype)
    pos = torch.rand(2, 50, 1, device=device)
    freqs = att.rotary_frequencies((32,))
    want = att.rotate(x[:, :, :5].contiguous(), pos, freqs, (32,))
    assert torch.equal(att.rotate(x[:, :, :5], pos, freqs, (32,)), want)
    t = x[:, :, :5].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(att.rotate(t, pos, freqs, (32,)), want)
    t = x[:, :, :5].permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)
    assert torch.equal(att.rotate(t, pos, freqs, (32,)), want)
    t = torch.empty(2, 50, 5, 67, dtype=dtype, device=device)[..., 1:65].copy_(x[:, :, :5])
    assert torch.equal(att.rotate(t, pos, freqs, (32,)), want)
    one = x[:1, :, :5].expand(2, -1, -1, -1)
    assert torch.equal(att.rotate(one, pos[:1].expand(2, -1, -1), freqs, (32,))[1], want[0])
    wide = torch.rand(2, 50, 3, device=device)
    wide[..., 1:2] = pos
    assert torch.equal(att.rotate(x[:, :, :5], wide[..., 1:2], freqs, (32,)), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(device, dtype, interleaved):
    x = torch.randn(2, 30, 3, 80, device=device).to(dtype).requires_grad_(True)
    pos = 30 * torch.rand(2, 30, 2, device=device)
    freqs = att.rotary_frequencies((8, 16))
    dy = torch.randn(2, 30, 3, 80, device=device).to(dtype)
    y = att.rotate(x, pos, freqs, (8, 16), interleaved=interleaved)
    (dx,) = torch.autograd.grad(y, x, dy)
    want = rotation(dy, pos, freqs, (8, 16), interleaved=interleaved, inverse=True)
    assert_within(dx, want, _bound(dy, want, dtype), "dx")
    # the gradient of a plain sum has stride 0
    (dx,) = torch.autograd.grad(
        att.rotate(x, pos, freqs, (8, 16), interleaved=interleaved).sum(), x)
    one = torch.ones_like(dy)
    want = rotation(one, pos, freqs, (8, 16), interleaved=interleaved, inverse=True)
    assert_within(dx, want, _bound(one, want, dtype), "dx of a sum")


def test_gradient_against_differences(device):
    """The rotation is linear: a difference is the derivative but for the float32 roundings
    of two sums, 2^-20 of their terms each."""
    x = torch.randn(1, 9, 2, 32, device=device)
    way = torch.randn(1, 9, 2, 32, device=device)
    w = torch.randn(1, 9, 2, 32, device=device).double()
    pos = 30 * torch.rand(1, 9, 1, device=device)
    freqs = att.rotary_frequencies((16,))

    def value(t):
        return (att.rotate(t, pos, freqs, (16,)).double() * w).sum()

    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(value(leaf), leaf)
    slope = (value(x + way) - value(x - way)) / 2
    assert (slope - (g.double() * way.double()).sum()).abs() <= 2.0**-19 * w.abs().sum() * 8


def test_captured(device):
    x = torch.randn(2, 3, 8, 64, device=device)
    pos = torch.rand(2, 3, 2, device=device)
    freqs = att.rotary_frequencies((16, 16))
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        att.rotate(x, pos, freqs, (16, 16))
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        y = att.rotate(x, pos, freqs, (16, 16))
    for _ in range(3):
        x.normal_()
        pos.uniform_(0, 9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, att.rotate(x, pos, freqs, (16, 16)))


def test_empty_and_refused(device):
    f = att.rotary_frequencies((4, 4))
    x = torch.randn(2, 3, 2, 16, device=device)
    pos = torch.zeros(2, 3, 2, device=device)
    assert att.rotate(x[:0], pos[:0], f, (4, 4)).shape == (0, 3, 2, 16)
    assert att.rotate(x[:, :0], pos[:, :0], f, (4, 4)).shape == (2, 0, 2, 16)
    assert torch.equal(att.rotate(x, pos[..., :1], f[:0], (0,)), x)
    with pytest.raises(ValueError, match="ROCm"):
        att.rotate(x.cpu(), pos, f, (4, 4))
    with pytest.raises(ValueError, match="4D"):
        att.rotate(x[0], pos, f, (4, 4))
    with pytest.raises(TypeError, match="float32"):
        att.rotate(x.double(), pos, f, (4, 4))
    with pytest.raises(ValueError, match="positions must be"):
        att.rotate(x, pos[:, :2], f, (4, 4))
    with pytest.raises(TypeError, match="int32"):
        att.rotate(x, pos.double(), f, (4, 4))
    with pytest.raises(ValueError, match="half"):
        att.rotate(x, pos, att.rotary_frequencies((4, 5)), (4, 5))
    with pytest.raises(ValueError, match="freqs"):
        att.rotate(x, pos, f[:7], (4, 4))
    with pytest.raises(ValueError, match="sections"):
        att.rotate(x, pos.repeat(1, 1, 3)[..., :5], f, (1, 1, 1, 1, 4))
    with pytest.raises(NotImplementedError, match="positions"):
        att.rotate(x, pos.clone().requires_grad_(True), f, (4, 4))
