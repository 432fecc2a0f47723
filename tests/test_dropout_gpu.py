"""attention.dropout on the GPU against the generator in numpy."""

from __future__ import annotations

import pytest
import torch

from attention_oracle import assert_within
from layers_oracle import dropout, stays
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rand(dtype, *shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p", [0.0, 2.0**-33, 0.1, 0.5, 0.999, 1.0 - 2.0**-33, 1.0])
@pytest.mark.parametrize("added", [False, True])
def test_values_and_gradients(device, dtype, p, added):
    x, r, dy = (_rand(dtype, 3, 7, 33, seed=s).to(device) for s in range(3))
    x.requires_grad_(True)
    r = r.requires_grad_(True) if added else None
    y = att.dropout(x, p, 1234567, 5, residual=r)
    assert y.dtype == dtype and y.is_contiguous()
    nothing = round(p * 2**32) >= 2**32
    want = dropout(x, 1.0 if nothing else p, 1234567, 5, r)
    assert_within(y, *want, "y")
    grads = torch.autograd.grad(y, (x, r) if added else (x,), dy)
    assert_within(grads[0], *dropout(dy, 1.0 if nothing else p, 1234567, 5), "dx")
    if added:
        assert torch.equal(grads[1], dy)
    if p == 0.0 and not added:
        assert torch.equal(y, x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [0, 1, 3, 4, 5, 7, 8, 9, 15, 16, 17, 255, 2047, 2049, 100003])
def test_lengths(device, dtype, count):
    x = _rand(dtype, count).to(device)
    y = att.dropout(x, 0.3, -1, 2**63 + 11)
    assert_within(y, *dropout(x, 0.3, -1, 2**63 + 11), "y")


@pytest.mark.parametrize("dtype", DTYPES)
def test_mask_goes_by_place(device, dtype):
    """Whatever the strides, the alignment, the residual and the type."""
    x = _rand(dtype, 6, 40).to(device).abs() + 1
    want = att.dropout(x, 0.4, 7)
    assert torch.equal(att.dropout(x.t().contiguous().t(), 0.4, 7), want)
    odd = torch.empty(241, dtype=dtype, device=device)[1:].view(6, 40).copy_(x)
    assert torch.equal(att.dropout(odd, 0.4, 7), want)
    assert torch.equal(att.dropout(x, 0.4, 7, residual=odd * 0), want)
    assert torch.equal(att.dropout(x[:1].expand(6, 40), 0.4, 7) != 0, want != 0)
    assert torch.equal(att.dropout(x.float(), 0.4, 7) != 0, want != 0)
    assert torch.equal(att.dropout(x, 0.4, 7).view(2, 3, 40), att.dropout(x.view(2, 3, 40), 0.4, 7))
    assert not torch.equal(att.dropout(x, 0.4, 8), want)
    assert not torch.equal(att.dropout(x, 0.4, 7, 1), want)


def test_seed_on_the_device(device):
    x = _rand(torch.float16, 5, 1001).to(device).requires_grad_(True)
    for seed in (0, 2**40 + 3, -5):
        at = torch.tensor([seed], device=device)
        y, z = att.dropout(x, 0.2, at, 9), att.dropout(x, 0.2, seed, 9)
        assert torch.equal(y, z)
        assert torch.equal(torch.autograd.grad(y.sum(), x)[0],
                           torch.autograd.grad(z.sum(), x)[0])
    y = att.dropout(x, 0.2, at)
    at += 1  # another mask than the forward pass's: refused, not wrong
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)


def test_captured(device):
    """A captured step follows the seed on the device from replay to replay."""
    x = _rand(torch.bfloat16, 4, 300, 8).to(device).requires_grad_(True)
    seed, dy = torch.zeros((), dtype=torch.int64, device=device), torch.randn_like(x)

    def once():
        y = att.dropout(x, 0.1, seed, 3, residual=dy)
        return (y.detach(), *torch.autograd.grad(y, x, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    masks = []
    for _ in range(3):
        seed += 1
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, once()):
            assert torch.equal(a, b)
        masks.append(got[1] != 0)
    assert not torch.equal(masks[0], masks[1]) and not torch.equal(masks[1], masks[2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_and_infinity_that_are_left_out(device, dtype):
    x = torch.full((64,), float("nan"), dtype=dtype, device=device)
    x[::2] = float("inf")
    keep = stays(0, 64, 0.5, 3, 0).to(device)
    y = att.dropout(x, 0.5, 3)
    assert not y[~keep].any() and not y[keep].isfinite().any()


def test_more_than_32_bits_of_elements(device):
    """The counter's second word, and offsets past 2^32."""
    count = 2**34 + 21
    x = torch.ones(count, dtype=torch.bfloat16, device=device)
    y = att.dropout(x, 0.25, 99, 1)
    for first, n in ((0, 1000), (2**32 - 500, 1000), (2**34 - 500, 521)):
        keep = stays(first, n, 0.25, 99, 1).to(device)
        assert torch.equal(y[first:first + n] != 0, keep)


def test_share_left_out(device):
    """1e6 elements at p: the share's standard deviation is sqrt(p (1 - p) / 1e6); six of them."""
    x = torch.ones(1_000_000, device=device)
    for p in (0.01, 0.1, 0.5, 0.9):
        gone = (att.dropout(x, p, 42) == 0).double().mean().item()
        assert abs(gone - p) <= 6 * (p * (1 - p) / 1e6) ** 0.5


def test_second_derivatives_and_tangents(device):
    x, r, t, s = (_rand(torch.float32, 50, seed=n).to(device) for n in range(4))
    x.requires_grad_(True)
    y = att.dropout(x, 0.3, 5)
    (g,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    (h,) = torch.autograd.grad(g.sum(), x)
    keep = stays(0, 50, 0.3, 5, 0).to(device)
    torch.testing.assert_close(h, keep * 2 / 0.7**2, rtol=1e-6, atol=0)
    x = x.detach()
    fn = lambda x, r: att.dropout(x, 0.3, 5, residual=r)  # noqa: E731
    y, tangent = torch.func.jvp(fn, (x, r), (t, s))
    assert torch.equal(y, fn(x, r)) and torch.equal(tangent, fn(t, s))
    _, tangent = torch.func.jvp(lambda r: fn(x, r), (r,), (s,))
    assert torch.equal(tangent, s)
    _, tangent = torch.func.jvp(lambda x: fn(x, r), (x,), (t,))
    assert torch.equal(tangent, att.dropout(t, 0.3, 5))


def test_refused(device):
    x = torch.randn(4, 8, device=device)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="p must be"):
            att.dropout(x, p, 0)
    with pytest.raises(TypeError, match="float32"):
        att.dropout(x.double(), 0.1, 0)
    with pytest.raises(ValueError, match="ROCm"):
        att.dropout(x.cpu(), 0.1, 0)
    with pytest.raises(ValueError, match="64 bits"):
        att.dropout(x, 0.1, 2**64)
    with pytest.raises(TypeError, match="int64"):
        att.dropout(x, 0.1, torch.zeros((), dtype=torch.int32, device=device))
    with pytest.raises(ValueError, match="one number"):
        att.dropout(x, 0.1, torch.zeros(2, dtype=torch.int64, device=device))
    with pytest.raises(ValueError, match="one number"):
        att.dropout(x, 0.1, torch.zeros((), dtype=torch.int64))
    with pytest.raises(ValueError, match="residual"):
        att.dropout(x, 0.1, 0, residual=x[:2])
    with pytest.raises(TypeError, match="residual"):
        att.dropout(x, 0.1, 0, residual=x.half())


def test_opcheck(device):
    x, r = (torch.randn(3, 5, device=device, requires_grad=True) for _ in range(2))
    seed = torch.tensor(3, device=device)
    for args in ((x, 0.1, 4, 2), (x, 0.1, 0, 0, seed, r)):
        torch.library.opcheck(torch.ops.attention.dropout.default, args,
                              test_utils=("test_schema", "test_faketensor",
                                          "test_aot_dispatch_dynamic"))
