"""attention.norm_rotate's gradient of the weight, which is summed over blocks, to a bound that a lost
or doubled block passes.

A sum's longest chain of additions: a lane's own terms (few, as the blocks are as many as fill
the card), the lanes of a block that hold one feature (256 at most), every 32nd of the blocks
(2048 + one a group, 65 of them) and the 32 of these: under 400.  The sum is off by 400 float32
roundings of its terms' sizes, each term by its sines and cosines (2^-18 for 16-bit types, 2^-21
for float32, of the turned pair) and 16 roundings.
"""

from __future__ import annotations

import pytest
import torch

from attention_oracle import assert_within, rotation
from torchmatch_amd import attention as att

CHAIN, ULP = 400, 2.0**-24
CASES = [(2, 2500, (8,)), (3, 700, (5, 2, 1)), (1, 30011, (4, 2)), (40, 123, (6, 2))]
D, SECTIONS = 64, (16, 16)


def _inputs(dtype, b, n, heads):
    g = torch.Generator().manual_seed(17)
    x = (torch.randn(b, n, sum(heads), D, generator=g)
         * torch.randn(b, n, 1, 1, generator=g).exp()).to(dtype)
    w = 1 + 0.3 * torch.randn(len(heads), D, generator=g)
    pos = 50 * torch.rand(b, n, len(SECTIONS), generator=g)
    dy = torch.randn(b, n, sum(heads), D, generator=g).to(dtype)
    freqs = torch.cat([10000.0 ** (-torch.arange(s).float() / s) for s in SECTIONS])
    return x, w, pos, freqs, dy


def _oracle(x, pos, freqs, dy, heads, without=None):
    """dw and its bound in float64; ``without``: tokens whose terms are left out."""
    x, dy, dtype = x.double(), dy.double(), x.dtype
    g = rotation(dy, pos, freqs, SECTIONS, inverse=True)
    u = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    pairs = sum(SECTIONS)
    size = torch.cat([dy[..., :pairs].abs() + dy[..., pairs:2 * pairs].abs()] * 2, -1)
    sine = 2.0**-21 if dtype == torch.float32 else 2.0**-18
    off = sine * size * u.abs() + (16 + CHAIN) * ULP * (g * u).abs()
    terms = g * u
    if without is not None:
        terms = terms.flatten(0, 1).clone()
        terms[without] = 0
    rows = lambda t: torch.stack([p.reshape(-1, D).sum(0) for p in t.split(heads, -2)])  # noqa: E731
    value = rows(terms)
    return value, rows(off) + ULP * value.abs()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,n,heads", CASES)
def test_the_bound_sees_a_lost_block(dtype, b, n, heads):
    """Without one block's terms the value is past its bound: some tokens of a row of the weight, one
    at least."""
    x, _, pos, freqs, dy = _inputs(dtype, b, n, heads)
    value, bound = _oracle(x, pos, freqs, dy, heads)
    for lost in (slice(0, 4), slice(b * n // 2, b * n // 2 + 2), slice(b * n - 1, None)):
        less, _ = _oracle(x, pos, freqs, dy, heads, without=lost)
        assert ((value - less).abs() > bound).any(1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,n,heads", CASES)
def test_gradient_of_the_weight(device, dtype, b, n, heads):
    x, w, pos, freqs, dy = _inputs(dtype, b, n, heads)
    value, bound = _oracle(x, pos, freqs, dy, heads)
    leaf = w.to(device).requires_grad_(True)
    y = att.norm_rotate(x.to(device), leaf, pos.to(device), freqs.to(device), SECTIONS, heads=heads)
    (dw,) = torch.autograd.grad(y, leaf, dy.to(device))
    assert_within(dw, value, bound, "dw")
