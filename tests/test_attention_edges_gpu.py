"""Calls at the edge of attention.attend's arguments: sets without points, batches of
millions of short rows, limits past 32 bits,
numbers that float32 does not hold."""

from __future__ import annotations

import pytest
import torch

from attention_oracle import assert_within, attention, visible
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("b,lq,lk", [(0, 3, 4), (2, 0, 4), (2, 3, 0), (2, 0, 0), (2, 40, 0),
                                     (2, 0, 200)])
@pytest.mark.parametrize("axes", [1, 2, 3])
@pytest.mark.parametrize("docs", [False, True])
def test_empty_sets_with_positions(device, b, lq, lk, axes, docs):
    """A set without points, or without points to match: zeros, and gradients of zero."""
    q, k, v = (torch.randn(b, n, 2, 32, device=device, requires_grad=True) for n in (lq, lk, lk))
    kw = {"slopes": torch.ones(2, device=device),
          "q_positions": torch.rand(b, lq, axes, device=device),
          "k_positions": torch.rand(b, lk, axes, device=device)}
    if docs:
        kw["q_docs"] = torch.zeros(b, lq, dtype=torch.int32, device=device)
        kw["k_docs"] = torch.zeros(b, lk, dtype=torch.int32, device=device)
    out, lse = att.attend(q, k, v, return_lse=True, **kw)
    assert out.shape == (b, lq, 2, 32) and (out == 0).all() and lse.isneginf().all()
    out.sum().backward()
    for t in (q, k, v):
        assert t.grad.shape == t.shape and (t.grad == 0).all()


@pytest.mark.parametrize("b,lq,lk", [(1 << 22, 2, 3), ((1 << 22) - 1, 1, 130),
                                     ((1 << 23) // 5, 130, 1)])
def test_millions_of_short_rows_of_documents(device, b, lq, lk):
    """As many batch rows as the limit on blocks admits, or half of it: each as in a call of a
    few rows, forward and backward."""
    d = 8
    g = torch.Generator(device=device).manual_seed(1)
    q, k, v, do = (torch.randn(b, n, 1, d, device=device, generator=g).half()
                   for n in (lq, lk, lk, lq))
    q_docs, k_docs = (torch.randint(-1, 2, (b, n), device=device, generator=g, dtype=torch.int32)
                      for n in (lq, lk))

    def run(rows):
        t = [x[rows].clone().requires_grad_(True) for x in (q, k, v)]
        out = att.attend(*t, q_docs=q_docs[rows], k_docs=k_docs[rows])
        return (out.detach(), *torch.autograd.grad(out, t, do[rows]))

    every = run(slice(0, b))
    for first in (0, b // 2 - 500, b - 1000):
        rows = slice(first, first + 1000)
        for x, y in zip(every, run(rows)):
            assert torch.equal(x[rows], y)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_limits_past_32_bits(device, dtype):
    """Lengths and prefixes of int64: those past the keys see all of them, negative ones none."""
    b, lq, lk = 5, 40, 70
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(b, n, 2, 64, generator=g).to(dtype).to(device) for n in (lq, lk, lk))
    far = [2**31, 2**32 + 5, 2**63 - 1, -2**31 - 1, -2**63]
    near = [lk, lk, lk, 0, 0]
    see = visible(b, lq, lk, lengths=near)
    want = attention(q, k, v, see, scale=64 ** -0.5)
    out = att.attend(q, k, v, lengths=torch.tensor(far, device=device))
    assert_within(out, *want["out"], "out by lengths")
    see = visible(b, lq, lk, causal=True, prefix=near)
    want = attention(q, k, v, see, scale=64 ** -0.5)
    out = att.attend(q, k, v, causal=True, prefix=torch.tensor(far, device=device))
    assert_within(out, *want["out"], "out by prefixes")


@pytest.mark.parametrize("dtype", DTYPES)
def test_numbers_that_float32_does_not_hold(device, dtype):
    q, k, v = (torch.randn(1, 9, 1, 64, device=device).to(dtype) for _ in range(3))
    for scale in (1e39, -1e300):
        with pytest.raises(ValueError, match="scale"):
            att.attend(q, k, v, scale=scale)
    with pytest.raises(ValueError, match="cap"):
        att.attend(q, k, v, cap=1e-46)  # not "no cap"
    with pytest.raises(ValueError, match="cap"):
        att.attend(q, k, v, cap=1e-39)  # scale / cap is infinite: 0 * inf where q.k is 0
    if dtype == torch.float32:
        with pytest.raises(ValueError, match="cap"):
            att.attend(q, k, v, cap=1e38)
    zero = torch.zeros_like(q)
    out = att.attend(zero, k, v, cap=1e-30)
    assert_within(out, *attention(zero, k, v, visible(1, 9, 9), scale=0.125, cap=1e-30)["out"],
                  "out")
