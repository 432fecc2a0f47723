"""Calls at the edge of attention.attend's arguments: sets without points."""

from __future__ import annotations

import pytest
import torch

from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu


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
