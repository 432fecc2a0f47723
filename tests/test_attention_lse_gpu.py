"""The gradient through the log of each row's sum, alone and next to the output's."""

from __future__ import annotations

import pytest
import torch

from attention_norms import assert_near, gradients
from attention_oracle import visible
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(dev, dtype, b, lq, lk, h, hkv, d, *, cap=0.0, causal=False, lengths=None, size=1.0,
           use_out=True):
    g = torch.Generator().manual_seed(b + lq + d)
    q = torch.randn(b, lq, h, d, generator=g).to(dtype)
    k, v = (torch.randn(b, lk, hkv, d, generator=g).to(dtype) for _ in range(2))
    do = torch.randn(b, lq, h, d, generator=g).to(dtype)
    dl = size * torch.randn(b, h, lq, generator=g)
    see = visible(b, lq, lk, causal=causal, lengths=lengths)
    empty = ~see.any(-1)[:, None].expand(b, h, lq)
    want = gradients(q, k, v, see, do if use_out else torch.zeros_like(do), scale=d ** -0.5,
                     cap=cap, dlse=dl.masked_fill(empty, 0.0))
    dl[empty] = float("nan")  # what a loss makes of -inf may be anything

    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    kw = {} if lengths is None else {"lengths": torch.tensor(lengths, dtype=torch.int32).to(dev)}
    out, lse = att.attend(*leaves, cap=cap, causal=causal, return_lse=True, **kw)
    assert torch.equal(lse.isneginf().cpu(), empty)
    if use_out:
        got = torch.autograd.grad((out, lse), leaves, (do.to(dev), dl.to(dev)))
    else:
        got = torch.autograd.grad(lse, leaves, dl.to(dev))
        assert not got[2].any()
    for name, x in zip(("dq", "dk", "dv"), got):
        assert_near(x, *want[name], dtype, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("use_out", [True, False])
@pytest.mark.parametrize("d", [40, 64, 128, 256])
def test_gradient_of_the_log_sum(device, dtype, use_out, d):
    _check(device, dtype, 1, 130, 200, 4, 2, d, use_out=use_out)
    _check(device, dtype, 2, 90, 70, 2, 1, d, causal=True, lengths=[70, 33], cap=4.0, size=20.0,
           use_out=use_out)


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_queries(device, dtype):
    _check(device, dtype, 2, 3, 900, 8, 2, 64, causal=True, lengths=[900, 2])


def test_against_differences(device):
    """float32; the step and what differences may be off as in the output's test."""
    g = torch.Generator().manual_seed(3)
    t = [torch.randn(1, n, 2, 32, generator=g).to(device) for n in (20, 70, 70)]
    w = torch.randn(1, 2, 20, generator=g).to(device)

    def value(q, k, v):
        return (att.attend(q, k, v, cap=4.0, return_lse=True)[1].double() * w.double()).sum()

    leaves = [x.clone().requires_grad_(True) for x in t]
    grads = torch.autograd.grad(value(*leaves), leaves)
    assert not grads[2].any()
    step = 2.0 ** -5
    for i in range(2):
        for _ in range(3):
            way = torch.randn(t[i].shape, generator=g).to(device)
            way = way / way.norm()
            plus, minus = list(t), list(t)
            plus[i], minus[i] = t[i] + step * way, t[i] - step * way
            slope = (value(*plus) - value(*minus)) / (2 * step)
            want = (grads[i].double() * way.double()).sum()
            assert (slope - want).abs() <= 2e-3 * grads[i].double().norm() + 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_joining_two_halves_of_the_keys(device, dtype):
    """Two calls joined by their log-sums have the gradients of one call over all keys."""
    g = torch.Generator().manual_seed(4)
    q, k, v, do = (torch.randn(1, n, 2, 64, generator=g).to(dtype) for n in (70, 200, 200, 70))
    want = gradients(q, k, v, visible(1, 70, 200), do, scale=64 ** -0.5)
    leaves = [t.to(device).requires_grad_(True) for t in (q, k, v)]
    parts = [att.attend(leaves[0], leaves[1][:, s], leaves[2][:, s], return_lse=True)
             for s in (slice(0, 90), slice(90, 200))]
    lse = torch.stack([p[1] for p in parts])
    share = torch.softmax(lse, 0).transpose(2, 3)[..., None]  # (2, B, Lq, H, 1)
    out = sum(w * p[0].float() for w, p in zip(share, parts))
    got = torch.autograd.grad(out, leaves, do.float().to(device))
    for name, x in zip(("dq", "dk", "dv"), got):
        # the parts' outputs and their gradients are rounded as well: about four independent
        # terms of one size in place of one, twice as much in squares
        assert_near(x, *want[name], dtype, name, times=2.0)


def test_the_output_alone_is_as_it_was(device):
    """Asking for the log-sum without using it changes nothing, nor does its gradient of zero."""
    q, k, v, do = (torch.randn(1, 70, 2, 64, device=device).half() for _ in range(4))
    for t in (q, k, v):
        t.requires_grad_(True)
    first = torch.autograd.grad(att.attend(q, k, v), (q, k, v), do)
    out, lse = att.attend(q, k, v, return_lse=True)
    second = torch.autograd.grad((out, lse), (q, k, v), (do, torch.zeros_like(lse)))
    for x, y in zip(first, second):
        assert torch.equal(x, y)
