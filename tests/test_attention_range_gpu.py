"""Gradients of attention.attend over the range of what half precision holds: output gradients
from 1e-4 to 1e4, of one size and of many, and weights that many keys share.  No bound grows
with the smallest number that the type holds, but for the result's own rounding."""

from __future__ import annotations

import pytest
import torch

from attention_norms import assert_near, gradients
from attention_oracle import visible
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(dev, dtype, sizes, size, *, qk=0.5, vk=1.0, docs=None, cap=0.0, causal=False, seed=0,
           names=("dq", "dk", "dv"), parts=(slice(None),)):
    """``size``: of the output's gradient, a number or one for each query; ``parts``: rows whose
    gradients are looked at by themselves."""
    b, lq, lk, h, hkv, d = sizes
    g = torch.Generator().manual_seed(seed)
    q = (qk * torch.randn(b, lq, h, d, generator=g)).to(dtype)
    k = torch.randn(b, lk, hkv, d, generator=g).to(dtype)
    v = (vk * torch.randn(b, lk, hkv, d, generator=g)).to(dtype)
    do = torch.randn(b, lq, h, d, generator=g)
    do = (do * torch.as_tensor(size).view(-1, 1, 1)).to(dtype)
    kw = {}
    if docs is not None:
        kw["q_docs"] = torch.tensor([docs] * b, dtype=torch.int32)
        kw["k_docs"] = kw["q_docs"]
    see = visible(b, lq, lk, causal=causal, **kw)
    want = gradients(q, k, v, see, do, scale=d ** -0.5, cap=cap)
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = att.attend(*leaves, cap=cap, causal=causal, **{n: t.to(dev) for n, t in kw.items()})
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do.to(dev))))
    for name in names:
        value, spread = want[name]
        assert value.abs().max() < 65504.0
        for at in parts:
            assert_near(got[name][:, at], value[:, at], spread[:, at], dtype, f"{name} {at}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e-2, 1.0, 1e3])
@pytest.mark.parametrize("d", [64, 128])
def test_sizes_of_the_output_gradient(device, dtype, size, d):
    """Weights of 2^-13: score gradients of 1e-7 and below."""
    _check(device, dtype, (1, 256, 8192, 2, 1, d), size)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-3, 1.0, 1e3])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_peaked_weights(device, dtype, size, d):
    _check(device, dtype, (1, 256, 256, 2, 2, d), size, qk=4.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_score_gradients_past_half_precision(device, dtype, d):
    """An output's gradient of 1e4: ds passes 65504, the gradients of q, k and v do not."""
    _check(device, dtype, (1, 256, 256, 1, 1, d), 1e4, qk=1.0, vk=4.0, names=("dq",))
    _check(device, dtype, (1, 256, 8192, 1, 1, d), 1e4, qk=1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 128])
def test_queries_of_unlike_sizes(device, dtype, d):
    """Rows from 2^-16 to 2^10 next to each other, small ones first and last; dq in parts."""
    n = 300
    size = 2.0 ** ((torch.arange(n) * 7) % 27 - 16)
    size[:40], size[-40:] = 2.0**-16, 2.0**-16
    _check(device, dtype, (1, n, n, 2, 2, d), size, qk=1.0)
    _check(device, dtype, (1, n, n, 2, 2, d), size, qk=1.0, names=("dq",),
           parts=(slice(0, 40), slice(40, n - 40), slice(n - 40, n)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_documents_of_unlike_sizes(device, dtype):
    """Keys of a document see its own queries alone, whose gradients differ by 2^20."""
    docs = [0] * 130 + [1] * 70 + [2] * 150
    size = torch.tensor([2.0**-12] * 130 + [2.0**8] * 70 + [2.0**-10] * 150)
    _check(device, dtype, (1, 350, 350, 2, 2, 64), size, qk=1.0, docs=docs,
           parts=(slice(0, 130), slice(130, 200), slice(200, 350)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_weights_that_many_keys_share(device, dtype, d):
    """Weights of 2^-17 for 100003 keys, below half precision's normal numbers."""
    _check(device, dtype, (1, 40, 100003, 1, 1, d), 1.0, qk=0.25, names=("dv",))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-3, 1e3])
def test_caps_and_shared_heads(device, dtype, size):
    _check(device, dtype, (2, 150, 150, 6, 2, 64), size, qk=1.0, cap=6.0, causal=True)
    _check(device, dtype, (1, 130, 130, 4, 1, 128), size, qk=1.0, cap=6.0,
           docs=[0] * 60 + [1] * 70)
