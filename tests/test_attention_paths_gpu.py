"""Ways through the attention kernels that take more rows or masks than the other tests have:
few queries with positions or documents over many tiles, more documents' tiles than a wave looks
at together, the largest cap, and the C entries themselves."""

from __future__ import annotations

import ctypes

import pytest
import torch

from attention_norms import assert_near, gradients
from attention_oracle import assert_within, attention, visible
from torchmatch_amd import _native
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(dtype, b, lq, lk, h, hkv, d, seed, qk=1.5):
    g = torch.Generator().manual_seed(seed)
    q = (qk * torch.randn(b, lq, h, d, generator=g)).to(dtype)
    k, v = (torch.randn(b, lk, hkv, d, generator=g).to(dtype) for _ in range(2))
    return g, q, k, v


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq", [1, 5, 16])
@pytest.mark.parametrize("axes", [1, 2, 3])
def test_few_queries_with_positions(device, dtype, lq, axes):
    """Positions of a wave's tiles change places, over a split of the keys and its join."""
    b, lk, h, hkv, d = 3, 3001, 8, 2, 64
    g, q, k, v = _inputs(dtype, b, lq, lk, h, hkv, d, axes)
    slopes = 2.0 ** -torch.arange(1.0, h + 1)
    pos = [9 * torch.rand(b, n, axes, generator=g) for n in (lq, lk)]
    for causal in (False, True):
        lengths = [3001, 1777, lq]
        see = visible(b, lq, lk, causal=causal, lengths=lengths)
        want = attention(q, k, v, see, scale=d ** -0.5, slopes=slopes, q_positions=pos[0],
                         k_positions=pos[1], lengths=lengths)
        out, lse = att.attend(*(t.to(device) for t in (q, k, v)), slopes=slopes.to(device),
                              q_positions=pos[0].to(device), k_positions=pos[1].to(device),
                              causal=causal, return_lse=True,
                              lengths=torch.tensor(lengths, dtype=torch.int32, device=device))
        assert_within(out, *want["out"], "out")
        assert_within(lse, *want["lse"], "lse")


def _ids(kind, n, g):
    if kind == "sorted":  # documents of 1 to 400 keys, padding between some
        ids, at = torch.full((n,), -1, dtype=torch.int32), 0
        for i in range(n):
            size = int(torch.randint(1, 400, (1,), generator=g))
            ids[at:at + size] = i % 9 if i % 5 else -1
            at += size
            if at >= n:
                return ids
    if kind == "sparse":  # nearly all padding: whole groups of 64 tiles without a key
        ids = torch.full((n,), -1, dtype=torch.int32)
        ids[n - 3:], ids[7], ids[n // 2] = 1, 1, 2
        return ids
    return torch.randint(-1, 6, (n,), generator=g, dtype=torch.int32)  # no order


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["sorted", "sparse", "mixed"])
@pytest.mark.parametrize("lq", [1, 5, 16])
def test_few_queries_of_documents(device, dtype, kind, lq):
    """More tiles than waves, so that each takes several turns, and a tile's second half."""
    b, lk, h, hkv, d = 2, 9001, 4, 2, 64
    g, q, k, v = _inputs(dtype, b, lq, lk, h, hkv, d, lq)
    k_docs = torch.stack([_ids(kind, lk, g) for _ in range(b)])
    q_docs = torch.tensor([[1, 2, 0, -1, 3] * 4] * b, dtype=torch.int32)[:, :lq].contiguous()
    lengths = [9001, 8990]
    see = visible(b, lq, lk, lengths=lengths, q_docs=q_docs, k_docs=k_docs)
    want = attention(q, k, v, see, scale=d ** -0.5)
    out, lse = att.attend(*(t.to(device) for t in (q, k, v)), q_docs=q_docs.to(device),
                          k_docs=k_docs.to(device), return_lse=True,
                          lengths=torch.tensor(lengths, dtype=torch.int32, device=device))
    assert_within(out, *want["out"], "out")
    assert_within(lse, *want["lse"], "lse")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["sorted", "sparse", "mixed"])
@pytest.mark.parametrize("causal", [False, True])
def test_long_rows_of_documents(device, dtype, kind, causal):
    """71 tiles a row and more blocks than run at once: the walk over tiles goes on after its
    first 64, and blocks are ordered by counts over more than 64.  The key heads' queries are
    the same, so that one head's exact values serve for all of them."""
    b, n, h, hkv, d = 1, 4500, 16, 16, 64
    g, q, k, v = _inputs(dtype, b, n, n, 1, 1, d, 3, qk=1.0)
    docs = torch.stack([_ids(kind, n, g) for _ in range(b)])
    do = torch.randn(b, n, 1, d, generator=g).to(dtype)
    see = visible(b, n, n, causal=causal, q_docs=docs, k_docs=docs)
    want = attention(q, k, v, see, scale=d ** -0.5)
    grads = gradients(q, k, v, see, do, scale=d ** -0.5)
    leaves = [t.to(device).expand(-1, -1, h, -1).detach().requires_grad_(True) for t in (q, k, v)]
    out = att.attend(*leaves, causal=causal, q_docs=docs.to(device))
    got = torch.autograd.grad(out, leaves, do.to(device).expand(-1, -1, h, -1))
    for t in (out, *got):
        assert torch.equal(t, t[:, :, :1].expand(-1, -1, h, -1))
    assert_within(out[:, :, :1], *want["out"], "out")
    for name, t in zip(("dq", "dk", "dv"), got):
        assert_near(t[:, :, :1], *grads[name], dtype, name)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("cap", [700.0, 1024.0])
def test_largest_caps_in_half_precision(device, cap, causal):
    """tanh by exp is good to 2e-7 of the cap, which is added to a score and so makes weights err
    by 2e-7 cap (2^-12.2 at 1024) on top of what the oracle allows: twice the sum of weights times
    values, as it may be of both signs, and its log-sum once."""
    b, lq, lk, h, d = 1, 90, 150, 2, 64
    g, q, k, v = _inputs(torch.float16, b, lq, lk, h, h, d, 4)
    do = torch.randn(b, lq, h, d, generator=g).half()
    see = visible(b, lq, lk, causal=causal)
    want = attention(q, k, v, see, scale=d ** -0.5, cap=cap)
    a = attention(q, k, v.abs(), see, scale=d ** -0.5, cap=cap)["out"][0]
    leaves = [t.to(device).requires_grad_(True) for t in (q, k, v)]
    out, lse = att.attend(*leaves, cap=cap, causal=causal, return_lse=True)
    value, bound = want["out"]
    assert_within(out, value, bound + 2 * 2e-7 * cap * a, "out")
    value, bound = want["lse"]
    assert_within(lse, value, bound + 2e-7 * cap, "lse")
    grads = gradients(q, k, v, see, do, scale=d ** -0.5, cap=cap)
    for name, t in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do.to(device))):
        # weights err by half of u more (2^-12.2 of 2^-11)
        assert_near(t, *grads[name], torch.float16, name, times=1.5)


def test_rows_of_heads_through_the_c_entries(device):
    """tm_attention_forward and tm_attention_backward give the bits that the ops give."""
    b, lq, lk, h, hkv, d = 2, 90, 333, 4, 2, 64
    g, *t = _inputs(torch.bfloat16, b, lq, lk, h, hkv, d, 6)
    q, k, v = (x.to(device).requires_grad_(True) for x in t)
    do = torch.randn(b, lq, h, d, generator=g).bfloat16().to(device)
    want, lse = att.attend(q, k, v, causal=True, cap=9.0, return_lse=True)
    grads = torch.autograd.grad(want, (q, k, v), do)
    a = _native.Attention(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_b=lq * h * d, q_l=h * d, q_h=d,
        k_b=lk * hkv * d, k_l=hkv * d, k_h=d, v_b=lk * hkv * d, v_l=hkv * d, v_h=d,
        dtype=_native.TM_BF16, B=b, Lq=lq, Lk=lk, H=h, Hkv=hkv, D=d, causal=1, scale=d ** -0.5,
        cap=9.0)
    lib, at = _native.lib(), ctypes.byref(a)
    stream = torch.cuda.current_stream().cuda_stream
    out, low = torch.empty_like(q), torch.empty_like(q)
    log_sum = torch.empty(b, h, lq, device=device)
    n = lib.tm_attention_workspace_bytes(at)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=device)
    assert lib.tm_attention_forward(at, out.data_ptr(), low.data_ptr(), log_sum.data_ptr(),
                                    ws.data_ptr(), n, stream) == _native.TM_OK
    assert torch.equal(out, want) and torch.equal(log_sum, lse)
    n = lib.tm_attention_backward_workspace_bytes(at)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=device)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    assert lib.tm_attention_backward(
        at, out.data_ptr(), low.data_ptr(), log_sum.data_ptr(), do.data_ptr(), lq * h * d, h * d,
        d, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), n, stream) == _native.TM_OK
    for x, y in zip((dq, dk, dv), grads):
        assert torch.equal(x, y)
    assert lib.tm_attention_backward(
        at, out.data_ptr(), low.data_ptr(), log_sum.data_ptr(), do.data_ptr(), lq * h * d, h * d,
        d, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), n - 1,
        stream) == _native.TM_ERR_WORKSPACE


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 2), (1, 2)])
def test_some_inputs_without_gradient(device, dtype, which):
    """The gradients of some of q, k and v are those of all of them."""
    _, *t = _inputs(dtype, 1, 70, 130, 4, 2, 64, 8)
    do = torch.randn(1, 70, 4, 64).to(dtype).to(device)
    every = [x.to(device).requires_grad_(True) for x in t]
    want = torch.autograd.grad(att.attend(*every, causal=True), every, do)
    some = [x.to(device).requires_grad_(i in which) for i, x in enumerate(t)]
    att.attend(*some, causal=True).backward(do)
    for i, x in enumerate(some):
        assert torch.equal(x.grad, want[i]) if i in which else x.grad is None


def test_traced_gradients(device):
    """The gradients' graph, traced with sizes that change, gives the eager values."""
    q = torch.randn(2, 40, 4, 32, device=device, requires_grad=True)
    k, v = (torch.randn(2, 70, 2, 32, device=device, requires_grad=True) for _ in range(2))
    torch.library.opcheck(torch.ops.attention.attend.default, (q, k, v),
                          {"scale": 0.2, "causal": True}, test_utils="test_aot_dispatch_dynamic")
    pos, freqs = torch.rand(2, 40, 2, device=device), att.rotary_frequencies((8, 8))
    torch.library.opcheck(torch.ops.attention.rotate.default, (q, pos, freqs, [8, 8]),
                          test_utils="test_aot_dispatch_dynamic")


def test_gradients_of_the_log_sum_are_checked(device):
    """attend_backward's last tensor: float32, shaped as lse, any strides."""
    _, *t = _inputs(torch.float32, 1, 20, 30, 2, 1, 64, 9)
    q, k, v = (x.to(device) for x in t)
    out, low, lse = torch.ops.attention.attend_forward(q, k, v, scale=0.125)
    dl = torch.randn(1, 20, 2, device=device).transpose(1, 2)
    back = lambda dlse: torch.ops.attention.attend_backward(  # noqa: E731
        torch.zeros_like(q), q, k, v, out, low, lse, dlse=dlse, scale=0.125)
    for x, y in zip(back(dl), back(dl.contiguous())):
        assert torch.equal(x, y)
    with pytest.raises(TypeError, match="float32"):
        back(dl.double())
    with pytest.raises(ValueError, match="as lse"):
        back(dl[:, :1])
    with pytest.raises(ValueError, match="as lse"):
        back(dl.cpu())
