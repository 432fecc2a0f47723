"""attention.attend on the GPU against the 64-bit oracle: types, head layouts, lengths from
one token on, masks that leave rows empty, garbage in masked places, strides, gradients."""

from __future__ import annotations

import pytest
import torch

from attention_oracle import assert_within, attention, visible
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _case(dev, dtype, b, lq, lk, h, hkv, d, *, cap=0.0, axes=-1, causal=False, prefix=None,
          lengths=None, docs=None, k_docs=None, seed=0, grads=True, qk=1.5):
    """Runs one call and its gradients against the oracle."""
    g = torch.Generator().manual_seed(seed)
    q = (qk * torch.randn(b, lq, h, d, generator=g)).to(dtype).to(dev).requires_grad_(grads)
    k = torch.randn(b, lk, hkv, d, generator=g).to(dtype).to(dev).requires_grad_(grads)
    v = torch.randn(b, lk, hkv, d, generator=g).to(dtype).to(dev).requires_grad_(grads)
    kw = {}
    if axes >= 0:
        kw["slopes"] = (2.0 ** -torch.arange(1, h + 1, dtype=torch.float32)).to(dev)
    if axes > 0:
        kw["q_positions"] = (9 * torch.rand(b, lq, axes, generator=g)).to(dev)
        kw["k_positions"] = (9 * torch.rand(b, lk, axes, generator=g)).to(dev)
    masks = {"prefix": prefix, "lengths": lengths, "q_docs": docs, "k_docs": k_docs}
    masks = {n: torch.as_tensor(t, dtype=torch.int32).to(dev) for n, t in masks.items()
             if t is not None}
    scale = d ** -0.5
    out, lse = att.attend(q, k, v, scale=scale, cap=cap, causal=causal, return_lse=True, **masks,
                          **kw)
    see = visible(b, lq, lk, causal=causal, prefix=prefix, lengths=lengths,
                  q_docs=masks.get("q_docs"),
                  k_docs=masks.get("k_docs", masks.get("q_docs")))
    do = torch.randn(b, lq, h, d, generator=g).to(dtype).to(dev) if grads else None
    want = attention(q, k, v, see, scale=scale, cap=cap, lengths=lengths, dout=do, **kw)
    assert_within(out, *want["out"], "out")
    assert_within(lse, *want["lse"], "lse")
    assert out.dtype == dtype and lse.dtype == torch.float32
    if grads:
        got = torch.autograd.grad(out, (q, k, v), do)
        for name, t in zip(("dq", "dk", "dv"), got):
            assert t.dtype == dtype
            assert_within(t, *want[name], name)
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 32, 40, 64, 80, 96, 128, 160, 256])
def test_head_dims(device, dtype, d):
    _case(device, dtype, 1, 70, 133, 2, 1, d, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 2), (2, 1), (1, 63), (1, 64), (1, 65), (31, 33),
                                   (32, 32), (63, 64), (65, 64), (128, 128), (129, 257),
                                   (300, 71), (5, 700)])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(device, dtype, lq, lk, causal):
    _case(device, dtype, 2, lq, lk, 2, 2, 64, causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hkv", [(1, 1), (6, 2), (4, 1), (8, 8), (3, 3)])
def test_shared_heads(device, dtype, h, hkv):
    _case(device, dtype, 2, 77, 77, h, hkv, 32, causal=True, axes=0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cap", [0.0, 3.0, 30.0])
@pytest.mark.parametrize("axes", [-1, 0, 1, 2, 3])
def test_cap_and_bias(device, dtype, cap, axes):
    _case(device, dtype, 2, 90, 150, 4, 2, 64, cap=cap, axes=axes, qk=4.0)
    _case(device, dtype, 1, 150, 150, 2, 2, 128, cap=cap, axes=axes, causal=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefix_and_lengths(device, dtype):
    # prefixes of nothing, of part and past the row's length; lengths of zero, fewer keys
    # than queries (the first queries see nothing), all
    _case(device, dtype, 4, 100, 200, 2, 1, 64, causal=True, prefix=[0, 37, 199, 500])
    _case(device, dtype, 5, 100, 200, 2, 1, 64, causal=True, prefix=[0, 3, 64, 9, 200],
          lengths=[0, 1, 99, 130, 200], axes=0)
    _case(device, dtype, 3, 70, 200, 2, 1, 64, lengths=[0, 65, 200])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cap", [0.25, 100.0, 1024.0])
def test_small_and_large_caps(device, dtype, cap):
    """Large caps leave scores nearly as they are: nothing may be lost to their size.  The
    16-bit kernels' tanh is good to 2^-22 of the cap; a cap of 1024 adds 2^-12 to what
    weights may be off, less than a float16 rounding."""
    if dtype == torch.float16 and cap > 500:
        cap = 500.0  # 2^-13: stays within the 2^-11 of a weight's rounding
    _case(device, dtype, 1, 90, 150, 2, 2, 64, cap=cap, causal=False)


def _ids(*parts):
    return [i for i, n in parts for _ in range(n)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_documents(device, dtype, causal):
    # sorted with padding inside and at the end, one document over many tiles, and ids
    # in no order
    rows = [_ids((0, 70), (1, 1), (-1, 9), (2, 200), (3, 20)),
            _ids((5, 128), (7, 64), (-1, 108)),
            [(7 * i) % 5 - 1 for i in range(300)]]
    _case(device, dtype, 3, 300, 300, 2, 1, 64, causal=causal, docs=rows)


@pytest.mark.parametrize("dtype", DTYPES)
def test_pairs_of_sets(device, dtype):
    # queries of one set against keys of the other; a pair without keys, one without queries
    q_docs = [_ids((0, 33), (1, 50), (2, 40), (4, 7)), _ids((0, 130))]
    k_docs = [_ids((0, 64), (2, 100), (3, 30), (4, 6)), _ids((-1, 100), (0, 100))]
    _case(device, dtype, 2, 130, 200, 4, 4, 64, docs=q_docs, k_docs=k_docs, cap=5.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_to_see(device, dtype):
    out = _case(device, dtype, 1, 40, 70, 2, 2, 64, docs=[[-1] * 40], k_docs=[[-1] * 70])
    assert (out == 0).all()
    out = _case(device, dtype, 2, 3, 900, 2, 2, 64, lengths=[0, 0])
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq", [1, 3, 16, 17, 40])
@pytest.mark.parametrize("h,hkv", [(8, 1), (4, 4), (32, 8)])
def test_few_tokens_over_a_cache(device, dtype, lq, h, hkv):
    _case(device, dtype, 3, lq, 3000, h, hkv, 128, causal=True, axes=0,
          lengths=[3000, 1777, lq], grads=False)
    _case(device, dtype, 1, lq, 2049, h, hkv, 64, causal=True, cap=8.0, grads=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -3e38])
@pytest.mark.parametrize("lq", [2, 96])
def test_garbage_past_the_keys(device, dtype, junk, lq):
    """Keys past the lengths, in padding and past the last causal query hold anything."""
    g = torch.Generator().manual_seed(3)
    b, lk, h, d = 2, 400, 2, 64
    junk = torch.tensor(junk).to(dtype).item()
    t = [torch.randn(b, n, h, d, generator=g).to(dtype).to(device) for n in (lq, lk, lk, lq)]
    lengths = torch.tensor([130, 301], dtype=torch.int32)
    docs = torch.zeros(b, lk, dtype=torch.int32)
    docs[0, 20:31] = -1
    docs[1, 256:] = -1
    q_docs = torch.zeros(b, lq, dtype=torch.int32)
    q_docs[1, lq // 2:] = -1
    see = visible(b, lq, lk, lengths=lengths, q_docs=q_docs, k_docs=docs)
    hidden = ~see.any(1)
    blind = ~see.any(2)
    t[0][blind.to(device)] = junk
    t[1][hidden.to(device)] = junk
    t[2][hidden.to(device)] = junk
    t[3][blind.to(device)] = junk
    q, k, v, do = t
    for x in (q, k, v):
        x.requires_grad_(True)
    out = att.attend(q, k, v, lengths=lengths.to(device), q_docs=q_docs.to(device),
                     k_docs=docs.to(device))
    want = attention(q, k, v, see, scale=d ** -0.5, dout=do)
    assert_within(out, *want["out"], "out")
    grads = torch.autograd.grad(out, (q, k, v), do)
    for name, x in zip(("dq", "dk", "dv"), grads):
        assert_within(x, *want[name], name)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(device, dtype):
    """Scores of hundreds: one key takes all of the weight, nothing overflows."""
    _case(device, dtype, 1, 65, 200, 2, 2, 64, qk=300.0, grads=False)
    q = torch.full((1, 3, 1, 32), 200.0, dtype=dtype, device=device)
    k = torch.full((1, 90, 1, 32), 200.0, dtype=dtype, device=device)
    k[:, 40] = 201.0
    v = torch.arange(90, device=device).view(1, 90, 1, 1).expand(1, 90, 1, 32).to(dtype)
    assert (att.attend(q, k, v, scale=1.0) == 40).all()
    assert (att.attend(q, -k, v, scale=1.0)[..., 0] != 40).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_and_nan_inputs_show(device, dtype):
    """NaN in what is seen is NaN in the rows that see it, and in no other."""
    q = torch.randn(1, 80, 1, 64, device=device).to(dtype)
    k = torch.randn(1, 80, 1, 64, device=device).to(dtype)
    v = torch.randn(1, 80, 1, 64, device=device).to(dtype)
    q[0, 70, 0, 5] = float("nan")
    out = att.attend(q, k, v)
    assert out[0, 70].isnan().all() and not out[0, :70].isnan().any()
    k[0, 64, 0, 0] = float("nan")
    out = att.attend(q, k, v, causal=True)
    assert not out[0, :64].isnan().any() and out[0, 64:].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(device, dtype):
    """Views of one projection, heads before rows, shared keys, odd offsets, odd strides."""
    g = torch.Generator().manual_seed(5)
    b, n, h, d = 2, 100, 2, 64
    qkv = torch.randn(b, n, 3 * h, d, generator=g).to(dtype).to(device)
    q, k, v = qkv.split(h, 2)
    base = att.attend(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    assert torch.equal(att.attend(q, k, v, causal=True), base)
    bhld = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(att.attend(*bhld, causal=True), base)
    dlast = [t.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2) for t in (q, k, v)]
    assert torch.equal(att.attend(*dlast, causal=True), base)
    odd = [torch.empty(t.numel() + 1, dtype=dtype, device=device)[1:].view(t.shape).copy_(t)
           for t in (q, k, v)]
    assert torch.equal(att.attend(*odd, causal=True), base)
    wide = [torch.empty(b, n, h, d + 3, dtype=dtype, device=device)[..., :d].copy_(t)
            for t in (q, k, v)]
    assert torch.equal(att.attend(*wide, causal=True), base)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 3, 20, 63])
def test_odd_head_dims(device, dtype, d):
    _case(device, dtype, 1, 30, 90, 2, 2, d)


def test_gradients_of_broadcast_inputs(device):
    """One key set for the whole batch, and the gradient of a plain sum (stride 0)."""
    g = torch.Generator().manual_seed(7)
    q = torch.randn(3, 50, 4, 32, generator=g).to(device).requires_grad_(True)
    k1 = torch.randn(1, 60, 2, 32, generator=g).to(device).requires_grad_(True)
    v1 = torch.randn(1, 60, 2, 32, generator=g).to(device).requires_grad_(True)
    att.attend(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1)).sum().backward()
    see = visible(3, 50, 60)
    do = torch.ones(3, 50, 4, 32)
    want = attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1), see,
                     scale=32 ** -0.5, dout=do)
    assert_within(q.grad, *want["dq"], "dq")
    for got, name in ((k1.grad, "dk"), (v1.grad, "dv")):
        value, bound = want[name]
        assert_within(got, value.sum(0, keepdim=True), bound.sum(0, keepdim=True), name)


@pytest.mark.parametrize("cap,axes,causal", [(0.0, -1, False), (4.0, 2, False), (2.0, 0, True)])
def test_gradient_against_differences(device, cap, axes, causal):
    """float32: central differences of a weighted sum of the output, in random directions.

    With step h the difference errs by h^2 / 6 times the third derivative along the
    direction (O(1) here, as the directions are of unit norm) and by the sum's float32
    error, 2^-20 times its terms, over h.  h = 2^-5: below 2e-3 of the gradient's norm."""
    g = torch.Generator().manual_seed(11)
    b, lq, lk, h, hkv, d = 1, 20, 70, 2, 1, 32
    t = [torch.randn(s, generator=g).to(device) for s in
         ((b, lq, h, d), (b, lk, hkv, d), (b, lk, hkv, d), (b, lq, h, d))]
    kw = {"cap": cap, "causal": causal}
    if axes >= 0:
        kw["slopes"] = torch.tensor([0.5, 0.1], device=device)
    if axes > 0:
        kw["q_positions"] = torch.rand(b, lq, axes, generator=g).to(device)
        kw["k_positions"] = torch.rand(b, lk, axes, generator=g).to(device)
    w = t.pop()

    def value(q, k, v):
        return (att.attend(q, k, v, **kw).double() * w.double()).sum()

    leaves = [x.clone().requires_grad_(True) for x in t]
    grads = torch.autograd.grad(value(*leaves), leaves)
    step = 2.0 ** -5
    for i in range(3):
        for _ in range(3):
            way = torch.randn(t[i].shape, generator=g).to(device)
            way = way / way.norm()
            plus, minus = list(t), list(t)
            plus[i], minus[i] = t[i] + step * way, t[i] - step * way
            slope = (value(*plus) - value(*minus)) / (2 * step)
            want = (grads[i].double() * way.double()).sum()
            assert (slope - want).abs() <= 2e-3 * grads[i].double().norm() + 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hkv,lq,lk,d", [(12, 1, 70, 130, 64), (7, 1, 513, 129, 32),
                                           (1, 1, 900, 40, 128), (10, 2, 257, 300, 256),
                                           (5, 1, 1, 33, 96), (1, 1, 641, 641, 80)])
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_of_few_key_blocks(device, dtype, h, hkv, lq, lk, d, causal):
    """Gradients of k and v that many query heads or queries share over few keys."""
    _case(device, dtype, 2, lq, lk, h, hkv, d, causal=causal, cap=5.0, axes=1,
          lengths=[lk, lk // 3])


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_few_key_blocks_of_documents(device, dtype):
    rows = [_ids((0, 3), (1, 200), (2, 1), (-1, 130), (3, 90))]
    _case(device, dtype, 1, 424, 424, 6, 1, 64, causal=True, docs=rows)


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits(device, dtype):
    """The same call gives the same bits, forward and backward, on any stream."""
    g = torch.Generator().manual_seed(13)
    q, k, v, do = (torch.randn(2, n, h, 64, generator=g).to(dtype).to(device)
                   for n, h in ((333, 4), (700, 2), (700, 2), (333, 4)))
    for t in (q, k, v):
        t.requires_grad_(True)

    def once():
        out = att.attend(q, k, v, cap=9.0)
        return (out, *torch.autograd.grad(out, (q, k, v), do))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_captured(device):
    """A captured call, replayed on new inputs with eager work between the replays."""
    q = torch.randn(2, 3, 8, 64, device=device).half()
    k = torch.randn(2, 2500, 2, 64, device=device).half()
    v = torch.randn(2, 2500, 2, 64, device=device).half()
    lengths = torch.tensor([2500, 900], dtype=torch.int32, device=device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        att.attend(q, k, v, lengths=lengths, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = att.attend(q, k, v, lengths=lengths, causal=True)
    for n in range(4):
        q.normal_()
        v.normal_()
        lengths.copy_(torch.tensor([2500 - n, 37 * n + 3], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, att.attend(q, k, v, lengths=lengths, causal=True))


def test_keys_past_32_bit_offsets(device):
    """A cache whose rows lie further apart than 32 bits of elements reach."""
    row = 1 << 22
    big = torch.zeros(1100 * row, dtype=torch.float16, device=device)  # 9.2 GB
    g = torch.Generator().manual_seed(17)
    q = torch.randn(1, 2, 1, 64, generator=g).half().to(device)
    k = torch.randn(1, 1100, 1, 64, generator=g).half().to(device)
    v = torch.randn(1, 1100, 1, 64, generator=g).half().to(device)
    far_k = big.as_strided((1, 1100, 1, 64), (0, row, 0, 1))
    far_v = big.as_strided((1, 1100, 1, 64), (0, row, 0, 1), 64)
    far_k.copy_(k)
    far_v.copy_(v)
    assert torch.equal(att.attend(q, far_k, far_v, causal=True),
                       att.attend(q, k, v, causal=True))
    q = torch.randn(1, 1100, 1, 64, generator=g).half().to(device).requires_grad_(True)
    grads = []
    for a, b in ((far_k, far_v), (k, v)):
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        grads.append(torch.autograd.grad(att.attend(q, a, b), (q, a, b), q.detach()))
    for x, y in zip(*grads):
        assert torch.equal(x, y)


def test_empty_sizes(device):
    for b, lq, lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q = torch.randn(b, lq, 2, 32, device=device, requires_grad=True)
        k = torch.randn(b, lk, 2, 32, device=device, requires_grad=True)
        v = torch.randn(b, lk, 2, 32, device=device, requires_grad=True)
        out, lse = att.attend(q, k, v, return_lse=True)
        assert out.shape == (b, lq, 2, 32) and (out == 0).all() and lse.isneginf().all()
        out.sum().backward()
        for t in (q, k, v):
            assert t.grad.shape == t.shape and (t.grad == 0).all()


def test_refusals(device):
    q = torch.randn(2, 5, 4, 64, device=device)
    k = torch.randn(2, 9, 2, 64, device=device)
    ids = torch.zeros(2, 5, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="ROCm"):
        att.attend(q.cpu(), k, k)
    with pytest.raises(ValueError, match="4D"):
        att.attend(q[0], k, k)
    with pytest.raises(TypeError, match="one dtype"):
        att.attend(q, k.half(), k.half())
    with pytest.raises(TypeError, match="bfloat16"):
        att.attend(q.double(), k.double(), k.double())
    with pytest.raises(ValueError, match="one shape"):
        att.attend(q, k, k[:, :8])
    with pytest.raises(ValueError, match="multiple"):
        att.attend(q[:, :, :3], k, k)
    with pytest.raises(ValueError, match="as q is"):
        att.attend(q, k[:1], k[:1])
    with pytest.raises(ValueError, match="features"):
        att.attend(torch.zeros(1, 1, 1, 300, device=device), *(2 * [torch.zeros(
            1, 1, 1, 300, device=device)]))
    with pytest.raises(ValueError, match="cap"):
        att.attend(q, k, k, cap=-1.0)
    with pytest.raises(ValueError, match="at most 1024"):
        att.attend(q.half(), k.half(), k.half(), cap=2000.0)
    with pytest.raises(ValueError, match="scale"):
        att.attend(q, k, k, scale=float("nan"))
    with pytest.raises(ValueError, match="causal"):
        att.attend(q, k, k, prefix=torch.zeros(2, dtype=torch.int32, device=device))
    with pytest.raises(ValueError, match="k_docs must be"):
        att.attend(q, k, k, q_docs=ids)
    with pytest.raises(TypeError, match="int32"):
        att.attend(q, k, k, q_docs=ids.float(), k_docs=ids.float())
    with pytest.raises(ValueError, match="lengths must be"):
        att.attend(q, k, k, lengths=torch.zeros(3, dtype=torch.int32, device=device))
    with pytest.raises(ValueError, match="slopes"):
        att.attend(q, k, k, q_positions=torch.zeros(2, 5, 1, device=device),
                   k_positions=torch.zeros(2, 9, 1, device=device))
    slopes = torch.ones(4, device=device)
    with pytest.raises(ValueError, match="both"):
        att.attend(q, k, k, slopes=slopes, q_positions=torch.zeros(2, 5, 1, device=device))
    with pytest.raises(ValueError, match="axes"):
        att.attend(q, k, k, slopes=slopes, q_positions=torch.zeros(2, 5, 4, device=device),
                   k_positions=torch.zeros(2, 9, 4, device=device))
    with pytest.raises(NotImplementedError, match="slopes"):
        att.attend(q, k, k, slopes=slopes.clone().requires_grad_(True))


def test_opcheck(device):
    """Schemas, fake kernels and autograd registration agree with the kernels."""
    q = torch.randn(2, 40, 4, 32, device=device, requires_grad=True)
    k = torch.randn(2, 70, 2, 32, device=device, requires_grad=True)
    v = torch.randn(2, 70, 2, 32, device=device, requires_grad=True)
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(torch.ops.attention.attend.default, (q, k, v), {"scale": 0.2},
                          test_utils=tests)
    lengths = torch.tensor([70, 9], dtype=torch.int32, device=device)
    torch.library.opcheck(torch.ops.attention.attend.default,
                          (q.bfloat16(), k.bfloat16(), v.bfloat16()),
                          {"scale": 0.2, "cap": 3.0, "causal": True, "lengths": lengths},
                          test_utils=tests)
    freqs = att.rotary_frequencies((8, 8))
    pos = torch.rand(2, 40, 2, device=device)
    torch.library.opcheck(torch.ops.attention.rotate.default, (q, pos, freqs, [8, 8]),
                          test_utils=tests)


def test_second_derivative_is_refused(device):
    q, k, v = (torch.randn(1, 8, 2, 32, device=device, requires_grad=True) for _ in range(3))
    (g,) = torch.autograd.grad(att.attend(q, k, v).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="derivative|not implemented"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hkv,b", [(2, 2, 4), (1, 1, 5), (16, 4, 2), (3, 1, 1)])
def test_many_heads_and_batches(device, dtype, h, hkv, b):
    """Heads that do and do not divide by the chip's eight dies."""
    _case(device, dtype, b, 260, 260, h, hkv, 64, causal=True, seed=h + b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_documents_of_every_head_dim(device, dtype, d):
    rows = [_ids((0, 70), (-1, 9), (2, 130), (3, 41))]
    _case(device, dtype, 1, 250, 250, 4, 2, d, causal=True, docs=rows, axes=2, cap=10.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_negative_and_zero_scale(device, dtype):
    g = torch.Generator().manual_seed(23)
    q, k, v, do = (torch.randn(1, n, 2, 64, generator=g).to(dtype).to(device)
                   for n in (50, 90, 90, 50))
    see = visible(1, 50, 90)
    for scale in (-0.2, 0.0):
        for t in (q, k, v):
            t.requires_grad_(True)
        out = att.attend(q, k, v, scale=scale)
        want = attention(q, k, v, see, scale=scale, dout=do)
        assert_within(out, *want["out"], "out")
        for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), do)):
            assert_within(x, *want[name], name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_many_blocks_of_documents(device, dtype, causal):
    """More blocks than run at once: those that see most tiles are started first."""
    rows = [_ids((3, 5), (0, 300), (1, 700), (2, 100)),
            _ids((0, 900), (-1, 50), (4, 155))]
    _case(device, dtype, 2, 1105, 1105, 32, 32, 32, causal=causal, docs=rows,
          lengths=[1105, 1000], qk=0.7)
