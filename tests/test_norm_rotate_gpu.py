"""attention.norm_rotate on the GPU against the 64-bit oracle."""

from __future__ import annotations

import pytest
import torch

from attention_oracle import assert_within
from layers_oracle import norm_rotate
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(dtype, b, n, heads, d, sections, seed, device, wide=False):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(b, n, sum(heads), d, generator=g)
         * torch.randn(b, n, 1, 1, generator=g).exp()).to(dtype).to(device)
    w = (1 + 0.3 * torch.randn(len(heads), d, generator=g)).to(torch.float32 if wide else dtype)
    pos = (50 * torch.rand(b, n, len(sections), generator=g)).to(device)
    dy = torch.randn(b, n, sum(heads), d, generator=g).to(dtype).to(device)
    return x, w.to(device), pos, att.rotary_frequencies(sections), dy


def _check(x, w, pos, freqs, sections, heads, dy, eps=1e-6, interleaved=False):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y = att.norm_rotate(x, w, pos, freqs, sections, heads=heads, eps=eps,
                        interleaved=interleaved)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dw.dtype == w.dtype and dw.shape == w.shape and dx.shape == x.shape
    want = norm_rotate(x, w, pos if pos.ndim == 3 else pos.expand(x.shape[0], *pos.shape), freqs,
                       sections, heads, eps, interleaved, dy, w.dtype)
    for name, got in (("y", y), ("dx", dx), ("dw", dw)):
        assert_within(got, *want[name], name)
    return y, dx, dw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,sections", [
    (128, (64,)), (128, (16, 24, 24)), (64, (8, 8)), (96, (48,)), (256, (128,)), (512, (256,)),
    (512, (0,)), (80, (20, 12)), (32, (16,)), (16, (3, 2, 1, 1)), (30, (7, 8)), (1, (0,)),
    (2, (1,)), (500, (249,)), (36, (10,)), (510, (1,))])
def test_head_layouts(device, dtype, interleaved, d, sections):
    heads = (4, 1)
    x, w, pos, freqs, dy = _inputs(dtype, 2, 37, heads, d, sections, 1, device)
    _check(x, w, pos, freqs, sections, heads, dy, interleaved=interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,n,heads", [(1, 1, (1,)), (1, 1, (32, 8)), (8, 1, (3, 1)),
                                       (1, 3001, (1,)), (3, 700, (5, 2, 1)), (2, 2500, (8,)),
                                       (2, 9, (1,) * 8), (300, 5, (2, 2))])
def test_shapes(device, dtype, b, n, heads):
    x, w, pos, freqs, dy = _inputs(dtype, b, n, heads, 64, (16, 16), 2, device, wide=True)
    _check(x, w, pos, freqs, (16, 16), heads, dy)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(device, dtype):
    """Views of a projection are read in place, others copied; results are the same bits."""
    heads, sections = (4, 1), (32,)
    x, w, pos, freqs, dy = _inputs(dtype, 2, 50, (4, 1, 3), 64, sections, 3, device)
    x, w, dy = x[:, :, :5], w[:2], dy[:, :, :5]
    want = _check(x.contiguous(), w, pos, freqs, sections, heads, dy.contiguous())

    def same(x, w=w, pos=pos, dy=dy):
        for a, b in zip(_check(x, w, pos, freqs, sections, heads, dy), want):
            assert torch.equal(a, b)

    same(x)
    same(x.transpose(1, 2).contiguous().transpose(1, 2))
    same(x.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2))
    same(torch.empty(2, 50, 5, 67, dtype=dtype, device=device)[..., 1:65].copy_(x))
    same(x, dy=torch.empty(2, 50, 5, 67, dtype=dtype, device=device)[..., 1:65].copy_(dy))
    same(x, w=w.t().contiguous().t())
    wide = torch.rand(2, 50, 3, device=device)
    wide[..., 1:2] = pos
    same(x, pos=wide[..., 1:2])
    one = _check(x[:1].expand(2, -1, -1, -1), w, pos[0], freqs, sections, heads, dy)
    assert torch.equal(one[0][0], want[0][0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_a_sum(device, dtype):
    """The output's gradient has stride 0."""
    x, w, pos, freqs, _ = _inputs(dtype, 2, 20, (2,), 32, (16,), 4, device)
    one = torch.ones((), dtype=dtype, device=device).expand(x.shape)
    _check(x, w, pos, freqs, (16,), (2,), one)


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_weight_and_shared_weight(device, dtype):
    x, w, pos, freqs, dy = _inputs(dtype, 1, 40, (3,), 64, (32,), 5, device)
    x.requires_grad_(True)
    y = att.norm_rotate(x, None, pos, freqs, (32,))
    want = norm_rotate(x, None, pos, freqs, (32,), (3,), 1e-6, False, dy)
    assert_within(y, *want["y"], "y")
    assert_within(torch.autograd.grad(y, x, dy)[0], *want["dx"], "dx")
    y = att.norm_rotate(x, w[0], pos, freqs, (32,))
    assert torch.equal(y, att.norm_rotate(x, w, pos, freqs, (32,), heads=(3,)))
    leaf = w[0].clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(att.norm_rotate(x, leaf, pos, freqs, (32,)), leaf, dy)
    assert dw.shape == (64,)


@pytest.mark.parametrize("dtype", DTYPES)
def test_only_some_gradients(device, dtype):
    x, w, pos, freqs, dy = _inputs(dtype, 2, 33, (2, 1), 64, (32,), 6, device)
    _, dx, dw = _check(x, w, pos, freqs, (32,), (2, 1), dy)
    for need_x in (True, False):
        a, b = x.detach().requires_grad_(need_x), w.detach().requires_grad_(not need_x)
        y = att.norm_rotate(a, b, pos, freqs, (32,), heads=(2, 1))
        (g,) = torch.autograd.grad(y, a if need_x else b, dy)
        assert torch.equal(g, dx if need_x else dw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sizes_of_rows(device, dtype):
    """Rows of zeros give zeros; rows far from one in size are normed all the same."""
    x, w, pos, freqs, dy = _inputs(dtype, 1, 6, (2,), 64, (32,), 7, device)
    x = x * torch.tensor([0.0, 1.0, 2.0**-6, 2.0**6, 2.0**10, 1.0], device=device,
                         dtype=dtype).view(1, 6, 1, 1)
    y, dx, _ = _check(x, w, pos, freqs, (32,), (2,), dy, eps=1e-3)
    assert not y[:, 0].any() and dx[:, 0].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_stays_in_its_head(device, dtype):
    x, w, pos, freqs, _ = _inputs(dtype, 1, 5, (2, 2), 64, (32,), 8, device)
    want = att.norm_rotate(x, w, pos, freqs, (32,), heads=(2, 2))
    x[0, 2, 1, 5] = float("nan")
    got = att.norm_rotate(x, w, pos, freqs, (32,), heads=(2, 2))
    assert got[0, 2, 1].isnan().all()
    got[0, 2, 1] = want[0, 2, 1]
    assert torch.equal(got, want)


def test_against_norm_then_rotate(device):
    """The two passes of a program that has no such call: float32, a few roundings apart."""
    x, w, pos, freqs, _ = _inputs(torch.float32, 2, 60, (3, 1), 96, (20, 20), 9, device)
    row = [0, 0, 0, 1]
    normed = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w[row]
    want = att.rotate(normed, pos, freqs, (20, 20))
    got = att.norm_rotate(x, w, pos, freqs, (20, 20), heads=(3, 1))
    assert (got - want).abs().max() <= 64 * 2.0**-24 * normed.abs().max()


def test_gradient_against_differences(device):
    """Central differences along random ways: off by the third derivative, h^2 times a number
    of the size of the value's terms, and by float32 roundings over h."""
    x, w, pos, freqs, dy = _inputs(torch.float32, 1, 7, (2, 1), 32, (16,), 10, device)
    x = x / x.square().mean(-1, keepdim=True).sqrt()
    wayx, wayw = torch.randn_like(x), torch.randn_like(w)

    def value(t):
        y = att.norm_rotate(x + t * wayx, w + t * wayw, pos, freqs, (16,), heads=(2, 1))
        return (y.double() * dy.double()).sum()

    x.requires_grad_(True)
    w.requires_grad_(True)
    y = att.norm_rotate(x, w, pos, freqs, (16,), heads=(2, 1))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x, w, h = x.detach(), w.detach(), 2.0**-6
    slope = (value(h) - value(-h)) / (2 * h)
    told = (dx.double() * wayx.double()).sum() + (dw.double() * wayw.double()).sum()
    terms = dy.double().abs().sum() * 4
    assert (slope - told).abs() <= terms * (16 * h * h + 64 * 2.0**-24 / h)


def test_same_bits_again_and_on_another_stream(device):
    x, w, pos, freqs, dy = _inputs(torch.bfloat16, 2, 1500, (4, 2), 128, (64,), 11, device)

    def once():
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = att.norm_rotate(a, b, pos, freqs, (64,), heads=(4, 2))
        return (y.detach(), *torch.autograd.grad(y, (a, b), dy))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, second, once()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured(device):
    """Forward and backward in one graph, replayed on new inputs with eager work between."""
    x, w, pos, freqs, dy = _inputs(torch.float16, 2, 70, (4, 2), 64, (16, 16), 12, device)
    x.requires_grad_(True)
    w.requires_grad_(True)

    def once():
        y = att.norm_rotate(x, w, pos, freqs, (16, 16), heads=(4, 2))
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    for _ in range(3):
        with torch.no_grad():
            x.normal_()
            w.uniform_(0.5, 1.5)
            pos.uniform_(0, 9)
            dy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, once()):
            assert torch.equal(a, b)


def test_far_positions(device):
    x, w, _, freqs, dy = _inputs(torch.bfloat16, 1, 64, (2,), 64, (32,), 13, device)
    pos = torch.arange(64, device=device).view(1, 64, 1) * 16381 + 1_000_000
    for kind in (torch.int32, torch.int64, torch.float32):
        _check(x, w, pos.to(kind), freqs, (32,), (2,), dy)


def test_rows_past_32_bit_offsets(device):
    """Tokens further apart than 32 bits of elements reach."""
    row = 1 << 22
    big = torch.zeros(1100 * row, dtype=torch.float16, device=device)
    x, w, pos, freqs, dy = _inputs(torch.float16, 1, 1100, (1,), 64, (32,), 14, device)
    far = big.as_strided((1, 1100, 1, 64), (0, row, 0, 1)).copy_(x)
    for a, b in zip(_check(far, w, pos, freqs, (32,), (1,), dy),
                    _check(x, w, pos, freqs, (32,), (1,), dy)):
        assert torch.equal(a, b)


def test_empty_and_refused(device):
    x, w, pos, f, dy = _inputs(torch.float32, 2, 3, (2, 1), 16, (4, 4), 15, device)
    s, h = (4, 4), (2, 1)
    for a, p in ((x[:0], pos[:0]), (x[:, :0], pos[:, :0])):
        a, b = a.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = att.norm_rotate(a, b, p, f, s, heads=h)
        assert y.shape == a.shape
        dx, dw = torch.autograd.grad(y, (a, b), torch.ones_like(y))
        assert dx.shape == a.shape and not dw.any() and dw.shape == w.shape
    with pytest.raises(ValueError, match="ROCm"):
        att.norm_rotate(x.cpu(), w, pos, f, s, heads=h)
    with pytest.raises(ValueError, match="4D"):
        att.norm_rotate(x[0], w, pos, f, s, heads=h)
    with pytest.raises(TypeError, match="float32"):
        att.norm_rotate(x.double(), w, pos, f, s, heads=h)
    with pytest.raises(TypeError, match="weight"):
        att.norm_rotate(x.half(), w.bfloat16(), pos, f, s, heads=h)
    with pytest.raises(ValueError, match="weight"):
        att.norm_rotate(x, w[:1], pos, f, s, heads=h)
    with pytest.raises(ValueError, match="weight"):
        att.norm_rotate(x, w.cpu(), pos, f, s, heads=h)
    with pytest.raises(ValueError, match="heads"):
        att.norm_rotate(x, w, pos, f, s, heads=(2, 2))
    with pytest.raises(ValueError, match="heads"):
        att.norm_rotate(x, w, pos, f, s, heads=(3, 0))
    with pytest.raises(ValueError, match="heads"):
        att.norm_rotate(x, None, pos, f, s, heads=())
    with pytest.raises(ValueError, match="eps"):
        att.norm_rotate(x, w, pos, f, s, heads=h, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        att.norm_rotate(x, w, pos, f, s, heads=h, eps=float("nan"))
    with pytest.raises(ValueError, match="positions must be"):
        att.norm_rotate(x, w, pos[:, :2], f, s, heads=h)
    with pytest.raises(ValueError, match="half"):
        att.norm_rotate(x, w, pos, att.rotary_frequencies((4, 5)), (4, 5), heads=h)
    wide = torch.zeros(1, 1, 1, 513, device=device)
    with pytest.raises(ValueError, match="512"):
        att.norm_rotate(wide, None, pos[:1, :1], f, s)
    with pytest.raises(NotImplementedError, match="positions"):
        att.norm_rotate(x, w, pos.clone().requires_grad_(True), f, s, heads=h)
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(att.norm_rotate(x, w, pos, f, s, heads=h).square().sum(), x,
                               create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(lambda t: att.norm_rotate(t, w, pos, f, s, heads=h), (x.detach(),),
                       (x.detach(),))


@pytest.mark.parametrize("weight", [False, True])
def test_opcheck(device, weight):
    x, w, pos, f, dy = _inputs(torch.float32, 2, 5, (2, 1), 16, (4, 4), 16, device)
    x.requires_grad_(True)
    args = (x, w.requires_grad_(True) if weight else None, pos, f, [4, 4], [2, 1], 1e-6)
    torch.library.opcheck(torch.ops.attention.norm_rotate.default, args,
                          test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))
    plain = [a.detach() if isinstance(a, torch.Tensor) else a for a in args]
    for need_x in (True, False):
        torch.library.opcheck(torch.ops.attention.norm_rotate_backward.default, (dy, *plain),
                              {"need_x": need_x, "need_weight": weight},
                              test_utils=("test_schema", "test_faketensor"))
