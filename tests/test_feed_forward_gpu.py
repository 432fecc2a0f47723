"""attention.feed_forward on the GPU against the 64-bit oracle."""

from __future__ import annotations

import pytest
import torch

from attention_norms import assert_near
from attention_oracle import assert_within
from layers_oracle import feed_forward
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NAMES = ("dx", "dgate", "dup", "ddown")


def _inputs(dtype, rows, c, f, o, seed, device, grad=0.02):
    g = torch.Generator(device=device).manual_seed(seed)

    def rand(size, *shape):
        return (size * torch.randn(*shape, generator=g, device=device)).to(dtype)

    rows = rows if isinstance(rows, tuple) else (rows,)
    return (rand(1.0, *rows, c), rand(c**-0.5, f, c), rand(c**-0.5, f, c), rand(f**-0.5, o, f),
            rand(grad, *rows, o))


def _check(x, gate, up, down, dy, activation="silu", norms=True):
    leaves = [t.detach().requires_grad_(True) for t in (x, gate, up, down)]
    y = att.feed_forward(*leaves, activation=activation)
    assert y.dtype == x.dtype and y.shape == dy.shape and y.is_contiguous()
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(att.feed_forward(x, gate, up, down, activation=activation), y)
    want = feed_forward(x, gate, up, down, activation, dy)
    for name, got in zip(("y", *NAMES), (y, *grads)):
        value, bound, spread = (t.cpu() for t in want[name])
        assert got.shape == value.shape and got.dtype == x.dtype and got.is_contiguous(), name
        assert_within(got, value, bound, name)
        if norms and value.numel() > 1000:
            assert_near(got, value, spread, x.dtype, name)
    return (y, *grads)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu"])
def test_activations(device, dtype, activation):
    x, *rest = _inputs(dtype, (3, 50), 96, 160, 96, 1, device)
    _check(x * 2, *rest, activation)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 5, 16, 17, 31, 33, 64, 65, 127, 128, 129, 257, 500])
def test_rows(device, dtype, rows):
    _check(*_inputs(dtype, rows, 128, 200, 72, 2, device))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c,f,o", [(1, 1, 1), (8, 8, 8), (4, 12, 20), (7, 9, 3), (33, 65, 31),
                                   (64, 63, 128), (65, 64, 129), (100, 130, 257), (256, 683, 256),
                                   (1000, 31, 2), (2, 1001, 40), (520, 264, 136)])
@pytest.mark.parametrize("rows", [3, 70])
def test_sizes(device, dtype, c, f, o, rows):
    _check(*_inputs(dtype, rows, c, f, o, 3, device))


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_tiles(device, dtype):
    """As many rows and hidden features as the large tiles are taken for, odd edges."""
    _check(*_inputs(dtype, 4097, 264, 2080, 1032, 4, device))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,f,o", [(300, 1032, 1000, 2056), (2050, 520, 1030, 1544),
                                        (4400, 136, 1100, 264), (700, 2049, 264, 2500)])
def test_split_tiles(device, dtype, rows, c, f, o):
    """Tiles past a whole number of rounds are split over k and joined, edges among them."""
    _check(*_inputs(dtype, rows, c, f, o, 18, device))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,f,o", [(2051, 1032, 140, 1032), (2060, 530, 4200, 260),
                                        (5000, 264, 130, 1100), (2300, 1160, 2060, 264)])
def test_tiles_of_more_rows(device, dtype, rows, c, f, o):
    """More rows than go in small groups: each kind of tile, split and not, in either direction."""
    _check(*_inputs(dtype, rows, c, f, o, 19, device))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c,f,o", [(136, 250, 72), (256, 683, 256), (1000, 520, 1030)])
@pytest.mark.parametrize("rows", [66, 113, 515, 1030, 2048])
def test_groups_of_rows(device, dtype, rows, c, f, o):
    """Groups of 16 and 32 rows, the last one with a part of its own."""
    _check(*_inputs(dtype, rows, c, f, o, 20, device))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,f,o", [(2049, 72, 137, 140), (3001, 40, 64, 65), (2500, 250, 33, 31),
                                        (200, 300, 700, 257), (1025, 65, 1030, 90)])
def test_small_tiles(device, dtype, rows, c, f, o):
    """Products that would give larger tiles too few blocks."""
    _check(*_inputs(dtype, rows, c, f, o, 21, device))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,f,o", [(2204, 2745, 27, 98), (2619, 47, 2591, 19), (733, 47, 5258, 630),
                                        (1821, 2255, 20, 67), (6264, 161, 16, 1725), (5270, 1484, 101, 309),
                                        (517, 2477, 1657, 183), (5959, 2805, 705, 1945)])
def test_long_and_narrow(device, dtype, rows, c, f, o):
    """One size of three far from the others: tiles of each kind, split ones past whole rounds."""
    _check(*_inputs(dtype, rows, c, f, o, 22, device))


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_weights_of_many_rows(device, dtype):
    """The weights' gradients are split over the rows."""
    _check(*_inputs(dtype, (3, 3001), 64, 100, 40, 5, device))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 9, 30])
def test_few_rows_of_long_weights(device, dtype, rows):
    _check(*_inputs(dtype, rows, 2056, 4104, 520, 6, device))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(device, dtype):
    """Views are read in place or copied; the results are the same bits."""
    x, gate, up, down, dy = _inputs(dtype, (2, 40), 64, 96, 48, 7, device)
    want = _check(x, gate, up, down, dy)

    def same(x=x, gate=gate, up=up, down=down, dy=dy):
        for a, b in zip(_check(x, gate, up, down, dy), want):
            assert torch.equal(a, b)

    both = torch.cat((gate, up))
    same(gate=both[:96], up=both[96:])
    side = torch.cat((gate, up), 1)
    same(gate=side[:, :64], up=side[:, 64:])
    same(gate=side[:, :64])
    pairs = torch.stack((gate, up), 1).flatten(0, 1)
    same(gate=pairs[::2], up=pairs[1::2])
    same(gate=gate.t().contiguous().t(), down=down.t().contiguous().t())
    same(x=x.transpose(0, 1).contiguous().transpose(0, 1))
    wide = torch.empty(2, 40, 67, dtype=dtype, device=device)
    same(x=wide[..., 1:65].copy_(x))
    wide = torch.empty(2, 40, 67, dtype=dtype, device=device)
    same(dy=wide[..., 2:50].copy_(dy))
    same(x=torch.cat((x, x), -1)[..., :64], dy=torch.cat((dy, dy), -1)[..., 48:])
    y = att.feed_forward(x[:1].expand(2, -1, -1), gate, up, down)
    assert torch.equal(y[0], want[0][0]) and torch.equal(y[1], want[0][0])
    assert torch.equal(att.feed_forward(x[0, 3], gate, up, down),
                       att.feed_forward(x[0, 3:4], gate, up, down)[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_a_sum(device, dtype):
    x, gate, up, down, _ = _inputs(dtype, 50, 64, 64, 64, 8, device)
    _check(x, gate, up, down, torch.ones((), dtype=dtype, device=device).expand(50, 64))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", [(0,), (1,), (2,), (3,), (0, 3), (1, 2)])
def test_only_some_gradients(device, dtype, which):
    *t, dy = _inputs(dtype, 90, 64, 100, 48, 9, device)
    want = _check(*t, dy)
    some = [x.detach().requires_grad_(i in which) for i, x in enumerate(t)]
    att.feed_forward(*some).backward(dy)
    for i, x in enumerate(some):
        assert torch.equal(x.grad, want[1 + i]) if i in which else x.grad is None


@pytest.mark.parametrize("size", [1e-6, 1e-4, 1e3])
def test_half_precision_gradients_of_any_size(device, size):
    """The hidden features' gradients keep their bits where the results have theirs."""
    *t, dy = _inputs(torch.float16, 600, 64, 96, 64, 10, device, grad=1.0)
    _, *want = _check(*t, dy)
    leaves = [x.detach().requires_grad_(True) for x in t]
    scale = 2.0 ** round(torch.log2(torch.tensor(size)).item())
    got = torch.autograd.grad(att.feed_forward(*leaves), leaves, dy * scale)
    for name, g, w in zip(NAMES, got, want):
        # exact but for what half precision's own range does to dy and to the result
        g, w = g.double() / scale, w.double()
        limit = 2.0**-25 / scale * (1 + 600**0.5 * 4)
        fits = w.abs() * scale < 65504
        off = (g - w).abs()[fits]
        assert (off <= 2.0**-10 * w.abs()[fits] + 8 * limit + 2.0**-9 * w.std()).all(), name


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_and_infinity_stay_in_their_rows(device, dtype):
    x, gate, up, down, _ = _inputs(dtype, 300, 72, 80, 64, 11, device)
    want = att.feed_forward(x, gate, up, down)
    x[7, 3], x[299, 71] = float("nan"), float("inf")
    got = att.feed_forward(x, gate, up, down)
    assert got[7].isnan().all() and not got[299].isfinite().any()
    got[7], got[299] = want[7], want[299]
    assert torch.equal(got, want)


def test_gradient_against_differences(device):
    """Central differences: off by the third derivative, h^2, and float32 roundings over h."""
    x, gate, up, down, dy = _inputs(torch.float32, 20, 24, 40, 16, 12, device, grad=1.0)
    t = [x, gate, up, down]
    way = [torch.randn_like(s) * s.std() for s in t]

    def value(h):
        y = att.feed_forward(*(s + h * w for s, w in zip(t, way)))
        return (y.double() * dy.double()).sum()

    leaves = [s.detach().requires_grad_(True) for s in t]
    grads = torch.autograd.grad(att.feed_forward(*leaves), leaves, dy)
    h = 2.0**-6
    slope = (value(h) - value(-h)) / (2 * h)
    told = sum((g.double() * w.double()).sum() for g, w in zip(grads, way))
    size = dy.double().abs().sum() * 4
    assert (slope - told).abs() <= size * (16 * h * h + 64 * 2.0**-24 / h)


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_again_and_on_another_stream(device, dtype):
    *t, dy = _inputs(dtype, 1500, 128, 384, 128, 13, device)

    def once():
        leaves = [x.detach().requires_grad_(True) for x in t]
        y = att.feed_forward(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, second, once()):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 12, 300])
def test_captured(device, dtype, rows):
    """Forward and backward in one graph, replayed on new inputs with eager work between."""
    *t, dy = _inputs(dtype, rows, 128, 264, 128, 14, device)
    for x in t:
        x.requires_grad_(True)

    def once():
        y = att.feed_forward(*t)
        with torch.no_grad():
            z = att.feed_forward(*t, activation="gelu")
        return (z, y.detach(), *torch.autograd.grad(y, t, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    for n in range(3):
        with torch.no_grad():
            t[0].normal_()
            t[3].normal_(0, 0.1)
            dy.normal_(0, 10.0**-n)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, once()):
            assert torch.equal(a, b)


def test_weights_past_32_bit_offsets(device):
    """Rows further apart than 32 bits of bytes reach in all."""
    row = 3 << 20
    big = torch.zeros(1100 * row, dtype=torch.float16, device=device)
    x, gate, up, down, dy = _inputs(torch.float16, 1100, 64, 1100, 64, 15, device)
    far = big.as_strided((1100, 64), (row, 1)).copy_(x)
    far_gate = big.as_strided((1100, 64), (row, 1), 64).copy_(gate)
    far_up = big.as_strided((1100, 64), (row, 1), 128).copy_(up)
    for a, b in zip(_check(far, far_gate, far_up, down, dy), _check(x, gate, up, down, dy)):
        assert torch.equal(a, b)


def test_empty_and_refused(device):
    x, gate, up, down, dy = _inputs(torch.float32, (2, 3), 16, 24, 8, 16, device)
    leaves = [t.detach().requires_grad_(True) for t in (x[:0], gate, up, down)]
    y = att.feed_forward(*leaves)
    assert y.shape == (0, 3, 8)
    for g, t in zip(torch.autograd.grad(y, leaves, dy[:0]), leaves):
        assert g.shape == t.shape and not g.any()
    with pytest.raises(ValueError, match="ROCm"):
        att.feed_forward(x.cpu(), gate, up, down)
    with pytest.raises(ValueError, match="one device"):
        att.feed_forward(x, gate.cpu(), up, down)
    with pytest.raises(TypeError, match="float32"):
        att.feed_forward(x.double(), gate, up, down)
    with pytest.raises(TypeError, match="one dtype"):
        att.feed_forward(x.half(), gate.half(), up, down.half())
    with pytest.raises(ValueError, match="activation"):
        att.feed_forward(x, gate, up, down, activation="tanh")
    with pytest.raises(ValueError, match="as x is"):
        att.feed_forward(x, gate[:, :8], up[:, :8], down)
    with pytest.raises(ValueError, match="as x is"):
        att.feed_forward(x, gate, up[:8], down)
    with pytest.raises(ValueError, match="as gate is"):
        att.feed_forward(x, gate, up, down[:, :8])
    with pytest.raises(ValueError, match="gate and up"):
        att.feed_forward(x, gate[0], up[0], down)
    with pytest.raises(ValueError, match="positive"):
        att.feed_forward(x, gate[:0], up[:0], down[:, :0])
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(att.feed_forward(x, gate, up, down).square().sum(), x,
                               create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(lambda t: att.feed_forward(t, gate, up, down), (x.detach(),),
                       (x.detach(),))
    saved = torch.zeros(1, dtype=torch.uint8, device=device)
    with pytest.raises(ValueError, match="saved"):
        torch.ops.attention.feed_forward_backward(dy, x.detach(), gate, up, down, saved, "silu")
    with pytest.raises(ValueError, match="dout"):
        torch.ops.attention.feed_forward_backward(dy[:1], x.detach(), gate, up, down, saved,
                                                  "silu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_opcheck(device, dtype):
    x, gate, up, down, dy = _inputs(dtype, (2, 5), 16, 20, 8, 17, device)
    args = [t.requires_grad_(True) for t in (x, gate, up, down)]
    torch.library.opcheck(torch.ops.attention.feed_forward.default, (*args, "silu"),
                          test_utils=("test_schema", "test_faketensor",
                                      "test_aot_dispatch_dynamic"))
    args = [t.detach() for t in args]
    torch.library.opcheck(torch.ops.attention.feed_forward_save.default, (*args, "silu"),
                          test_utils=("test_schema", "test_faketensor"))
    _, saved = torch.ops.attention.feed_forward_save(*args, "silu")
    torch.library.opcheck(torch.ops.attention.feed_forward_backward.default,
                          (dy, *args, saved, "silu"), {"need_up": False, "need_x": False},
                          test_utils=("test_schema", "test_faketensor"))
