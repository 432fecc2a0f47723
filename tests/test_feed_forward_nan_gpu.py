"""attention.feed_forward where NaN and infinities are in the weights, against the formula's places."""

from __future__ import annotations

import pytest
import torch

from layers_oracle import _activation
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTIVATIONS = ["silu", "gelu", "gelu_tanh", "relu"]
ROWS = [5, 2100]  # rows in groups; tiles, which calls of more than 2048 rows always take


def _inputs(dtype, rows, seed, device, c=72, f=80, o=64):
    g = torch.Generator(device=device).manual_seed(seed)

    def rand(size, *shape):
        return (size * torch.randn(*shape, generator=g, device=device)).to(dtype)

    return (rand(1.0, rows, c), rand(c**-0.5, f, c), rand(c**-0.5, f, c), rand(f**-0.5, o, f),
            rand(0.02, rows, o))


def _formula(x, gate, up, down, activation, dy):
    """y, dx, dgate, dup, ddown in float64."""
    x, gate, up, down, dy = (t.detach().double() for t in (x, gate, up, down, dy))
    a, b = x @ gate.t(), x @ up.t()
    # the oracle's relu keeps NaN (clamp), its slope there is 0
    act, slope, _ = _activation(a, activation)
    h, dh = act * b, dy @ down
    da, db = dh * b * slope, dh * act
    return h @ down.t(), da @ gate + db @ up, da.t() @ x, db.t() @ x, dy.t() @ h


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("which", ["gate", "up", "down"])
def test_nan_in_one_weight_is_seen(device, dtype, activation, rows, which):
    *t, dy = _inputs(dtype, rows, 1, device)
    t[("x", "gate", "up", "down").index(which)][11, 7] = float("nan")
    leaves = [v.detach().requires_grad_(True) for v in t]
    y = att.feed_forward(*leaves, activation=activation)
    got = (y, *torch.autograd.grad(y, leaves, dy))
    with torch.no_grad():
        assert torch.equal(att.feed_forward(*t, activation=activation).isnan(), y.isnan())
    want = _formula(*t, activation, dy)
    for name, a, b in zip(("y", "dx", "dgate", "dup", "ddown"), got, want):
        assert b.isnan().any() or which != "gate" or name == "dgate"
        assert torch.equal(a.isnan(), b.isnan()), name
        assert not a.isinf().any(), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinite_gate_weight(device, dtype, activation, rows, sign):
    """Infinite where the formula is, not a number where it is not one, and rows that relu closes
    as they are with a weight row of zeros."""
    x, gate, up, down, dy = _inputs(dtype, rows, 2, device)
    gate[11, 7] = sign * float("inf")
    got = att.feed_forward(x, gate, up, down, activation=activation)
    want = _formula(x, gate, up, down, activation, dy)[0]
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isposinf(), want.isposinf())
    assert torch.equal(got.isneginf(), want.isneginf())
    if activation == "relu":
        shut = x[:, 7] * sign < 0
        assert shut.any() and want[shut].isfinite().all()
        gate[11] = 0
        zero = att.feed_forward(x, gate, up, down, activation=activation)
        assert torch.equal(got[shut], zero[shut])


@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_a_float32_infinity_is_seen(device, activation):
    """In tiles, whose products are of parts, it is NaN for every row; in groups as in the formula."""
    x, gate, up, down, dy = _inputs(torch.float32, 2100, 3, device)
    gate[11, 7] = float("inf")
    assert att.feed_forward(x, gate, up, down, activation=activation).isnan().all()
    got = att.feed_forward(x[:5], gate, up, down, activation=activation)
    want = _formula(x[:5], gate, up, down, activation, dy[:5])[0]
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isposinf(), want.isposinf())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("rows", ROWS)
def test_gates_far_from_zero(device, dtype, activation, rows):
    """a = 2^70 and its like, whose square float32 does not hold, with b = 0: nothing is infinite.
    dx is db U alone there (da = dh b act' = 0), db rounded once and dx once."""
    x, gate, up, down, dy = _inputs(dtype, rows, 4, device)
    up[:, 0] = 0
    x[3] = 0
    x[3, 0] = 2.0**70
    dy[3] *= 2.0**-40
    leaves = [v.detach().requires_grad_(True) for v in (x, gate, up, down)]
    y = att.feed_forward(*leaves, activation=activation)
    got = (y, *torch.autograd.grad(y, leaves, dy))
    want = _formula(x, gate, up, down, activation, dy)
    for name, a, b in zip(("y", "dx", "dgate", "dup", "ddown"), got, want):
        assert b.isfinite().all() and a.isfinite().all(), name
    assert not got[0][3].any()
    # each term of a sum is off by u of itself, and sums of 64 and 80 terms by their float32 roundings
    u = torch.finfo(dtype).eps / 2
    dh = dy[3].double() @ down.double()
    act = _activation(2.0**70 * gate[:, 0].double(), activation)[0]
    terms = (dy[3].double().abs() @ down.double().abs()) * act.abs() @ up.double().abs()
    limit = (2 * u + 160 * 2.0**-23) * terms + 2.0**-18 * (dh * act).abs() @ up.double().abs()
    assert ((got[1][3].double() - want[1][3]).abs() <= limit).all()
