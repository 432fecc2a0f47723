"""attention.feed_forward's gradients in half precision over its whole range.

The gradients of the hidden features are held in half precision times one power of two, chosen so that
none of them is infinite that is not so without it, and that none loses bits that it has without it:
what each element is off by is at most half a step of its own (u = 2^-11) or half of the smallest
subnormal number (z = 2^-25).  A row of dx is then off by u of the squares' root of its terms and by z of
those of the weights; each gradient is rounded once more.  Independent roundings add in squares; one
is off by its bound over sqrt(3) on average, which is left for everything else.
"""

from __future__ import annotations

import pytest
import torch

from attention_norms import assert_near
from layers_oracle import feed_forward
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

U, Z = 2.0**-11, 2.0**-25
HALF = torch.float16


def _rand(g, size, *shape):
    return (size * torch.randn(*shape, generator=g, device=g.device)).to(HALF)


def _grads(t, dy, activation="silu", which=(0, 1, 2, 3)):
    leaves = [v.detach().requires_grad_(i in which) for i, v in enumerate(t)]
    y = att.feed_forward(*leaves, activation=activation)
    return torch.autograd.grad(y, [leaves[i] for i in which], dy)


def _rows_near(got, t, want):
    """Each row of dx on its own."""
    value, _, spread = want["dx"]
    floor = Z * (t[1].double().square().sum() + t[2].double().square().sum()).sqrt()
    limit = (value.to(HALF).double() - value).norm(dim=-1) + U * spread.norm(dim=-1) + floor
    off = (got.double() - value).norm(dim=-1)
    assert got.isfinite().all()
    assert (off <= limit).all(), (off / limit).max().item()


@pytest.mark.parametrize("rows", [64, 700, 2500])
@pytest.mark.parametrize("outlier", [8, 11, 13])
def test_rows_of_mixed_size(device, rows, outlier):
    """One row of the output's gradient 2^18 to 2^23 times as large as the others."""
    g = torch.Generator(device=device).manual_seed(1)
    t = (_rand(g, 1.0, rows, 256), _rand(g, 1 / 16, 512, 256), _rand(g, 1 / 16, 512, 256),
         _rand(g, 512**-0.5, 256, 512))
    dy = torch.randn(rows, 256, generator=g, device=device).clamp(-4, 4) * 2.0**-10
    dy[5] *= 2.0**(outlier + 10) / 4
    dy = dy.to(HALF)
    want = feed_forward(*t, "silu", dy)
    got = _grads(t, dy)
    _rows_near(got[0], t, want)
    for name, a in zip(("dgate", "dup", "ddown"), got[1:]):
        assert_near(a, *(v.cpu() for v in (want[name][0], want[name][2])), HALF, name)


# rows, width, hidden features, outputs: products of dy and down in each kind of tile, whole and split
SHAPES = [(64, 256, 512, 1024), (1030, 256, 512, 1024), (300, 264, 137, 2056), (733, 48, 5258, 630),
          (4097, 64, 2080, 72), (4500, 64, 1100, 1032), (508, 40, 3979, 5745),
          (3565, 24, 4815, 3991)]


def _amplified(device, rows, c, f, o, size, seed):
    """A gate near zero beside large features of up: h and y are of ordinary size, da is far larger
    than dy."""
    g = torch.Generator(device=device).manual_seed(seed)
    t = (_rand(g, 1.0, rows, c), _rand(g, 0.01 * c**-0.5, f, c), _rand(g, 8000 * c**-0.5, f, c),
         _rand(g, 1.0, o, f))
    return t, _rand(g, size, rows, o)


@pytest.mark.parametrize("rows,c,f,o", SHAPES)
@pytest.mark.parametrize("size", [1e-5, 3e-4])
def test_large_features_beside_small_gradients(device, rows, c, f, o, size):
    t, dy = _amplified(device, rows, c, f, o, size, 2)
    want = feed_forward(*t, "silu", dy)
    for name in ("y", "dx", "dgate", "dup", "ddown"):
        assert want[name][0].abs().max() < 65504, name
    got = _grads(t, dy)
    _rows_near(got[0], t, want)
    for name, a in zip(("dgate", "dup", "ddown"), got[1:]):
        assert_near(a, *(v.cpu() for v in (want[name][0], want[name][2])), HALF, name)


@pytest.mark.parametrize("rows,c,f,o", SHAPES[:3])
def test_hidden_gradients_past_the_range(device, rows, c, f, o):
    """Past 65504 as they are, the inputs' gradients within: scaled down."""
    t, dy = _amplified(device, rows, c, f, o, 1.0, 3)
    want = feed_forward(*t, "silu", dy)
    value, _, spread = want["dx"]
    dh = dy.double() @ t[3].double()
    assert (dh * (t[0].double() @ t[2].double().t()) / 2).abs().max() > 2 * 65504
    fits = value.abs() < 60000
    dx, dup = _grads(t, dy, which=(0, 2))
    assert dx[fits].isfinite().all() and fits.double().mean() > 0.99
    # the scale is 2^-7 or more, and what it leaves in db, which is far smaller than da, is off by z
    floor = 2.0**7 * Z * rows**0.5 * (t[1].double().square().sum()
                                      + t[2].double().square().sum()).sqrt()
    limit = (value.to(HALF).double() - value)[fits].norm() + U * spread[fits].norm() + floor
    assert (dx.double() - value)[fits].norm() <= limit
    value, _, spread = want["dup"]
    limit = (value.to(HALF).double() - value).norm() + U * spread.norm() \
        + 2.0**7 * Z * t[0].double().norm() * f**0.5
    assert (dup.double() - value).norm() <= limit


def test_infinite_and_nan_gradients_leave_the_others(device):
    """Rows of the output's gradient that are no numbers do not choose the scale."""
    t, dy = _amplified(device, 300, 64, 136, 72, 1e-3, 4)
    want = _grads(t, dy)[0]
    bad = dy.clone()
    bad[7, 3], bad[200, 1] = float("nan"), float("inf")
    got = _grads(t, bad)[0]
    assert got[7].isnan().all() and not got[200].isfinite().all()
    rest = [i for i in range(300) if i not in (7, 200)]
    assert got[rest].isfinite().all()
    off = (got[rest].double() - want[rest].double()).norm()
    assert off <= 2 * U * want[rest].double().norm()


def test_replays_choose_their_own_scale(device):
    """A captured backward pass: each replay as the eager call, whether the one before overflowed or
    not."""
    t, dy = _amplified(device, 515, 128, 520, 264, 1e-3, 5)
    for v in t:
        v.requires_grad_(True)

    def once():
        return torch.autograd.grad(att.feed_forward(*t), t, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    for n, (up, size) in enumerate([(500.0, 1e-3), (0.1, 1e-3), (500.0, 1e-4), (0.1, 1e-6), (500.0, 3.0)]):
        with torch.no_grad():
            t[2].normal_(0, up)
            dy.normal_(0, size)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, once()):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)), n
            assert n == 4 or a.isfinite().all(), n
