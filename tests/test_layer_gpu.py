"""A layer of a matching network out of the attention entry points, as they are used together."""

from __future__ import annotations

import pytest
import torch

from layers_oracle import stays
from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu

H, KV, D, F, SECTIONS = 4, 2, 32, 96, (8, 8)
C = H * D
P = 0.2


def _parameters(dtype, device):
    g = torch.Generator().manual_seed(0)
    rand = lambda size, *s: (size * torch.randn(*s, generator=g)).to(dtype).to(device)  # noqa: E731
    return {"qkv": rand(C**-0.5, (H + 2 * KV) * D, C), "norm": 1 + rand(0.1, 2, D),
            "out": rand(C**-0.5, C, C), "gate": rand(C**-0.5, F, C), "up": rand(C**-0.5, F, C),
            "down": rand(F**-0.5, C, F)}


def _layer(x, p, pos, freqs, docs, seed):
    b, n, _ = x.shape
    qkv = torch.nn.functional.linear(x, p["qkv"]).view(b, n, H + 2 * KV, D)
    qk = att.norm_rotate(qkv[:, :, :H + KV], p["norm"], pos, freqs, SECTIONS, heads=(H, KV))
    a = att.attend(qk[:, :, :H], qk[:, :, H:], qkv[:, :, H + KV:], q_docs=docs)
    x = att.dropout(torch.nn.functional.linear(a.flatten(2), p["out"]), P, seed, 0, residual=x)
    y = att.feed_forward(x, p["gate"], p["up"], p["down"])
    return att.dropout(y, P, seed, 1, residual=x)


def _reference(x, p, pos, freqs, docs, seed):
    """The same in the tensors' own type (float64) by plain operations."""
    b, n, _ = x.shape
    axis = [a for a, s in enumerate(SECTIONS) for _ in range(s)]
    angle = pos.double()[..., axis] * freqs.double()
    c, s = angle.cos()[:, :, None], angle.sin()[:, :, None]
    qkv = (x @ p["qkv"].t()).view(b, n, H + 2 * KV, D)
    qk = qkv[:, :, :H + KV]
    qk = qk * (qk.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * p["norm"][[0] * H + [1] * KV]
    u, v = qk.split(D // 2, -1)
    qk = torch.cat((u * c - v * s, v * c + u * s), -1)
    q, k = qk[:, :, :H], qk[:, :, H:].repeat_interleave(H // KV, 2)
    v = qkv[:, :, H + KV:].repeat_interleave(H // KV, 2)
    w = torch.einsum("bihd,bjhd->bhij", q, k) * D**-0.5
    w = w.masked_fill((docs[:, :, None] != docs[:, None])[:, None], -torch.inf).softmax(-1)
    a = torch.einsum("bhij,bjhd->bihd", w, v).flatten(2)

    def dropped(t, offset):
        keep = stays(0, t.numel(), P, seed, offset).view(t.shape).to(t.device)
        return torch.where(keep, t / (1 - P), 0.0)

    x = x + dropped(a @ p["out"].t(), 0)
    h = torch.nn.functional.silu(x @ p["gate"].t()) * (x @ p["up"].t())
    return x + dropped(h @ p["down"].t(), 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,n", [(1, 1), (2, 70)])
def test_forward_and_gradients(device, dtype, b, n):
    """Against 64 bits: eight roundings of the layer's results follow one another forward, as many
    backward, each of half a step of its own size or less, with sizes near one throughout."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(b, n, C, generator=g).to(dtype).to(device)
    dy = torch.randn(b, n, C, generator=g).to(dtype).to(device)
    pos = (20 * torch.rand(b, n, 2, generator=g)).to(device)
    docs = (torch.arange(n, dtype=torch.int32) // 40).expand(b, n).contiguous().to(device)
    freqs, p = att.rotary_frequencies(SECTIONS), _parameters(dtype, device)
    leaves = [x, *p.values()]

    def run(layer, leaves):
        leaves = [t.detach().requires_grad_(True) for t in leaves]
        y = layer(leaves[0], dict(zip(p, leaves[1:])), pos, freqs, docs, 7)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy.to(y.dtype)))

    got = run(_layer, leaves)
    want = run(_reference, [t.double() for t in leaves])
    u = torch.finfo(dtype).eps / 2
    limit = 16 * u
    # A query that sees one key has a weight of 1, and the gradients of its query, its key and their
    # norm are zero: what is left of ds = do v - sum(out do), where out is v but for u^2 of it (its
    # rounding is carried along) and sums of D products are off by D 2^-24 at most.  With |q|, |k|
    # <= 1.3 sqrt(D), |v| <= 1.5 sqrt(D) and sum_h |do_h| <= 2 sqrt(H) |dy|, the norm's gradient is
    # scale |ds| |k| |q| <= (u^2 + D 2^-24) 4 sqrt(H) D |dy| at most.
    left = (u * u + D * 2.0**-24) * 4 * H**0.5 * D * dy.double().norm()
    for name, a, w in zip(("y", "x", *p), got, want):
        assert a.dtype == dtype and a.shape == w.shape
        # independent roundings: their norms add in squares, eight and eight of them
        assert (a.double() - w).norm() <= (limit * w.norm() if w.any() else left), name


def test_captured_training_step(device):
    """One graph of forward and backward, the seed on the device: replays follow it."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 60, C, generator=g).bfloat16().to(device)
    pos = (20 * torch.rand(2, 60, 2, generator=g)).to(device)
    docs = torch.zeros(2, 60, dtype=torch.int32, device=device)
    freqs, p = att.rotary_frequencies(SECTIONS), _parameters(torch.bfloat16, device)
    for t in p.values():
        t.requires_grad_(True)
    seed = torch.zeros((), dtype=torch.int64, device=device)

    def once():
        y = _layer(x, p, pos, freqs, docs, seed)
        return (y.detach(), *torch.autograd.grad(y, list(p.values()), x))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    last = None
    for _ in range(3):
        seed += 1
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, once()):
            assert torch.equal(a, b)
        assert last is None or not torch.equal(last, got[0])
        last = got[0].clone()


def test_two_graphs_and_a_side_stream(device):
    """Captured calls have their own workspaces: two graphs run one after the other, on their
    streams, and beside eager calls, and give what each gives alone."""
    p = _parameters(torch.float16, device)
    x = [torch.randn(1, n, C, device=device).half() for n in (40, 900)]
    feed = lambda t: att.feed_forward(t, p["gate"], p["up"], p["down"])  # noqa: E731
    want = [feed(t) for t in x]
    graphs, got, streams = [], [], [torch.cuda.Stream() for _ in x]
    for t, stream in zip(x, streams):
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got.append(feed(t))
        graphs.append(graph)
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        beside = feed(x[1])
        torch.cuda.synchronize()
        assert torch.equal(beside, want[1])
        for a, b in zip(got, want):
            assert torch.equal(a, b)
