"""A small matching network end to end: attention, then transport, then assignment.

Two sets of points with noisy descriptors are matched.  Both sets of every pair lie in one
row of a packed batch: the points' features are turned by their image coordinates
(``attention.rotate``), each set attends to itself with a bias by distance and then to the
other one (``attention.attend``, documents keep pairs apart), and the products of the features
are the scores.  Training follows the negative log of a softmax over rows and columns;
matching solves the transport problem on the scores (``transport.matrix.solve``) and rounds
its plan to a one-to-one mapping (``assignment.solve``).

    python examples/match_points.py [--steps 60] [--points 96] [--pairs 8]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from torchmatch_amd import assignment, attention, transport  # noqa: E402

HEADS, HEAD_DIM, SECTIONS = 4, 32, (8, 8)
WIDTH = HEADS * HEAD_DIM


class Block(nn.Module):
    """Attention within the sets, attention across, and a feed-forward part."""

    def __init__(self) -> None:
        super().__init__()
        self.norm_self, self.norm_cross, self.norm_mlp = (nn.LayerNorm(WIDTH) for _ in range(3))
        self.qkv = nn.Linear(WIDTH, 3 * WIDTH)
        self.q, self.kv = nn.Linear(WIDTH, WIDTH), nn.Linear(WIDTH, 2 * WIDTH)
        self.out_self, self.out_cross = nn.Linear(WIDTH, WIDTH), nn.Linear(WIDTH, WIDTH)
        self.mlp = nn.Sequential(nn.Linear(WIDTH, 2 * WIDTH), nn.GELU(),
                                 nn.Linear(2 * WIDTH, WIDTH))

    def forward(self, x, other, pos, docs, other_docs, slopes, freqs):
        """``x``: (1, rows, WIDTH) of one side; ``other``: the other side's features."""
        rows = x.shape[1]
        qkv = self.qkv(self.norm_self(x)).view(1, rows, 3 * HEADS, HEAD_DIM)
        # queries and keys lie side by side: one call turns both
        qk = attention.rotate(qkv[:, :, :2 * HEADS], pos, freqs, SECTIONS)
        a = attention.attend(qk[:, :, :HEADS], qk[:, :, HEADS:], qkv[:, :, 2 * HEADS:],
                             q_docs=docs, slopes=slopes, q_positions=pos, k_positions=pos)
        x = x + self.out_self(a.flatten(2))
        q = self.q(self.norm_cross(x)).view(1, rows, HEADS, HEAD_DIM)
        kv = self.kv(self.norm_cross(other)).view(1, other.shape[1], 2 * HEADS, HEAD_DIM)
        a = attention.attend(q, kv[:, :, :HEADS], kv[:, :, HEADS:], cap=30.0, q_docs=docs,
                             k_docs=other_docs)
        x = x + self.out_cross(a.flatten(2))
        return x + self.mlp(self.norm_mlp(x))


class Matcher(nn.Module):
    """Scores (pairs, points, points) of packed pairs of point sets."""

    def __init__(self, features: int, blocks: int = 2) -> None:
        super().__init__()
        self.embed = nn.Linear(features, WIDTH)
        self.blocks = nn.ModuleList(Block() for _ in range(blocks))
        self.head = nn.Linear(WIDTH, WIDTH)
        self.register_buffer("freqs", attention.rotary_frequencies(SECTIONS, device="cpu"))
        self.register_buffer("slopes", 0.5 ** torch.arange(1.0, HEADS + 1))

    def forward(self, left, right, left_pos, right_pos):
        pairs, n, m = left.shape[0], left.shape[1], right.shape[1]
        ids = torch.arange(pairs, dtype=torch.int32, device=left.device)
        docs_l, docs_r = (ids.repeat_interleave(k)[None] for k in (n, m))
        x, y = (self.embed(t).flatten(0, 1)[None] for t in (left, right))
        pos_l, pos_r = (t.flatten(0, 1)[None] for t in (left_pos, right_pos))
        for block in self.blocks:
            x, y = (block(x, y, pos_l, docs_l, docs_r, self.slopes, self.freqs),
                    block(y, x, pos_r, docs_r, docs_l, self.slopes, self.freqs))
        x = self.head(x).view(pairs, n, WIDTH)
        y = self.head(y).view(pairs, m, WIDTH)
        return x @ y.transpose(1, 2).contiguous() / WIDTH ** 0.5


def match(scores: torch.Tensor) -> torch.Tensor:
    """One-to-one mapping (pairs, points): the transport plan's best assignment."""
    cost = scores.amax((1, 2), keepdim=True) - scores
    log_plan = transport.matrix.solve(cost.float().contiguous(), reg=1.0, n_iter=50)
    return assignment.solve((-log_plan).clamp(max=1e6).contiguous())


def sample(pairs: int, n: int, features: int, generator: torch.Generator, device):
    """Points, the same points turned, moved and shuffled, and which is which."""
    pos = 20 * torch.rand(pairs, n, 2, generator=generator)
    desc = torch.randn(pairs, n, features, generator=generator)
    order = torch.stack([torch.randperm(n, generator=generator) for _ in range(pairs)])
    turn = 0.3 * torch.randn(pairs, 1, generator=generator)
    c, s = turn.cos(), turn.sin()
    moved = torch.stack((pos[..., 0] * c - pos[..., 1] * s, pos[..., 0] * s + pos[..., 1] * c), -1)
    at = order[..., None]
    right_pos = moved.gather(1, at.expand(-1, -1, 2))
    noise = torch.randn(pairs, n, features, generator=generator)
    right = desc.gather(1, at.expand(-1, -1, features)) + 0.8 * noise
    truth = order.argsort(1)  # left point i is right point truth[i]
    return [t.to(device) for t in (desc, right, pos, right_pos, truth)]


def train(steps: int = 60, pairs: int = 8, points: int = 96, features: int = 16, seed: int = 0,
          log=print):
    """Trains a matcher on sampled pairs; returns the losses and the share of new points that
    it matches right."""
    torch.manual_seed(seed)
    device = torch.device("cuda")
    generator = torch.Generator().manual_seed(seed)
    model = Matcher(features).to(device)
    adam = torch.optim.Adam(model.parameters(), lr=1e-3)
    losses = []
    for step in range(steps):
        *batch, truth = sample(pairs, points, features, generator, device)
        scores = model(*batch)
        log_p = scores.log_softmax(2) + scores.log_softmax(1)
        loss = -log_p.gather(2, truth[..., None]).mean()
        adam.zero_grad()
        loss.backward()
        adam.step()
        losses.append(loss.item())
        if step % 10 == 0:
            log(f"step {step:3d}  loss {losses[-1]:.3f}")
    *batch, truth = sample(pairs, points, features, generator, device)
    with torch.no_grad():
        found = match(model(*batch))
    right = (found == truth).float().mean().item()
    log(f"matched right: {right:.1%}")
    return losses, right


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--points", type=int, default=96)
    parser.add_argument("--pairs", type=int, default=8)
    args = parser.parse_args()
    train(args.steps, args.pairs, args.points)
