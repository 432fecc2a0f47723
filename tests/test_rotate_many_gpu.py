"""attention.rotate over more tokens than a launch has blocks."""

from __future__ import annotations

import pytest
import torch

from torchmatch_amd import attention as att

pytestmark = pytest.mark.gpu


def test_more_tokens_than_blocks(device):
    """17 million tokens of features that cannot be read 16 bytes at a time (a token a block
    where they are few): each as in a call of a few tokens."""
    tokens, heads, d, sections = (1 << 24) + 5, 19, 54, (20, 7)
    g = torch.Generator(device=device).manual_seed(1)
    one = torch.randn(1, 1, heads, d, device=device, generator=g).half()
    x = one.expand(1, tokens, heads, d)  # 34 GB of outputs from one token's features
    pos = 100 * torch.rand(1, tokens, 2, device=device, generator=g)
    freqs = att.rotary_frequencies(sections)
    y = att.rotate(x, pos, freqs, sections)
    for first in (0, tokens // 2 - 50, tokens - 100):
        rows = slice(first, first + 100)
        assert torch.equal(y[:, rows], att.rotate(x[:, rows], pos[:, rows], freqs, sections))


@pytest.mark.parametrize("sections,d", [((32,), 64), ((9,), 20)])
def test_many_tokens_of_few_features(device, sections, d):
    """One feature row a token, 16-byte reads or not: several tokens a block."""
    tokens = (1 << 24) + 3
    g = torch.Generator(device=device).manual_seed(2)
    x = torch.randn(1, 1, 1, d, device=device, generator=g).half().expand(1, tokens, 1, d)
    pos = 100 * torch.rand(1, tokens, 1, device=device, generator=g)
    freqs = att.rotary_frequencies(sections)
    y = att.rotate(x, pos, freqs, sections)
    for first in (0, tokens // 2 - 50, tokens - 100):
        rows = slice(first, first + 100)
        assert torch.equal(y[:, rows], att.rotate(x[:, rows], pos[:, rows], freqs, sections))
