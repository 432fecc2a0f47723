"""What stands around attention in a layer of a matching network (no reference counterpart):
queries and keys normed and turned in one pass, the gated feed-forward block, dropout.

Arguments are checked by the ops (``csrc/torch_layers.cpp``).  Device tensors only:
there is no host fallback.
"""

from __future__ import annotations

import torch

from torchmatch_amd.attention import ops
from torchmatch_amd.attention._attend import _on_device

_NORM_ROTATE, _DROPOUT = ops.norm_rotate.default, ops.dropout.default
_FEED_FORWARD = ops.feed_forward.default


def norm_rotate(  # noqa: PLR0913
    x: torch.Tensor,
    weight: torch.Tensor | None,
    positions: torch.Tensor,
    freqs: torch.Tensor,
    sections: list[int] | tuple[int, ...],
    *,
    heads: list[int] | tuple[int, ...] | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> torch.Tensor:
    """``x`` (B, L, H, D) with each head divided by its root mean square and multiplied with
    ``weight``, then turned by ``positions`` as :func:`rotate` does, in one pass.

    ``weight`` is (D,), shared by all heads, or (n, D) with ``heads``: row g is for
    ``heads[g]`` heads, which follow each other (queries and keys that lie side by side in a
    projection take one call); None for no weight.  The mean of the squares has ``eps`` added
    before its root.  ``positions``, ``freqs``, ``sections`` and ``interleaved`` are those of
    :func:`rotate`.

    bfloat16, float16 or float32, D up to 512, any strides; ``weight`` is of x's type or
    float32.  Sums are float32 and the result is rounded once.  Differentiable in x and weight,
    with the same bits each time; reverse mode, once.
    """
    _on_device(x, "norm_rotate", "x")
    if positions.ndim == 2 and x.ndim == 4:
        positions = positions.unsqueeze(0).expand(x.shape[0], -1, -1)
    if heads is None:
        heads = (x.shape[2] if x.ndim == 4 else 1,)
        if weight is not None and weight.ndim == 1:
            weight = weight.unsqueeze(0)
    return _NORM_ROTATE(x, weight, positions, freqs, sections, heads, eps, interleaved)


def feed_forward(
    x: torch.Tensor,
    gate: torch.Tensor,
    up: torch.Tensor,
    down: torch.Tensor,
    *,
    activation: str = "silu",
) -> torch.Tensor:
    """``(act(x @ gate.T) * (x @ up.T)) @ down.T``: the gated feed-forward block.

    ``x`` is (..., C), ``gate`` and ``up`` are (F, C) and ``down`` is (O, F), as linear layers hold
    them; gate and up may be the halves of one matrix.  ``activation`` is "silu", "gelu",
    "gelu_tanh" (its approximation) or "relu".  Features contiguous and rows at multiples of 16
    bytes are read in place, else copied; sizes that do not fill 16 bytes are padded.

    bfloat16, float16 or float32, all of one type.  Products are summed in float32; the hidden
    features are rounded to the type once, as are their gradients.  Half precision's hidden
    features have its range (65504).  Their gradients are held times one power of two a call: up
    where the output's gradient is small, down where one of theirs would pass the range; none is
    infinite and none loses bits that would not without it.  Those 2^15 times smaller than the
    output's largest gradient may lose some.  Differentiable in all four, with the same bits each
    time; only the gradients that are asked for are computed.
    Reverse mode, once.
    """
    _on_device(x, "feed_forward", "x")
    return _FEED_FORWARD(x, gate, up, down, activation)


def dropout(
    x: torch.Tensor,
    p: float,
    seed: int | torch.Tensor,
    offset: int = 0,
    *,
    residual: torch.Tensor | None = None,
) -> torch.Tensor:
    """``x / (1 - p)`` with elements left out (zero) with probability ``p``, added to
    ``residual`` where it is given.

    The mask is a function of ``seed``, ``offset`` and the elements' row-major places, whatever
    the type and strides, and is never stored: the gradient makes it again.  Element i stays where
    word ``i % 4`` of the ten-round Philox 4x32 generator is at least ``round(p * 2**32)``; its
    counter is ``i // 4`` and ``offset`` in 64 bits each, its key the seed.  Layers and steps that
    shall differ take another ``offset`` or ``seed`` (integers of up to 64 bits).  A seed may be an
    int64 tensor of one element on x's device, read when the kernel runs: a captured call follows
    it from replay to replay.

    bfloat16, float16 or float32.  Differentiable in x and residual, in both modes and any number
    of times.
    """
    _on_device(x, "dropout", "x")
    if isinstance(seed, torch.Tensor):
        return _DROPOUT(x, p, 0, _signed(offset, "offset"), seed, residual)
    return _DROPOUT(x, p, _signed(seed, "seed"), _signed(offset, "offset"), None, residual)


def _signed(n: int, name: str) -> int:
    """64 bits as the ops take them."""
    if not -(2**63) <= n < 2**64:
        msg = f"torchmatch_amd.attention.dropout: {name} must fit 64 bits, got {n}"
        raise ValueError(msg)
    return n - 2**64 if n >= 2**63 else n
