"""Attention for matching networks on MI355X: the layers that produce the scores which
:mod:`torchmatch_amd.assignment` and :mod:`torchmatch_amd.transport` solve on.

Attention itself, and what a layer has around it.  Registers ``torch.ops.attention.attend``,
``rotate``, ``norm_rotate``, ``feed_forward`` and ``dropout``.
"""

from __future__ import annotations

from torchmatch_amd.attention import ops
from torchmatch_amd.attention._attend import attend, rotary_frequencies, rotate
from torchmatch_amd.attention._layers import dropout, feed_forward, norm_rotate

__all__ = ["attend", "dropout", "feed_forward", "norm_rotate", "ops", "rotary_frequencies",
           "rotate"]
