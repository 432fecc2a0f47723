"""Attention for matching networks on MI355X: the layers that produce the scores which
:mod:`torchmatch_amd.assignment` and :mod:`torchmatch_amd.transport` solve on.

Registers ``torch.ops.attention.attend`` and ``torch.ops.attention.rotate``.
"""

from __future__ import annotations

from torchmatch_amd.attention import ops
from torchmatch_amd.attention._attend import attend, rotary_frequencies, rotate

__all__ = ["attend", "ops", "rotary_frequencies", "rotate"]
