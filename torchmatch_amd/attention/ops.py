"""Direct handles for the ``torch.ops.attention.*`` ops, and their shapes for fake tensors."""

from __future__ import annotations

import torch

from torchmatch_amd._loader import load as _load

_load()

attend = torch.ops.attention.attend
attend_backward = torch.ops.attention.attend_backward
rotate = torch.ops.attention.rotate


@torch.library.register_fake("attention::attend")
def _attend_fake(q, k, v, *masks, scale, cap=0.0, causal=False):  # noqa: ANN002
    del masks, scale, cap, causal
    torch._check(q.dim() == 4 and k.dim() == 4 and v.dim() == 4,
                 lambda: "q, k and v must be 4D (B, L, heads, D)")
    b, length, heads, d = q.shape
    return (q.new_empty(b, length, heads, d),
            q.new_empty(b, heads, length, dtype=torch.float32))


@torch.library.register_fake("attention::attend_forward")
def _attend_forward_fake(q, k, v, *masks, scale, cap=0.0, causal=False):  # noqa: ANN002
    out, lse = _attend_fake(q, k, v, *masks, scale=scale, cap=cap, causal=causal)
    low = q.new_empty(0) if q.dtype == torch.float32 else torch.empty_like(out)
    return out, low, lse


@torch.library.register_fake("attention::attend_backward")
def _attend_backward_fake(dout, q, k, v, *rest, scale, cap=0.0, causal=False):  # noqa: ANN002
    del dout, rest, scale, cap, causal
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


@torch.library.register_fake("attention::rotate")
def _rotate_fake(x, positions, freqs, sections, interleaved=False, inverse=False):
    del positions, freqs, sections, interleaved, inverse
    torch._check(x.dim() == 4, lambda: "x must be 4D (B, L, heads, D)")
    return x.new_empty(x.shape)


__all__ = ["attend", "attend_backward", "rotate"]
