"""Direct handles for the ``torch.ops.attention.*`` ops, and their shapes for fake tensors."""

from __future__ import annotations

import torch

from torchmatch_amd._loader import load as _load

_load()

attend = torch.ops.attention.attend
attend_forward = torch.ops.attention.attend_forward
attend_backward = torch.ops.attention.attend_backward
rotate = torch.ops.attention.rotate
norm_rotate = torch.ops.attention.norm_rotate
norm_rotate_backward = torch.ops.attention.norm_rotate_backward
dropout = torch.ops.attention.dropout
feed_forward = torch.ops.attention.feed_forward
feed_forward_save = torch.ops.attention.feed_forward_save
feed_forward_backward = torch.ops.attention.feed_forward_backward


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


@torch.library.register_fake("attention::norm_rotate")
def _norm_rotate_fake(x, weight, positions, freqs, sections, heads, eps, interleaved=False):
    del weight, positions, freqs, sections, heads, eps, interleaved
    torch._check(x.dim() == 4, lambda: "x must be 4D (B, L, heads, D)")
    return x.new_empty(x.shape)


@torch.library.register_fake("attention::norm_rotate_backward")
def _norm_rotate_backward_fake(dout, x, weight, positions, freqs, sections, heads, eps,
                               interleaved=False, need_x=True, need_weight=True):
    del dout, positions, freqs, sections, heads, eps, interleaved
    return (x.new_empty(x.shape if need_x else (0,)),
            weight.new_empty(weight.shape) if need_weight and weight is not None
            else x.new_empty(0))


@torch.library.register_fake("attention::dropout")
def _dropout_fake(x, p, seed=0, offset=0, seed_at=None, residual=None):
    del p, seed, offset, seed_at, residual
    return x.new_empty(x.shape)


@torch.library.register_fake("attention::feed_forward")
def _feed_forward_fake(x, gate, up, down, activation):
    del gate, up, activation
    return x.new_empty((*x.shape[:-1], down.shape[0]))


@torch.library.register_fake("attention::feed_forward_save")
def _feed_forward_save_fake(x, gate, up, down, activation):
    rows, hidden = x.numel() // x.shape[-1], (gate.shape[0] + 7) // 8 * 8
    size = 12 if x.dtype == torch.float32 else 8  # bytes for each hidden feature
    return (_feed_forward_fake(x, gate, up, down, activation),
            x.new_empty(rows * hidden * size, dtype=torch.uint8))


@torch.library.register_fake("attention::feed_forward_backward")
def _feed_forward_backward_fake(dout, x, gate, up, down, saved, activation,  # noqa: PLR0913
                                need_x=True, need_gate=True, need_up=True, need_down=True):
    del dout, saved, activation
    return tuple(x.new_empty(t.shape if need else (0,)) for t, need in
                 ((x, need_x), (gate, need_gate), (up, need_up), (down, need_down)))


__all__ = ["attend", "attend_backward", "attend_forward", "dropout", "feed_forward",
           "feed_forward_backward", "feed_forward_save", "norm_rotate", "norm_rotate_backward",
           "rotate"]
