"""The attention entry points of a matching network (no reference counterpart).

Arguments are checked by the ops (``csrc/torch_attention.cpp``); this module turns
what programs hold (masks of any integer type, shared by the batch or not) into
what the ops take.  Device tensors only: there is no host fallback.
"""

from __future__ import annotations

import torch

from torchmatch_amd.attention import ops

# the overloads themselves: resolving them takes microseconds of every call
_ATTEND, _ROTATE = ops.attend.default, ops.rotate.default


def _on_device(t: torch.Tensor, who: str, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        msg = f"torchmatch_amd.attention.{who}: {name} must be a tensor, got {type(t).__name__}"
        raise TypeError(msg)
    if t.device.type != "cuda":
        msg = (f"torchmatch_amd.attention.{who}: runs on ROCm devices only "
               f"({name} is on {t.device})")
        raise ValueError(msg)


def _rows(t: torch.Tensor | None, batch: int, ndim: int, dtype: torch.dtype):
    """``t`` with a batch dimension (rows shared by the batch are repeated), as ``dtype``."""
    if t is None:
        return None
    if t.ndim == ndim - 1:
        t = t.unsqueeze(0).expand(batch, *t.shape)
    if dtype == torch.int32 and t.dtype in (torch.int64, torch.int16, torch.int8, torch.uint8):
        t = t.to(dtype)
    return t.contiguous()


def _limits(t: torch.Tensor | None, batch: int):
    """Numbers of keys: past 32 bits they mean all of them, as any number past the keys does."""
    if t is not None and t.dtype == torch.int64:
        t = t.clamp(0, 2**31 - 1)
    return _rows(t, batch, 1, torch.int32)


def attend(  # noqa: PLR0913
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    scale: float | None = None,
    cap: float = 0.0,
    causal: bool = False,
    prefix: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    q_docs: torch.Tensor | None = None,
    k_docs: torch.Tensor | None = None,
    slopes: torch.Tensor | None = None,
    q_positions: torch.Tensor | None = None,
    k_positions: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """Attention of ``q`` (B, Lq, H, D) over ``k``, ``v`` (B, Lk, Hkv, D); Hkv divides H
    and query head h reads key head ``h // (H // Hkv)``.

    Scores are ``scale * q.k`` (``scale`` is ``D ** -0.5`` by default), then
    ``cap * tanh(score / cap)`` where ``cap > 0`` (at most 1024 for 16-bit types), then less
    ``slopes[h]`` times the distance of the pair: of ``q_positions`` (B, Lq, axes) and
    ``k_positions`` (B, Lk, axes), summed over 1 to 3 axes, or of the indices where no
    positions are given.  What a query sees:

    * ``lengths`` (B,): the first ``lengths[b]`` keys (all by default, and where it is larger);
    * ``causal``: query i stands at ``i + length - Lq`` and sees keys up to there, and the
      first ``prefix[b]`` keys wherever it stands;
    * ``q_docs`` (B, Lq), ``k_docs`` (B, Lk): keys of the same document; negative ids are
      padding, and ids fit 32 bits.  ``k_docs`` is ``q_docs`` where it is not given.

    A query that sees nothing gets zeros, and ``-inf`` for its log-sum.  Any strides;
    features contiguous and rows 16-byte aligned are read in place, else copied.
    bfloat16, float16 or float32; sums and softmax are float32.  Differentiable in q, k
    and v, with the same bits each time.  Returns ``out`` (B, Lq, H, D), with
    ``return_lse`` also the logarithm of each row's sum, (B, H, Lq) float32, which is
    differentiable too (a row that sees nothing passes no gradient on).
    Reverse mode, once: second derivatives and forward mode are refused.
    """
    _on_device(q, "attend", "q")
    _on_device(k, "attend", "k")
    _on_device(v, "attend", "v")
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.ndim and q.shape[-1] else 1.0
    if q_docs is not None or k_docs is not None or prefix is not None or lengths is not None \
            or q_positions is not None or k_positions is not None:
        batch = q.shape[0] if q.ndim else 0
        q_docs = _rows(q_docs, batch, 2, torch.int32)
        k_docs = q_docs if k_docs is None else _rows(k_docs, batch, 2, torch.int32)
        prefix, lengths = _limits(prefix, batch), _limits(lengths, batch)
        q_positions = _rows(q_positions, batch, 3, torch.float32)
        k_positions = _rows(k_positions, batch, 3, torch.float32)
    out, lse = _ATTEND(q, k, v, slopes, q_positions, k_positions, q_docs, k_docs, prefix,
                       lengths, scale=scale, cap=cap, causal=causal)
    return (out, lse) if return_lse else out


def rotary_frequencies(
    sections: list[int] | tuple[int, ...],
    *,
    theta: float = 10000.0,
    device: torch.device | str = "cuda",
) -> torch.Tensor:
    """The angle per unit of position of each pair: ``theta ** (-p / n)`` for pair p of an
    axis's n, axis after axis (float32)."""
    if theta <= 0:
        msg = f"torchmatch_amd.attention.rotary_frequencies: theta must be positive, got {theta}"
        raise ValueError(msg)
    freqs = [theta ** (-p / n) for n in sections for p in range(n)]
    return torch.tensor(freqs, dtype=torch.float32, device=device)


def rotate(
    x: torch.Tensor,
    positions: torch.Tensor,
    freqs: torch.Tensor,
    sections: list[int] | tuple[int, ...],
    *,
    interleaved: bool = False,
    inverse: bool = False,
) -> torch.Tensor:
    """``x`` (B, L, H, D) with its feature pairs turned by ``positions`` (B, L, axes).

    ``sections[a]`` pairs turn by axis a (time, height, width, ...): pair p of a token by
    the angle ``positions[axis(p)] * freqs[p]``, and by its opposite with ``inverse``.
    Pair p is features p and P + p, P the number of pairs, or 2p and 2p + 1 where
    ``interleaved``; features past 2 P pass as they are.  Queries and keys that lie side
    by side in a projection can be turned by one call on the view that holds both.

    bfloat16, float16 or float32, any strides; positions are float32, int32 or int64,
    (L, axes) where the batch shares them.  Angles are exact to float32 at any position.
    Differentiable in x, in both modes and any number of times.
    """
    _on_device(x, "rotate", "x")
    if positions.ndim == 2 and x.ndim == 4:
        positions = positions.unsqueeze(0).expand(x.shape[0], -1, -1)
    return _ROTATE(x, positions, freqs, sections, interleaved, inverse)
