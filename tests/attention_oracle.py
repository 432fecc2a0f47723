"""Attention and rotation in 64 bits on the CPU, with what a kernel may be off.

The bounds follow the roundings a kernel is allowed.  u is the unit roundoff of the inputs'
type (2^-8 bfloat16, 2^-11 float16; float32 rounds nothing on the way), f = 2^-16 + 2^-22 max |s|
covers float32 scores (off by a few roundings of themselves, which the exponential makes
relative), sums over up to a few thousand terms and hardware exponentials.  z is half of
the type's smallest subnormal number: what any rounding to it may be off by, however small
the value (2^-25 for float16; bfloat16 and float32 reach below what counts).

* out: weights rounded (u, z), scores and sums (f), the result rounded (u, z):
      (u + f) sum_j p |v| + z sum_j |v| over what is seen + u |out| + z
* dv:  the same with the sum over queries of p |do|.
* ds = p (dp - delta) slant: rounded (u |ds| + z); delta comes from the rounded output, off by
      E = (2u + f) sum_d (sum_j p |v|) |do|, and dp by f sum_d |v| |do|:
      e_ij = (u + f) |ds| + z + p (E + f sum_d |v| |do|)   where seen
* dq = scale ds k: scale sum_j e |k| + u |dq| + z; dk the same over queries.
"""

from __future__ import annotations

import torch

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 0.0}
HALF_SUBNORMAL = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}
F32 = 2.0**-16


def visible(b, lq, lk, *, causal=False, prefix=None, lengths=None, q_docs=None, k_docs=None):
    """(B, Lq, Lk): which keys each query sees."""
    see = torch.zeros(b, lq, lk, dtype=torch.bool)
    for n in range(b):
        length = lk if lengths is None else min(max(int(lengths[n]), 0), lk)
        for i in range(lq):
            reach = length
            if causal:
                reach = max(i + length - lq + 1, 0 if prefix is None else int(prefix[n]))
            see[n, i, :max(0, min(reach, length))] = True
        if q_docs is not None:
            qd, kd = q_docs[n].cpu(), k_docs[n].cpu()
            see[n] &= (qd[:, None] == kd[None]) & (qd[:, None] >= 0)
    return see


def attention(q, k, v, see, *, scale, cap=0.0, slopes=None, q_positions=None, k_positions=None,
              lengths=None, dout=None):
    """out, lse (and dq, dk, dv) in float64, each with its bound: a dict name -> (value,
    bound).  Values nobody sees are never touched."""
    u, z = UNIT[q.dtype], HALF_SUBNORMAL[q.dtype]
    qd, kd, vd = (t.detach().double().cpu() for t in (q, k, v))
    b, lq, h, d = qd.shape
    lk, hkv = kd.shape[1], kd.shape[2]
    group = h // hkv
    seen = see.any(1)  # (B, Lk): by anybody
    kd = kd.masked_fill(~seen[:, :, None, None], 0.0)
    vd = vd.masked_fill(~seen[:, :, None, None], 0.0)
    qd = qd.masked_fill(~see.any(2)[:, :, None, None], 0.0)
    kk = kd.repeat_interleave(group, 2).permute(0, 2, 1, 3)  # (B, H, Lk, D)
    vv = vd.repeat_interleave(group, 2).permute(0, 2, 1, 3)
    qq = qd.permute(0, 2, 1, 3)
    s = scale * (qq @ kk.transpose(2, 3))
    f = F32 + (2.0**-22 * s.abs().nan_to_num(0.0).max().item() if s.numel() else 0.0)
    slant = torch.ones_like(s)
    if cap:
        t = torch.tanh(s / cap)
        slant = 1 - t * t
        s = cap * t
    if slopes is not None:
        if q_positions is not None:
            dist = (q_positions.double().cpu()[:, :, None]
                    - k_positions.double().cpu()[:, None]).abs().sum(-1)
        else:
            i = torch.arange(lq, dtype=torch.float64)
            off = [(lk if lengths is None else min(max(int(lengths[n]), 0), lk)) - lq
                   for n in range(b)]
            dist = torch.stack([(i[:, None] + o - torch.arange(lk)).abs() for o in off])
        s = s - slopes.double().cpu()[None, :, None, None] * dist[:, None]
    s = s.masked_fill(~see[:, None], -torch.inf)
    lse = torch.logsumexp(s, -1) if lk else torch.full((b, h, lq), -torch.inf).double()
    p = torch.exp(s - lse.masked_fill(lse == -torch.inf, 0.0)[..., None])
    o = p @ vv
    a = p @ vv.abs()  # (B, H, Lq, D)
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    sees = see[:, None].double()
    res = {"out": (back(o), back((u + f) * a + z * (sees @ vv.abs()) + u * o.abs() + z)),
           "lse": (lse, f * (1 + lse.masked_fill(lse == -torch.inf, 0.0).abs()))}
    if dout is None:
        return res
    do = dout.detach().double().cpu().masked_fill(~see.any(2)[:, :, None, None], 0.0)
    do = do.permute(0, 2, 1, 3)
    ds = p * (do @ vv.transpose(2, 3) - (o * do).sum(-1, keepdim=True)) * slant
    e = (2 * u + f) * (a * do.abs()).sum(-1, keepdim=True)
    e = (u + f) * ds.abs() + z * sees + p * (e + f * (do.abs() @ vv.abs().transpose(2, 3)))
    shared = lambda t: t.unflatten(1, (hkv, group)).sum(2).permute(0, 2, 1, 3)  # noqa: E731
    dq = scale * (ds @ kk)
    res["dq"] = (back(dq), back(abs(scale) * (e @ kk.abs()) + u * dq.abs() + z))
    dk = shared(scale * (ds.transpose(2, 3) @ qq))
    res["dk"] = (dk, shared(abs(scale) * (e.transpose(2, 3) @ qq.abs())) + u * dk.abs() + z)
    dv = shared(p.transpose(2, 3) @ do)
    w = (u + f) * p + z * sees
    res["dv"] = (dv, shared(w.transpose(2, 3) @ do.abs()) + u * dv.abs() + z)
    return res


def rotation(x, positions, freqs, sections, *, interleaved=False, inverse=False):
    """The turned features in float64."""
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = positions.double().cpu()[..., axis] * freqs.double().cpu()
    if inverse:
        angle = -angle
    c, s = angle.cos()[:, :, None], angle.sin()[:, :, None]
    x = x.detach().double().cpu()
    y, p = x.clone(), len(axis)
    one = slice(0, 2 * p, 2) if interleaved else slice(0, p)
    two = slice(1, 2 * p, 2) if interleaved else slice(p, 2 * p)
    y[..., one] = x[..., one] * c - x[..., two] * s
    y[..., two] = x[..., two] * c + x[..., one] * s
    return y


def assert_within(got, value, bound, label):
    """Every element within its bound (and a rounding of float32, 2^-23, and denormals)."""
    got = got.detach().double().cpu()
    same = (got == value) | (torch.isnan(got) & torch.isnan(value))
    off = (got - value).abs()
    limit = bound + 2.0**-23 * value.abs() + 1e-30
    bad = ~(same | (off <= limit))
    if bad.any():
        worst = torch.where(bad, off / limit, 0.0).nan_to_num(torch.inf).argmax()
        at = torch.unravel_index(worst, got.shape)
        at = tuple(int(x) for x in at)
        raise AssertionError(f"{label}: {int(bad.sum())} of {bad.numel()} off, at {at} "
                             f"{got[at]:.6g} for {value[at]:.6g}, bound {limit[at]:.3g}")
