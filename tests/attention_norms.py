"""Gradients of attention in 64 bits, with how far roundings that are independent put them off.

A kernel for 16-bit types rounds weights p and score gradients ds to its type (relative error u, the
type's unit roundoff, at most, each on its own).  Errors of independent terms add in squares:

* dv_j = sum_i p_ij do_i:            u sqrt(sum_i (p_ij do_i)^2)
* dk_j = scale sum_i ds_ij q_i:      u scale sqrt(sum_i (ds_ij q_i)^2), dq the same over keys
* delta_i = sum_d out_i do_i comes from weights that the forward pass rounded, off by
  E_i = u sqrt(sum_j (p_ij dp_ij)^2), which enters all of a row's ds:
      dq: scale E_i |sum_j p_ij slant_ij k_j|;  dk: scale sqrt(sum_i (E_i p_ij slant_ij q_i)^2)

A rounding is off by u / sqrt(3) on average where u is what it may be off by: that factor is left
for everything else (float32 scores and sums).  float32 inputs take u = 2^-16, for scores off by a
few of their own roundings.  The final rounding to the type is counted as what it is.
"""

from __future__ import annotations

import torch

from attention_oracle import UNIT


def gradients(q, k, v, see, do, *, scale, cap=0.0, dlse=None):
    """name -> (value, spread): the exact gradient and the root of the squares above over u."""
    qd, kd, vd = (t.detach().double().cpu().transpose(1, 2) for t in (q, k, v))
    hkv, group = kd.shape[1], qd.shape[1] // kd.shape[1]
    kd, vd = (t.repeat_interleave(group, 1) for t in (kd, vd))
    do = do.detach().double().cpu().transpose(1, 2)
    s = scale * (qd @ kd.transpose(2, 3))
    slant = torch.ones(())
    if cap:
        t = torch.tanh(s / cap)
        s, slant = cap * t, 1 - t * t
    s = s.masked_fill(~see[:, None], -torch.inf)
    lse = torch.logsumexp(s, -1, keepdim=True)
    p = torch.exp(s - lse.masked_fill(lse == -torch.inf, 0.0))
    dp = do @ vd.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    if dlse is not None:
        ds = ds + p * dlse.double().cpu()[..., None]
    ds, ps = ds * slant, p * slant
    e = (p * dp).square().sum(-1, keepdim=True)
    shared = lambda t: t.unflatten(1, (hkv, group)).sum(2).transpose(1, 2)  # noqa: E731
    dq = scale * (ds @ kd)
    dk = scale * (ds.transpose(2, 3) @ qd)
    dv = p.transpose(2, 3) @ do
    q2 = scale ** 2 * (ds.square() @ kd.square() + e * (ps @ kd).square())
    k2 = scale ** 2 * ((ds.square() + e * ps.square()).transpose(2, 3) @ qd.square())
    v2 = p.square().transpose(2, 3) @ do.square()
    return {"dq": (dq.transpose(1, 2), q2.sqrt().transpose(1, 2)),
            "dk": (shared(dk), shared(k2).sqrt()), "dv": (shared(dv), shared(v2).sqrt())}


def assert_near(got, value, spread, dtype, label, times=1.0):
    """The norm of what ``got`` is off by, against the final rounding's and u times the spread's."""
    got = got.detach().double().cpu()
    assert got.isfinite().all(), f"{label}: not finite"
    limit = (value.to(dtype).double() - value).norm() + max(UNIT[dtype], 2.0**-16) * spread.norm()
    off = (got - value).norm()
    assert off <= times * limit, (f"{label}: off by {off / value.norm():.3g} of its norm, "
                                  f"{times * limit / value.norm():.3g} allowed")
