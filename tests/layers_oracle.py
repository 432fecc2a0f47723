"""The layer's operators around attention in 64 bits, with what a kernel may be off.

u is the unit roundoff of the inputs' type.  A cosine or sine is off by e: 2^-18 for 16-bit types
(hardware sines) and 2^-21 for float32, angles and products included.  A float32 sum over a head adds
at most 22 numbers one after the other (16 of a lane, 6 exchanges), so it is off by 22 of its roundings
(2^-24), a root mean square by 11 of them; four more roundings multiply the factors.
"""

from __future__ import annotations

import numpy as np
import torch

from attention_oracle import UNIT, rotation

SINE = {torch.bfloat16: 2.0**-18, torch.float16: 2.0**-18, torch.float32: 2.0**-21}
ULP = 2.0**-24
# the smallest subnormal number's half: what any rounding may be off by
FLOOR = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}


def norm_rotate(x, weight, pos, freqs, sections, heads, eps, interleaved, dy=None, wdtype=None):
    """name -> (value, bound) of y (and dx, dw) in float64."""
    dtype = x.dtype
    u, e, z = UNIT[dtype] or ULP, SINE[dtype], FLOOR[dtype]
    xd = x.detach().double().cpu()
    b, n, h, d = xd.shape
    groups = len(heads)
    row = [g for g, k in enumerate(heads) for _ in range(k)]
    w = torch.ones(h, d, dtype=torch.float64) if weight is None else \
        weight.detach().double().cpu()[row]
    r = (xd.square().mean(-1, keepdim=True) + eps).rsqrt()
    normed = xd * r * w
    y = rotation(normed, pos, freqs, sections, interleaved=interleaved)
    size = 2 * normed.abs().amax(-1, keepdim=True)
    found = {"y": (y, u * y.abs() + z + (e + 16 * ULP) * size)}
    if dy is None:
        return found
    g = rotation(dy.detach(), pos, freqs, sections, interleaved=interleaved, inverse=True)
    gs = 2 * dy.detach().double().cpu().abs().amax(-1, keepdim=True)
    mean = (g * w * xd * r).mean(-1, keepdim=True)
    dx = r * (g * w - xd * r * mean)
    spread = ((g * w * xd).abs() * r).mean(-1, keepdim=True)
    off = r * e * gs * (w.abs() + (xd * r).abs() * ((w * xd).abs() * r).mean(-1, keepdim=True))
    off = off + 64 * ULP * r * ((g * w).abs() + (xd * r).abs() * spread)
    found["dx"] = (dx, u * dx.abs() + z + off)
    dw, bound = torch.zeros(groups, d).double(), torch.zeros(groups, d).double()
    terms, about = g * xd * r, e * gs * (xd * r).abs() + 16 * ULP * (g * xd * r).abs()
    chain = b * n * max(heads) + 64  # additions in one sum, at most
    for k, q in enumerate(row):
        dw[q] += terms[:, :, k].sum((0, 1))
        bound[q] += about[:, :, k].sum((0, 1)) + chain * ULP * terms[:, :, k].abs().sum((0, 1))
    uw = UNIT[wdtype] or ULP if wdtype is not None else ULP
    found["dw"] = (dw, bound + uw * dw.abs() + (FLOOR[wdtype] if wdtype is not None else 0.0))
    return found


# ---- dropout -------------------------------------------------------------------------


def philox(counter, key):
    """Ten rounds of Philox 4x32 on rows of four counter words (uint64 arrays of 32-bit values)."""
    low = np.uint64(0xFFFFFFFF)
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    k0, k1 = np.uint64(key[0]), np.uint64(key[1])
    for _ in range(10):
        m, n = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(n >> np.uint64(32)) ^ c[1] ^ k0, n & low, (m >> np.uint64(32)) ^ c[3] ^ k1, m & low]
        k0, k1 = (k0 + np.uint64(0x9E3779B9)) & low, (k1 + np.uint64(0xBB67AE85)) & low
    return np.stack(c, 1)


def stays(first, count, p, seed, offset):
    """Which of the elements first .. first + count - 1 dropout leaves in."""
    seed, offset = seed % 2**64, offset % 2**64
    begin = first // 4
    at = np.arange(begin, (first + count + 3) // 4, dtype=np.uint64)
    counter = np.stack([at & np.uint64(0xFFFFFFFF), at >> np.uint64(32),
                        np.full_like(at, offset & 0xFFFFFFFF), np.full_like(at, offset >> 32)], 1)
    words = philox(counter, (seed & 0xFFFFFFFF, seed >> 32)).reshape(-1)
    words = words[first - 4 * begin:][:count]
    return torch.from_numpy(words >= np.uint64(round(p * 2**32)))


def dropout(x, p, seed, offset=0, residual=None):
    """The value and its bound: a float32 product and sum, then the result's rounding."""
    u, z = UNIT[x.dtype] or ULP, FLOOR[x.dtype]
    keep = stays(0, x.numel(), p, seed, offset).view(x.shape)
    xd = x.detach().double().cpu()
    kept = torch.where(keep, xd / (1 - p) if p < 1 else xd, 0.0)
    r = residual.detach().double().cpu() if residual is not None else torch.zeros_like(kept)
    y = r + kept
    return y, u * y.abs() + z + 4 * ULP * (kept.abs() + r.abs())
