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


# ---- feed_forward --------------------------------------------------------------------


def _activation(a, name):
    """Value, slope, and how much the slope changes with a, at most."""
    if name == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s)), 0.5
    if name == "relu":
        return a.clamp(min=0), (a > 0).double(), 0.0
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-a / 2**0.5)
        return a * cdf, cdf + a * torch.exp(-a * a / 2) / (2 * torch.pi) ** 0.5, 0.8
    k = (2 / torch.pi) ** 0.5
    t = torch.tanh(k * (a + 0.044715 * a**3))
    return 0.5 * a * (1 + t), \
        0.5 * (1 + t) + 0.5 * a * (1 - t * t) * k * (1 + 3 * 0.044715 * a * a), 0.8


def feed_forward(x, gate, up, down, activation, dy=None):
    """name -> (value, bound, spread) of y (and dx, dgate, dup, ddown) in float64, on x's device.

    bound: every product's sum is off by its length times 2^-23 of its terms' sizes (float32), an
    activation by 2^-19 |a| (16 bits: hardware exponentials; float32 2^-21), a slope by as much of
    1 + |a|; h, da and db are rounded (u); a and b are saved with 2^-15 (16-bit types).
    spread: what independent roundings of h, da and db by one part put a result off by, in squares.
    """
    dtype, c = x.dtype, x.shape[-1]
    u, z = UNIT[dtype] or ULP, FLOOR[dtype]
    half = dtype != torch.float32
    cut, act_off = (2.0**-15, 2.0**-19) if half else (0.0, 2.0**-21)
    xd, g, w, d = (t.detach().double() for t in (x, gate, up, down))
    xd = xd.reshape(-1, c)
    length = lambda n: n * 2.0**-23  # noqa: E731
    a, b = xd @ g.t(), xd @ w.t()
    ea, eb = (length(c) * (xd.abs() @ m.abs().t()) for m in (g, w))
    act, slope, bend = _activation(a, activation)

    def slope_off(ea):
        if activation == "relu":
            return (a.abs() <= ea).double()
        return bend * ea + act_off * (1 + a.abs())

    h = act * b
    eh = (slope.abs() * ea + bend * ea * ea + act_off * a.abs()) * (b.abs() + eb) + act.abs() * eb
    eh = eh + u * h.abs() + z
    y = h @ d.t()
    ey = eh @ d.abs().t() + length(len(gate)) * (h.abs() @ d.abs().t()) + u * y.abs() + z
    found = {"y": (y.view(*x.shape[:-1], -1), ey.view(*x.shape[:-1], -1),
                   (h.square() @ d.square().t()).sqrt().view(*x.shape[:-1], -1))}
    if dy is None:
        return found
    dyd = dy.detach().double().reshape(len(xd), -1)
    dh = dyd @ d
    edh = length(len(down)) * (dyd.abs() @ d.abs())
    ea, eb = ea + cut * a.abs(), eb + cut * b.abs()
    es = slope_off(ea)
    da, db = dh * b * slope, dh * act
    top = dyd.abs().max().item() if dyd.numel() else 1.0
    zg = z * 2 * top  # float16: held times a power of two that brings dy to 1 .. 2
    eda = edh * (b * slope).abs() + dh.abs() * (eb * slope.abs() + (b.abs() + eb) * es) \
        + (u + 4 * ULP) * da.abs() + zg
    edb = edh * act.abs() + dh.abs() * (slope.abs() * ea + bend * ea * ea + act_off * a.abs()) \
        + (u + 4 * ULP) * db.abs() + zg
    # h again, from what was saved
    eh = (slope.abs() * ea + bend * ea * ea + act_off * a.abs()) * (b.abs() + eb) \
        + act.abs() * eb + u * h.abs() + z

    def product(terms, n):
        value = sum(p @ q for p, q, _ in terms)
        size = sum(p.abs() @ q.abs() for p, q, _ in terms)
        off = sum(e @ q.abs() for _, q, e in terms)
        spread = sum(p.square() @ q.square() for p, q, _ in terms).sqrt()
        return value, off + length(n) * size + u * value.abs() + z, spread

    v = product([(da, g, eda), (db, w, edb)], 2 * len(gate))
    found["dx"] = tuple(t.view(x.shape) for t in v)
    n = len(xd)
    found["dgate"] = product([(da.t(), xd, eda.t())], n)
    found["dup"] = product([(db.t(), xd, edb.t())], n)
    found["ddown"] = tuple(t.t() for t in product([(h.t(), dyd, eh.t())], n))
    return found
