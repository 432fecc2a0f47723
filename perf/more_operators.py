"""The operators around attention that this framework is timed on.

A matching network's layer is attention between rotated queries and keys and a
feed-forward part, each added to what came in.  Three operators of such a layer
are measured: the norm of queries and keys for each head with the rotation by
positions in the same pass, the gated feed-forward block, and dropout whose mask
is made again wherever it is needed; forward, with gradients, and for single
tokens.

With ``own`` false :func:`run` computes them in plain float32 torch
operations; with ``own`` true it calls ``torchmatch_amd.attention``.
"""

from __future__ import annotations

import math

import torch

own = False

_DEV = "cuda"
_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_EPS = 1e-6


def _norm(name, b, length, heads, d, sections, *, dtype="bfloat16", interleaved=False, grid=(),
          train=False, packed=False, start=0, wide=False):
    """``heads``: how many heads each row of the weight is for (queries, keys); ``grid``: integer
    positions on a grid of these sides, else uniform float positions; ``packed``: x is the
    query and key part of a wider projection; ``wide``: the weight is float32."""
    return {"name": name, "op": "norm_rotate", "B": b, "L": length,
            "heads": ",".join(map(str, heads)), "D": d, "sections": ",".join(map(str, sections)),
            "dtype": dtype, "interleaved": interleaved, "grid": ",".join(map(str, grid)),
            "train": train, "packed": packed, "start": start, "wide": wide}


def _feed(name, b, length, c, f, *, o=0, dtype="bfloat16", activation="silu", train=False):
    """(B, L, C) features through F hidden ones to O (C where it is 0)."""
    return {"name": name, "op": "feed_forward", "B": b, "L": length, "C": c, "F": f, "O": o or c,
            "dtype": dtype, "activation": activation, "train": train}


def _drop(name, b, length, c, p, *, dtype="bfloat16", residual=True, train=False, on_device=False):
    """``residual``: what the result is added to; ``on_device``: the seed lies in a tensor, as a
    captured training step needs it."""
    return {"name": name, "op": "dropout", "B": b, "L": length, "C": c, "p": p, "dtype": dtype,
            "residual": residual, "train": train, "on_device": on_device}


def listed():
    return [
        # one new token for each of eight streams: latency only
        _norm("norm_rotate_token_8x1x40x128", 8, 1, (32, 8), 128, (64,), grid=(70001,),
              start=70000, packed=True),
        # a video clip on a time, height and width grid, odd sides, queries and keys out of one
        # projection
        _norm("norm_rotate_video_2x9x37x41", 2, 13653, (24, 8), 128, (16, 24, 24),
              grid=(9, 37, 41), interleaved=True, packed=True),
        # key points with image coordinates and packed documents' tokens, in a training step
        _norm("norm_rotate_train_4x4099", 4, 4099, (16, 4), 128, (32, 32), train=True,
              packed=True, wide=True),
        # one new token, a single stream: every weight is read once
        _feed("feed_token_1x2048x5632", 1, 1, 2048, 5632),
        # a few tokens of each of some streams: weights bound it still
        _feed("feed_tokens_3x5x4096x11264", 3, 5, 4096, 11264, dtype="float16"),
        # a small matching layer in float32 as a training step needs it, an odd hidden size
        _feed("feed_points_train_f32_16x2048", 16, 2048, 256, 683, dtype="float32",
              activation="gelu", train=True),
        # prompts of an odd length
        _feed("feed_prompt_2x4097", 2, 4097, 2048, 5632, activation="gelu_tanh"),
        # odd sizes throughout, half precision, with gradients
        _feed("feed_odd_train_3x1237", 3, 1237, 1000, 2731, dtype="float16", activation="relu",
              train=True),
        # a training step's long rows
        _feed("feed_train_1x8192", 1, 8192, 2048, 5632, train=True),
        # a small layer's step: latency
        _drop("dropout_points_4x301x256", 4, 301, 256, 0.1, dtype="float32"),
        # a training step, the seed on the device
        _drop("dropout_train_1x8192x2048", 1, 8192, 2048, 0.1, train=True, on_device=True),
        # all of a large step's hidden features
        _drop("dropout_large_16x2047x4099", 16, 2047, 4099, 0.25, dtype="float16",
              residual=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    kind = rng.random()
    if kind < 0.3:
        d = rng.choice((32, 64, 64, 96, 128, 128, 256))
        axes = rng.choice((1, 2, 3))
        left = d // 2 if rng.random() < 0.8 else d // 4  # all, or half, of each head is rotated
        sections = []
        for a in range(axes, 0, -1):
            sections.append(left if a == 1 else max(1, left // a + rng.choice((-1, 0, 1))))
            left -= sections[-1]
        length = _log_int(rng, 1, 20000)
        kv = rng.choice((1, 2, 4, 8))
        heads = (kv * rng.choice((1, 2, 4)), kv) if rng.random() < 0.8 else (kv,)
        b = _log_int(rng, 1, max(1, min(32, 60_000_000 // (length * sum(heads) * d))))
        if rng.random() < 0.5 and (dtype != "float32" or axes > 1):
            side = max(1, math.ceil(length ** (1 / axes)))
            grid = (math.ceil(length / side ** (axes - 1)),) + (side,) * (axes - 1)
        else:
            grid = ()
        c = _norm("", b, length, heads, d, sections, dtype=dtype,
                  interleaved=rng.random() < 0.5, grid=grid, train=rng.random() < 0.4,
                  packed=rng.random() < 0.5,
                  start=rng.choice((0, 0, 5000)) if grid and dtype != "float32" else 0,
                  wide=rng.random() < 0.5)
    elif kind < 0.75:
        activation = rng.choice(("silu", "silu", "gelu", "gelu_tanh", "relu"))
        train = rng.random() < 0.45
        width = _log_int(rng, 64, 4096)
        hidden = int(width * rng.uniform(1.5, 4.5))
        if rng.random() < 0.7:  # most networks keep to multiples of 64
            width, hidden = max(64, width // 64 * 64), max(64, hidden // 64 * 64)
        budget = (9.4e10 if dtype != "float32" else 1.2e10) / (1 if train else 1 / 3)
        most = max(1, int(budget / (width * hidden)))
        tokens = _log_int(rng, 1, min(16, most)) if rng.random() < 0.35 else \
            _log_int(rng, min(17, most), min(60000, most))
        b = rng.choice((1, 1, 2, 3))
        c = _feed("", b, max(1, tokens // b), width, hidden,
                  o=width if rng.random() < 0.8 else max(8, width // 2 + rng.choice((-3, 0, 8))),
                  dtype=dtype, activation=activation, train=train)
    else:
        length, width = _log_int(rng, 1, 16384), _log_int(rng, 16, 4099)
        b = _log_int(rng, 1, max(1, min(64, 120_000_000 // (length * width))))
        c = _drop("", b, length, width, rng.choice((0.0, 0.05, 0.1, 0.3, 0.5)), dtype=dtype,
                  residual=rng.random() < 0.6, train=rng.random() < 0.5,
                  on_device=rng.random() < 0.5)
    del c["name"]
    return c


# ---- inputs --------------------------------------------------------------------------


def _ints(text):
    return [int(t) for t in text.split(",")] if text else []


def _prepare_norm(case, g):
    b, n, d = case["B"], case["L"], case["D"]
    heads, sections, grid = _ints(case["heads"]), _ints(case["sections"]), _ints(case["grid"])
    dtype, h = _DTYPES[case["dtype"]], sum(heads)
    full = torch.randn(b, n, h + heads[-1] if case["packed"] else h, d, device=_DEV, generator=g)
    # tokens' projections differ in size
    full = full * torch.exp(torch.randn(b, n, 1, 1, device=_DEV, generator=g))
    if grid:
        at = (torch.arange(n, device=_DEV) + case["start"]) % math.prod(grid)
        cols = []
        for side in reversed(grid):
            cols.append(at % side)
            at = at // side
        pos = torch.stack(cols[::-1], -1).expand(b, n, len(grid)).contiguous()
        # each stream is at another place
        pos = pos + torch.randint(0, 3, (b, 1, 1), device=_DEV, generator=g)
    else:
        pos = 640 * torch.rand(b, n, len(sections), device=_DEV, generator=g)
    freqs = torch.cat([10000.0 ** (-torch.arange(s, device=_DEV, dtype=torch.float32) / s)
                       for s in sections])
    weight = 1 + 0.2 * torch.randn(len(heads), d, device=_DEV, generator=g)
    st = {"case": case, "x": full.to(dtype)[:, :, :h], "pos": pos, "freqs": freqs,
          "sections": sections, "heads": heads,
          "weight": weight if case["wide"] else weight.to(dtype)}
    if case["train"]:
        st["dy"] = torch.randn(b, n, h, d, device=_DEV, generator=g).to(dtype)
        st["x"].requires_grad_(True)
        st["weight"].requires_grad_(True)
    return st


def _prepare_feed(case, g):
    b, n, c, f, o = (case[k] for k in ("B", "L", "C", "F", "O"))
    dtype = _DTYPES[case["dtype"]]

    def rand(size, *shape):
        return (size * torch.randn(*shape, device=_DEV, generator=g)).to(dtype)

    # normed features, weights that keep their size
    st = {"case": case, "x": rand(1.0, b, n, c), "gate": rand(c ** -0.5, f, c),
          "up": rand(c ** -0.5, f, c), "down": rand(f ** -0.5, o, f)}
    if case["train"]:
        st["dy"] = rand(0.02, b, n, o)
        for k in ("x", "gate", "up", "down"):
            st[k].requires_grad_(True)
    return st


def _prepare_drop(case, g):
    shape, dtype = (case["B"], case["L"], case["C"]), _DTYPES[case["dtype"]]

    def rand():
        return torch.randn(*shape, device=_DEV, generator=g).to(dtype)

    seed = torch.randint(0, 2**62, (), device=_DEV, generator=g)
    st = {"case": case, "x": rand(), "residual": rand() if case["residual"] else None,
          "seed": seed if case["on_device"] else int(seed), "offset": 3}
    if case["train"]:
        st["dy"] = rand()
        st["x"].requires_grad_(True)
    return st


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    if case["op"] == "norm_rotate":
        return _prepare_norm(case, g)
    return _prepare_feed(case, g) if case["op"] == "feed_forward" else _prepare_drop(case, g)


# ---- plain forms ---------------------------------------------------------------------


def _turn(x, cos, sin, interleaved):
    """Pairs of x's leading features turned by angles whose cos and sin are given."""
    p = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :p], x[..., p:2 * p]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * p:]), -1)


def _plain_norm(st):
    case, heads = st["case"], st["heads"]
    axis = [a for a, s in enumerate(st["sections"]) for _ in range(s)]
    # far positions: a float32 angle would be off by more than the result's rounding
    angle = st["pos"].double()[..., axis] * st["freqs"].double()
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    row = [i for i, n in enumerate(heads) for _ in range(n)]
    w = st["weight"].detach().float()[row]
    x = st["x"].detach().float()
    size = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
    y = _turn(x * size * w, cos, sin, case["interleaved"]).to(st["x"].dtype)
    if not case["train"]:
        return y
    g = _turn(st["dy"].float(), cos, -sin, case["interleaved"])
    gw = g * w
    dx = size * (gw - x * size.square() * (gw * x).mean(-1, keepdim=True))
    dw = (g * x * size).sum((0, 1))
    dw = torch.zeros_like(w[:len(heads)]).index_add_(0, torch.tensor(row, device=_DEV), dw)
    return y, dx.to(st["x"].dtype), dw.to(st["weight"].dtype)


def _activate(a, name):
    """The activation and its slope."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-a))
        return a * s, s * (1 + a * (1 - s))
    if name == "relu":
        return a.clamp(min=0), (a > 0).to(a.dtype)
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-a * math.sqrt(0.5))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) * (2 * math.pi) ** -0.5
    inner = math.sqrt(2 / math.pi)
    t = torch.tanh(inner * (a + 0.044715 * a ** 3))
    return 0.5 * a * (1 + t), \
        0.5 * (1 + t) + 0.5 * a * (1 - t * t) * inner * (1 + 3 * 0.044715 * a * a)


def _plain_feed(st):
    case, dtype = st["case"], st["x"].dtype
    x = st["x"].detach().float().flatten(0, 1)
    gate, up, down = (st[k].detach().float() for k in ("gate", "up", "down"))
    a, b = x @ gate.t(), x @ up.t()
    act, slope = _activate(a, case["activation"])
    h = act * b
    y = (h @ down.t()).view(case["B"], case["L"], case["O"]).to(dtype)
    if not case["train"]:
        return y
    dy = st["dy"].float().flatten(0, 1)
    dh = dy @ down
    da, db = dh * b * slope, dh * act
    dx = (da @ gate + db @ up).view_as(st["x"])
    return tuple(t.to(dtype) for t in (y, dx, da.t() @ x, db.t() @ x, dy.t() @ h))


def _kept(count, p, seed, offset, dev):
    """Which elements stay: four 32-bit words of the ten-round Philox generator (Salmon and
    others, "Parallel random numbers: as easy as 1, 2, 3", 2011) for each four elements."""
    low = 0xFFFFFFFF
    i = torch.arange((count + 3) // 4, device=dev)
    c0, c1 = i & low, i >> 32
    c2, c3 = (torch.full_like(i, offset >> s & low) for s in (0, 32))
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        # 64-bit products wrap, their bits are those of the unsigned ones
        m, n = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = n >> 32 & low ^ c1 ^ k0, n & low, m >> 32 & low ^ c3 ^ k1, m & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack((c0, c1, c2, c3), 1).flatten()[:count]
    return words >= round(p * 2.0**32)


def _plain_drop(st):
    case, x = st["case"], st["x"].detach()
    seed = st["seed"]
    keep = _kept(x.numel(), case["p"], seed, st["offset"], x.device).view(x.shape)
    scale = 1 / (1 - case["p"])
    zero = torch.zeros((), device=x.device)
    y = torch.where(keep, x.float() * scale, zero)
    if st["residual"] is not None:
        y = y + st["residual"].float()
    y = y.to(x.dtype)
    if not case["train"]:
        return y
    return y, torch.where(keep, st["dy"].float() * scale, zero).to(x.dtype)


def run(state):
    case, op = state["case"], state["case"]["op"]
    if not own:
        if op == "norm_rotate":
            return _plain_norm(state)
        return _plain_feed(state) if op == "feed_forward" else _plain_drop(state)
    from torchmatch_amd import attention

    if op == "norm_rotate":
        inputs = (state["x"], state["weight"])
        y = attention.norm_rotate(*inputs, state["pos"], state["freqs"], state["sections"],
                                  heads=state["heads"], eps=_EPS,
                                  interleaved=case["interleaved"])
    elif op == "feed_forward":
        inputs = tuple(state[k] for k in ("x", "gate", "up", "down"))
        y = attention.feed_forward(*inputs, activation=case["activation"])
    else:
        inputs = (state["x"],)
        y = attention.dropout(state["x"], case["p"], state["seed"], state["offset"],
                              residual=state["residual"])
    if not case["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, inputs, state["dy"]))


# ---- work and exact values -----------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    n = case["B"] * case["L"]
    if case["op"] == "norm_rotate":
        axes, pairs, h = len(_ints(case["sections"])), sum(_ints(case["sections"])), \
            sum(_ints(case["heads"]))
        rows = n * h * case["D"]
        places = n * axes * (8 if case["grid"] else 4)
        # read, square, scale and turn; x and dy to dx and dw
        if not case["train"]:
            return {"bytes": 2 * rows * size + places, "flops": 4 * rows + 6 * n * h * pairs}
        return {"bytes": 4 * rows * size + places, "flops": 15 * rows + 12 * n * h * pairs}
    if case["op"] == "feed_forward":
        c, f, o = case["C"], case["F"], case["O"]
        weights, rows = 2 * c * f + o * f, n * (c + o)
        # with gradients: inputs and the output's gradient read, output and gradients written,
        # two products backward for each one forward
        return {"bytes": (2 if case["train"] else 1) * (weights + rows) * size,
                "flops": (6 if case["train"] else 2) * n * weights}
    count = n * case["C"]
    reads = 2 if case["residual"] else 1
    passes = reads + 1 + (2 if case["train"] else 0)
    return {"bytes": passes * count * size, "flops": 3 * count}


def _exact_norm(st):
    x, w = st["x"].detach().double(), st["weight"].detach().double()
    pos, freqs, heads = st["pos"].double(), st["freqs"].double(), st["heads"]
    owner = torch.repeat_interleave(torch.arange(len(st["sections"]), device=_DEV),
                                    torch.tensor(st["sections"], device=_DEV))
    unit = torch.polar(torch.ones((), dtype=torch.float64, device=_DEV),
                       pos.index_select(-1, owner) * freqs)[:, :, None]
    pairs, d = len(owner), st["case"]["D"]

    def turned(t, u):
        head = t[..., :2 * pairs]
        if st["case"]["interleaved"]:
            z = torch.view_as_complex(head.unflatten(-1, (pairs, 2)).contiguous()) * u
            head = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(head[..., :pairs].contiguous(), head[..., pairs:].contiguous()) * u
            head = torch.cat((z.real, z.imag), -1)
        return torch.cat((head, t[..., 2 * pairs:]), -1)

    parts = list(zip(x.split(heads, 2), w))
    norms = [((part * part).sum(-1, keepdim=True) / d + _EPS).sqrt() for part, _ in parts]
    y = torch.cat([turned(part / r * v, unit) for (part, v), r in zip(parts, norms)], 2)
    if not st["case"]["train"]:
        return y
    dx, dw = [], []
    for (part, v), r, g in zip(parts, norms, st["dy"].double().split(heads, 2)):
        g = turned(g, unit.conj())
        u = part / r
        dw.append(torch.einsum("blhd,blhd->d", g, u))
        g = g * v
        dx.append((g - u * ((g * u).sum(-1, keepdim=True) / d)) / r)
    return y, torch.cat(dx, 2), torch.stack(dw)


def _exact_feed(st):
    """Gradients by torch's own differentiation of the formula in 64 bits."""
    from torch.nn import functional as fn

    case = st["case"]
    leaves = [st[k].detach().double().requires_grad_(case["train"])
              for k in ("x", "gate", "up", "down")]
    x, gate, up, down = leaves
    act = {"silu": fn.silu, "relu": fn.relu, "gelu": fn.gelu,
           "gelu_tanh": lambda t: fn.gelu(t, approximate="tanh")}[case["activation"]]
    y = fn.linear(act(fn.linear(x, gate)) * fn.linear(x, up), down)
    if not case["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, leaves, st["dy"].double()))


def _exact_drop(st):
    """The generator by 16-bit halves, one word of the four at a time."""
    case, x = st["case"], st["x"].detach()
    seed, low = int(st["seed"]), 0xFFFFFFFF

    def product(c, m):
        """High and low 32 bits of c m."""
        t = (c & 0xFFFF) * m
        u = (c >> 16) * m + (t >> 16)
        return u >> 16, (u & 0xFFFF) << 16 | t & 0xFFFF

    n = x.numel()
    at = torch.arange(-(-n // 4), device=x.device)
    ctr = [at & low, at >> 32, torch.full_like(at, st["offset"] & low),
           torch.full_like(at, st["offset"] >> 32)]
    for turn in range(10):
        key = [(seed + turn * 0x9E3779B9) & low, ((seed >> 32) + turn * 0xBB67AE85) & low]
        hi0, lo0 = product(ctr[0], 0xD2511F53)
        hi1, lo1 = product(ctr[2], 0xCD9E8D57)
        ctr = [hi1 ^ ctr[1] ^ key[0], lo1, hi0 ^ ctr[3] ^ key[1], lo0]
    gone = torch.empty(len(at), 4, dtype=torch.bool, device=x.device)
    for k, word in enumerate(ctr):
        gone[:, k] = word < int(case["p"] * 2**32 + 0.5)
    gone = gone.flatten()[:n].view(x.shape)

    def thinned(t):
        return (t.double() / (1 - case["p"])).masked_fill_(gone, 0.0)

    y = thinned(x)
    if st["residual"] is not None:
        y += st["residual"].double()
    return (y, thinned(st["dy"])) if case["train"] else y


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm_rotate":
        return _exact_norm(st)
    return _exact_feed(st) if case["op"] == "feed_forward" else _exact_drop(st)
