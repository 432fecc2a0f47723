"""The attention-side operators this framework is timed on.

Matching networks put a few layers of attention between the features of two
point sets and the assignment or transport problem solved on their scores.
Two operators are measured: the rotation of feature pairs by positions on
several axes, and attention with a capped score, a bias that falls with
distance, and document, prefix, causal and length masks; forward, with
gradients, and for a few new tokens against a long cache.

With ``own`` false :func:`run` computes them in plain float32 torch
operations; with ``own`` true it calls ``torchmatch_amd.attention``.
"""

from __future__ import annotations

import math

import torch

own = False

_DEV = "cuda"
_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def _rot(name, b, length, heads, d, sections, *, dtype="bfloat16", interleaved=False, grid=(),
         train=False, packed=False, start=0):
    """``grid``: integer positions on a grid of these sides (their product is at
    least ``length``), else uniform float positions; ``packed``: x is the query and
    key part of a wider projection, so its rows are strided."""
    return {"name": name, "op": "rotate", "B": b, "L": length, "H": heads, "D": d,
            "sections": ",".join(map(str, sections)), "dtype": dtype, "interleaved": interleaved,
            "grid": ",".join(map(str, grid)), "train": train, "packed": packed, "start": start}


def _att(name, b, lq, lk, heads, kv, d, *, dtype="bfloat16", cap=0.0, axes=-1, causal=False,
         prefix=0, docs=0, ragged=False, train=False):
    """``axes``: -1 no distance bias, 0 distance between indices, 1 to 3 distance
    between float positions; ``docs``: number of documents or pairs packed in a row (with
    a padded tail); ``ragged``: each row of the batch holds fewer keys than Lk."""
    return {"name": name, "op": "attend", "B": b, "Lq": lq, "Lk": lk, "H": heads, "Hkv": kv,
            "D": d, "dtype": dtype, "cap": cap, "axes": axes, "causal": causal, "prefix": prefix,
            "docs": docs, "ragged": ragged, "train": train}


def listed():
    return [
        # one new token for each of eight streams: launch and host latency only
        _rot("rotate_token_8x1x40x128", 8, 1, 40, 128, (64,), grid=(70001,), start=70000,
             packed=True),
        # a video clip on a time, height and width grid, odd sides, queries and keys
        # out of one projection
        _rot("rotate_video_2x9x37x41", 2, 13653, 32, 128, (16, 24, 24), grid=(9, 37, 41),
             interleaved=True, packed=True),
        # key points with image coordinates, float32, as a training step needs it
        _rot("rotate_points_train_16x2048", 16, 2048, 4, 64, (16, 16), dtype="float32",
             train=True),
        # one new token against a short cache, a single stream: latency
        _att("attend_token_1x300", 1, 1, 300, 8, 8, 64, dtype="float16", axes=0, causal=True),
        # one new token against long caches of unequal lengths, shared heads
        _att("attend_token_16x16384", 16, 1, 16384, 32, 8, 128, axes=0, causal=True, ragged=True),
        # a few drafted tokens against a long cache, capped scores
        _att("attend_tokens_4x5x50001", 4, 5, 50001, 16, 2, 128, cap=30.0, causal=True),
        # a matching layer's self-attention over key points, float32, bias by image distance
        _att("attend_points_f32_16x2048", 16, 2048, 2048, 4, 4, 64, dtype="float32", axes=2),
        # cross-attention between the two sets of many packed pairs, with gradients
        _att("attend_pairs_train_4x2900x3700", 4, 2900, 3700, 8, 8, 64, dtype="float16", docs=7,
             train=True),
        # a prompt whose first part sees itself both ways, capped scores, shared heads
        _att("attend_prefix_cap_2x4097", 2, 4097, 4097, 16, 4, 128, cap=30.0, causal=True,
             prefix=700),
        # packed documents, causal, shared heads, with gradients: a training step
        _att("attend_docs_train_2x8192", 2, 8192, 8192, 16, 4, 128, causal=True, docs=9,
             train=True),
        # capped scores and the bias by index distance with gradients, long rows
        _att("attend_cap_bias_train_1x8191", 1, 8191, 8191, 16, 16, 128, cap=20.0, axes=0,
             causal=True, train=True),
        # the longest prompt
        _att("attend_long_1x32768", 1, 32768, 32768, 16, 2, 128, causal=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    if rng.random() < 0.3:
        d = rng.choice((32, 64, 64, 96, 128, 128, 256))
        axes = rng.choice((1, 2, 3))
        left = d // 2 if rng.random() < 0.8 else d // 4  # all, or half, of each head is rotated
        sections = []
        for a in range(axes, 0, -1):
            sections.append(left if a == 1 else max(1, left // a + rng.choice((-1, 0, 1))))
            left -= sections[-1]
        length = _log_int(rng, 1, 20000)
        heads = rng.choice((1, 4, 8, 24, 40))
        b = _log_int(rng, 1, max(1, min(32, 100_000_000 // (length * heads * d))))
        # float32 angles of positions in the thousands are good to 3 digits only
        if rng.random() < 0.5 and (dtype != "float32" or axes > 1):
            side = max(1, math.ceil(length ** (1 / axes)))
            grid = (math.ceil(length / side ** (axes - 1)),) + (side,) * (axes - 1)
        else:
            grid = ()
        c = _rot("", b, length, heads, d, sections, dtype=dtype, interleaved=rng.random() < 0.5,
                 grid=grid, train=rng.random() < 0.4, packed=rng.random() < 0.5,
                 start=rng.choice((0, 0, 5000)) if grid and dtype != "float32" else 0)
        del c["name"]
        return c
    kv = rng.choice((1, 2, 4, 8))
    heads = kv * rng.choice((1, 1, 2, 4, 8))
    d = rng.choice((32, 64, 64, 80, 128, 128))
    cap = rng.choice((0.0, 0.0, 20.0, 50.0))
    axes = rng.choice((-1, -1, 0, 1, 2, 3))
    if rng.random() < 0.35:  # new tokens against a cache
        lk = _log_int(rng, 64, 60000)
        lq = min(lk, rng.choice((1, 1, 1, 2, 5, 16)))
        b = _log_int(rng, 1, max(1, min(64, 500_000_000 // (lk * kv * d))))
        c = _att("", b, lq, lk, heads, kv, d, dtype=dtype, cap=cap, axes=axes, causal=True,
                 ragged=rng.random() < 0.6)
    else:
        train = rng.random() < 0.45
        lq = _log_int(rng, 17, 8192 if dtype != "float32" else 4096)
        same = rng.random() < 0.7
        lk = lq if same else max(16, int(lq * math.exp(rng.uniform(-0.7, 0.7))))
        causal = same and rng.random() < 0.6
        budget = 1.0e12 if dtype != "float32" else 2.0e11
        b = _log_int(rng, 1, max(1, min(32, int(budget / (4 * d * heads * lq * lk)
                                                / (3.5 if train else 1)))))
        while heads > kv and 4 * d * heads * lq * lk * (3.5 if train else 1) > budget:
            heads -= kv
        c = _att("", b, lq, lk, heads, kv, d, dtype=dtype, cap=cap, axes=axes, causal=causal,
                 prefix=rng.choice((0, lq // 5)) if causal else 0,
                 docs=rng.choice((0, 0, 3, 12)) if lq >= 100 and lk >= 100 else 0,
                 ragged=rng.random() < 0.2, train=train)
    del c["name"]
    return c


# ---- inputs --------------------------------------------------------------------------


def _ints(text):
    return [int(t) for t in text.split(",")] if text else []


def _cuts(length, docs, shift):
    """Document edges of a row: unequal parts, the last hundredth of the row padding."""
    used = length - length // 100
    edges = [0]
    for i in range(1, docs):
        edges.append(min(used, max(edges[-1], int(used * (i + 0.4 * math.sin(i + shift)) / docs))))
    return edges + [used]


def _lengths(case):
    lk, lq = case["Lk"], case["Lq"]
    if not case["ragged"]:
        return [lk] * case["B"]
    return [max(min(lq, lk), lk - (lk * (5 * b % 8)) // 11 - b) for b in range(case["B"])]


def _doc_ids(length, docs, shift):
    ids = torch.full((length,), -1, dtype=torch.int32)
    cuts = _cuts(length, docs, shift)
    for i in range(docs):
        ids[cuts[i]:cuts[i + 1]] = i
    return ids


def _prepare_rotate(case, g):
    b, n, h, d = case["B"], case["L"], case["H"], case["D"]
    dtype = _DTYPES[case["dtype"]]
    sections, grid = _ints(case["sections"]), _ints(case["grid"])
    full = torch.randn(b, n, h + (h + 3) // 4 if case["packed"] else h, d, device=_DEV,
                       generator=g).to(dtype)
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
    st = {"case": case, "x": full[:, :, :h], "pos": pos, "freqs": freqs, "sections": sections}
    if case["train"]:
        st["dy"] = torch.randn(b, n, h, d, device=_DEV, generator=g).to(dtype)
        st["x"].requires_grad_(True)
    return st


def _prepare_attend(case, g):
    b, lq, lk, h, kv, d = (case[x] for x in ("B", "Lq", "Lk", "H", "Hkv", "D"))
    dtype = _DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.randn(*shape, device=_DEV, generator=g)

    st = {"case": case, "scale": d ** -0.5, "slopes": None, "q_positions": None,
          "k_positions": None, "q_docs": None, "k_docs": None, "prefix": None, "lengths": None,
          "q": (2.0 * rand(b, lq, h, d)).to(dtype), "k": rand(b, lk, kv, d).to(dtype),
          "v": rand(b, lk, kv, d).to(dtype)}
    if case["axes"] >= 0:
        slopes = 2.0 ** (-8.0 * torch.arange(1, h + 1, dtype=torch.float32) / h)
        st["slopes"] = slopes.to(_DEV)
    if case["axes"] > 0:
        st["q_positions"] = 40 * torch.rand(b, lq, case["axes"], device=_DEV, generator=g)
        st["k_positions"] = 40 * torch.rand(b, lk, case["axes"], device=_DEV, generator=g)
    if case["docs"]:
        st["q_docs"] = torch.stack([_doc_ids(lq, case["docs"], i) for i in range(b)]).to(_DEV)
        # pairs of sets: their parts are cut elsewhere on the key side
        shift = 0 if case["causal"] else 3
        st["k_docs"] = torch.stack([_doc_ids(lk, case["docs"], i + shift)
                                    for i in range(b)]).to(_DEV)
    if case["prefix"]:
        st["prefix"] = torch.tensor([case["prefix"] - i for i in range(b)], dtype=torch.int32,
                                    device=_DEV).clamp_(min=0)
    if case["ragged"]:
        st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=_DEV)
    if case["train"]:
        st["do"] = rand(b, lq, h, d).to(dtype)
        for n in ("q", "k", "v"):
            st[n].requires_grad_(True)
    return st


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    return _prepare_rotate(case, g) if case["op"] == "rotate" else _prepare_attend(case, g)


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


def _plain_rotate(st):
    case = st["case"]
    axis = [a for a, s in enumerate(st["sections"]) for _ in range(s)]
    angle = st["pos"].float()[..., axis] * st["freqs"]
    cos, sin = angle.cos()[:, :, None], angle.sin()[:, :, None]
    y = _turn(st["x"].detach().float(), cos, sin, case["interleaved"]).to(st["x"].dtype)
    if not case["train"]:
        return y
    return y, _turn(st["dy"].float(), cos, -sin, case["interleaved"]).to(st["x"].dtype)


def _mask_and_bias(st, b, dev):
    """What queries may see of the keys of batch row b, and the distance of each pair."""
    case = st["case"]
    lq, lk = case["Lq"], case["Lk"]
    length = st["lengths"][b] if st["lengths"] is not None else lk
    j = torch.arange(lk, device=dev)
    i = torch.arange(lq, device=dev)[:, None] + (length - lq)
    see = (j < length).expand(lq, lk)
    if case["causal"]:
        past = j <= i
        if st["prefix"] is not None:
            past = past | (j < st["prefix"][b])
        see = see & past
    if st["q_docs"] is not None:
        see = see & (st["q_docs"][b][:, None] == st["k_docs"][b]) & (st["k_docs"][b] >= 0)
    dist = None
    if case["axes"] == 0:
        dist = (i - j).abs().float()
    elif case["axes"] > 0:
        dist = sum((st["q_positions"][b, :, a, None] - st["k_positions"][b, None, :, a]).abs()
                   for a in range(case["axes"]))
    return see, dist


def _plain_attend(st):
    case = st["case"]
    bs, lq, lk, h, kv, d = (case[x] for x in ("B", "Lq", "Lk", "H", "Hkv", "D"))
    group, cap, scale = h // kv, case["cap"], st["scale"]
    q, k, v = (st[n].detach() for n in ("q", "k", "v"))
    out = torch.empty_like(q)
    if case["train"]:
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    step = max(1, (1 << 28) // (group * lq * lk))  # kv heads at a time
    for b in range(bs):
        see, dist = _mask_and_bias(st, b, q.device)
        for g0 in range(0, kv, step):
            n = min(step, kv - g0)
            heads = slice(g0 * group, (g0 + n) * group)
            # (n, group * Lq, D) against (n, Lk, D)
            qf = q[b, :, heads].float().view(lq, n, group, d).permute(1, 2, 0, 3)
            qf = qf.reshape(n, group * lq, d)
            kf = k[b, :, g0:g0 + n].float().transpose(0, 1)
            vf = v[b, :, g0:g0 + n].float().transpose(0, 1)
            s = (qf @ kf.transpose(1, 2)).mul_(scale).view(n, group, lq, lk)
            if cap:
                s = s.div_(cap).tanh_()
                slope = 1 - s * s if case["train"] else None  # of the cap, for the gradient
                s = s.mul_(cap)
            if dist is not None:
                s = s - st["slopes"][heads].view(n, group, 1, 1) * dist
            s = s.masked_fill_(~see, float("-inf"))
            top = s.amax(-1, keepdim=True)
            s = s.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
            total = s.sum(-1, keepdim=True)
            p = s.div_(torch.where(total == 0, 1.0, total)).view(n, group * lq, lk)
            o = p @ vf

            def back(t):
                return t.view(n, group, lq, d).permute(2, 0, 1, 3).reshape(lq, n * group, d)

            out[b, :, heads] = back(o).to(q.dtype)
            if not case["train"]:
                continue
            do = st["do"][b, :, heads].float().view(lq, n, group, d).permute(1, 2, 0, 3)
            do = do.reshape(n, group * lq, d)
            dv[b, :, g0:g0 + n] = (p.transpose(1, 2) @ do).transpose(0, 1).to(q.dtype)
            ds = do @ vf.transpose(1, 2)
            ds = ds.sub_((o * do).sum(-1, keepdim=True)).mul_(p)
            if cap:
                ds = ds.mul_(slope.view_as(ds))
            dq[b, :, heads] = back((ds @ kf).mul_(scale)).to(q.dtype)
            dk[b, :, g0:g0 + n] = (ds.transpose(1, 2) @ qf).mul_(scale).transpose(0, 1).to(q.dtype)
    return (out, dq, dk, dv) if case["train"] else out


def run(state):
    case = state["case"]
    if not own:
        return _plain_rotate(state) if case["op"] == "rotate" else _plain_attend(state)
    from torchmatch_amd import attention

    if case["op"] == "rotate":
        y = attention.rotate(state["x"], state["pos"], state["freqs"], state["sections"],
                             interleaved=case["interleaved"])
        if not case["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, state["x"], state["dy"]))
    masks = {n: state[n] for n in ("slopes", "q_positions", "k_positions", "q_docs", "k_docs",
                                   "prefix", "lengths")}
    out = attention.attend(state["q"], state["k"], state["v"], scale=state["scale"],
                           cap=case["cap"], causal=case["causal"], **masks)
    if not case["train"]:
        return out
    grads = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["do"])
    return (out.detach(), *grads)


# ---- work and exact values -----------------------------------------------------------


def _pairs(case):
    """Query-key pairs of one head that the masks leave, over the batch, and the keys
    that any query sees."""
    lq, lk = case["Lq"], case["Lk"]
    total, keys = 0, 0
    for b, length in enumerate(_lengths(case)):
        i = torch.arange(lq, dtype=torch.int64)
        lo, hi = torch.zeros_like(i), torch.full_like(i, length)
        if case["causal"]:
            hi = (i + length - lq + 1).clamp(max=length)
            if case["prefix"]:
                hi = hi.clamp(min=min(length, max(0, case["prefix"] - b)))
        if case["docs"]:
            ids = _doc_ids(lq, case["docs"], b).long()
            cuts = torch.tensor(_cuts(lk, case["docs"], b + (0 if case["causal"] else 3)))
            lo = cuts[ids.clamp(min=0)]
            hi = torch.where(ids < 0, lo, torch.minimum(hi, cuts[ids.clamp(min=0) + 1]))
        total += int((hi - lo).clamp(min=0).sum())
        keys += min(length, int(cuts[-1])) if case["docs"] else length
    return total, keys


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    b, d, h = case["B"], case["D"], case["H"]
    if case["op"] == "rotate":
        axes, pairs = len(_ints(case["sections"])), sum(_ints(case["sections"]))
        passes = 2 if case["train"] else 1
        n = b * case["L"]
        return {"bytes": passes * 2 * n * h * d * size + n * axes * (8 if case["grid"] else 4),
                "flops": passes * 6 * n * h * pairs}
    pairs, keys = _pairs(case)
    rows = b * case["Lq"] * h * d * size  # q or out
    cols = keys * case["Hkv"] * d * size  # k or v that is seen
    if not case["train"]:
        return {"bytes": 2 * rows + 2 * cols, "flops": 4 * d * h * pairs}
    # q, k, v and do read, out and the three gradients written; two products
    # forward, five backward
    whole = b * case["Lk"] * case["Hkv"] * d * size
    return {"bytes": 4 * rows + 2 * cols + 2 * whole, "flops": 14 * d * h * pairs}


def _exact_rotate(st):
    x = st["x"].detach().double()
    pos, freqs = st["pos"].double(), st["freqs"].double()
    owner = torch.repeat_interleave(torch.arange(len(st["sections"]), device=x.device),
                                    torch.tensor(st["sections"], device=x.device))
    unit = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       pos.index_select(-1, owner) * freqs)[:, :, None]
    pairs = len(owner)

    def turned(t, u):
        head = t[..., :2 * pairs]
        if st["case"]["interleaved"]:
            z = torch.view_as_complex(head.unflatten(-1, (pairs, 2)).contiguous()) * u
            head = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(head[..., :pairs], head[..., pairs:]) * u
            head = torch.cat((z.real, z.imag), -1)
        return torch.cat((head, t[..., 2 * pairs:]), -1)

    y = turned(x, unit)
    return (y, turned(st["dy"].double(), unit.conj())) if st["case"]["train"] else y


def _exact_terms(st, b, part):
    """Of the queries ``part`` of batch row b: which keys each one sees, and the L1
    distances in 64 bits (None without a bias)."""
    case, dev = st["case"], st["q"].device
    lq, lk = case["Lq"], case["Lk"]
    length = lk if st["lengths"] is None else int(st["lengths"][b])
    at = torch.arange(part.start, part.stop, device=dev, dtype=torch.float64) + (length - lq)
    key = torch.arange(lk, device=dev, dtype=torch.float64)
    hidden = torch.zeros(len(at), lk, dtype=torch.bool, device=dev)
    hidden[:, length:] = True
    if case["causal"]:
        open_to = 0 if st["prefix"] is None else int(st["prefix"][b])
        hidden[:, open_to:] |= key[open_to:] > at[:, None]
    if st["q_docs"] is not None:
        mine, theirs = st["q_docs"][b, part, None].double(), st["k_docs"][b].double()
        hidden |= (mine - theirs != 0) | (mine < 0)
    if case["axes"] < 0:
        return hidden, None
    mine, theirs = at[:, None], key[:, None]
    if case["axes"] > 0:
        mine, theirs = st["q_positions"][b, part].double(), st["k_positions"][b].double()
    dist = torch.zeros(len(at), lk, dtype=torch.float64, device=dev)
    for x, y in zip(mine.unbind(1), theirs.unbind(1)):
        dist += torch.abs(torch.sub(x.unsqueeze(1), y))
    return hidden, dist


def _exact_attend(st):
    """Row blocks of one head at a time: weights from the log of their sum."""
    case = st["case"]
    lq, h, kv = case["Lq"], case["H"], case["Hkv"]
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    out = torch.zeros_like(q)
    train = case["train"]
    grads = (torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)) if train else ()
    rows = max(1, (1 << 26) // case["Lk"])
    for b in range(case["B"]):
        for r in range(0, lq, rows):
            part = slice(r, min(lq, r + rows))
            hidden, dist = _exact_terms(st, b, part)
            for head in range(h):
                kb, vb = k[b, :, head * kv // h], v[b, :, head * kv // h]
                qb = q[b, part, head]
                raw = torch.einsum("id,jd->ij", qb, kb) * st["scale"]
                t = torch.tanh(raw / case["cap"]) if case["cap"] else None
                logit = raw if t is None else case["cap"] * t
                if dist is not None:
                    logit = logit - st["slopes"][head].double() * dist
                logit = logit.masked_fill(hidden, -torch.inf)
                norm = torch.logsumexp(logit, 1, keepdim=True)
                w = torch.exp(logit - norm.masked_fill(norm == -torch.inf, 0.0))
                out[b, part, head] = w @ vb
                if train:
                    do = st["do"][b, part, head].double()
                    g = do @ vb.T
                    g = w * (g - (w * g).sum(1, keepdim=True))
                    if t is not None:
                        g = g * (1 - t.square())
                    grads[0][b, part, head] = g @ kb * st["scale"]
                    grads[1][b, :, head * kv // h] += g.T @ qb * st["scale"]
                    grads[2][b, :, head * kv // h] += w.T @ do
    return (out, *grads) if train else out


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_rotate(st) if case["op"] == "rotate" else _exact_attend(st)
