"""Operators of prompts with images and of a cache in 4 bits: what is measured of them, their plain forms in torch, and their values in 64 bits.

rope_rows    norm, rotation by positions of several axes (time, height, width) and rounding to 16 bits of a prompt's query, key and value rows
attn_prompt  causal attention of whole prompts, packed one behind the other, with grouped heads, in f16 or bf16
kv_append    rows with positions of several axes into pages of 4 bits (read back with kv_read, since codes are compared as values)
kv_read      tokens of such pages back as f16
attn_paged   attention of a ragged batch of rows over such pages

A cache in 4 bits is k, v u8 [n_pages][n_kv][page * (dim / 2 + dim / 32)] and k_scale, v_scale f32 [n_pages][n_kv][page]. Of a page and head, first the codes c of its tokens,
two to a byte (the even dim in the low half), then a byte per token and 32 dims: the code z of zero in the low half, a factor u of 1 to 15 in the high one. A value is scale * u * (c - z).
"""
import math

import torch

own = False
EPS = 1e-6


def listed():
    return [
        # verify rows of eight slots in a chat about an image: 24 heads of 256 over 4, a quarter of the dims rotated, by time, height and width in turn
        dict(name="rows_verify", op="rows", seqs=8, rows=6, past=2000, ragged=False, heads=24, kv=4, dim=256, rot=64, axes=3, turns=True, inter=False, norm=True, type="f16"),
        # prompts with images: 32 heads of 128 over 8, all dims rotated, the axes one after the other
        dict(name="rows_image", op="rows", seqs=3, rows=2801, past=0, ragged=True, heads=32, kv=8, dim=128, rot=128, axes=3, turns=False, inter=False, norm=False, type="bf16"),
        # the verify rows of eight slots of the mixture-of-experts model (24 heads over 2), appended
        dict(name="append_slots", op="append", seqs=8, rows=3, past=2048, ragged=True, heads=24, kv=2, dim=256, page=16, rot=64, axes=3, turns=True, inter=False, norm=True),
        # prompts of several sequences, each with an image, heads of 128
        dict(name="append_image", op="append", seqs=4, rows=1000, past=500, ragged=True, heads=32, kv=8, dim=128, page=32, rot=128, axes=3, turns=False, inter=False, norm=True),
        # one slot's cache handed to the f16 attention
        dict(name="read_slot", op="read", seqs=1, rows=4096, past=0, ragged=False, kv=4, dim=256, page=64),
        # the caches of a batch taken out
        dict(name="read_batch", op="read", seqs=16, rows=5000, past=0, ragged=True, kv=8, dim=128, page=16),
        # one token of one sequence at the benchmark's context: latency
        dict(name="attn_one", op="attn", seqs=1, rows=1, past=4096, ragged=False, heads=24, kv=4, dim=256, page=64, window=0, sinks=0, gate=True),
        # the verify rows of eight slots: six rows each, two blocks of heads and rows and a rest
        dict(name="attn_verify", op="attn", seqs=8, rows=6, past=4093, ragged=True, heads=24, kv=4, dim=256, page=64, window=0, sinks=0, gate=True),
        # a full serving batch of single tokens with long contexts: bytes
        dict(name="attn_batch", op="attn", seqs=64, rows=1, past=12000, ragged=True, heads=32, kv=8, dim=128, page=32, window=0, sinks=0, gate=False),
        # short prompts of a few users at once, 24 heads of 256 over 4, gated
        dict(name="prompt_short", op="prompt", seqs=5, rows=77, ragged=True, heads=24, kv=4, dim=256, type="f16", packed=False, gate=True),
        # prompts of a batch, packed, rows of q, k and v side by side as one projection gives them
        dict(name="prompt_packed", op="prompt", seqs=7, rows=3001, ragged=True, heads=32, kv=8, dim=128, type="bf16", packed=True, gate=False),
        # one long document, 24 heads of 256 over 4
        dict(name="prompt_long", op="prompt", seqs=1, rows=8190, ragged=False, heads=24, kv=4, dim=256, type="f16", packed=False, gate=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 6.5e12, w["flops"] / (1.4e15 if c["op"] == "prompt" else 4e14))   # paged rows: operations at a rate that kernels of 32-bit results reach


def draw(rng):
    most = 0.8 * max(_cost(c) for c in listed())
    while True:
        c = _drawn(rng)
        if _cost(c) <= most:
            return c


def _drawn(rng):
    op = rng.choice(["attn", "attn", "prompt", "prompt", "append", "rows", "read"])
    dim, kv = rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 6, 8, 12] if kv < 8 else [1, 2, 4, 5])
    c = dict(op=op, ragged=rng.random() < 0.7, kv=kv, dim=dim)
    if op == "prompt":
        rows = _log(rng, 1, 6000)
        return dict(c, heads=heads, seqs=rng.randint(1, 10 if rows < 3500 else 2), rows=rows, type=rng.choice(["f16", "bf16"]), packed=rng.random() < 0.5, gate=rng.random() < 0.3)
    page = rng.choice([16, 32, 64, 128])
    if op == "read":
        return dict(c, seqs=rng.randint(1, 16), rows=_log(rng, 1, 6000), past=0, page=page)
    if op == "attn":
        if rng.random() < 0.25:   # prompt chunks
            rows, seqs, past = _log(rng, 9, 500), rng.randint(1, 2), _log(rng, 1, 2000)
        else:
            rows, seqs, past = rng.choice([1, 1, rng.randint(2, 8)]), rng.randint(1, 40), _log(rng, 1, 10000)
        window = rng.choice([0, 0, _log(rng, 1, 4000)])
        return dict(c, heads=heads, page=page, seqs=seqs, rows=rows, past=past, window=window, sinks=rng.choice([0, 1, 4, 100]) if window else 0, gate=rng.random() < 0.5)
    rows = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 900)])
    c.update(heads=heads, seqs=rng.randint(1, 4 if rows > 8 else 64), rows=rows, past=_log(rng, 1, 3000), rot=rng.choice([dim, dim // 4, dim // 2]), axes=rng.choice([1, 2, 3, 3, 4]), turns=rng.random() < 0.5,
             inter=rng.random() < 0.3, norm=rng.random() < 0.6)
    return dict(c, page=page) if op == "append" else dict(c, type=rng.choice(["f16", "bf16", "f32"]))


def _lengths(c):
    """Rows and tokens of each sequence: all alike, or spread from the largest down to one row and a quarter of the tokens."""
    S, T = c["seqs"], c["rows"]
    L = T + c.get("past", 0)
    if not c["ragged"]:
        return [T] * S, [L] * S
    if c["op"] == "read":   # whole sequences
        ln = [max(1, L - (3 * L // 4) * ((7 * s) % S) // S) for s in range(S)]
        return ln, ln
    rows = [max(1, T - (T - 1) * ((3 * s) % S) // S) for s in range(S)]
    return rows, [max(r, L - (3 * L // 4) * ((7 * s) % S) // S) for s, r in enumerate(rows)]


def _visible(c):
    """Per sequence: keys that some row sees, and pairs of a row and a key that it sees."""
    out, w, k = [], c["window"], c["sinks"]
    for t, n in zip(*_lengths(c)):
        pairs = 0
        for pos in range(n - t, n):
            lo = max(0, pos - w + 1) if w else 0
            pairs += pos + 1 - lo + min(lo, k)
        lo = max(0, n - t - w + 1) if w else 0
        out.append((n - lo + min(lo, k), pairs))
    return out


def work(c):
    rows, _ = _lengths(c)
    R, kv, D, H = sum(rows), c["kv"], c["dim"], c.get("heads", 0)
    token = 2 * kv * (D // 2 + D // 32 + 4)   # codes, bytes of the groups and scales of K and V
    if c["op"] == "prompt":
        return {"bytes": R * (2 * H + 2 * kv) * D * 2 + (R * H * D * 4 if c["gate"] else 0), "flops": sum(2 * H * D * t * (t + 1) for t in rows)}
    if c["op"] == "rows":
        return {"bytes": R * (H + 2 * kv) * D * (8 if c["type"] == "f32" else 6), "flops": 0}
    if c["op"] == "read":
        return {"bytes": R * (token + 4 * kv * D), "flops": 0}
    if c["op"] == "append":   # rows in, q and codes out, codes in and f16 out
        return {"bytes": R * (4 * (2 * H + 2 * kv) * D + 2 * token + 4 * kv * D), "flops": 0}
    v = _visible(c)
    return {"bytes": sum(n for n, _ in v) * token + R * H * D * 4 * (3 if c["gate"] else 2), "flops": 4 * H * D * sum(p for _, p in v)}


TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _axis_of_pairs(c):
    """The axis whose position turns each pair of dims: sections one after the other, or in turn until a section is used up, the rest to the first axis."""
    half, n = c["rot"] // 2, c["axes"]
    small = half // (n + 1) if n > 1 else 0
    if not c["turns"]:
        return [min(i // small, n - 1) if small else 0 for i in range(half)]
    return [i % n if i < n * small else 0 for i in range(half)]


def _positions(c):
    """[axes][R]: a sequence's rows are text with an image in their middle half, in rows of up to 32 patches; behind it the text goes on from the largest position."""
    out = [[] for _ in range(c["axes"])]
    for t, n in zip(*_lengths(c)):
        p, first = n - t, t // 4
        patches = t // 2
        width = max(1, min(32, int(math.sqrt(patches)))) if patches else 1
        rows = -(-patches // width)
        after = p + first + max(rows, width) if patches else p + first
        for i in range(t):
            j = i - first
            for a in range(c["axes"]):
                if j < 0:
                    x = p + i
                elif j < patches:
                    x = p + first + (j // width if a == 1 else j % width if a == 2 else 0)
                else:
                    x = after + j - patches
                out[a].append(x)
    return out


def _turns(st, c, dev):
    pos = _positions(c)
    st["positions"] = torch.tensor(pos, dtype=torch.int32, device=dev)
    half = c["rot"] // 2
    f = 1e7 ** (-2 * torch.arange(half, device=dev, dtype=torch.float64) / c["rot"])
    a = torch.arange(max(map(max, pos)) + 1, device=dev, dtype=torch.float64)[:, None] * f
    st["rope"] = torch.stack([a.cos(), a.sin()], -1).float().contiguous()
    st["axes"] = _axis_of_pairs(c)


def _quantise(x):
    """Codes, bytes of the groups and scales of x [..., D] in 32 bits."""
    g = x.unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
    half = 0.5 * hi - 0.5 * lo
    most = half.amax(-1)
    scale = most / 112.5
    live = scale > 0
    u = torch.where(live[..., None], (15 * half / torch.where(live, most, torch.ones_like(most))[..., None]).ceil().clamp(0, 15), torch.zeros_like(half))
    t = scale[..., None] * u
    t = torch.where(t > 0, t, torch.ones_like(t))
    z = torch.where(u > 0, (-lo / t).round().clamp(0, 15), torch.zeros_like(u))
    c = ((g / t[..., None]).round() + z[..., None]).clamp(0, 15)
    c = torch.where(u[..., None] > 0, c, torch.zeros_like(c)).flatten(-2).to(torch.uint8)
    return c[..., 0::2] | c[..., 1::2] << 4, (z.to(torch.uint8) | u.to(torch.uint8) << 4), scale


def _parts(pool, page, dim):
    """Views of the codes [..., page, dim / 2] and of the bytes of the groups [..., page, dim / 32]."""
    n = page * dim // 2
    return pool[..., :n].unflatten(-1, (page, dim // 2)), pool[..., n:].unflatten(-1, (page, dim // 32))


def _values(codes, groups, scale):
    """Codes [..., D / 2], bytes [..., D / 32] and scales [...] as values [..., D] in the scales' type."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 32)).to(scale.dtype)
    return (scale[..., None, None] * ((groups >> 4).to(scale.dtype)[..., None] * (c - (groups & 15).to(scale.dtype)[..., None]))).flatten(-2)


def prepare(c, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rows, lens = _lengths(c)
    S, R, kv, D, H = c["seqs"], sum(rows), c["kv"], c["dim"], c.get("heads", 0)
    st = {"c": c, "R": R, "max_rows": max(rows), "max_kv": max(lens)}
    st["row_start"] = torch.tensor([sum(rows[:s]) for s in range(S + 1)], dtype=torch.int32, device=dev)
    sigma = torch.rand(D, generator=g, device=dev)   # rows as projections give them: normal, a few dims larger than the others; what is quantised on its way comes from a projection whose heads are even
    sigma = 1 + 0.2 * sigma if c["op"] == "append" else 1 + 2 * (sigma > 0.95).float()
    if c["op"] == "prompt":
        kind = TYPES[c["type"]]
        x = (torch.randn((R, H + 2 * kv, D), generator=g, device=dev) * sigma).to(kind)
        q, k, v = x.split([H, kv, kv], 1)
        st["q"], st["k"], st["v"] = (q, k, v) if c["packed"] else (q.contiguous(), k.contiguous(), v.contiguous())
        st["gate"] = torch.randn((R, H, D), generator=g, device=dev) if c["gate"] else None
        return st
    if c["op"] in ("rows", "append"):   # projection rows: q, k and v side by side
        st["rows"] = torch.randn((R, H + 2 * kv, D), generator=g, device=dev) * sigma
        for n in ("q_norm", "k_norm"):
            st[n] = (1 + 0.1 * torch.randn(D, generator=g, device=dev)).bfloat16() if c["norm"] else None
        _turns(st, c, dev)
        if c["op"] == "rows":
            return st
    P = c["page"]
    cols = -(-max(lens) // P)
    n_pages = sum(-(-n // P) for n in lens) + 3
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)   # pages as a pool hands them out
    used = torch.tensor([-(-n // P) for n in lens], device=dev)
    first = torch.cumsum(used, 0) - used
    col = torch.arange(cols, device=dev)
    st["table"] = torch.where(col < used[:, None], order[(first[:, None] + col).clamp(max=n_pages - 1)], torch.full((), -1, dtype=torch.int32, device=dev)).contiguous()
    st["kv_len"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    step = max(1, (1 << 25) // (kv * P * D))
    for n in ("k", "v"):
        st[n] = torch.zeros((n_pages, kv, P * (D // 2 + D // 32)), dtype=torch.uint8, device=dev)
        st[n + "_scale"] = torch.zeros((n_pages, kv, P), device=dev)
        if c["op"] == "append":   # empty pages
            continue
        codes, groups = _parts(st[n], P, D)   # pages as appended tokens left them
        for i in range(0, n_pages, step):
            m = min(step, n_pages - i)
            x = torch.randn((m, kv, P, D), generator=g, device=dev) * sigma * torch.exp(0.3 * torch.randn((m, kv, P, 1), generator=g, device=dev))
            codes[i:i + m], groups[i:i + m], st[n + "_scale"][i:i + m] = _quantise(x)
    if c["op"] == "attn":   # q and its gate side by side per head, as the projection of a gated model gives them
        st["qg"] = torch.randn((R, H, 2 * D if c["gate"] else D), generator=g, device=dev)
    if own:
        from hipster_b200 import kernels
        st["pages"] = kernels.KVPages(st["k"], st["v"], st["k_scale"], st["v_scale"])
    return st


def _seq_of_rows(st):
    """Sequence, index in it and position of every row."""
    rs = st["row_start"].long()
    r = torch.arange(st["R"], device=rs.device)
    s = torch.searchsorted(rs[1:].contiguous(), r, right=True)
    t = r - rs[s]
    return s, t, st["kv_len"].long()[s] - (rs[s + 1] - rs[s]) + t


def _slots(st):
    """Page and place in it of every row."""
    P = st["c"]["page"]
    s, _, pos = _seq_of_rows(st)
    return st["table"].long()[s, pos // P], pos % P


def _read_rows(st):
    page, at = _slots(st)
    out = []
    for n in ("k", "v"):
        codes, groups = _parts(st[n], st["c"]["page"], st["c"]["dim"])
        out.append(_values(codes[page, :, at], groups[page, :, at], st[n + "_scale"][page, :, at]).half())
    return tuple(out)


def _turn(st, x):
    """The rotation of the first dims of x [R][heads][D] by each pair's axis."""
    rot, inter = st["c"]["rot"], st["c"]["inter"]
    half = rot // 2
    axis = torch.tensor(st["axes"], device=x.device)
    cs = st["rope"][st["positions"].long()[axis].T, torch.arange(half, device=x.device)]   # [R][half][2]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :half], x[..., half:rot])
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    u, w = a * c - b * s, b * c + a * s
    turned = torch.stack([u, w], -1).flatten(-2) if inter else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _rms(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.to(x.dtype)


def _plain_rows(st):
    c = st["c"]
    q, k, v = st["rows"].split([c["heads"], c["kv"], c["kv"]], 1)
    kind = TYPES[c["type"]]
    return _turn(st, _rms(q, st["q_norm"])).to(kind), _turn(st, _rms(k, st["k_norm"])).to(kind), v.to(kind, copy=True)


def _plain_append(st):
    c = st["c"]
    q, k, v = st["rows"].split([c["heads"], c["kv"], c["kv"]], 1)
    page, at = _slots(st)
    for n, x in (("k", _turn(st, _rms(k, st["k_norm"]))), ("v", v)):
        codes, groups = _parts(st[n], c["page"], c["dim"])
        codes[page, :, at], groups[page, :, at], st[n + "_scale"][page, :, at] = _quantise(x)
    return (_turn(st, _rms(q, st["q_norm"])), *_read_rows(st), st["k_scale"], st["v_scale"])


def _weigh(x, v):
    """Weights of scores x (masked ones -inf) times values, over their sum."""
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    return (x @ v) / x.sum(-1, keepdim=True).clamp(min=1e-37)


def _plain_attn(st):
    c = st["c"]
    S, T, H, kv, D, G = c["seqs"], st["max_rows"], c["heads"], c["kv"], c["dim"], c["heads"] // c["kv"]
    s, t, pos = _seq_of_rows(st)
    table = st["table"].long().clamp(min=0)
    q = torch.zeros((S, T, H, D), device="cuda")
    q[s, t] = st["qg"][..., :D]
    q = q.view(S, T, kv, G, D).permute(0, 2, 3, 1, 4).reshape(S, kv, G * T, D)
    at = torch.full((S, T), -1, dtype=torch.int64, device="cuda")
    at[s, t] = pos
    j, at = torch.arange(table.shape[1] * c["page"], device="cuda"), at[..., None]
    see = j <= at
    if c["window"]:
        see &= (j > at - c["window"]) | (j < c["sinks"])
    o = torch.empty((S, kv, G * T, D), device="cuda")
    for i in range(0, S, 8):   # a few sequences at a time
        k, v = (_values(*(p[table[i:i + 8]] for p in _parts(st[n], c["page"], D)), st[n + "_scale"][table[i:i + 8]]).transpose(1, 2).reshape(-1, kv, len(j), D) for n in ("k", "v"))
        m = k.shape[0]
        mask = see[i:i + 8, None, None].expand(m, 1, G, T, -1).reshape(m, 1, G * T, -1)
        o[i:i + 8] = _weigh(((q[i:i + 8] @ k.transpose(-1, -2)) * (1 / math.sqrt(D))).masked_fill(~mask, -math.inf), v)
    o = o.view(S, kv, G, T, D).permute(0, 3, 1, 2, 4).reshape(S, T, H, D)[s, t]
    return o * torch.sigmoid(st["qg"][..., D:]) if c["gate"] else o


def _plain_prompt(st):
    c = st["c"]
    H, kv, D = c["heads"], c["kv"], c["dim"]
    out, r0 = torch.empty((st["R"], H, D), dtype=TYPES[c["type"]], device="cuda"), 0
    for t in _lengths(c)[0]:
        hidden = torch.ones((t, t), dtype=torch.bool, device="cuda").triu(1)
        for h in range(kv):   # the query heads of a kv head together
            k, v = (st[n][r0:r0 + t, h].float() for n in ("k", "v"))
            hs = slice(h * (H // kv), (h + 1) * (H // kv))
            o = _weigh(((st["q"][r0:r0 + t, hs].float().transpose(0, 1) @ k.T) * (1 / math.sqrt(D))).masked_fill(hidden, -math.inf), v).transpose(0, 1)
            out[r0:r0 + t, hs] = o * torch.sigmoid(st["gate"][r0:r0 + t, hs]) if c["gate"] else o
        r0 += t
    return out


def run(st):
    c = st["c"]
    if own:
        from hipster_b200 import kernels as K
        H, kv, D = c.get("heads"), c["kv"], c["dim"]
        if c["op"] == "prompt":
            return K.attn_prompt(st["q"], st["k"], st["v"], st["row_start"], max_rows=st["max_rows"], gate=st["gate"])[0]
        if c["op"] == "rows":
            x = st["rows"]
            return K.rope_rows(x[:, :H], x[:, H:H + kv], x[:, H + kv:], st["rope"], st["positions"], axes=st["axes"], interleaved=c["inter"], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS,
                               dtype=TYPES[c["type"]])
        if c["op"] == "read":
            return K.kv_read(st["pages"], st["table"], st["row_start"], st["kv_len"], R=st["R"])
        if c["op"] == "append":
            x = st["rows"]
            q = K.kv_append(st["pages"], x[:, H:H + kv], x[:, H + kv:], st["table"], st["row_start"], st["kv_len"], st["rope"], q=x[:, :H], interleaved=c["inter"], q_norm=st["q_norm"], k_norm=st["k_norm"],
                            eps=EPS, positions=st["positions"], axes=st["axes"])
            return (q, *K.kv_read(st["pages"], st["table"], st["row_start"], st["kv_len"], R=st["R"]), st["k_scale"], st["v_scale"])
        return K.attn_paged(st["qg"][..., :D], st["pages"], st["table"], st["row_start"], st["kv_len"], max_rows=st["max_rows"], max_kv=st["max_kv"], window=c["window"], n_sink=c["sinks"],
                            gate=st["qg"][..., D:] if c["gate"] else None)[0]
    return {"rows": _plain_rows, "read": _read_rows, "append": _plain_append, "attn": _plain_attn, "prompt": _plain_prompt}[c["op"]](st)


# ---- in 64 bits, written from the definitions, a sequence at a time
def _softmax_rows(q, k, v, hidden, D):
    return torch.softmax((q @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf), -1) @ v


def exact(c, seed):
    st = prepare(c, seed)
    d = torch.float64
    rows, lens = _lengths(c)
    kv, D, H = c["kv"], c["dim"], c.get("heads", 0)
    if c["op"] == "prompt":
        out, r0 = torch.empty((st["R"], H, D), device="cuda", dtype=d), 0
        for t in rows:
            for h in range(H):
                k, v = st["k"][r0:r0 + t, h // (H // kv)].to(d), st["v"][r0:r0 + t, h // (H // kv)].to(d)
                for a in range(0, t, 2048):   # rows a .. b - 1 see the keys in front of b
                    b = min(t, a + 2048)
                    hidden = torch.arange(b, device="cuda")[None] > torch.arange(a, b, device="cuda")[:, None]
                    out[r0 + a:r0 + b, h] = _softmax_rows(st["q"][r0 + a:r0 + b, h].to(d), k[:b], v[:b], hidden, D)
            r0 += t
        return out / (1 + torch.exp(-st["gate"].to(d))) if c["gate"] else out

    def tokens(s, n):
        """A sequence's values [kv][len][D], dim by dim from the bytes."""
        pages = st["table"][s, :-(-lens[s] // P)].long()
        b = st[n][pages].long()
        i = torch.arange(D, device="cuda")
        tok = torch.arange(P, device="cuda")[:, None]
        code = (b[..., tok * (D // 2) + i // 2] >> (4 * (i % 2))) % 16
        group = b[..., P * (D // 2) + tok * (D // 32) + i // 32]
        x = st[n + "_scale"][pages].to(d)[..., None] * ((group // 16) * (code - group % 16)).to(d)
        return x.permute(1, 0, 2, 3).reshape(kv, -1, D)[:, :lens[s]]

    P = c.get("page")
    if c["op"] == "read":
        return tuple(torch.cat([tokens(s, n)[:, lens[s] - rows[s]:].transpose(0, 1) for s in range(c["seqs"])]) for n in ("k", "v"))
    if c["op"] == "attn":
        G, out, r0 = H // kv, [], 0
        for s in range(c["seqs"]):
            k, v, n, t = tokens(s, "k"), tokens(s, "v"), lens[s], rows[s]
            p, j = torch.arange(n - t, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
            hidden = (j > p) | ((p - j >= c["window"]) & (j >= c["sinks"])) if c["window"] else j > p
            o = torch.stack([_softmax_rows(st["qg"][r0:r0 + t, h, :D].to(d), k[h // G], v[h // G], hidden, D) for h in range(H)], 1)
            out.append(o / (1 + torch.exp(-st["qg"][r0:r0 + t, :, D:].to(d))) if c["gate"] else o)
            r0 += t
        return torch.cat(out)
    # rows and append
    rot, half, x = c["rot"], c["rot"] // 2, st["rows"].to(d)
    axis = _axis_of_pairs(c)

    def turned(y, w):
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.to(d)
        z = y.clone()
        for i in range(half):   # the table is an input
            angle = st["rope"][st["positions"][axis[i]].long(), i].to(d)
            a, b = (2 * i, 2 * i + 1) if c["inter"] else (i, i + half)
            z[..., a] = y[..., a] * angle[:, None, 0] - y[..., b] * angle[:, None, 1]
            z[..., b] = y[..., a] * angle[:, None, 1] + y[..., b] * angle[:, None, 0]
        return z

    q, k, v = turned(x[:, :H], st["q_norm"]), turned(x[:, H:H + kv], st["k_norm"]), x[:, H + kv:]
    if c["op"] == "rows":
        return q, k, v
    back, scales = [], []
    for n, y in (("k", k), ("v", v)):
        span = torch.stack([y[..., i:i + 32].amax(-1).clamp(min=0) - y[..., i:i + 32].amin(-1).clamp(max=0) for i in range(0, D, 32)], -1)
        scale = span.amax(-1) / 225
        val = torch.empty_like(y)
        for i in range(D // 32):
            g = y[..., 32 * i:32 * i + 32]
            step = (scale * (15 * span[..., i] / span.amax(-1)).ceil().clamp(max=15))[..., None]
            zero = (-g.amin(-1, keepdim=True).clamp(max=0) / step).round()
            val[..., 32 * i:32 * i + 32] = step * (((g / step).round() + zero).clamp(0, 15) - zero)
        back.append(val)
        pool, r0 = st[n + "_scale"].to(d), 0
        for s, (t, m) in enumerate(zip(rows, lens)):
            at = torch.arange(m - t, m, device="cuda")
            pool[st["table"][s].long()[at // P], :, at % P] = scale[r0:r0 + t]
            r0 += t
        scales.append(pool)
    return (q, *back, *scales)
