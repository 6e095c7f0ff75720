"""The operators of the paged 8-bit cache: what is measured of them, their plain forms in torch, and their values in 64 bits.

rope_table   cos and sin of scaled rotary angles
kv_append    norm, rotation and quantisation of new rows into the pages of their sequences (read back with kv_read, since 8-bit codes are compared as values)
attn_paged   attention of a ragged batch of rows over those pages, with window and first tokens that stay visible
kv_read      tokens of the pages back as f16

A cache is k, v [n_pages][n_kv][page][dim] in int8 or e4m3 and k_scale, v_scale [n_pages][n_kv][page] in f32: one scale per token and head. table [S][columns]
gives the page of a sequence's positions; row_start [S + 1] and kv_len [S] say which rows are a sequence's newest tokens and how many it has with them.
"""
import math

import torch

own = False
EPS = 1e-6


def listed():
    return [
        # a rotary table at load: the engine's own context and rotated dims
        dict(name="table_8k", op="table", pos=8192, rot=64, scaling="none"),
        # and one for a long context, scaled by parts
        dict(name="table_long", op="table", pos=262144, rot=128, scaling="yarn"),
        # one decode row of the dense model (24 heads of 256 over 4), appended
        dict(name="append_one", op="append", seqs=1, rows=1, ctx=4097, ragged=False, heads=24, kv=4, dim=256, page=64, type="i8", rot=64, inter=False, norm=True),
        # the verify rows of eight slots of the mixture-of-experts model (24 heads over 2)
        dict(name="append_slots", op="append", seqs=8, rows=3, ctx=2051, ragged=True, heads=24, kv=2, dim=256, page=16, type="e4m3", rot=64, inter=False, norm=True),
        # prompts of several sequences at once, heads of 128, whole heads rotated in pairs of neighbours, no norm
        dict(name="append_prompts", op="append", seqs=4, rows=1000, ctx=1500, ragged=True, heads=32, kv=8, dim=128, page=32, type="i8", rot=128, inter=True, norm=False),
        # one token of one sequence at the benchmark's context: latency
        dict(name="attn_one", op="attn", seqs=1, rows=1, ctx=4097, ragged=False, heads=24, kv=4, dim=256, page=64, type="i8", window=0, sinks=0, gate=True),
        # the verify rows of eight slots: mixture-of-experts model, three rows each
        dict(name="attn_slots", op="attn", seqs=8, rows=3, ctx=2051, ragged=True, heads=24, kv=2, dim=256, page=16, type="e4m3", window=0, sinks=0, gate=True),
        # a full serving batch of single tokens with long contexts: bytes
        dict(name="attn_batch", op="attn", seqs=48, rows=1, ctx=8192, ragged=True, heads=24, kv=4, dim=256, page=64, type="i8", window=0, sinks=0, gate=True),
        # many short rows of a long chat behind a window with its first tokens kept, heads of 128
        dict(name="attn_window", op="attn", seqs=32, rows=2, ctx=8000, ragged=True, heads=32, kv=8, dim=128, page=32, type="e4m3", window=1000, sinks=4, gate=False),
        # a prompt chunk of the dense model behind 4096 tokens
        dict(name="attn_prompt", op="attn", seqs=1, rows=509, ctx=4605, ragged=False, heads=24, kv=4, dim=256, page=64, type="i8", window=0, sinks=0, gate=True),
        # one slot's cache handed to the f16 attention
        dict(name="read_slot", op="read", seqs=1, rows=4096, ctx=4096, ragged=False, kv=4, dim=256, page=64, type="i8"),
        # the caches of a batch taken out
        dict(name="read_batch", op="read", seqs=16, rows=5000, ctx=5000, ragged=True, kv=8, dim=128, page=16, type="e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 6.5e12, w["flops"] / 4e14)   # operations at a rate that kernels of 32-bit results reach


def draw(rng):
    most = 0.8 * max(_cost(c) for c in listed())
    while True:
        c = _drawn(rng)
        if _cost(c) <= most:
            return c


def _drawn(rng):
    op = rng.choice(["attn", "attn", "attn", "append", "append", "read", "table"])
    if op == "table":
        return dict(op=op, pos=_log(rng, 100, 262144), rot=2 * rng.randint(8, 64), scaling=rng.choice(["none", "linear", "yarn"]))
    dim = rng.choice([64, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    c = dict(op=op, ragged=rng.random() < 0.7, kv=kv, dim=dim, page=rng.choice([16, 32, 64, 128]), type=rng.choice(["i8", "e4m3"]))
    if op == "read":
        ctx = _log(rng, 1, 6000)
        return dict(c, seqs=rng.randint(1, 16), rows=ctx, ctx=ctx)
    c["heads"] = kv * rng.choice([1, 2, 3, 4, 6, 8, 12] if kv < 8 else [1, 2, 4, 5])
    if op == "append":
        rows = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 900)])
        return dict(c, seqs=rng.randint(1, 4 if rows > 8 else 64), rows=rows, ctx=rows + _log(rng, 1, 2000), rot=rng.choice([dim, dim // 4, dim // 2]), inter=rng.random() < 0.5, norm=rng.random() < 0.5)
    if rng.random() < 0.25:   # prompt chunks
        rows, seqs, past = _log(rng, 9, 500), rng.randint(1, 2), _log(rng, 1, 2000)
    else:
        rows, seqs, past = rng.choice([1, 1, rng.randint(2, 8)]), rng.randint(1, 40), _log(rng, 1, 8000)
    window = rng.choice([0, 0, _log(rng, 1, 4000)])
    return dict(c, seqs=seqs, rows=rows, ctx=rows + past, window=window, sinks=rng.choice([0, 1, 4, 100]) if window else 0, gate=rng.random() < 0.5)


def _lengths(c):
    """Rows and tokens of each sequence: all alike, or spread from the largest down to one row and a quarter of the tokens."""
    S, T, L = c["seqs"], c["rows"], c["ctx"]
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
    if c["op"] == "table":
        return {"bytes": c["pos"] * c["rot"] * 4, "flops": 0}
    rows, lens = _lengths(c)
    R, kv, D = sum(rows), c["kv"], c["dim"]
    token = 2 * kv * (D + 4)   # codes and scales of K and V
    if c["op"] == "read":
        return {"bytes": R * (token + 4 * kv * D), "flops": 0}
    if c["op"] == "append":   # rows in, q and codes out, codes in and f16 out
        H = c["heads"]
        return {"bytes": R * (4 * (2 * H + 2 * kv) * D + 2 * token + 4 * kv * D), "flops": 0}
    v, H = _visible(c), c["heads"]
    return {"bytes": sum(n for n, _ in v) * token + R * H * D * 4 * (3 if c["gate"] else 2), "flops": 4 * H * D * sum(p for _, p in v)}


def _quantise(x, kind):
    amax = x.abs().amax(-1)
    scale = amax / (127.0 if kind == "i8" else 448.0)
    y = x / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    return (y.round().clamp(-127, 127).to(torch.int8) if kind == "i8" else y.clamp(-448, 448).to(torch.float8_e4m3fn)), scale


def _base(seed):
    return 1e7 * (1 + (seed % 9973) / 9973)


def _norm_rows(shape, g, dim_sigma, device):
    """Rows as projections give them: normal, a few dims larger than the others."""
    x = torch.randn(shape, generator=g, device=device)
    return x * dim_sigma


def prepare(c, seed):
    dev = "cuda"
    if c["op"] == "table":
        return {"c": c, "base": _base(seed), "factor": 8.0, "orig": max(1, c["pos"] // 8)}
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rows, lens = _lengths(c)
    S, R, kv, D, P = c["seqs"], sum(rows), c["kv"], c["dim"], c["page"]
    cols = -(-max(lens) // P)
    n_pages = sum(-(-n // P) for n in lens) + 3
    st = {"c": c, "R": R, "max_rows": max(rows), "max_kv": max(lens)}
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)   # pages as a pool hands them out
    used = torch.tensor([-(-n // P) for n in lens], device=dev)
    first = torch.cumsum(used, 0) - used
    col = torch.arange(cols, device=dev)
    st["table"] = torch.where(col < used[:, None], order[(first[:, None] + col).clamp(max=n_pages - 1)], torch.full((), -1, dtype=torch.int32, device=dev)).contiguous()
    st["row_start"] = torch.tensor([sum(rows[:s]) for s in range(S + 1)], dtype=torch.int32, device=dev)
    st["kv_len"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    kind = torch.int8 if c["type"] == "i8" else torch.float8_e4m3fn
    sigma = 1 + 2 * (torch.rand(D, generator=g, device=dev) > 0.95).float()
    if c["op"] == "append":   # empty pages
        for n in ("k", "v"):
            st[n] = torch.zeros((n_pages, kv, P, D), dtype=torch.uint8, device=dev).view(kind)
            st[n + "_scale"] = torch.zeros((n_pages, kv, P), device=dev)
        H, n_pos = c["heads"], max(lens)
        # projection rows: q, k and v side by side
        st["rows"] = _norm_rows((R, (H + 2 * kv), D), g, sigma, dev)
        f = _base(seed) ** (-2 * torch.arange(c["rot"] // 2, device=dev, dtype=torch.float64) / c["rot"])
        a = torch.arange(n_pos, device=dev, dtype=torch.float64)[:, None] * f
        st["rope"] = torch.stack([a.cos(), a.sin()], -1).float().contiguous()
        for n in ("q_norm", "k_norm"):
            st[n] = (1 + 0.1 * torch.randn(D, generator=g, device=dev)).bfloat16() if c["norm"] else None
    else:   # pages as appended tokens left them
        step = max(1, (1 << 26) // (kv * P * D))
        for n in ("k", "v"):
            st[n] = torch.empty((n_pages, kv, P, D), dtype=kind, device=dev)
            st[n + "_scale"] = torch.empty((n_pages, kv, P), device=dev)
            for i in range(0, n_pages, step):
                m = min(step, n_pages - i)
                x = _norm_rows((m, kv, P, D), g, sigma, dev) * torch.exp(0.3 * torch.randn((m, kv, P, 1), generator=g, device=dev))
                q, s = _quantise(x, c["type"])
                st[n].view(torch.uint8)[i:i + m] = q.view(torch.uint8)
                st[n + "_scale"][i:i + m] = s
    if c["op"] == "attn":   # q and its gate side by side per head, as the projection of a gated model gives them
        st["qg"] = torch.randn((R, c["heads"], 2 * D if c["gate"] else D), generator=g, device=dev)
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
    return st["table"].long()[s, pos // P], pos % P, pos


def _read_rows(st):
    page, at, _ = _slots(st)
    return tuple((st[n][page, :, at].float() * st[n + "_scale"][page, :, at][..., None]).half() for n in ("k", "v"))


def _plain_table(st):
    c = st["c"]
    i = torch.arange(c["rot"] // 2, device="cuda", dtype=torch.float64)
    f, m = st["base"] ** (-2 * i / c["rot"]), 1.0
    if c["scaling"] == "linear":
        f = f / st["factor"]
    elif c["scaling"] == "yarn":
        g = ((st["orig"] * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f, m = f * ((1 - g) / st["factor"] + g), 0.1 * math.log(st["factor"]) + 1
    a = torch.arange(c["pos"], device="cuda", dtype=torch.float64)[:, None] * f
    return torch.stack([a.cos() * m, a.sin() * m], -1).float()


def _turn(x, cs, inter, rot):
    """The rotation of the first `rot` dims of x [R][heads][D] by cs [R][rot / 2][2]."""
    half = rot // 2
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :half], x[..., half:rot])
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    u, w = a * c - b * s, b * c + a * s
    turned = torch.stack([u, w], -1).flatten(-2) if inter else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _rms(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.to(x.dtype)


def _plain_append(st):
    c = st["c"]
    H, kv = c["heads"], c["kv"]
    q, k, v = st["rows"].split([H, kv, kv], 1)
    page, at, pos = _slots(st)
    cs = st["rope"][pos]
    q = _turn(_rms(q, st["q_norm"]), cs, c["inter"], c["rot"])
    k = _turn(_rms(k, st["k_norm"]), cs, c["inter"], c["rot"])
    for n, x in (("k", k), ("v", v)):
        codes, scale = _quantise(x, c["type"])
        st[n].view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
        st[n + "_scale"][page, :, at] = scale
    return (q, *_read_rows(st), st["k_scale"], st["v_scale"])


def _plain_attn(st):
    c = st["c"]
    S, T, H, kv, D, G = c["seqs"], st["max_rows"], c["heads"], c["kv"], c["dim"], c["heads"] // c["kv"]
    s, t, pos = _seq_of_rows(st)
    table = st["table"].long().clamp(min=0)
    k, v = ((st[n][table].float() * st[n + "_scale"][table][..., None]).transpose(1, 2).reshape(S, kv, -1, D) for n in ("k", "v"))
    q = torch.zeros((S, T, H, D), device="cuda")
    q[s, t] = st["qg"][..., :D]
    q = q.view(S, T, kv, G, D).permute(0, 2, 3, 1, 4).reshape(S, kv, G * T, D)
    at = torch.full((S, T), -1, dtype=torch.int64, device="cuda")
    at[s, t] = pos
    j, at = torch.arange(k.shape[2], device="cuda"), at[..., None]
    see = j <= at
    if c["window"]:
        see &= (j > at - c["window"]) | (j < c["sinks"])
    see = see[:, None, None].expand(S, 1, G, T, -1).reshape(S, 1, G * T, -1)
    x = (q @ k.transpose(-1, -2)) * (1 / math.sqrt(D))
    x = x.masked_fill(~see, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    o = (x @ v) / x.sum(-1, keepdim=True).clamp(min=1e-37)
    o = o.view(S, kv, G, T, D).permute(0, 3, 1, 2, 4).reshape(S, T, H, D)[s, t]
    return o * torch.sigmoid(st["qg"][..., D:]) if c["gate"] else o


def run(st):
    c = st["c"]
    if own:
        from hipster_b200 import kernels as K
        if c["op"] == "table":
            return K.rope_table(c["pos"], c["rot"], st["base"], scaling=c["scaling"], factor=st["factor"], orig_ctx=st["orig"])
        if c["op"] == "read":
            return K.kv_read(st["pages"], st["table"], st["row_start"], st["kv_len"], R=st["R"])
        if c["op"] == "append":
            H, kv = c["heads"], c["kv"]
            x = st["rows"]
            q = K.kv_append(st["pages"], x[:, H:H + kv], x[:, H + kv:], st["table"], st["row_start"], st["kv_len"], st["rope"], q=x[:, :H], interleaved=c["inter"],
                            q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS)
            return (q, *K.kv_read(st["pages"], st["table"], st["row_start"], st["kv_len"], R=st["R"]), st["k_scale"], st["v_scale"])
        D = c["dim"]
        return K.attn_paged(st["qg"][..., :D], st["pages"], st["table"], st["row_start"], st["kv_len"], max_rows=st["max_rows"], max_kv=st["max_kv"], window=c["window"], n_sink=c["sinks"],
                            gate=st["qg"][..., D:] if c["gate"] else None)[0]
    return {"table": _plain_table, "read": _read_rows, "append": _plain_append, "attn": _plain_attn}[c["op"]](st)


# ---- in 64 bits, written from the definitions, a sequence at a time
def exact(c, seed):
    st = prepare(c, seed)
    d = torch.float64
    if c["op"] == "table":
        pos, out, rot = torch.arange(c["pos"], device="cuda", dtype=d), [], c["rot"]
        for i in range(rot // 2):
            f, m = math.exp(-2.0 * i / rot * math.log(st["base"])), 1.0
            if c["scaling"] == "linear":
                f /= st["factor"]
            if c["scaling"] == "yarn":
                turns = st["orig"] * f / (2 * math.pi)   # of the original context
                keep = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
                f, m = keep * f + (1 - keep) * f / st["factor"], 1 + math.log(st["factor"]) / 10
            out.append(torch.stack([torch.cos(pos * f) * m, torch.sin(pos * f) * m], 1))
        return torch.stack(out, 1)
    rows, lens = _lengths(c)
    kv, D, P = c["kv"], c["dim"], c["page"]

    def tokens(s, n):
        pages = st["table"][s, :-(-lens[s] // P)].long()
        x = st[n][pages].to(d) * st[n + "_scale"][pages].to(d)[..., None]
        return x.permute(1, 0, 2, 3).reshape(kv, -1, D)[:, :lens[s]]

    if c["op"] == "read":
        return tuple(torch.cat([tokens(s, n)[:, lens[s] - rows[s]:].transpose(0, 1) for s in range(c["seqs"])]) for n in ("k", "v"))
    if c["op"] == "attn":
        G, out, r0 = c["heads"] // kv, [], 0
        for s in range(c["seqs"]):
            k, v, n, t = tokens(s, "k"), tokens(s, "v"), lens[s], rows[s]
            p, j = torch.arange(n - t, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
            hidden = (j > p) | ((p - j >= c["window"]) & (j >= c["sinks"])) if c["window"] else j > p
            o = torch.empty((t, c["heads"], D), device="cuda", dtype=d)
            for h in range(c["heads"]):
                a = st["qg"][r0:r0 + t, h, :D].to(d) @ k[h // G].T / math.sqrt(D)
                o[:, h] = torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v[h // G]
            if c["gate"]:
                o = o / (1 + torch.exp(-st["qg"][r0:r0 + t, :, D:].to(d)))
            out.append(o)
            r0 += t
        return torch.cat(out)
    # append
    H, rot, half, x = c["heads"], c["rot"], c["rot"] // 2, st["rows"].to(d)
    first = [2 * i if c["inter"] else i for i in range(half)]
    second = [2 * i + 1 if c["inter"] else i + half for i in range(half)]
    place = torch.cat([torch.arange(n - t, n) for t, n in zip(rows, lens)]).cuda()
    angle = st["rope"].to(d)[place]   # the table is an input

    def turned(y, w):
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.to(d)
        z = y.clone()
        z[..., first] = y[..., first] * angle[:, None, :, 0] - y[..., second] * angle[:, None, :, 1]
        z[..., second] = y[..., first] * angle[:, None, :, 1] + y[..., second] * angle[:, None, :, 0]
        return z

    q, scales, back = turned(x[:, :H], st["q_norm"]), [], []
    for n, y in (("k", turned(x[:, H:H + kv], st["k_norm"])), ("v", x[:, H + kv:])):
        a = y.abs().amax(-1, keepdim=True) / (127 if c["type"] == "i8" else 448)
        z = y / a
        back.append((z.round() if c["type"] == "i8" else z.float().to(torch.float8_e4m3fn).to(d)) * a)
        pool, r0 = st[n + "_scale"].to(d), 0
        for s, (t, m) in enumerate(zip(rows, lens)):
            at = torch.arange(m - t, m, device="cuda")
            pool[st["table"][s].long()[at // P], :, at % P] = a[r0:r0 + t, :, 0]
            r0 += t
        scales.append(pool)
    return (q, *back, *scales)
