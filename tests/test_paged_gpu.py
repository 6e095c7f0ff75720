"""The paged 8-bit cache on the GPU (hp_rope_table, hp_kv_append, hp_kv_read, hp_attn_paged) against plain implementations in 64 bits."""
import ctypes
import itertools
import math
import os
import subprocess
import sys

import pytest
import torch

import hipster_b200 as hb
from hipster_b200 import _lib, kernels as K_

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24     # half a step of f32, relative
KINDS = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


class Setup:
    """A pool with random contents, and a ragged batch with scattered pages."""

    def __init__(self, rows, lens, n_kv, D, page, kind, seed=0, spare=3, cols=None):
        g = gen(seed)
        self.rows, self.lens, self.R, self.D, self.kind, self.page = rows, lens, sum(rows), D, kind, page
        need = [-(-max(n, 0) // page) for n in lens]
        n_pages = sum(need) + spare
        cols = cols or max(need + [1])
        order = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        t = [[-1] * cols for _ in rows]
        for s, n in enumerate(need):
            for c in range(n):
                t[s][c] = order.pop()
        self.spare = order
        i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.table, self.kv_len = i(t), i(lens)
        self.row_start = i([sum(rows[:s]) for s in range(len(rows) + 1)])
        shape = (n_pages, n_kv, page, D)
        if kind == "i8":
            codes = [torch.randint(-127, 128, shape, generator=g, device="cuda").to(torch.int8) for _ in range(2)]
        else:
            codes = [(torch.randn(shape, generator=g, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
        unit = 1 / 70 if kind == "i8" else 1 / 100
        scales = [unit * torch.exp(0.5 * torch.randn(shape[:3], generator=g, device="cuda")) for _ in range(2)]
        self.pool = K_.KVPages(*codes, *scales)

    @property
    def batch(self):
        return self.table, self.row_start, self.kv_len

    def slot(self, s, pos):
        return int(self.table[s, pos // self.page]), pos % self.page

    def tokens(self, s, which, lo=0):
        """[n_kv][len][D] in 64 bits"""
        codes, scale = (self.pool.k, self.pool.k_scale) if which == "k" else (self.pool.v, self.pool.v_scale)
        ids = self.table[s].clamp(min=0).long()
        x = codes[ids].double() * scale[ids].double()[..., None]
        return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, self.D)[:, lo:max(self.lens[s], lo)]


    def scales(self, s):
        """Scales of v, [n_kv][len]"""
        return self.pool.v_scale[self.table[s].clamp(min=0).long()].double().permute(1, 0, 2).reshape(self.pool.n_kv, -1)


# ------------------------------------------------------------------ rotary tables
@pytest.mark.parametrize("n_pos,n_rot", [(1, 2), (100, 64), (517, 6), (1000, 256), (70000, 128)])
@pytest.mark.parametrize("scaling", [None, "linear", "yarn"])
def test_rope_table(n_pos, n_rot, scaling):
    base, factor, orig = 5e5, 6.5, 500
    got = K_.rope_table(n_pos, n_rot, base, scaling, factor=factor, orig_ctx=orig).double()
    i = torch.arange(n_rot // 2, device="cuda", dtype=torch.float64)
    f, m = torch.exp(-2 * i / n_rot * math.log(base)), 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        turns = orig * f / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        f, m = keep * f + (1 - keep) * f / factor, 1 + 0.1 * math.log(factor)
    a = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * f
    want = torch.stack([a.cos(), a.sin()], -1) * m
    assert got.shape == (n_pos, n_rot // 2, 2)
    # one rounding; angles of up to n_pos radians in 64 bits (a relative 2^-51 of the frequency and of the product)
    assert ((got - want).abs() <= U32 * want.abs() + n_pos * 2.0 ** -49 + 1e-40).all()
    hb.kernels.device_status()


def test_rope_table_is_the_engines_table():
    t = K_.rope_table(300, 64, 1e7).cpu().double()
    want = torch.tensor([[(math.cos(p * 1e7 ** (-2.0 * i / 64)), math.sin(p * 1e7 ** (-2.0 * i / 64))) for i in range(32)] for p in range(300)], dtype=torch.float64)
    assert ((t - want).abs() <= U32 * want.abs() + 1e-13).all()


# ------------------------------------------------------------------ append and read back
def turned64(x, w, eps, cs, inter, n_rot):
    """Norm and rotation in 64 bits -> values, and the sum of magnitudes that each is made of."""
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    y, mag = x.clone(), x.abs()
    if n_rot:
        h = n_rot // 2
        first = torch.arange(h, device=x.device) * (2 if inter else 1)
        second = first + (1 if inter else h)
        a, b, c, s = x[..., first], x[..., second], cs[:, None, :, 0], cs[:, None, :, 1]
        y[..., first], y[..., second] = a * c - b * s, b * c + a * s
        mag[..., first], mag[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, mag


def check_append(rows, lens, H, n_kv, D, page, kind, n_rot, inter, norm, seed=0, tail=0, in_place=False):
    st = Setup(rows, lens, n_kv, D, page, kind, seed)
    g, R = gen(seed + 1), st.R
    wide = torch.randn((R + tail, (2 * H + 2 * n_kv) * D + 8), generator=g, device="cuda") * torch.exp(torch.randn((R + tail, 1), generator=g, device="cuda"))
    # rows as a gated projection leaves them: q and its gate by head, then k, then v
    q = wide[:, :2 * H * D].view(R + tail, H, 2 * D)[..., :D]
    k, v = (wide[:, (2 * H + i * n_kv) * D:(2 * H + (i + 1) * n_kv) * D].view(R + tail, n_kv, D) for i in (0, 1))
    qn, kn = ((1 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16() if norm else None for _ in range(2))
    rope = K_.rope_table(max(lens), n_rot, 1e4) if n_rot else None
    q64, k64, v64 = q.double(), k.double(), v.double()
    before = [t.view(torch.uint8).clone() if t.dtype != torch.float32 else t.clone() for t in (st.pool.k, st.pool.v, st.pool.k_scale, st.pool.v_scale)]
    out = q if in_place else torch.full((R + tail, H, D), 7.0, device="cuda")
    old_tail = wide[R:].clone()
    got = K_.kv_append(st.pool, k, v, *st.batch, rope, q=q, q_out=out, interleaved=inter, q_norm=qn, k_norm=kn)
    K_.device_status()
    pos = torch.tensor([n - t + i for t, n in zip(rows, lens) for i in range(t)], device="cuda")
    cs = rope.double()[pos] if n_rot else None
    # 32-bit steps: up to 14 roundings in the sum of squares (halved by the root), 6 in norm and weight, 3 in the rotation
    lost = 16 * U32
    want, mag = turned64(q64[:R], qn, 1e-6, cs, inter, n_rot)
    assert ((got[:R].double() - want).abs() <= lost * mag).all()
    assert torch.equal(wide[R:], old_tail) if in_place else (out[R:] == 7).all()
    where = [st.slot(s, n - t + i) for s, (t, n) in enumerate(zip(rows, lens)) for i in range(t)]
    pg, at = (torch.tensor(x, device="cuda", dtype=torch.long) for x in zip(*where))
    top = 127.0 if kind == "i8" else 448.0
    ko, vo = (torch.full((R + tail, n_kv, D), 9.0, device="cuda", dtype=torch.float16) for _ in range(2))
    K_.kv_read(st.pool, *st.batch, k_out=ko, v_out=vo)
    for codes, scale, back, x64, w, turn in ((st.pool.k, st.pool.k_scale, ko, k64, kn, True), (st.pool.v, st.pool.v_scale, vo, v64, None, False)):
        want, mag = turned64(x64[:R], w, 1e-6, cs, inter, n_rot) if turn else (x64[:R], x64[:R].abs())
        amax, off = want.abs().amax(-1, keepdim=True), lost * mag.amax(-1, keepdim=True)
        s = scale[pg, :, at].double()[..., None]
        assert ((s - amax / top).abs() <= off / top + 2 * U32 * amax / top).all()
        value = codes[pg, :, at].double() * s
        # half a step of the code, a step's worth of shift where the 32-bit value lies on the other side of a border
        half = s / 2 if kind == "i8" else torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10)
        assert ((value - want).abs() <= half * (1 + 1e-5) + 2 * off + 4 * U32 * amax).all()
        assert ((back[:R].double() - value).abs() <= value.abs() * (2.0 ** -11 + 2 * U32) + 2.0 ** -25).all() and (back[R:] == 9).all()
    # nothing else was written
    for old, t in zip(before, (st.pool.k, st.pool.v, st.pool.k_scale, st.pool.v_scale)):
        now = t.view(torch.uint8) if t.dtype != torch.float32 else t
        old[pg, :, at] = now[pg, :, at]
        assert torch.equal(old, now)
    return st


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("D,H,n_kv,page,n_rot,inter,norm", [(256, 24, 4, 64, 64, False, True), (128, 5, 5, 16, 128, True, False), (64, 8, 1, 32, 64, False, False), (256, 2, 2, 128, 6, True, True),
                                                            (128, 12, 2, 1024, 2, False, True), (64, 1, 1, 16, 0, False, True), (256, 3, 1, 16, 256, False, False)])
def test_append(kind, D, H, n_kv, page, n_rot, inter, norm):
    check_append([1, 3, 0, 8, 17], [1, 40, 5, 8, 133], H, n_kv, D, page, kind, n_rot, inter, norm, tail=3)


def test_append_in_place_and_one_row():
    check_append([1], [1], 4, 2, 128, 16, "i8", 32, False, True, in_place=True)
    check_append([2, 5], [70, 9], 4, 2, 256, 32, "e4m3", 64, True, True, in_place=True, tail=2)


def test_append_many_rows_and_sequences():
    check_append([301], [400], 6, 1, 256, 64, "i8", 64, False, True)
    check_append([1] * 100, list(range(1, 101)), 3, 1, 64, 16, "e4m3", 64, False, False)


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_append_special_values(kind):
    st = Setup([6], [6], 1, 64, 16, kind)
    x = torch.randn((6, 1, 64), generator=gen(3), device="cuda")
    x[1] = 0
    x[2, 0, 5], x[3, 0, 63], x[4, 0, 0] = math.nan, -math.inf, 3e38
    x[5] = 1e-44   # a scale that is zero in 32 bits
    K_.kv_append(st.pool, x, x, *st.batch)
    k, v = K_.kv_read(st.pool, *st.batch, R=6)
    K_.device_status()
    assert torch.equal(k.view(torch.int16), v.view(torch.int16))
    assert torch.isfinite(k[[0, 1, 5]]).all() and (k[[1, 5]] == 0).all() and torch.isnan(k[2:4]).all()   # whole tokens, and their neighbours not
    page, at = st.slot(0, 4)
    top = 127 if kind == "i8" else 448
    assert float(st.pool.k[page, 0, at].double()[0]) == top and abs(float(st.pool.k_scale[page, 0, at]) * top / 3e38 - 1) < 1e-6


def test_appending_again_leaves_no_trace():
    """Rows that are appended, rejected and overwritten: the pages hold what appending the kept rows alone gives, bit for bit."""
    a, b = Setup([4], [20], 2, 128, 16, "i8"), Setup([4], [20], 2, 128, 16, "i8")
    x, wild = (torch.randn((4, 2, 128), generator=gen(s), device="cuda") for s in (1, 2))
    K_.kv_append(a.pool, torch.cat([x[:1], 1e3 * wild[1:]]), torch.cat([x[:1], 1e3 * wild[1:]]), *a.batch)
    K_.kv_append(a.pool, x, x, *a.batch)
    K_.kv_append(b.pool, x, x, *b.batch)
    for n in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(a.pool, n), getattr(b.pool, n))


def status():
    try:
        K_.device_status()
        return 0
    except hb.HipsterError as e:
        return e.code


def test_indexes_that_do_not_fit():
    """Bad pages, lengths and rows are left out and told; their neighbours are served. The kernels check every index before they use it."""
    st = Setup([2, 2, 2], [20, 20, 20], 1, 64, 16, "i8")
    x = torch.randn((6, 1, 64), generator=gen(1), device="cuda")
    rope = K_.rope_table(20, 64, 1e4)
    assert status() == 0
    good = st.table.clone()
    for bad in (-1, st.pool.n_pages, 1 << 30):
        st.table[1, 1] = bad
        before = st.pool.k.clone()
        K_.kv_append(st.pool, x, x, *st.batch, rope)
        assert status() == 1 and status() == 0
        changed = {tuple(i) for i in (st.pool.k != before).any(-1).nonzero().tolist()}
        assert changed <= {(p, 0, i) for s in (0, 2) for p, i in (st.slot(s, 18), st.slot(s, 19))}
        back = torch.full((6, 1, 64), 5.0, device="cuda", dtype=torch.float16)
        K_.kv_read(st.pool, *st.batch, k_out=back, v_out=back.clone())
        assert status() == 1 and (back[2:4] == 5).all() and (back[[0, 1, 4, 5]] != 5).any(-1).all()
        out, _ = K_.attn_paged(x, st.pool, *st.batch, max_rows=2, max_kv=20)
        assert status() == 1
        st.table.copy_(good)
        want, _ = K_.attn_paged(x, st.pool, *st.batch, max_rows=2, max_kv=20)
        assert torch.equal(out[[0, 1, 4, 5]], want[[0, 1, 4, 5]]) and status() == 0
        st.table.copy_(good)
    for what, at, value in (("kv_len", 1, 33), ("kv_len", 1, -5), ("kv_len", 1, 1 << 30), ("row_start", 3, 7), ("row_start", 3, 1 << 30), ("row_start", 1, -4), ("row_start", 2, 0), ("kv_len", 2, 1)):
        t = getattr(st, what)
        old = t.clone()
        t[at] = value
        K_.kv_append(st.pool, x, x, *st.batch, rope)   # 33 tokens: more than the columns hold; 1 token of 2 rows: no position
        assert status() == 1, (what, at, value)
        K_.kv_read(st.pool, *st.batch, R=6)
        assert status() == 1, (what, at, value)
        K_.attn_paged(x, st.pool, *st.batch, max_rows=2, max_kv=20)
        assert status() == (0 if (what, value) == ("kv_len", 1) else 1), (what, at, value)
        t.copy_(old)
    K_.attn_paged(x, st.pool, *st.batch, max_rows=1, max_kv=20)
    assert status() == 1
    K_.attn_paged(x, st.pool, *st.batch, max_rows=2, max_kv=19)
    assert status() == 1
    K_.kv_append(st.pool, x, x, *st.batch, rope[:19].contiguous())   # a position beyond the rotary table
    assert status() == 1


# ------------------------------------------------------------------ attention
def attn64(st, q, scale, window, n_sink, gate):
    """-> values and tolerances of every output, in 64 bits.

    With A_j = scale * sum |q_d k_jd| over the dims: a score is off by its 2 D / 16 additions on the tensor pipe (two chains of D / 16, each off by a step
    2^-23 of what has been summed), the rests of q (2^-22) and four roundings: |ds_j| <= (D / 16 + 8) 2^-23 A_j, and a shift of the scores by ds moves the result
    by at most 2 ds sum p |v|. The weights (2^-22 of ex2, 2^-22 of their rests, two roundings) and the sums (a step per 32 keys and per split of 256,
    counted on both sides of the quotient), gate and quotient (8 roundings) come on top.

    Weights far below the largest: w_j = p_j times the scale of v goes in as two f16 each on a common scale on which the largest is above 2^7 (the reference is whole and
    moves to 8 below the largest logarithm; it only grows, and what was added earlier is scaled down with its error), and f16 ends in steps of 2^-24. So each weight
    may be off by half such a step, 2^-25 / 2^7 = 2^-32 of the largest, and an output by 2^-32 max_j w_j sum_j |code_jd|: this is what is left where the
    code of a key that takes nearly all of the weight is zero."""
    H, n_kv, D = q.shape[1], st.pool.n_kv, st.D
    G = H // n_kv
    out, tol = torch.zeros((st.R, H, D), dtype=torch.float64, device="cuda"), torch.zeros((st.R, H, D), dtype=torch.float64, device="cuda")
    r0 = 0
    for s, (T, n) in enumerate(zip(st.rows, st.lens)):
        for t in range(T):
            pos = n - T + t
            if pos < 0:
                continue
            j = torch.arange(pos + 1, device="cuda")
            j = j[(j > pos - window) | (j < n_sink)] if window else j
            k, v = st.tokens(s, "k")[:, j].repeat_interleave(G, 0), st.tokens(s, "v")[:, j].repeat_interleave(G, 0)
            x = q[r0 + t].double()
            sc = torch.einsum("hd,hjd->hj", x, k) * scale
            A = (torch.einsum("hd,hjd->hj", x.abs(), k.abs()) * scale).amax(-1)
            p = torch.softmax(sc, -1)
            out[r0 + t] = torch.einsum("hj,hjd->hd", p, v)
            mag = torch.einsum("hj,hjd->hd", p, v.abs())
            steps = (2 * (D / 16 + 8) * A[:, None] + 2 * (len(j) / 32 + len(j) / 256 + 8) + 12)
            vs = st.scales(s)[:, j].repeat_interleave(G, 0)
            small = 2.0 ** -32 * (p * vs).amax(-1)[:, None] * (v.abs() / vs.clamp(min=1e-300)[..., None]).sum(1)
            tol[r0 + t] = steps * 2.0 ** -23 * mag + small
        r0 += T
    if gate is not None:
        g = torch.sigmoid(gate.double())
        out, tol = out * g, tol * g
    return out, tol


def check_attn(rows, lens, H, n_kv, D, page, kind, window=0, n_sink=0, gate=False, seed=0, tail=0, st=None, spread=1.0):
    st = st or Setup(rows, lens, n_kv, D, page, kind, seed)
    g = gen(seed + 5)
    qg = torch.randn((st.R + tail, H, 2 * D), generator=g, device="cuda") * torch.exp(spread * torch.randn((st.R + tail, H, 1), generator=g, device="cuda")).clamp(max=4)
    q, gt = qg[..., :D], qg[..., D:] if gate else None
    got, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=max(max(rows), 1), max_kv=max(max(lens), 1), window=window, n_sink=n_sink, gate=gt)
    assert status() == 0
    want, tol = attn64(st, q[:st.R], D ** -0.5, window, n_sink, None if gt is None else gt[:st.R])
    bad = (got[:st.R].double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(((got[:st.R].double() - want).abs() / tol.clamp(min=1e-30)).max()))
    return st, q, got


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows,lens", [([1], [1]), ([1, 1, 1], [64, 65, 63]), ([3, 1, 0, 8], [700, 257, 9, 8]), ([8, 2], [256, 1025])])
def test_attention_shapes(kind, D, rows, lens):
    check_attn(rows, lens, 12, 2, D, 16, kind, gate=True)


@pytest.mark.parametrize("H,n_kv", [(1, 1), (5, 5), (17, 1), (24, 4), (70, 2), (128, 1)])
def test_attention_heads(H, n_kv):
    check_attn([2, 1, 7], [300, 31, 90], H, n_kv, 64, 32, "i8")


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_attention_pages(page):
    check_attn([1, 4], [555, 130], 6, 2, 128, page, "e4m3")


@pytest.mark.parametrize("D,kind", [(64, "i8"), (128, "e4m3"), (256, "i8")])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (5, 4), (64, 0), (100, 300), (300, 70), (257, 1), (1000, 4), (5000, 0)])
def test_attention_window(D, kind, window, n_sink):
    check_attn([1, 8, 3, 2], [1500, 620, 3, 513], 6, 2, D, 16, kind, window=window, n_sink=n_sink)


@pytest.mark.parametrize("D,kind,H,n_kv", [(256, "i8", 24, 4), (128, "e4m3", 7, 1), (64, "i8", 4, 4)])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (50, 3), (200, 0), (129, 300)])
def test_attention_prompts(D, kind, H, n_kv, window, n_sink):
    check_attn([33, 9, 0, 100], [33, 400, 70, 217], H, n_kv, D, 32, kind, window=window, n_sink=n_sink, gate=True)


@pytest.mark.parametrize("D,kind,H,n_kv,page", [(256, "e4m3", 12, 2, 16), (128, "i8", 2, 1, 1024), (64, "e4m3", 49, 1, 64)])
def test_attention_long_prompts(D, kind, H, n_kv, page):
    check_attn([17], [3001], H, n_kv, D, page, kind)                    # few blocks: the keys in several splits
    check_attn([301, 1], [2301, 2000], H, n_kv, D, page, kind, window=1000, n_sink=130)


def test_attention_long_context():
    check_attn([1, 2], [20000, 9000], 6, 1, 128, 64, "i8")
    check_attn([1], [40000], 2, 2, 64, 256, "e4m3", window=33000, n_sink=600)


@pytest.mark.parametrize("H,n_kv,most", [(6, 2, 3), (2, 2, 16), (3, 1, 40)])
def test_attention_many_sequences(H, n_kv, most):
    rows = [1 + (7 * i) % most for i in range(75)]
    check_attn(rows, [r + (37 * i) % 300 for i, r in enumerate(rows)], H, n_kv, 64, 16, "i8")


def test_sequences_that_share_pages():
    st = Setup([2, 2, 1], [140, 140, 100], 2, 128, 16, "e4m3")
    st.table[1], st.table[2, :6] = st.table[0], st.table[0, :6]
    q = torch.randn((5, 4, 128), generator=gen(1), device="cuda")
    q[2:4] = q[:2]
    got, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=2, max_kv=140)
    want, tol = attn64(st, q, 128 ** -0.5, 0, 0, None)
    assert torch.equal(got[:2], got[2:4]) and ((got.double() - want).abs() <= tol).all() and status() == 0


def test_largest_window_and_first_tokens():
    big = 2 ** 31 - 1
    st = Setup([2, 20], [3, 300], 1, 64, 16, "i8")
    q = torch.randn((22, 2, 64), generator=gen(1), device="cuda")
    for mr, rs in ((20, st.row_start), (2, torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"))):
        a, b, c = (K_.attn_paged(q, st.pool, st.table, rs, st.kv_len, max_rows=mr, max_kv=300, window=w, n_sink=k)[0] for w, k in ((0, 0), (big, big), (big, 0)))
        n = int(rs[-1])
        assert status() == 0 and torch.equal(b[:n], c[:n])
        assert ((a[:n] - b[:n]).abs() <= 1e-5 * a[:n].abs().amax()).all()   # other splits: the same but for rounding


def test_rows_without_a_key_and_rows_behind_the_last():
    st = Setup([3, 1, 2], [1, 0, 40], 1, 64, 16, "i8", cols=3)
    q = torch.randn((20, 4, 64), generator=gen(2), device="cuda")
    for mr in (3, 17):   # both forms
        ws = torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda")
        out = torch.full((20, 4, 64), 3.0, device="cuda")
        v, z = ctypes.c_void_p, ctypes.c_longlong
        hb.check(hb.lib().hp_attn_paged(hb.ptr(q), z(256), z(64), None, z(0), z(0), 4, hb.ptr(st.table), 3, hb.ptr(st.row_start), hb.ptr(st.kv_len), 3, 20, mr, 40, v(st.pool._at), ctypes.c_float(0.125), 0, 0,
                                        hb.ptr(out), None, None, hb.ptr(ws), K_._stream()))
        assert status() == 0
        want, tol = attn64(st, q[:6], 0.125, 0, 0, None)
        assert (out[:2] == 0).all() and (out[3] == 0).all() and ((out[:6].double() - want).abs() <= tol).all() and (out[6:] == 3).all()


def test_what_no_row_sees_does_not_count():
    """Codes and scales of masked, unused and foreign slots: NaN, infinity, huge; pages in front of the window are not even in the table."""
    for kind in ("i8", "e4m3"):
        for window, n_sink in ((0, 0), (70, 3)):
            rows, lens = [2, 1, 20], [300, 201, 250]
            a = Setup(rows, lens, 2, 128, 16, kind, seed=4)
            q = torch.randn((23, 4, 128), generator=gen(1), device="cuda")
            want = [K_.attn_paged(q[i:j], a.pool, a.table[s:s + 1], torch.tensor([0, j - i], dtype=torch.int32, device="cuda"), a.kv_len[s:s + 1], max_rows=j - i, max_kv=300, window=window, n_sink=n_sink)[0]
                    for s, (i, j) in enumerate(((0, 2), (2, 3), (3, 23)))]
            seen = torch.zeros(a.pool.k.shape[:3], dtype=torch.bool, device="cuda")
            for s, (t, n) in enumerate(zip(rows, lens)):
                for pos in range(n):
                    if not window or pos > n - t - window or pos < n_sink:
                        pg, at = a.slot(s, pos)
                        seen[pg, :, at] = True
                for c in range(a.table.shape[1]):   # pages that no row sees
                    pg = int(a.table[s, c])
                    if pg >= 0 and not seen[pg].any():
                        a.table[s, c] = -7
            for codes in (a.pool.k, a.pool.v):
                codes.view(torch.uint8)[~seen] = 0x7f
            a.pool.k_scale[~seen] = math.nan
            a.pool.v_scale[~seen] = math.inf
            for s, (i, j) in enumerate(((0, 2), (2, 3), (3, 23))):
                got, _ = K_.attn_paged(q[i:j], a.pool, a.table[s:s + 1], torch.tensor([0, j - i], dtype=torch.int32, device="cuda"), a.kv_len[s:s + 1], max_rows=j - i, max_kv=300, window=window, n_sink=n_sink)
                assert status() == 0 and torch.isfinite(got).all() and torch.equal(got, want[s])


def test_non_finite_tokens_reach_the_rows_that_see_them():
    st = Setup([4], [100], 1, 64, 16, "i8")
    q = torch.randn((4, 2, 64), generator=gen(1), device="cuda")
    clean, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=4, max_kv=100)
    for scale, bad in ((st.pool.k_scale, math.nan), (st.pool.v_scale, math.nan), (st.pool.v_scale, math.inf)):
        pg, at = st.slot(0, 98)   # seen by the last two rows
        old = scale.clone()
        scale[pg, 0, at] = bad
        got, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=4, max_kv=100)
        assert torch.equal(got[:2], clean[:2]) and torch.isnan(got[2:]).all()
        scale.copy_(old)
    q[1] = math.nan
    got, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=4, max_kv=100)
    assert torch.isnan(got[1]).all() and torch.equal(got[[0, 2, 3]], clean[[0, 2, 3]])


@pytest.mark.parametrize("k_up,v_up", [(1e-12, 1e-12), (1e10, 1e15), (1.0, 1e-25), (1e-30, 1.0)])
def test_magnitudes(k_up, v_up):
    """Scales far from 1, and of very different size from token to token (some of them zero)."""
    st = Setup([2, 1], [150, 40], 2, 64, 16, "e4m3")
    st.pool.k_scale.mul_(k_up)
    st.pool.v_scale.mul_(v_up * torch.exp(3 * torch.randn(st.pool.v_scale.shape, generator=gen(8), device="cuda")))
    st.pool.v_scale[:, :, 3] = 0
    g = gen(5)
    q = torch.randn((3, 4, 64), generator=g, device="cuda") / k_up
    got, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=2, max_kv=150)
    want, tol = attn64(st, q, 0.125, 0, 0, None)
    assert status() == 0 and ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("D,kind,G,window,n_sink", [(256, "i8", 6, 0, 0), (128, "e4m3", 12, 0, 0), (64, "i8", 5, 300, 4), (256, "e4m3", 12, 100, 1)])
def test_a_rows_bits_depend_on_nothing_else(D, kind, G, window, n_sink):
    """Up to 16 rows per sequence: the same bits alone, in a verify pass, and among other sequences."""
    rows, lens, H = [16, 1, 5, 8], [1300, 600, 271, 1025], 2 * G
    st, q, got = check_attn(rows, lens, H, 2, D, 32, kind, window=window, n_sink=n_sink)
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    r = 0
    for s, (t, n) in enumerate(zip(rows, lens)):
        for i in range(t):
            alone, _ = K_.attn_paged(q[r:r + 1], st.pool, st.table[s:s + 1], one, torch.tensor([n - t + i + 1], dtype=torch.int32, device="cuda"), max_rows=1, max_kv=n, window=window, n_sink=n_sink)
            assert torch.equal(alone[0], got[r]), (s, i)
            r += 1
    again, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=16, max_kv=4000, window=window, n_sink=n_sink)
    assert torch.equal(again, got)


def test_quantised_output_is_the_quantised_f32_output():
    st = Setup([3, 1, 4], [100, 40, 77], 2, 128, 16, "i8")
    q = torch.randn((8, 6, 128), generator=gen(1), device="cuda")
    out, xq = K_.attn_paged(q, st.pool, *st.batch, max_rows=4, max_kv=100, want_q8=True)
    want = K_.quantize_x_q8(out.view(8, -1)).unpack()
    assert all(torch.equal(a, b) for a, b in zip(xq.unpack(), want))
    none, xq = K_.attn_paged(q, st.pool, *st.batch, max_rows=4, max_kv=100, want_f32=False, want_q8=True)
    assert none is None and all(torch.equal(a, b) for a, b in zip(xq.unpack(), want))


def test_offsets_beyond_32_bits():
    """A pool of 5.4 GB per tensor, used at both ends."""
    page, n_kv, D = 1024, 8, 256
    n_pages = 2600
    k, v = (torch.empty((n_pages, n_kv, page, D), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty((n_pages, n_kv, page), device="cuda") for _ in range(2))
    small = Setup([3], [1500], n_kv, D, page, "i8")
    pool = K_.KVPages(k, v, ks, vs)
    table = torch.tensor([[n_pages - 1, 0]], dtype=torch.int32, device="cuda")
    for a, b in zip((k, v, ks, vs), (small.pool.k, small.pool.v, small.pool.k_scale, small.pool.v_scale)):
        for c in range(2):
            a[int(table[0, c])] = b[int(small.table[0, c])]
    x = torch.randn((3, 8, D), generator=gen(1), device="cuda")
    for p, t in ((pool, table), (small.pool, small.table)):
        K_.kv_append(p, x, 2 * x, t, small.row_start, small.kv_len)
    got, want = (K_.attn_paged(x, p, t, small.row_start, small.kv_len, max_rows=3, max_kv=1500)[0] for p, t in ((pool, table), (small.pool, small.table)))
    assert torch.equal(got, want)
    rs, ln = torch.tensor([0, 1500], dtype=torch.int32, device="cuda"), torch.tensor([1500], dtype=torch.int32, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(K_.kv_read(pool, table, rs, ln, R=1500), K_.kv_read(small.pool, small.table, rs, ln, R=1500)))
    assert status() == 0


# ------------------------------------------------------------------ together
def test_captured_steps_replay_with_other_lengths():
    st = Setup([1, 1], [90, 40], 2, 128, 16, "i8", cols=7, spare=8)
    for s in range(2):
        for c in range(7):
            if st.table[s, c] < 0:
                st.table[s, c] = st.spare.pop()
    rope = K_.rope_table(112, 128, 1e4)
    x = torch.randn((2, 8, 128), generator=gen(1), device="cuda")

    def step():
        q = K_.kv_append(st.pool, x[:, 4:6], x[:, 6:8], *st.batch, rope, q=x[:, :4])
        return K_.attn_paged(q, st.pool, *st.batch, max_rows=1, max_kv=112)[0]

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):   # two captures, each with a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = step()
        graphs.append((g, y))
    for i in range(8):
        st.kv_len += 1
        x.normal_(generator=gen(10 + i))
        g, y = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, step())
    assert status() == 0


def test_the_first_call_of_a_process_may_be_captured():
    code = ("import torch\n"
            "from hipster_b200 import kernels as K\n"
            "pool = K.KVPages.empty(4, 1, 16, 64)\n"
            "i = lambda x: torch.tensor(x, dtype=torch.int32, device='cuda')\n"
            "t, rs, kl = i([[0, 1]]), i([0, 1]), i([20])\n"
            "x = torch.randn((1, 1, 64), device='cuda')\n"
            "torch.cuda.synchronize()\n"
            "g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g):\n"
            "    rope = K.rope_table(32, 64, 1e4)\n"
            "    q = K.kv_append(pool, x, x, t, rs, kl, rope, q=x)\n"
            "    y, _ = K.attn_paged(q, pool, t, rs, kl, max_rows=1, max_kv=20)\n"
            "    k, v = K.kv_read(pool, t, rs, kl, R=1)\n"
            "g.replay()\n"
            "torch.cuda.synchronize()\n"
            "K.device_status()\n"
            "z, _ = K.attn_paged(q, pool, t, rs, kl, max_rows=1, max_kv=20)\n"
            "assert torch.equal(y, z) and (v.float() - x).abs().max() < 0.02 * x.abs().max()\n"
            "print('fine')\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_captured_prompts():
    st = Setup([40, 3], [90, 40], 2, 64, 16, "i8", cols=7, spare=6)
    for s in range(2):
        for c in range(7):
            if st.table[s, c] < 0:
                st.table[s, c] = st.spare.pop()
    q = torch.randn((43, 4, 64), generator=gen(1), device="cuda")
    step = lambda: K_.attn_paged(q, st.pool, *st.batch, max_rows=40, max_kv=112)[0]  # noqa: E731
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step()
    for i in range(5):
        st.kv_len += 4
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, step())
    assert status() == 0


@pytest.fixture(params=["native", "python"])
def form(request, monkeypatch):
    """The calls in C++ where they were built (they are, here), and without them."""
    assert _lib.tensors() is not None
    if request.param == "python":
        monkeypatch.setattr(_lib, "_tensor_calls", False)
    return request.param


def test_both_forms_of_the_calls(form):
    st = Setup([3, 0, 18], [50, 7, 200], 2, 128, 16, "e4m3")
    g = gen(2)
    x = torch.randn((23, 8, 128), generator=g, device="cuda")   # two rows behind the last
    rope = K_.rope_table(300, 64, 1e4, "yarn", factor=4, orig_ctx=64)
    assert torch.equal(rope, K_.rope_table(300, 64, 1e4, "yarn", factor=4.0, orig_ctx=64, beta_fast=32, beta_slow=1.0, attn_factor=0))
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    into = torch.full((23, 4, 256), 2.0, device="cuda")[..., :128]
    q = K_.kv_append(st.pool, x[:, 4:6], x[:, 6:], *st.batch, rope, q=x[:, :4], q_out=into, interleaved=True, q_norm=w, k_norm=w.view(torch.int16))
    assert q.data_ptr() == into.data_ptr() and (q[21:] == 2).all()
    assert torch.equal(K_.kv_append(st.pool, x[:, 4:6], x[:, 6:], *st.batch, rope, q=x[:, :4], interleaved=1, q_norm=w, k_norm=w)[:21], q[:21])
    assert K_.kv_append(st.pool, x[:, 4:6], x[:, 6:], *st.batch, rope, interleaved=True, k_norm=w) is None
    k, v = K_.kv_read(st.pool, *st.batch, R=21)
    a, xq = K_.attn_paged(q, st.pool, *st.batch, max_rows=18, max_kv=200, window=60, n_sink=2, gate=x[:, :4])
    b, xr = K_.attn_paged(q, st.pool, *st.batch, max_rows=18, max_kv=200, scale=128 ** -0.5, window=60, n_sink=2, gate=x[:, :4], want_q8=True)
    assert xq is None and torch.equal(a[:21], b[:21]) and k.shape == v.shape == (21, 2, 128) and status() == 0
    have = torch.cat([q[:21].flatten(), k.float().flatten(), v.float().flatten(), a[:21].flatten()])
    if form == "native":
        test_both_forms_of_the_calls.seen = have
    else:
        assert torch.equal(have, test_both_forms_of_the_calls.seen)


def test_refusals_of_the_python_calls(form):
    st = Setup([2], [20], 2, 64, 16, "i8")
    q = torch.randn((2, 4, 64), device="cuda")
    kv = q[:, :2]
    rope = K_.rope_table(32, 64, 1e4)
    t, rs, kl = st.batch
    cpu = K_.KVPages.empty(2, 2, 16, 64, device="cpu")
    bad = [lambda: K_.attn_paged(q, cpu, t, rs, kl, 2, 20), lambda: K_.attn_paged(q, st.pool, t.cpu(), rs, kl, 2, 20), lambda: K_.attn_paged(q, st.pool, t, rs.long(), kl, 2, 20),
           lambda: K_.attn_paged(q, st.pool, t, rs[:1], kl, 2, 20), lambda: K_.attn_paged(q, st.pool, t.expand(2, -1), rs, kl, 2, 20), lambda: K_.attn_paged(q.half(), st.pool, t, rs, kl, 2, 20),
           lambda: K_.attn_paged(q[..., :32], st.pool, t, rs, kl, 2, 20), lambda: K_.attn_paged(q.transpose(1, 2).contiguous().transpose(1, 2), st.pool, t, rs, kl, 2, 20), lambda: K_.attn_paged(q.cpu(), st.pool, t, rs, kl, 2, 20),
           lambda: K_.attn_paged(q[:, :3], st.pool, t, rs, kl, 2, 20), lambda: K_.attn_paged(q, st.pool, t, rs, kl, 2, 20, gate=q[:, :2]), lambda: K_.attn_paged(q, st.pool, t, rs, kl, 0, 20),
           lambda: K_.attn_paged(q, st.pool, t, rs, kl, 2, 20, n_sink=3), lambda: K_.attn_paged(q, st.pool, t, rs, kl, 2, 20, want_f32=False),
           lambda: K_.kv_append(st.pool, q, q, t, rs, kl), lambda: K_.kv_append(st.pool, kv, kv[:1], t, rs, kl), lambda: K_.kv_append(st.pool, kv, kv, t, rs, kl, rope.half()), lambda: K_.kv_append(st.pool, kv, kv, t, rs, kl, rope[:, ::2]),
           lambda: K_.kv_append(st.pool, kv, kv, t, rs, kl, K_.rope_table(32, 128, 1e4)), lambda: K_.kv_append(st.pool, kv, kv, t, rs, kl, rope, q=q, q_out=q[:, :2]), lambda: K_.kv_append(st.pool, kv, kv, t, rs, kl, q_norm=q[0, 0]),
           lambda: K_.kv_append(st.pool, kv, kv, t, rs, kl, k_norm=torch.ones(64, dtype=torch.float16, device="cuda")), lambda: K_.kv_read(st.pool, t, rs, kl), lambda: K_.kv_read(st.pool, t, rs, kl, R=0),
           lambda: K_.kv_read(st.pool, t, rs, kl, k_out=kv.half()), lambda: K_.kv_read(st.pool, t, rs, kl, k_out=kv, v_out=kv), lambda: K_.rope_table(0, 64, 1e4), lambda: K_.rope_table(8, 64, -1.0), lambda: K_.rope_table(8, 64, 1e4, device="cpu")]
    for i, f in enumerate(bad):
        with pytest.raises(hb.HipsterError):
            f()
            pytest.fail(f"call {i} was not refused")
    assert status() == 0


def test_streams():
    st = Setup([2], [500], 2, 256, 64, "i8")
    q = torch.randn((2, 12, 256), generator=gen(1), device="cuda")
    want, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=2, max_kv=500)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(4)], []
    for i in range(12):
        with torch.cuda.stream(streams[i % 4]):
            got.append(K_.attn_paged(q, st.pool, *st.batch, max_rows=2, max_kv=500)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_a_sequence_from_prompt_to_rejected_drafts():
    """Prompt chunk, verify passes of which a part is accepted, and the same tokens one at a time: the same pages and the same outputs, bit for bit."""
    H, n_kv, D, page, n = 6, 2, 256, 16, 60
    g = gen(11)
    stream = torch.randn((n, H + 2 * n_kv, D), generator=g, device="cuda")
    qn, kn = ((1 + 0.1 * torch.randn(D, generator=g, device="cuda")).bfloat16() for _ in range(2))
    rope = K_.rope_table(n + 8, 64, 1e7)
    table = torch.tensor([[2, 0, 5, 1, 4]], dtype=torch.int32, device="cuda")

    def run(plan):
        pool, pos, outs = K_.KVPages.empty(6, n_kv, page, D), 0, []
        for rows, keep in plan:
            x = stream[pos:pos + rows].clone()
            if rows > keep:   # rejected drafts: other rows than the stream's
                x = torch.cat([x[:keep], 30 * torch.randn((rows - keep, H + 2 * n_kv, D), generator=g, device="cuda")])
            rs = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
            ln = torch.tensor([pos + rows], dtype=torch.int32, device="cuda")
            q = K_.kv_append(pool, x[:, H:H + n_kv], x[:, H + n_kv:], table, rs, ln, rope, q=x[:, :H], q_norm=qn, k_norm=kn)
            outs.append(K_.attn_paged(q, pool, table, rs, ln, max_rows=rows, max_kv=pos + rows)[0][:keep])
            pos += keep
        assert pos == n and status() == 0
        return pool, outs

    pool, spec = run([(30, 30)] + [(6, 3)] * 10)
    ref, plain = run([(30, 30)] + [(1, 1)] * 30)
    assert torch.equal(torch.cat(spec[1:]), torch.cat(plain[1:])) and torch.equal(spec[0], plain[0])
    whole = torch.tensor([0, n], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(K_.kv_read(pool, table, *whole, R=n), K_.kv_read(ref, table, *whole, R=n)))

    # and the f16 attention on the cache that kv_read hands over, next to this one on the pages: the same tokens up to f16's rounding of them
    kc, vc = torch.zeros((2, n_kv, n + 8, D), dtype=torch.float16, device="cuda")
    K_.kv_read(pool, table, *whole, k_out=kc.transpose(0, 1)[:n], v_out=vc.transpose(0, 1)[:n])
    x = torch.randn((1, H + 2 * n_kv, D), generator=g, device="cuda")
    gate = torch.randn((1, H, D), generator=g, device="cuda")
    rs, ln = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([n + 1], dtype=torch.int32, device="cuda")
    qkv = torch.cat([torch.stack([x[:, :H], gate], 2).flatten(1), x[:, H:].flatten(1)], 1).contiguous()
    want, _ = K_.attn_decode(qkv, n, H, n_kv, 64, qn.view(torch.int16), kn.view(torch.int16), rope, kc, vc, n + 8, want_q8=False)
    q = K_.kv_append(pool, x[:, H:H + n_kv], x[:, H + n_kv:], table, rs, ln, rope, q=x[:, :H], q_norm=qn, k_norm=kn)
    # the new token itself is 8 bits here and f16 there: put the 8-bit one into the f16 cache too
    K_.kv_read(pool, table, rs, ln, k_out=kc.transpose(0, 1)[n:n + 1], v_out=vc.transpose(0, 1)[n:n + 1])
    k8, v8 = kc[:, n].clone(), vc[:, n].clone()
    got, _ = K_.attn_paged(q, pool, table, rs, ln, max_rows=1, max_kv=n + 1, gate=gate)
    # weights: f16 keys move a score by 2^-12 of sum |q k| / 16 (below 16 at unit rows); the token that differs has one weight of 61
    st = Setup([1], [n + 1], n_kv, D, page, "i8")
    st.pool, st.table = pool, table
    exact, tol = attn64(st, q, 1 / 16, 0, 0, gate)
    assert ((got.double() - exact).abs() <= tol).all() and k8.isfinite().all() and v8.isfinite().all()
    assert float((want.view(1, H, D).double() - exact).norm() / exact.norm()) < 0.05


@pytest.mark.parametrize("D,H,n_kv", [(64, 5, 1), (128, 3, 3), (256, 6, 2)])
@pytest.mark.parametrize("rows,lens,window,n_sink", [([3, 0, 1, 2], [700, 10, 1, 300], 0, 0), ([3, 1, 2], [900, 40, 513], 300, 20), ([40, 3, 0], [600, 3, 9], 0, 0), ([40, 19], [600, 777], 200, 5),
                                                       ([3, 0, 1, 16], [256, 10, 1, 40], 0, 0), ([8, 2], [2, 33], 0, 0)])
def test_gates_and_outputs_at_odd_places(D, H, n_kv, rows, lens, window, n_sink):
    # Gates are read four at a time where they lie so, and one at a time elsewhere; a single split writes the outputs itself where it can. The same bits, quantised rows too, and
    # with more splits (max_kv). The last row has no key.
    lens = [*lens, 0]
    rows = [*rows, 1]
    st = Setup(rows, lens, n_kv, D, 16, "e4m3", 3, cols=-(-4 * max(lens) // 16))
    g = gen(7)
    q = torch.randn((st.R, H, D), generator=g, device="cuda")
    gate = torch.randn((st.R, H, D), generator=g, device="cuda")
    odd = torch.zeros(st.R * (H * (D + 1) + 2) + 1, device="cuda")[1:].as_strided((st.R, H, D), (H * (D + 1) + 2, D + 1, 1))
    odd.copy_(gate)
    run = lambda x: K_.attn_paged(q, st.pool, *st.batch, max_rows=max(rows), max_kv=max(lens), window=window, n_sink=n_sink, gate=x, want_q8=True)  # noqa: E731
    (a, xa), (b, xb) = run(gate), run(odd)
    assert torch.equal(a, b) and torch.equal(xa.q, xb.q) and torch.equal(xa.sc, xb.sc)
    if max(rows) <= 16:
        c, xc = K_.attn_paged(q, st.pool, *st.batch, max_rows=max(rows), max_kv=4 * max(lens), window=window, n_sink=n_sink, gate=gate, want_q8=True)
        assert torch.equal(a, c) and torch.equal(xa.q, xc.q) and torch.equal(xa.sc, xc.sc)
    exact, tol = attn64(st, q, D ** -0.5, window, n_sink, gate)
    assert ((a.double() - exact).abs() <= tol).all() and (a[-1] == 0).all()


@pytest.mark.parametrize("window", [0, 5000])   # several splits; one, which writes the outputs itself
@pytest.mark.parametrize("D,kind", [(64, "i8"), (128, "e4m3"), (256, "i8")])
def test_non_finite_tokens_in_prompts(D, kind, window):
    st = Setup([70], [300], 1, D, 16, kind)
    q = torch.randn((70, 5, D), generator=gen(1), device="cuda")
    run = lambda: K_.attn_paged(q, st.pool, *st.batch, max_rows=70, max_kv=300, window=window)[0]  # noqa: E731
    clean = run()
    for scale, bad in itertools.product((st.pool.k_scale, st.pool.v_scale), (math.nan, math.inf)):
        pg, at = st.slot(0, 290)   # seen by the last ten rows
        old = scale.clone()
        scale[pg, 0, at] = bad
        got = run()
        assert torch.equal(got[:60], clean[:60]) and (scale is st.pool.k_scale and bad == math.inf or torch.isnan(got[60:]).all())
        scale.copy_(old)
    q[33, 2] = math.nan
    got = run()
    assert torch.isnan(got[33, 2]).all()
    got[33, 2] = clean[33, 2]
    assert torch.equal(got, clean) and status() == 0


@pytest.mark.parametrize("k_up,v_up", [(1e-12, 1e-12), (1e10, 1e15), (1.0, 1e-25), (1e-30, 1.0)])
@pytest.mark.parametrize("D,window", [(64, 0), (256, 0), (128, 5000), (256, 5000)])
def test_magnitudes_in_prompts(D, window, k_up, v_up):
    st = Setup([40, 17], [250, 90], 2, D, 16, "e4m3")
    st.pool.k_scale.mul_(k_up)
    st.pool.v_scale.mul_(v_up * torch.exp(3 * torch.randn(st.pool.v_scale.shape, generator=gen(8), device="cuda")))
    st.pool.v_scale[:, :, 3] = 0
    q = torch.randn((57, 8, D), generator=gen(5), device="cuda") / k_up
    got, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=40, max_kv=250, scale=0.125, window=window)
    want, tol = attn64(st, q, 0.125, 0, 0, None)
    assert status() == 0 and ((got.double() - want).abs() <= tol).all()


def test_prompts_and_steps_at_once():
    # calls that hold all accumulator memory of an SM and calls that hold none, on four streams
    st, few = Setup([150, 40], [1500, 700], 2, 256, 64, "i8"), Setup([2, 1], [900, 30], 2, 256, 16, "i8", 1)
    q = torch.randn((190, 12, 256), generator=gen(1), device="cuda")
    prompt = lambda: K_.attn_paged(q, st.pool, *st.batch, max_rows=150, max_kv=1500)[0]  # noqa: E731
    step = lambda: K_.attn_paged(q[:3], few.pool, *few.batch, max_rows=2, max_kv=900)[0]  # noqa: E731
    want = prompt(), step()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(4)], []
    for i in range(24):
        with torch.cuda.stream(streams[i % 4]):
            got.append((prompt if i % 3 else step)())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[0 if i % 3 else 1]) for i, g in enumerate(got)) and status() == 0
