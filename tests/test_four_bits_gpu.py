"""The paged cache in 4 bits (HP_KV_I4) and positions of several axes on the GPU, against plain implementations in 64 bits. The oracles of attention and rotation are those of the 8-bit cache."""
import ctypes
import math

import pytest
import torch

import hipster_b200 as hb
from hipster_b200 import _lib, kernels as K_
import test_paged_gpu as P

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
gen, status = P.gen, P.status
form = P.form


def parts(t, page, D):
    """Views of the codes [..., page, D / 2] and of the groups' bytes [..., page, D / 32] of a 4-bit tensor [..., page * 17 * D / 32]."""
    n = page * D // 2
    return t[..., :n].unflatten(-1, (page, D // 2)), t[..., n:].unflatten(-1, (page, D // 32))


def whole(codes, groups):
    """The whole numbers u * (c - z) [..., D] in 64 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 32)).double()
    return ((groups >> 4).double()[..., None] * (c - (groups & 15).double()[..., None])).flatten(-2)


class Setup(P.Setup):
    """P.Setup with every code and byte of a group that there is, factors of zero among them."""

    def __init__(self, rows, lens, n_kv, D, page, seed=0, spare=3, cols=None):
        super().__init__(rows, lens, n_kv, D, page, "i8", seed, spare, cols)
        g = gen(seed + 100)
        n_pages = self.pool.n_pages
        codes = [torch.randint(0, 256, (n_pages, n_kv, page * 17 * D // 32), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
        scales = [1 / 90 * torch.exp(0.5 * torch.randn((n_pages, n_kv, page), generator=g, device="cuda")) for _ in range(2)]
        self.kind, self.pool = "i4", K_.KVPages(*codes, *scales)

    def tokens(self, s, which, lo=0):
        codes, scale = (self.pool.k, self.pool.k_scale) if which == "k" else (self.pool.v, self.pool.v_scale)
        ids = self.table[s].clamp(min=0).long()
        x = whole(*parts(codes[ids], self.page, self.D)) * scale[ids].double()[..., None]
        return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, self.D)[:, lo:max(self.lens[s], lo)]


def check_attn(rows, lens, H, n_kv, D, page, window=0, n_sink=0, gate=False, seed=0, tail=0, spread=1.0):
    return P.check_attn(rows, lens, H, n_kv, D, page, "i4", window, n_sink, gate, seed, tail, Setup(rows, lens, n_kv, D, page, seed), spread)


# ------------------------------------------------------------------ append and read back
def positions(n_axes, R, n_pos, seed=0):
    return torch.randint(0, n_pos, (n_axes, R), generator=gen(seed + 50), device="cuda", dtype=torch.int32)


def angles64(rope, pos, axes):
    """[R][n_rot / 2][2]: each pair by the position on its axis."""
    a = torch.tensor(list(axes), device="cuda")
    return rope.double()[pos.long()[a].T, torch.arange(len(a), device="cuda")]


def held(x, off, codes, groups, scale):
    """What 4 bits hold of x (64 bits; off: how far the 32-bit values may be from it, by element) where the definition leaves no choice, and where it does, one of the choices."""
    D = x.shape[-1]
    g, og = x.unflatten(-1, (-1, 32)), off.unflatten(-1, (-1, 32)).amax(-1)
    lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
    span = hi - lo
    most, omost = span.amax(-1), 2 * og.amax(-1)
    s = scale.double()
    assert ((s - most / 225).abs() <= omost / 225 + 4 * U32 * most / 225 + 1e-44).all()
    u, z = (groups >> 4).double(), (groups & 15).double()
    ratio = 15 * span / most.clamp(min=1e-300)[..., None]
    wob = (30 * og / most.clamp(min=1e-300)[..., None] + 15 * (omost / most.clamp(min=1e-300))[..., None] + 1e-5)
    assert ((u >= (ratio - wob).ceil().clamp(0, 15)) & (u <= (ratio + wob).ceil().clamp(0, 15)))[most > 0].all()
    step = (s[..., None] * u).clamp(min=1e-300)
    rel = 8 * U32   # of step, reciprocal, products
    at = -lo / step
    assert ((z - at).abs() <= 0.5 + 2 * og / step + rel * at + 1e-6)[u > 0].all()
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 32)).double()
    t = g / step[..., None] + z[..., None]
    assert ((c - t.clamp(0, 15)).abs() <= 0.5 + (2 * og / step)[..., None] + rel * 16 + 1e-6)[(u > 0)[..., None].expand_as(c)].all()
    assert (c[(u == 0)[..., None].expand_as(c)] == 0).all()
    return whole(codes, groups) * s[..., None]


def check_append(rows, lens, H, n_kv, D, page, n_rot, inter, norm, axes=None, seed=0, tail=0, in_place=False, kind="i4"):
    st = Setup(rows, lens, n_kv, D, page, seed) if kind == "i4" else P.Setup(rows, lens, n_kv, D, page, kind, seed)
    g, R = gen(seed + 1), st.R
    wide = torch.randn((R + tail, (2 * H + 2 * n_kv) * D + 8), generator=g, device="cuda") * torch.exp(torch.randn((R + tail, 1), generator=g, device="cuda"))
    q = wide[:, :2 * H * D].view(R + tail, H, 2 * D)[..., :D]   # rows as a gated projection leaves them: q and its gate by head, then k, then v
    k, v = (wide[:, (2 * H + i * n_kv) * D:(2 * H + (i + 1) * n_kv) * D].view(R + tail, n_kv, D) for i in (0, 1))
    qn, kn = ((1 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16() if norm else None for _ in range(2))
    n_pos = 77 if axes is not None else max(lens)
    rope = K_.rope_table(n_pos, n_rot, 1e4) if n_rot else None
    pos = positions(1 + max(axes), R + tail, n_pos, seed) if axes is not None else None
    x64 = q.double(), k.double(), v.double()
    pools = lambda: (st.pool.k, st.pool.v, st.pool.k_scale, st.pool.v_scale)  # noqa: E731
    before = [t.clone() for t in pools()]
    out = q if in_place else torch.full((R + tail, H, D), 7.0, device="cuda")
    old_tail = wide[R:].clone()
    got = K_.kv_append(st.pool, k, v, *st.batch, rope, q=q, q_out=out, interleaved=inter, q_norm=qn, k_norm=kn, positions=pos, axes=axes)
    assert status() == 0
    place = torch.tensor([n - t + i for t, n in zip(rows, lens) for i in range(t)], device="cuda")
    cs = None if not n_rot else angles64(rope, pos[:, :R], axes) if axes is not None else rope.double()[place]
    lost = 16 * U32   # 32-bit steps: up to 14 roundings in the sum of squares (halved by the root), 6 in norm and weight, 3 in the rotation
    want, mag = P.turned64(x64[0][:R], qn, 1e-6, cs, inter, n_rot)
    assert ((got[:R].double() - want).abs() <= lost * mag).all()
    assert torch.equal(wide[R:], old_tail) if in_place else (out[R:] == 7).all()
    pg, at = (torch.tensor(x, device="cuda", dtype=torch.long) for x in zip(*[st.slot(s, n - t + i) for s, (t, n) in enumerate(zip(rows, lens)) for i in range(t)]))
    ko, vo = (torch.full((R + tail, n_kv, D), 9.0, device="cuda", dtype=torch.float16) for _ in range(2))
    K_.kv_read(st.pool, *st.batch, k_out=ko, v_out=vo)
    if kind != "i4":
        return st
    for pool, scale, back, x, w, turn in ((st.pool.k, st.pool.k_scale, ko, x64[1], kn, True), (st.pool.v, st.pool.v_scale, vo, x64[2], None, False)):
        want, mag = P.turned64(x[:R], w, 1e-6, cs, inter, n_rot) if turn else (x[:R], torch.zeros_like(x[:R]))
        codes, groups = (p[pg, :, at] for p in parts(pool, page, D))
        value = held(want, lost * mag, codes, groups, scale[pg, :, at])
        assert ((back[:R].double() - value).abs() <= value.abs() * (2.0 ** -11 + 2 * U32) + 2.0 ** -25).all() and (back[R:] == 9).all()
    old = before   # nothing else was written
    for o, now in zip(old, pools()):
        if o.dtype == torch.uint8:
            for a, b in zip(parts(o, page, D), parts(now, page, D)):
                a[pg, :, at] = b[pg, :, at]
        else:
            o[pg, :, at] = now[pg, :, at]
        assert torch.equal(o, now)
    return st


SHAPES = [(256, 24, 4, 64, 64, False, True), (128, 5, 5, 16, 128, True, False), (64, 8, 1, 32, 64, False, False), (256, 2, 2, 128, 6, True, True), (128, 12, 2, 1024, 2, False, True), (256, 3, 1, 16, 256, False, False),
          (64, 2, 2, 16, 20, False, True), (128, 3, 1, 32, 44, True, True)]


@pytest.mark.parametrize("D,H,n_kv,page,n_rot,inter,norm", SHAPES + [(64, 1, 1, 16, 0, False, True)])
def test_append(D, H, n_kv, page, n_rot, inter, norm):
    check_append([1, 3, 0, 8, 17], [1, 40, 5, 8, 133], H, n_kv, D, page, n_rot, inter, norm, tail=3)


@pytest.mark.parametrize("D,H,n_kv,page,n_rot,inter,norm", SHAPES)
@pytest.mark.parametrize("n_axes", [1, 3, 4])
def test_append_with_axes(D, H, n_kv, page, n_rot, inter, norm, n_axes):
    axes = [(i * i + i // 3) % n_axes for i in range(n_rot // 2)]
    axes[-1] = n_axes - 1
    check_append([1, 3, 0, 8, 17], [1, 40, 5, 8, 133], H, n_kv, D, page, n_rot, inter, norm, axes=axes, tail=3)


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_axes_in_eight_bits_and_positions_that_are_places(kind):
    """Positions that are the rows' places give the pages and queries of the call without positions, bit for bit."""
    rows, lens = [2, 9], [31, 9]
    place = torch.tensor([29, 30, *range(9)], dtype=torch.int32, device="cuda")
    rope = K_.rope_table(40, 64, 1e4)
    for k in (kind, "i4"):
        a, b, c = (Setup(rows, lens, 2, 128, 16) if k == "i4" else P.Setup(rows, lens, 2, 128, 16, k) for _ in range(3))
        x = torch.randn((11, 6, 128), generator=gen(1), device="cuda")
        for inter in (False, True):
            qs = [K_.kv_append(st.pool, x[:, 2:4], x[:, 4:], *st.batch, rope, q=x[:, :2], interleaved=inter, **kw)
                  for st, kw in ((a, {}), (b, dict(positions=place)), (c, dict(positions=place.expand(3, -1).contiguous(), axes=[i % 3 for i in range(32)])))]
            for st, q in zip((b, c), qs[1:]):
                assert torch.equal(q, qs[0]) and all(torch.equal(getattr(st.pool, n).view(torch.uint8), getattr(a.pool, n).view(torch.uint8)) for n in ("k", "v", "k_scale", "v_scale"))
    check_append([1, 5], [3, 40], 4, 2, 128, 16, 64, False, True, axes=[i % 3 for i in range(32)], kind=kind)


def test_append_in_place_one_row_and_many():
    check_append([1], [1], 4, 2, 128, 16, 32, False, True, in_place=True)
    check_append([2, 5], [70, 9], 4, 2, 256, 32, 64, True, True, in_place=True, tail=2)
    check_append([301], [400], 6, 1, 256, 64, 64, False, True)
    check_append([1] * 100, list(range(1, 101)), 3, 1, 64, 16, 64, False, False)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_append_special_values(D):
    st = Setup([10], [10], 1, D, 16)
    x = torch.randn((10, 1, D), generator=gen(3), device="cuda")
    x[1] = 0
    x[2, 0, 5], x[3, 0, D - 1] = math.nan, -math.inf
    x[4, 0, 0], x[4, 0, 1] = 3e38, -3e38        # a span beyond the largest number
    x[5] = 1e-44                                # a scale that is zero in 32 bits
    x[6] = x[6].abs() + 1                       # zero is the lowest code
    x[7] = -x[7].abs() - 1                      # and the highest
    x[8, 0, 32:] = 0                            # groups of nothing but zeros
    x[9] = 0
    x[9, 0, 33] = -2.5                          # one element, held exactly
    K_.kv_append(st.pool, x, x, *st.batch)
    k, v = K_.kv_read(st.pool, *st.batch, R=10)
    assert status() == 0 and torch.equal(k.view(torch.int16), v.view(torch.int16))
    assert torch.isnan(k[2:4]).all() and torch.isfinite(k[[0, 1, 5, 6, 7, 8, 9]]).all() and (k[[1, 5]] == 0).all() and (k[8, 0, 32:] == 0).all()
    assert abs(float(k[9, 0, 33]) + 2.5) <= 2.5 * 2.0 ** -11 and (k[9, 0, :33] == 0).all() and (k[9, 0, 34:] == 0).all()
    pg, at = st.slot(0, 4)
    codes, groups = (p[pg, 0, at] for p in parts(st.pool.k, 16, D))
    big = whole(codes, groups) * float(st.pool.k_scale[pg, 0, at])
    assert abs(float(st.pool.k_scale[pg, 0, at]) * 225 / 6e38 - 1) < 1e-6 and abs(float(big[0]) / 3e38 - 1) <= 1 / 14 and abs(float(big[1]) / -3e38 - 1) <= 1 / 14 and (big[2:] == 0).all()
    for r in (6, 7):
        assert ((k[r].double() - x[r].double()).abs() <= x[r].abs().amax().double() / 15 / 2 * 1.001 + x[r].abs().double() * 2.0 ** -11).all()


def test_appending_again_leaves_no_trace():
    a, b = Setup([4], [20], 2, 128, 16), Setup([4], [20], 2, 128, 16)
    x, wild = (torch.randn((4, 2, 128), generator=gen(s), device="cuda") for s in (1, 2))
    K_.kv_append(a.pool, torch.cat([x[:1], 1e3 * wild[1:]]), torch.cat([x[:1], 1e3 * wild[1:]]), *a.batch)
    K_.kv_append(a.pool, x, x, *a.batch)
    K_.kv_append(b.pool, x, x, *b.batch)
    assert all(torch.equal(getattr(a.pool, n), getattr(b.pool, n)) for n in ("k", "v", "k_scale", "v_scale"))


def test_indexes_that_do_not_fit():
    """Bad pages, lengths and positions are left out and told; their neighbours are served. The kernels check every index before they use it."""
    st = Setup([2, 2, 2], [20, 20, 20], 1, 64, 16)
    x = torch.randn((6, 1, 64), generator=gen(1), device="cuda")
    rope = K_.rope_table(20, 64, 1e4)
    good = st.table.clone()
    want = K_.kv_append(st.pool, x, x, *st.batch, rope, q=x)
    full = K_.attn_paged(x, st.pool, *st.batch, max_rows=2, max_kv=20)[0]
    assert status() == 0
    for bad in (-1, st.pool.n_pages, 1 << 30):
        st.table[1, 1] = bad
        before = [t.clone() for t in (st.pool.k, st.pool.k_scale)]
        K_.kv_append(st.pool, x, x, *st.batch, rope)
        assert status() == 1 and status() == 0 and all(torch.equal(a, b) for a, b in zip(before, (st.pool.k, st.pool.k_scale)))   # the others as they were appended before
        back = torch.full((6, 1, 64), 5.0, device="cuda", dtype=torch.float16)
        K_.kv_read(st.pool, *st.batch, k_out=back, v_out=back.clone())
        assert status() == 1 and (back[2:4] == 5).all() and (back[[0, 1, 4, 5]] != 5).any(-1).all()
        for mr in (2, 20):
            out, _ = K_.attn_paged(x, st.pool, *st.batch, max_rows=mr if mr == 2 else 17, max_kv=20)
            assert status() == 1 and (mr == 20 or torch.equal(out[[0, 1, 4, 5]], full[[0, 1, 4, 5]]))
        st.table.copy_(good)
    pos = torch.arange(6, dtype=torch.int32, device="cuda").repeat(3, 1)
    axes = [i % 3 for i in range(32)]
    want = K_.kv_append(st.pool, x, x, *st.batch, rope, q=x, positions=pos, axes=axes)
    for a, value in ((0, -1), (1, 20), (2, 2 ** 31 - 1), (2, -2 ** 31)):
        p = pos.clone()
        p[a, 3] = value
        before = st.pool.k.clone()
        out = torch.full((6, 1, 64), 5.0, device="cuda")
        K_.kv_append(st.pool, x, x, *st.batch, rope, q=x, q_out=out, positions=p, axes=axes)
        assert status() == 1 and (out[3] == 5).all() and torch.equal(out[[0, 1, 2, 4, 5]], want[[0, 1, 2, 4, 5]]) and torch.equal(st.pool.k, before)
        q, k, v = K_.rope_rows(x, x, x, rope, p, axes, dtype=torch.float32)
        assert status() == 1 and torch.equal(q[[0, 1, 2, 4, 5]], want[[0, 1, 2, 4, 5]])


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows,lens", [([1], [1]), ([1, 1, 1], [64, 65, 63]), ([3, 1, 0, 8], [700, 257, 9, 8]), ([8, 2], [256, 1025]), ([16, 5], [16, 333])])
def test_attention_shapes(D, rows, lens):
    check_attn(rows, lens, 12, 2, D, 16, gate=True)


@pytest.mark.parametrize("H,n_kv", [(1, 1), (5, 5), (17, 1), (24, 4), (70, 2), (128, 1)])
def test_attention_heads(H, n_kv):
    check_attn([2, 1, 7], [300, 31, 90], H, n_kv, 64, 32)
    check_attn([1, 6], [300, 90], H, n_kv, 256, 32)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_pages(page, D):
    check_attn([1, 4], [555, 130], 6, 2, D, page)
    check_attn([1, 20], [555, 130], 6, 2, D, page)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (5, 4), (64, 0), (100, 300), (257, 1), (1000, 4), (5000, 0)])
def test_attention_window(D, window, n_sink):
    check_attn([1, 8, 3, 2], [1500, 620, 3, 513], 6, 2, D, 16, window=window, n_sink=n_sink)


@pytest.mark.parametrize("D,H,n_kv", [(256, 24, 4), (128, 7, 1), (64, 4, 4)])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (50, 3), (129, 300)])
def test_attention_prompts(D, H, n_kv, window, n_sink):
    check_attn([33, 9, 0, 100], [33, 400, 70, 217], H, n_kv, D, 32, window=window, n_sink=n_sink, gate=True)


def test_attention_long():
    check_attn([1, 2], [20000, 9000], 6, 1, 128, 64)
    check_attn([1], [40000], 2, 2, 64, 256, window=33000, n_sink=600)
    check_attn([17], [3001], 12, 2, 256, 16)
    check_attn([1 + 7 * i % 3 for i in range(75)], [40 + (37 * i) % 300 for i in range(75)], 6, 2, 64, 16)


@pytest.mark.parametrize("rows", [[2, 1], [20, 3]])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_no_row_sees_does_not_count(D, rows):
    """Codes, groups and scales of slots that are unused, masked or foreign: any bytes, NaN and infinite scales."""
    lens = [300, 201]
    st = Setup(rows, lens, 2, D, 16, seed=4)
    q = torch.randn((sum(rows), 4, D), generator=gen(1), device="cuda")
    run = lambda: K_.attn_paged(q, st.pool, *st.batch, max_rows=max(rows), max_kv=300)[0]  # noqa: E731
    want = run()
    seen = torch.zeros(st.pool.k_scale.shape, dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        for pos in range(n):
            pg, at = st.slot(s, pos)
            seen[pg, :, at] = True
    for pool, scale, bad in ((st.pool.k, st.pool.k_scale, math.nan), (st.pool.v, st.pool.v_scale, math.inf)):
        scale[~seen] = bad
        for p in parts(pool, 16, D):
            p[~seen] = 255
    assert torch.equal(run(), want) and torch.isfinite(want).all() and status() == 0


@pytest.mark.parametrize("rows", [4, 40])
def test_non_finite_tokens_reach_the_rows_that_see_them(rows):
    st = Setup([rows], [100], 1, 128, 16)
    q = torch.randn((rows, 2, 128), generator=gen(1), device="cuda")
    run = lambda: K_.attn_paged(q, st.pool, *st.batch, max_rows=rows, max_kv=100)[0]  # noqa: E731
    clean = run()
    for scale, bad in ((st.pool.k_scale, math.nan), (st.pool.v_scale, math.nan), (st.pool.v_scale, math.inf)):
        pg, at = st.slot(0, 98)   # seen by the last two rows
        old = scale.clone()
        scale[pg, 0, at] = bad
        got = run()
        assert torch.equal(got[:-2], clean[:-2]) and torch.isnan(got[-2:]).all()
        scale.copy_(old)


@pytest.mark.parametrize("k_up,v_up", [(1e-12, 1e-12), (1e10, 1e15), (1.0, 1e-25), (1e-30, 1.0)])
@pytest.mark.parametrize("rows", [[2, 1], [40, 1]])
def test_magnitudes(rows, k_up, v_up):
    st = Setup(rows, [150, 40], 2, 64, 16)
    st.pool.k_scale.mul_(k_up)
    st.pool.v_scale.mul_(v_up * torch.exp(3 * torch.randn(st.pool.v_scale.shape, generator=gen(8), device="cuda")))
    st.pool.v_scale[:, :, 3] = 0
    q = torch.randn((sum(rows), 4, 64), generator=gen(5), device="cuda") / k_up
    got, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=max(rows), max_kv=150)
    want, tol = P.attn64(st, q, 0.125, 0, 0, None)
    assert status() == 0 and ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("D,G,window,n_sink", [(256, 6, 0, 0), (128, 12, 0, 0), (64, 5, 300, 4), (256, 12, 100, 1)])
def test_a_rows_bits_depend_on_nothing_else(D, G, window, n_sink):
    rows, lens, H = [16, 1, 5, 8], [1300, 600, 271, 1025], 2 * G
    st, q, got = check_attn(rows, lens, H, 2, D, 32, window=window, n_sink=n_sink)
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    r = 0
    for s, (t, n) in enumerate(zip(rows, lens)):
        for i in range(t):
            alone, _ = K_.attn_paged(q[r:r + 1], st.pool, st.table[s:s + 1], one, torch.tensor([n - t + i + 1], dtype=torch.int32, device="cuda"), max_rows=1, max_kv=n, window=window, n_sink=n_sink)
            assert torch.equal(alone[0], got[r]), (s, i)
            r += 1


def test_rows_without_a_key_and_rows_behind_the_last():
    st = Setup([3, 1, 2], [1, 0, 40], 1, 64, 16, cols=3)
    q = torch.randn((20, 4, 64), generator=gen(2), device="cuda")
    for mr in (3, 17):
        ws = torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda")
        out = torch.full((20, 4, 64), 3.0, device="cuda")
        v, z = ctypes.c_void_p, ctypes.c_longlong
        hb.check(hb.lib().hp_attn_paged(hb.ptr(q), z(256), z(64), None, z(0), z(0), 4, hb.ptr(st.table), 3, hb.ptr(st.row_start), hb.ptr(st.kv_len), 3, 20, mr, 40, v(st.pool._at), ctypes.c_float(0.125), 0, 0,
                                        hb.ptr(out), None, None, hb.ptr(ws), K_._stream()))
        assert status() == 0
        want, tol = P.attn64(st, q[:6], 0.125, 0, 0, None)
        assert (out[:2] == 0).all() and (out[3] == 0).all() and ((out[:6].double() - want).abs() <= tol).all() and (out[6:] == 3).all()


def test_offsets_beyond_32_bits():
    """A pool of 5.4 GB per tensor, used at both ends."""
    page, n_kv, D, n_pages = 1024, 8, 256, 4800
    k, v = (torch.empty((n_pages, n_kv, page * 136), dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty((n_pages, n_kv, page), device="cuda") for _ in range(2))
    small = Setup([3], [1500], n_kv, D, page)
    pool = K_.KVPages(k, v, ks, vs)
    table = torch.tensor([[n_pages - 1, 0]], dtype=torch.int32, device="cuda")
    for a, b in zip((k, v, ks, vs), (small.pool.k, small.pool.v, small.pool.k_scale, small.pool.v_scale)):
        for c in range(2):
            a[int(table[0, c])] = b[int(small.table[0, c])]
    x = torch.randn((3, 8, D), generator=gen(1), device="cuda")
    for p, t in ((pool, table), (small.pool, small.table)):
        K_.kv_append(p, x, 2 * x, t, small.row_start, small.kv_len)
    for rows in (3, 17):
        got, want = (K_.attn_paged(x, p, t, small.row_start, small.kv_len, max_rows=rows, max_kv=1500)[0] for p, t in ((pool, table), (small.pool, small.table)))
        assert torch.equal(got, want)
    rs, ln = torch.tensor([0, 1500], dtype=torch.int32, device="cuda"), torch.tensor([1500], dtype=torch.int32, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(K_.kv_read(pool, table, rs, ln, R=1500), K_.kv_read(small.pool, small.table, rs, ln, R=1500)))
    assert status() == 0


def test_read_of_many_rows():
    for lens, n_kv, D in (([3000, 2500], 1, 64), ([5000], 2, 256), ([100] * 60, 1, 128)):   # both block sizes
        st = Setup(lens, lens, n_kv, D, 32)
        k, v = K_.kv_read(st.pool, *st.batch, R=st.R)
        for got, n in ((k, "k"), (v, "v")):
            want = torch.cat([st.tokens(s, n).transpose(0, 1) for s in range(len(lens))])
            assert ((got.double() - want).abs() <= want.abs() * (2.0 ** -11 + U32) + 2.0 ** -25).all()
    assert status() == 0


def test_captured_steps_replay_with_other_lengths_and_positions():
    st = Setup([1, 1], [90, 40], 2, 128, 16, cols=7, spare=8)
    for s in range(2):
        for c in range(7):
            if st.table[s, c] < 0:
                st.table[s, c] = st.spare.pop()
    rope, axes = K_.rope_table(512, 128, 1e4), K_.rope_axes((24, 20, 20), interleaved=True)
    pos = positions(3, 2, 500)
    x = torch.randn((2, 8, 128), generator=gen(1), device="cuda")

    def step():
        q = K_.kv_append(st.pool, x[:, 4:6], x[:, 6:8], *st.batch, rope, q=x[:, :4], positions=pos, axes=axes)
        return K_.attn_paged(q, st.pool, *st.batch, max_rows=1, max_kv=112)[0]

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = step()
        graphs.append((g, y))
    for i in range(6):
        st.kv_len += 1
        pos += 2
        x.normal_(generator=gen(10 + i))
        g, y = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, step())
    assert status() == 0


def test_tables_that_are_part_of_wider_ones():
    st = Setup([2, 1], [100, 60], 2, 128, 16)
    q = torch.randn((3, 4, 128), generator=gen(1), device="cuda")
    wide = torch.full((2, 40), 1 << 29, dtype=torch.int32, device="cuda")
    wide[:, 5:12] = st.table
    for mr in (2, 17):
        got, want = (K_.attn_paged(q, st.pool, t, st.row_start, st.kv_len, max_rows=mr, max_kv=100)[0] for t in (wide[:, 5:12], st.table))
        assert torch.equal(got, want) and status() == 0


def test_both_forms_of_the_calls(form):
    st = Setup([3, 0, 18], [50, 7, 200], 2, 128, 16)
    x = torch.randn((23, 8, 128), generator=gen(2), device="cuda")   # two rows behind the last
    rope, pos, axes = K_.rope_table(300, 64, 1e4), positions(3, 23, 300), K_.rope_axes((12, 10, 10))
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    kw = dict(interleaved=True, q_norm=w, k_norm=w, positions=pos)
    into = torch.zeros((23, 4, 128), device="cuda")
    q = K_.kv_append(st.pool, x[:, 4:6], x[:, 6:], *st.batch, rope, q=x[:, :4], q_out=into, axes=axes, **kw)
    assert torch.equal(K_.kv_append(st.pool, x[:, 4:6], x[:, 6:], *st.batch, rope, q=x[:, :4], axes=list(axes), **kw)[:21], q[:21])
    assert K_.kv_append(st.pool, x[:, 4:6], x[:, 6:], *st.batch, rope, axes=tuple(axes), k_norm=w, interleaved=True, positions=pos) is None
    k, v = K_.kv_read(st.pool, *st.batch, R=21)
    a, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=18, max_kv=200, window=60, n_sink=2, gate=x[:, :4])
    rows = K_.rope_rows(x[:, :4], x[:, 4:6], x[:, 6:], rope, pos, axes, interleaved=True, q_norm=w, k_norm=w, dtype=torch.bfloat16)
    assert status() == 0
    have = torch.cat([t.float().flatten() for t in (q[:21], k, v, a[:21], *rows)])
    if form == "native":
        test_both_forms_of_the_calls.seen = have
    else:
        assert torch.equal(have, test_both_forms_of_the_calls.seen)


def test_refusals_of_the_python_calls(form):
    st = Setup([2], [20], 2, 64, 16)
    x = torch.randn((2, 4, 64), device="cuda")
    kv, rope, b = x[:, :2], K_.rope_table(32, 64, 1e4), st.batch
    pos = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    axes = [i % 3 for i in range(32)]
    app = lambda **kw: K_.kv_append(st.pool, kv, kv, *b, **{**dict(rope=rope, positions=pos, axes=axes), **kw})  # noqa: E731
    row = lambda **kw: K_.rope_rows(x, **{**dict(rope=rope, positions=pos, axes=axes), **kw})  # noqa: E731
    app()
    row()
    bad = []
    for f in (app, row):
        bad += [lambda f=f, kw=kw: f(**kw) for kw in (dict(positions=pos.long()), dict(positions=pos.cpu()), dict(positions=pos[:, :1]), dict(positions=pos.T.contiguous().T), dict(axes=None), dict(axes=axes[:-1]), dict(axes=axes[:-1] + [3]),
                                                      dict(axes=axes[:-1] + [-1]), dict(axes=axes[:-1] + [0.5]), dict(rope=None), dict(positions=None), dict(rope=rope.half()), dict(rope=rope[:, :, :1]), dict(positions=torch.zeros((5, 2), dtype=torch.int32, device="cuda")),
                                                      dict(rope=K_.rope_table(32, 128, 1e4), axes=axes + axes), dict(positions=None, rope=None))]
    bad += [lambda: row(dtype=torch.float64), lambda: K_.rope_rows(), lambda: K_.rope_rows(x.half()), lambda: K_.rope_rows(x[0]), lambda: K_.rope_rows(x, k=x[:1]), lambda: K_.rope_rows(x, k=x[:, :2], v=x[:, :1]), lambda: K_.rope_rows(x[..., :32]),
            lambda: K_.rope_rows(x, k=x.cpu()), lambda: K_.rope_rows(x, q_norm=x[0, 0]), lambda: K_.rope_rows(x.transpose(1, 2).contiguous().transpose(1, 2)), lambda: K_.rope_rows(x[..., 1:], None, None),
            lambda: K_.rope_rows(torch.zeros((2, 4, 65), device="cuda")[..., 1:])]
    bad += [lambda f=f, kw=kw: f(**kw) for f in (app, row) for kw in (dict(positions=pos[None]), dict(positions=pos[0, 0]), dict(rope=rope[0]), dict(rope=rope[None]))]
    for i, f in enumerate(bad):
        with pytest.raises(hb.HipsterError):
            f()
            pytest.fail(f"call {i} was not refused")
    assert status() == 0


# ------------------------------------------------------------------ rows that stay rows
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,H,n_kv,page,n_rot,inter,norm", SHAPES)
def test_rope_rows(dtype, D, H, n_kv, page, n_rot, inter, norm):
    g = gen(D + H)
    for R, n_axes in ((1, 3), (7, 4), (1100, 2)):
        wide = torch.randn((R, H + 2 * n_kv, D + 4), generator=g, device="cuda")[..., :D]
        q, k, v = wide[:, :H], wide[:, H:H + n_kv], wide[:, H + n_kv:]
        qn, kn = ((1 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16() if norm else None for _ in range(2))
        axes = [(i // 2) % n_axes for i in range(n_rot // 2)]
        pos, rope = positions(n_axes, R, 90, R), K_.rope_table(90, n_rot, 1e4)
        out = K_.rope_rows(q, k, v, rope, pos, axes, interleaved=inter, q_norm=qn, k_norm=kn, dtype=dtype)
        cs, half = angles64(rope, pos, axes), torch.finfo(dtype).eps / 2
        for got, x, w, turn in ((out[0], q, qn, True), (out[1], k, kn, True), (out[2], v, None, False)):
            want, mag = P.turned64(x.double(), w, 1e-6, cs, inter, n_rot) if turn else (x.double(), 0 * x.double())
            assert got.dtype == dtype and got.is_contiguous() and ((got.double() - want).abs() <= half * want.abs() * 1.001 + 16 * U32 * mag + (2.0 ** -25 if dtype == torch.float16 else 0)).all()
        assert status() == 0
        only = K_.rope_rows(None, k, None, rope, pos, axes, interleaved=inter, k_norm=kn, dtype=dtype)
        assert only[0] is None and only[2] is None and torch.equal(only[1], out[1])
        plain = K_.rope_rows(q, None, v, dtype=dtype)
        assert torch.equal(plain[0], q.to(dtype)) and torch.equal(plain[2], v.to(dtype))


def test_rope_rows_into_views_and_in_place():
    """The library's call with outputs side by side, rows in heads, and f32 rows in their own place; what lies between is left alone."""
    R, H, n_kv, D = 5, 3, 1, 64
    x = torch.randn((R, H + 2 * n_kv, D), generator=gen(1), device="cuda")
    rope, pos, axes = K_.rope_table(50, 64, 1e4), positions(2, R, 50), bytes(i % 2 for i in range(32))
    want = K_.rope_rows(x[:, :3], x[:, 3:4], x[:, 4:], rope, pos, axes, dtype=torch.float16)
    out = torch.full((H + 2 * n_kv, R + 2, D + 8), 3.0, device="cuda", dtype=torch.float16)
    t = lambda a: (a.data_ptr(), a.stride(0), a.stride(1))  # noqa: E731
    o = [out[i:j, :R, :D].transpose(0, 1) for i, j in ((0, 3), (3, 4), (4, 5))]
    call = lambda ins, outs, kind: hb.check(_lib.more().hp_rope_rows(*t(ins[0]), *t(outs[0]), H, *t(ins[1]), *t(outs[1]), *t(ins[2]), *t(outs[2]), n_kv, D, kind, None, None, rope.data_ptr(), 50, 64, 0, pos.data_ptr(), R, axes, 2, R, 1e-6,  # noqa: E731
                                                                     torch.cuda.current_stream().cuda_stream))
    call((x[:, :3], x[:, 3:4], x[:, 4:]), o, 1)
    assert all(torch.equal(a, b) for a, b in zip(o, want)) and (out[:, R:] == 3).all() and (out[:, :, D:] == 3).all()
    y = x.clone()
    f32 = K_.rope_rows(x[:, :3], x[:, 3:4], x[:, 4:], rope, pos, axes, dtype=torch.float32)
    call((y[:, :3], y[:, 3:4], y[:, 4:]), (y[:, :3], y[:, 3:4], y[:, 4:]), 0)
    assert torch.equal(y, torch.cat(f32, 1)) and status() == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("mr", [2, 16, 17, 40])
@pytest.mark.parametrize("kind", ["i4", "i8", "e4m3"])
def test_sequences_beside_one_with_a_bad_page_are_served(D, mr, kind):
    """The same bits as without the bad page, in decode steps and in prompts (more than 16 rows)."""
    n = min(mr, 20)
    st = Setup([n, n, n], [100, 300, 50], 2, D, 16) if kind == "i4" else P.Setup([n, n, n], [100, 300, 50], 2, D, 16, kind)
    x = torch.randn((3 * n, 4, D), generator=gen(1), device="cuda")
    run = lambda: K_.attn_paged(x, st.pool, *st.batch, max_rows=mr, max_kv=300)[0]  # noqa: E731
    want = run()
    assert status() == 0
    keep = [*range(n), *range(2 * n, 3 * n)]
    for column, bad in ((0, -1), (7, st.pool.n_pages), (18, 1 << 30), (3, -2 ** 31)):
        old = int(st.table[1, column])
        st.table[1, column] = bad
        got = run()
        assert status() == 1 and torch.equal(got[keep], want[keep])
        st.table[1, column] = old
    assert torch.equal(run(), want) and status() == 0
