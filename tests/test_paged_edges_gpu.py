"""Edges of the paged 8-bit cache on the GPU: entries that do not fit, extreme scales, tables that are views, bits that must not move."""
import ctypes
import math

import pytest
import torch

import hipster_b200 as hb
from hipster_b200 import _lib, kernels as K_
from test_paged_gpu import Setup, attn64, gen, status

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.fixture(params=["native", "python"])
def form(request, monkeypatch):
    """The calls in C++ where they were built, and without them."""
    if request.param == "python":
        monkeypatch.setattr(_lib, "_tensor_calls", False)
    elif _lib.tensors() is None:
        pytest.skip("the calls on torch tensors were not built")
    return request.param


@pytest.mark.parametrize("rows", [2, 20])
@pytest.mark.parametrize("max_kv", [2 ** 31 - 1, 2 ** 31 - 1023, 4096])
def test_bounds_beyond_every_sequence(form, rows, max_kv):
    """max_kv as a caller without a bound gives it: the same values as with the true one."""
    st = Setup([rows], [700], 2, 64, 16, "i8")
    q = torch.randn((rows, 4, 64), generator=gen(1), device="cuda")
    want, tol = attn64(st, q, 0.125, 0, 0, None)
    for q8 in (False, True):
        got, xq = K_.attn_paged(q, st.pool, *st.batch, max_rows=rows, max_kv=max_kv, want_q8=q8)
        assert status() == 0 and ((got.double() - want).abs() <= tol).all()
        if q8:
            assert all(torch.equal(a, b) for a, b in zip(xq.unpack(), K_.quantize_x_q8(got.view(rows, -1)).unpack()))


@pytest.mark.parametrize("a,b", [(0, 3), (2, 5), (5, 8)])
def test_tables_that_are_part_of_wider_ones(form, a, b):
    """table[:, a:b]: the same bits as with a table of its own; lengths beyond its columns are told, and the neighbouring columns' pages neither written nor read."""
    page, D = 16, 64
    st = Setup([2, 2], [20, 40], 1, D, page, "i8", cols=3, spare=12)
    foreign = torch.tensor(st.spare[:12], dtype=torch.int32, device="cuda")
    wide = foreign[torch.arange(16, device="cuda") % 12].view(2, 8).contiguous()
    wide[:, a:b] = st.table
    view = wide[:, a:b]
    x = torch.randn((4, 2, D), generator=gen(1), device="cuda")
    k = x[:, :1]
    pool = lambda: [t.view(torch.uint8).clone() if t.dtype != torch.float32 else t.clone() for t in (st.pool.k, st.pool.v, st.pool.k_scale, st.pool.v_scale)]  # noqa: E731
    outs = []
    for t in (st.table, view):
        K_.kv_append(st.pool, k, k, t, st.row_start, st.kv_len)
        outs.append((*K_.kv_read(st.pool, t, st.row_start, st.kv_len, R=4), K_.attn_paged(x, st.pool, t, st.row_start, st.kv_len, max_rows=2, max_kv=100)[0],
                     K_.attn_paged(x, st.pool, t, st.row_start, st.kv_len, max_rows=20, max_kv=100, want_q8=True)[0], *pool()))
        assert status() == 0
    assert all(torch.equal(u, w) for u, w in zip(*outs))
    for n in (49, 60, 128, 129, 2 ** 31 - 1):   # beyond three pages; of each sequence in turn
        for s in (0, 1):
            kl = st.kv_len.clone()
            kl[s] = n
            st.pool.k_scale[foreign.long()] = math.nan   # what reads them shows
            before = pool()
            K_.kv_append(st.pool, k, k, view, st.row_start, kl)
            assert status() == 1
            for old, now in zip(before, pool()):
                assert torch.equal(old[foreign.long()].view(torch.uint8), now[foreign.long()].view(torch.uint8))
            back = K_.kv_read(st.pool, view, st.row_start, kl, R=4)[0]
            assert status() == 1 and torch.isfinite(back[[2, 3] if s == 0 else [0, 1]]).all()
            for mr in (2, 20):
                got = K_.attn_paged(x, st.pool, view, st.row_start, kl, max_rows=mr, max_kv=2 ** 31 - 1)[0]
                assert status() == 1 and torch.isfinite(got[2:] if s == 0 else got).all()   # the first one's third column is -1


@pytest.mark.parametrize("rows", [2, 20])   # both kernels
@pytest.mark.parametrize("first", [-4, -(2 ** 31)])
def test_a_bad_first_row_leaves_the_other_sequences_alone(rows, first):
    """A sequence that begins in front of row 0 owns no row of the others, and takes no block of theirs."""
    st = Setup([rows] * 3, [60] * 3, 1, 64, 16, "i8")
    q = torch.randn((3 * rows, 12, 64), generator=gen(1), device="cuda")
    run = lambda: K_.attn_paged(q, st.pool, *st.batch, max_rows=3 * rows if rows < 4 else 60, max_kv=60)[0]  # noqa: E731
    want = run()
    assert status() == 0
    st.row_start[0] = first
    for _ in range(4):
        got = run()
        assert status() == 1 and torch.equal(got[rows:], want[rows:])


@pytest.mark.parametrize("what,at,value,places", [   # places: position of each row of the second and third sequence, None where it is left out
    ("kv_len", 1, 33, (31, None, 18, 19)), ("kv_len", 1, 34, (None, None, 18, 19)), ("kv_len", 1, 1 << 30, (None, None, 18, 19)), ("kv_len", 1, 2 ** 31 - 1, (None, None, 18, 19)),
    ("kv_len", 1, 1, (None, 0, 18, 19)), ("kv_len", 1, -5, (None, None, 18, 19)), ("kv_len", 1, -(2 ** 31), (None, None, 18, 19)),
    ("row_start", 3, 9, (18, 19, 15, 16)), ("row_start", 3, 2 ** 31 - 1, (18, 19, None, None))])
def test_rows_go_to_their_own_places_or_nowhere(what, at, value, places):
    """Row t of T of a sequence of n tokens has position n - T + t, whatever else does not fit: no kept token is overwritten, and none is read back for another."""
    st = Setup([2, 2, 2], [20, 20, 20], 1, 64, 16, "i8")
    x = torch.randn((6, 1, 64), generator=gen(1), device="cuda")
    getattr(st, what)[at] = value
    before = st.pool.k.clone()
    K_.kv_append(st.pool, x, 2 * x, *st.batch)
    assert status() == 1
    where = {2 + i: st.slot(1 + i // 2, p) for i, p in enumerate(places) if p is not None} | {0: st.slot(0, 18), 1: st.slot(0, 19)}
    changed = {tuple(i) for i in (st.pool.k != before).any(-1).nonzero().tolist()}
    assert changed == {(p, 0, i) for p, i in where.values()}
    got_k, got_v = (torch.full((6, 1, 64), 5.0, device="cuda", dtype=torch.float16) for _ in range(2))
    K_.kv_read(st.pool, *st.batch, k_out=got_k, v_out=got_v)
    assert status() == 1
    for r in range(6):
        if r in where:
            p, i = where[r]
            k, v = ((codes[p, 0, i].float() * scale[p, 0, i]).half() for codes, scale in ((st.pool.k, st.pool.k_scale), (st.pool.v, st.pool.v_scale)))
            assert torch.equal(got_k[r, 0], k) and torch.equal(got_v[r, 0], v) and (k.float() - x[r, 0]).abs().max() <= x[r].abs().max() / 250
        else:
            assert (got_k[r] == 5).all() and (got_v[r] == 5).all()


@pytest.mark.parametrize("rows,n,window", [(2, 250, 0), (2, 600, 0), (1, 3000, 0), (2, 600, 400), (40, 300, 0), (40, 3000, 0), (40, 600, 400)])   # one split, few and many; decode and prompts
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("low,high", [(0.0, 1e15), (1e-25, 1e18), (0.0, 1e30)])
def test_tokens_of_tiny_values_count_beside_huge_ones(D, rows, n, window, low, high):
    """Scales of v as far apart as 32 bits allow: the first tokens' values are nothing beside the others', but their weights are as large."""
    st = Setup([rows], [n], 2, D, 16, "i8")
    up = torch.full(st.pool.v_scale.shape[:1], high, device="cuda")
    up[st.table[0, :min(n // 2, 320) // 16].long()] = low   # whole slices, and where there are several splits a whole one
    st.pool.v_scale.mul_(up[:, None, None])
    q = torch.randn((rows, 4, D), generator=gen(1), device="cuda")
    got, _ = K_.attn_paged(q, st.pool, *st.batch, max_rows=rows, max_kv=n, window=window)
    want, tol = attn64(st, q, D ** -0.5, window, 0, None)
    assert status() == 0 and ((got.double() - want).abs() <= tol).all(), float(((got.double() - want).abs() / tol).max())


def near_the_limit(S, T, seed):
    """S sequences of 200 tokens whose last row has one factor x, such that the logarithm of the key at 64 lies within 4e-6 of the place where the reference of the row's weights, which the key
    at 0 set, moves: 15 above it. The last row's distances from the reference and its logarithms round in different steps there.
    -> q [S][T][64] (the other rows are zeros), pool, table."""
    g, f = torch.Generator(), torch.float32
    g.manual_seed(seed)
    rand = lambda lo, hi: lo + (hi - lo) * torch.rand(S, generator=g, dtype=torch.float64)  # noqa: E731
    x, v = rand(1, 1.9).to(f), torch.exp2(rand(-40, -20)).to(f)
    per = x.double() * 100 * 0.125 * math.log2(math.e)   # logarithm per unit of the key's scale, codes of 100
    z0, lv = rand(10, 40), torch.log2(v.double())
    z1 = torch.ceil(z0 + lv) - 8 + 15 - lv + rand(-4e-6, 4e-6)
    pool = K_.KVPages.empty(S, 1, 256, 64)
    pool.v_scale[:] = v.cuda()[:, None, None]
    pool.k_scale.fill_(1.0)
    pool.k[:, 0, 0, 0] = pool.k[:, 0, 64:200, 0] = 100
    pool.k_scale[:, 0, 0], pool.k_scale[:, 0, 64] = (z0 / per).to(f).cuda(), (z1 / per).to(f).cuda()
    # the tokens behind these alone have values; their distances round in other steps from another reference
    pool.k_scale[:, 0, 65:200] = pool.k_scale[:, 0, 64, None] * (0.3 + 0.25 * torch.rand((S, 135), generator=g)).cuda()
    pool.v[:, 0, 65:200] = torch.randint(-127, 128, (S, 135, 64), generator=g, dtype=torch.int8).cuda()
    q = torch.zeros((S, T, 64), device="cuda")
    q[:, -1, 0] = x.cuda()
    return q, pool, torch.arange(S, dtype=torch.int32, device="cuda")[:, None]


def test_a_references_move_hangs_on_its_own_row():
    """Rows whose reference is about to move, alone and beside a head whose reference does move: the same bits."""
    S = 2048
    q, pool, table = near_the_limit(S, 1, 1)
    rs, kl = i32(list(range(S + 1))), i32([200] * S)
    run = lambda q: K_.attn_paged(q, pool, table, rs, kl, max_rows=1, max_kv=200, scale=0.125)[0]  # noqa: E731
    both, alone = run(torch.cat([q, 10 * q], 1)), run(q)
    assert status() == 0 and torch.equal(both[:, :1], alone), int((both[:, :1] != alone).any(-1).sum())


def test_a_references_move_hangs_on_its_own_row_in_prompts():
    """The same in a prompt, beside rows whose references move."""
    S, T = 1024, 24
    q, pool, table = near_the_limit(S, T, 2)
    rs, kl = i32([T * s for s in range(S + 1)]), i32([200] * S)
    run = lambda: K_.attn_paged(q.view(S * T, 1, 64), pool, table, rs, kl, max_rows=T, max_kv=200, scale=0.125)[0].view(S, T, 64)[:, -1]  # noqa: E731
    alone = run()
    q[:, :-1, 0] = 10 * q[:, -1:, 0]
    beside = run()
    assert status() == 0 and torch.equal(beside, alone), int((beside != alone).any(-1).sum())


def test_both_kinds_of_status_are_reported():
    """A wait that gave up and an index that does not fit, before anyone asks: one after the other."""
    st = Setup([1], [20], 1, 64, 16, "i8")
    x = torch.randn((1, 1, 64), generator=gen(1), device="cuda")
    assert status() == 0
    flags = torch.zeros(8, dtype=torch.int32, device="cuda")
    hb.check(_lib.lib().hp_ep_wait_probe(_lib.ptr(flags), 2, 0, ctypes.c_uint(5), K_._stream()))   # a wait for a flag that nothing sets: ends by itself
    st.kv_len[0] = 40
    K_.kv_append(st.pool, x, x, *st.batch)
    assert [status() for _ in range(3)] == [4, 1, 0]


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("D,n,window", [(64, 300, 0), (256, 3000, 0), (128, 700, 500)])
@pytest.mark.parametrize("up", [1e6, 1e7, 1e8, 1e9, 1e12, 1e20, 1e30])
def test_scores_of_any_size(rows, D, n, window, up):
    """Finite scores have finite outputs: those of the largest one alone where it stands out of what 32 bits resolve, and never beyond the values there are."""
    st = Setup([rows] * 3, [n] * 3, 2, D, 16, "i8")
    q = torch.randn((3 * rows, 8, D), generator=gen(1), device="cuda") * up
    got = K_.attn_paged(q, st.pool, *st.batch, max_rows=rows, max_kv=n, window=window)[0].double()
    assert status() == 0
    stands_out = 0
    for s in range(3):
        k, v = st.tokens(s, "k").repeat_interleave(4, 0), st.tokens(s, "v").repeat_interleave(4, 0)
        for t in range(rows):
            pos = n - rows + t
            j = slice(max(0, pos - window + 1) if window else 0, pos + 1)
            x, o = q[s * rows + t].double(), got[s * rows + t]
            z = torch.einsum("hd,hjd->hj", x, k[:, j]) * (D ** -0.5 * math.log2(math.e))
            A = (torch.einsum("hd,hjd->hj", x.abs(), k[:, j].abs()) * (D ** -0.5 * math.log2(math.e))).amax(-1)
            top = z.topk(2, -1)
            # twice a score's error (the tensor pipe's additions, roundings), the steps by which a reference is lowered, and weights that are nothing beside the first
            clear = top.values[:, 0] - top.values[:, 1] > 2 * (D / 16 + 8) * 2.0 ** -23 * A + 8 * 2.0 ** -23 * top.values[:, 0].abs() + 60
            want = v[torch.arange(8, device="cuda"), top.indices[:, 0] + j.start]
            assert ((o - want).abs() <= 1e-5 * want.abs().amax(-1, keepdim=True))[clear].all()
            assert (o.abs() <= v[:, j].abs().amax((1, 2), keepdim=True)[:, 0] * (1 + 1e-5)).all()   # not for NaN
            stands_out += int(clear.sum())
    assert stands_out > 12 * rows


@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("up", [1.0, 1e10, 1e28, 1e32, 1e35])
def test_a_single_key_takes_all_whatever_its_score(rows, up):
    """Rows that see themselves alone, with scores as far below zero as 32 bits go: the value is their own."""
    st = Setup([rows] * 2, [rows + 70] * 2, 2, 64, 16, "e4m3")
    at = torch.arange(70, 70 + rows, device="cuda")
    k, v = (torch.cat([st.tokens(s, w)[:, at].transpose(0, 1) for s in range(2)]) for w in "kv")   # [row][kv head][dim]
    q = (-up * k.repeat_interleave(2, 1)).float()
    got = K_.attn_paged(q, st.pool, *st.batch, max_rows=rows, max_kv=rows + 70, window=1)[0].double()
    want = v.repeat_interleave(2, 1)
    # a weight as two f16 is off by 2^-22 of itself; its product with the scale, the sum, the quotient and the factor of e4m3 are rounded, by 2^-24 each
    assert status() == 0 and ((got - want).abs() <= 8 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True) + 2.0 ** -22 * want.abs()).all()
