"""Causal attention of packed prompts in 16 bits (hp_attn_prompt) on the GPU against a plain implementation in 64 bits, and a run of the prompt's and the cache's calls together."""
import math
import os
import subprocess
import sys

import pytest
import torch

import hipster_b200 as hb
from hipster_b200 import kernels as K_
import test_paged_gpu as P

pytestmark = pytest.mark.gpu

gen, status, form = P.gen, P.status, P.form
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts(rows):
    return i32([sum(rows[:s]) for s in range(len(rows) + 1)])


def prompt64(q, k, v, rows, scale, gate=None):
    """-> values and tolerances of every output, in 64 bits.

    h: half a step of the inputs' type. The output is rounded once (h of it, at most h sum p |v|), each weight once (h of it: together h sum p |v|), below f16's smallest normal to steps of 2^-24, where the largest
    weight is 1 or more, as is their sum (2^-25 sum |v|; bf16 has no such steps). A score is the sum of D products, formed 16 at a time: D / 16 additions and a rounding of each 16, each a step 2^-23 of at most A = scale sum |q k|,
    and the factor's three roundings: ds <= (D / 8 + 4) 2^-23 A, and moves the result by at most 2 ds sum p |v|. Reference, exponential (2^-22) and the sums (keys / 16 steps on the tensor pipe; 2^-24 times 64 + keys / 128 for the
    weights), the rescaling of a row at most once per tile on both sides of the quotient, and 8 for quotient and gate."""
    R, H, D = q.shape
    G = H // k.shape[1]
    h = torch.finfo(q.dtype).eps / 2
    out, tol = (torch.zeros((R, H, D), dtype=torch.float64, device="cuda") for _ in range(2))
    r0 = 0
    for T in filter(None, rows):
        hidden = torch.ones((T, T), dtype=torch.bool, device="cuda").triu(1)
        for i in range(H):
            x, y, z = q[r0:r0 + T, i].double(), k[r0:r0 + T, i // G].double(), v[r0:r0 + T, i // G].double()
            p = torch.softmax((x @ y.T * scale).masked_fill(hidden, -math.inf), -1)
            A = (x.abs() @ y.abs().T * scale).masked_fill(hidden, 0).amax(-1, keepdim=True)
            mag = p @ z.abs()
            n = torch.arange(1, T + 1, device="cuda", dtype=torch.float64)[:, None]
            out[r0:r0 + T, i] = p @ z
            tol[r0:r0 + T, i] = mag * (2 * h + (2 * (D / 8 + 4) * A + n / 16 + 2 * n / 128 + 64 + 16) * 2.0 ** -23) + (2.0 ** -25 * (z.abs().cumsum(0) + 1) if q.dtype == torch.float16 else 0)
        r0 += T
    if gate is not None:
        g = torch.sigmoid(gate.double())
        out, tol = out * g, tol * g
        if q.dtype == torch.float16:
            tol += 2.0 ** -25
    return out, tol


def make(rows, H, n_kv, D, kind, seed=0, tail=0, packed=True, up=1.0):
    R = sum(rows) + tail
    x = torch.randn((R, H + 2 * n_kv, D), generator=gen(seed), device="cuda") * torch.exp(0.5 * torch.randn((R, H + 2 * n_kv, 1), generator=gen(seed + 1), device="cuda"))
    x[:, :H] *= up
    x = x.to(TYPES[kind])
    q, k, v = x.split([H, n_kv, n_kv], 1)
    return (q, k, v) if packed else (q.contiguous(), k.contiguous(), v.contiguous())


def check(rows, H, n_kv, D, kind, gate=False, seed=0, tail=0, packed=True, up=1.0, scale=None, max_rows=None):
    q, k, v = make(rows, H, n_kv, D, kind, seed, tail, packed, up)
    R = sum(rows)
    g = torch.randn((R + tail, H, D + 4), generator=gen(seed + 2), device="cuda")[..., :D] if gate else None
    got, none = K_.attn_prompt(q, k, v, starts(rows), max_rows=max_rows or max(max(rows), 1), gate=g, scale=scale)
    assert status() == 0 and none is None and got.dtype == q.dtype
    want, tol = prompt64(q[:R], k[:R], v[:R], rows, D ** -0.5 if scale is None else scale, None if g is None else g[:R])
    bad = ~((got[:R].double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(((got[:R].double() - want).abs() / tol).max()))
    return q, k, v, got


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [[1], [2], [127], [128], [129], [255, 1, 0, 257], [300, 64, 33], [1] * 40, [700]])
def test_shapes(kind, D, rows):
    check(rows, 6, 2, D, kind, gate=len(rows) == 1)


@pytest.mark.parametrize("H,n_kv", [(1, 1), (5, 5), (17, 1), (24, 4), (32, 8), (70, 2)])
@pytest.mark.parametrize("D", [64, 256])
def test_heads(H, n_kv, D):
    check([140, 3], H, n_kv, D, "bf16")
    check([5], H, n_kv, D, "f16", packed=False)


@pytest.mark.parametrize("D,kind", [(64, "f16"), (128, "bf16"), (256, "f16"), (256, "bf16")])
def test_long_prompts(D, kind):
    check([2500, 1111], 2, 1, D, kind)
    check([5001], 1, 1, D, kind, gate=True, packed=False)


def test_many_prompts_in_any_order():
    rows = [(37 * i) % 300 for i in range(150)]   # more than a warp has lanes; empty ones
    check(rows, 2, 1, 64, "f16")
    check(sorted(rows), 1, 1, 128, "bf16", max_rows=5000)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_references_that_move(D, kind):
    """Scores that grow along the keys, so that the reference of a row moves tile by tile, and large ones: nearly all of the weight on one key."""
    rows, H = [700, 300], 2
    q, k, v = make(rows, H, 1, D, kind, 3, packed=False)
    k *= torch.linspace(0.1, 6, 1000, device="cuda")[:, None, None].to(k.dtype)
    for up in (1.0, 8.0):
        y = q * up
        got, _ = K_.attn_prompt(y, k, v, starts(rows), max_rows=700)
        want, tol = prompt64(y, k, v, rows, D ** -0.5)
        assert ((got.double() - want).abs() <= tol).all() and status() == 0


def test_rows_behind_the_last_and_between_are_left_as_they_were():
    rows, H, D = [130, 0, 5], 3, 64
    q, k, v = make(rows, H, 1, D, "f16", tail=60)
    for extra in (0, 60):
        out = torch.full((195, H, D), 3.0, device="cuda", dtype=torch.float16)
        rs = starts(rows)
        from hipster_b200 import _lib
        hb.check(_lib.more().hp_attn_prompt(q.data_ptr(), *q.stride()[:2], k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2], 1, None, 0, 0, H, 1, D, rs.data_ptr(), 3, 135 + extra, 130, D ** -0.5, out.data_ptr(), None, None,
                                            torch.cuda.current_stream().cuda_stream))
        want, tol = prompt64(q[:135], k[:135], v[:135], rows, D ** -0.5)
        assert status() == 0 and (out[135:] == 3).all() and ((out[:135].double() - want).abs() <= tol).all()


def test_a_prompts_result_depends_on_itself_alone():
    rows = [400, 77, 128, 1]
    q, k, v, got = check(rows, 4, 2, 128, "bf16")
    r = 0
    for t in rows:
        alone, _ = K_.attn_prompt(q[r:r + t], k[r:r + t], v[r:r + t], i32([0, t]), max_rows=t)
        assert torch.equal(alone, got[r:r + t])
        r += t
    head, _ = K_.attn_prompt(q[:200], k[:200], v[:200], i32([0, 200]), max_rows=200)   # causal: the first rows know nothing of the others
    assert torch.equal(head, got[:200])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("at", [0, 1, 127, 128, 200, 383, 391])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(kind, D, at, bad):
    rows, H = [392, 150], 2
    q, k, v = make(rows, H, 1, D, kind, 7, packed=False)
    clean, _ = K_.attn_prompt(q, k, v, starts(rows), max_rows=392)
    v[at, 0, 5] = bad
    v[at, 0, D - 1] = bad
    got, _ = K_.attn_prompt(q, k, v, starts(rows), max_rows=392)
    hit = torch.zeros((542, H, D), dtype=torch.bool, device="cuda")
    hit[at:392, :, [5, D - 1]] = True
    assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit]).any() and status() == 0
    if bad == math.inf:   # the key's own row: its weight is not zero
        assert (got[at, :, 5] == math.inf).all()


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("at", [0, 130, 391])
def test_keys_and_queries_that_are_not_finite(D, at):
    rows, H = [392, 150], 2
    q, k, v = make(rows, H, 1, D, "bf16", 7, packed=False)
    clean, _ = K_.attn_prompt(q, k, v, starts(rows), max_rows=392)
    old = k[at].clone()
    k[at, 0, 3] = math.nan
    got, _ = K_.attn_prompt(q, k, v, starts(rows), max_rows=392)
    assert torch.equal(got[:at], clean[:at]) and torch.isnan(got[at:392]).all() and torch.equal(got[392:], clean[392:])
    k[at] = old
    q[at, 1, 0] = math.inf
    got, _ = K_.attn_prompt(q, k, v, starts(rows), max_rows=392)
    keep = torch.ones((542, H), dtype=torch.bool, device="cuda")
    keep[at, 1] = False
    assert torch.equal(got[keep], clean[keep]) and status() == 0


@pytest.mark.parametrize("kind,up", [("f16", 200.0), ("bf16", 1e12)])
@pytest.mark.parametrize("D", [64, 256])
def test_a_row_with_scores_of_another_size_leaves_its_neighbours_as_they_were(D, kind, up):
    """Queries so large that a row's scores pass 2^26, where the kernel rounds otherwise: rows beside it, and their bits in 32-bit sums, know nothing of it."""
    q, k, v = make([150], 2, 1, D, kind, 8, packed=False)
    k[:, 0, 0] = 300
    clean, xc = K_.attn_prompt(q, k, v, i32([0, 150]), max_rows=150, want_q8=True)
    q[77, 0, 0] = 300 * up
    got, xq = K_.attn_prompt(q, k, v, i32([0, 150]), max_rows=150, want_q8=True)
    keep = [i for i in range(150) if i != 77]
    assert torch.equal(got[keep], clean[keep]) and all(torch.equal(a[keep], b[keep]) for a, b in zip(xq.unpack(), xc.unpack())) and torch.isfinite(got[77]).all() and status() == 0


def test_another_prompts_non_finite_rows_do_not_count():
    """Tiles reach over a prompt's end into the next one's rows, and past the last row of the buffers."""
    rows = [50, 200, 10]
    q, k, v = make(rows, 2, 1, 128, "f16", 5, packed=False)
    clean, _ = K_.attn_prompt(q, k, v, starts(rows), max_rows=200)
    for t in (q, k, v):
        t[50:250] = math.nan
    got, _ = K_.attn_prompt(q, k, v, starts(rows), max_rows=200)
    keep = [*range(50), *range(250, 260)]
    assert torch.equal(got[keep], clean[keep]) and torch.isnan(got[50:250]).all() and status() == 0


@pytest.mark.parametrize("up", [1e15, 1e18])
def test_scores_of_any_size(up):
    """Scores up to 1e36: the largest one takes it all, and outputs are finite."""
    T, D = 300, 64
    q, k, v = make([T], 2, 1, D, "bf16", 9, packed=False)
    q, k = (q.float() * up).bfloat16(), (k.float() * up).bfloat16()
    got, _ = K_.attn_prompt(q, k, v, i32([0, T]), max_rows=T)
    s = torch.einsum("ihd,jd->hij", q.double(), k[:, 0].double()).masked_fill(torch.ones((T, T), dtype=torch.bool, device="cuda").triu(1), -math.inf)
    want = v[:, 0][s.argmax(-1)].permute(1, 0, 2)
    assert status() == 0 and ((got.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs()).all()


def test_no_weight_at_all():
    """Scores that are all minus infinity: zeros, as elsewhere."""
    q, k, v = make([3], 1, 1, 64, "bf16", packed=False)
    q.fill_(1)
    k.fill_(-math.inf)
    got, _ = K_.attn_prompt(q, k, v, i32([0, 3]), max_rows=3)
    assert (got == 0).all() and status() == 0


def test_strides():
    T, H, n_kv, D = 200, 4, 2, 128
    q, k, v = make([T], H, n_kv, D, "f16", packed=False)
    want, _ = K_.attn_prompt(q, k, v, i32([0, T]), max_rows=T)
    heads_first = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    padded = lambda t: torch.nn.functional.pad(t, (0, 8, 0, 1))[:, :-1, :D]  # noqa: E731
    for f in (heads_first, padded):
        got, _ = K_.attn_prompt(f(q), f(k), f(v), i32([0, T]), max_rows=T, gate=None)
        assert torch.equal(got, want)
    one = k[:, :1]
    got, _ = K_.attn_prompt(q[:1], one[:1], v[:1, :1], i32([0, 1]), max_rows=7)
    assert torch.equal(got[:1, 0], v[:1, 0]) and status() == 0


def test_quantised_output_is_the_quantised_output():
    """Rows of the next projection: int8 of the outputs in 32 bits, which lie half a step of f16 from those in 16 bits."""
    rows, H, D = [150, 3], 6, 64
    q, k, v = make(rows, H, 2, D, "f16")
    gate = torch.randn((153, H, D), generator=gen(1), device="cuda")
    out, xq = K_.attn_prompt(q, k, v, starts(rows), max_rows=150, gate=gate, want_q8=True)
    none, only = K_.attn_prompt(q, k, v, starts(rows), max_rows=150, gate=gate, want_out=False, want_q8=True)
    assert none is None and torch.equal(xq.q, only.q) and torch.equal(xq.sc, only.sc)
    c, d, s = xq.unpack()
    x = out.view(153, -1).float()
    amax = x.unflatten(1, (-1, 32)).abs().amax(-1)
    assert ((d * 127 - amax).abs() <= 2.0 ** -10 * amax).all() and torch.equal(s, d * c.float().unflatten(1, (-1, 32)).sum(-1))
    assert ((c.float().unflatten(1, (-1, 32)) * d[..., None] - x.unflatten(1, (-1, 32))).abs() <= (0.5 + 127 * 2.0 ** -10) * d[..., None]).all() and status() == 0


def test_bad_row_starts_are_told():
    q, k, v = make([40], 2, 1, 64, "f16", packed=False)
    want, _ = K_.attn_prompt(q, k, v, i32([0, 30, 40]), max_rows=30)
    assert status() == 0
    for rs, kept in (([0, 30, 41], 40), ([-1, 30, 40], 0), ([0, 30, 1 << 30], 40), ([0, 30, 20], 30), ([0, -5, 40], 0)):
        got, _ = K_.attn_prompt(q, k, v, i32(rs), max_rows=30)
        assert status() == 1, rs
        assert torch.equal(got[:kept], want[:kept])
    K_.attn_prompt(q, k, v, i32([0, 30, 40]), max_rows=29)
    assert status() == 1


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("heads", [1, 6])
def test_gates_of_any_strides(D, heads):
    rows = [130, 0, 33, 1, 257]
    q, k, v = make(rows, heads, 1, D, "bf16", 21, tail=2)
    n = sum(rows) + 2
    wide = torch.randn((heads, n, 3 * D), generator=gen(3), device="cuda")
    got = []
    for gate in (wide[..., D:2 * D].transpose(0, 1), wide[..., D:2 * D].transpose(0, 1).contiguous(), torch.cat([wide[..., D:2 * D].transpose(0, 1), torch.full((n, heads, 8), math.nan, device="cuda")], 2)[..., :D]):
        got.append(K_.attn_prompt(q, k, v, starts(rows), max_rows=257, gate=gate)[0][:n - 2])
    want, tol = prompt64(q[:n - 2], k[:n - 2], v[:n - 2], rows, D ** -0.5, wide[:, :n - 2, D:2 * D].transpose(0, 1))
    assert ((got[0].double() - want).abs() <= tol).all() and torch.equal(got[0], got[1]) and torch.equal(got[0], got[2]) and status() == 0


@pytest.mark.parametrize("D", [64, 256])
def test_gates_at_their_ends(D):
    """Infinite gates and NaN of one row: 0, the ungated result, NaN, and nothing of it in other rows or behind the last."""
    q, k, v = make([140], 2, 1, D, "f16", 5, tail=1)
    plain, _ = K_.attn_prompt(q, k, v, i32([0, 140]), max_rows=140)
    gate = torch.full((141, 2, D), math.inf, device="cuda")
    gate[3], gate[4, 1], gate[140] = -math.inf, math.nan, math.nan
    got, _ = K_.attn_prompt(q, k, v, i32([0, 140]), max_rows=140, gate=gate)
    keep = [i for i in range(140) if i not in (3, 4)]
    assert torch.equal(got[keep], plain[keep]) and (got[3] == 0).all() and torch.equal(got[4, 0], plain[4, 0]) and got[4, 1].isnan().all() and status() == 0


# same lengths (a number for every block), few of very different ones, and many: blocks are counted in three ways
@pytest.mark.parametrize("rows", [[100] * 50, [128] * 33, [130] * 20, [0, 1, 900, 3, 0, 129], [700] + [5] * 40, [5] * 40 + [700], [1, 0, 127, 128, 129, 0, 256, 257] * 9 + [1500], [0] * 100 + [300] + [0] * 100 + [2]])
@pytest.mark.parametrize("D", [64, 256])
def test_blocks_of_many_prompts(rows, D):
    q, k, v = make(rows, 2, 1, D, "f16", 11, tail=3)
    got, _ = K_.attn_prompt(q, k, v, starts(rows), max_rows=max(rows))
    at = 0
    for T in rows:
        if T:
            part = slice(at, at + T)
            assert torch.equal(got[part], K_.attn_prompt(q[part], k[part], v[part], i32([0, T]), max_rows=T)[0]), (at, T)
        at += T
    assert status() == 0


def test_bad_row_starts_among_many_prompts_are_told():
    rows = [5] * 60 + [400]
    q, k, v = make(rows, 2, 1, 64, "f16", packed=False)
    good = starts(rows)
    want, _ = K_.attn_prompt(q, k, v, good, max_rows=400)
    assert status() == 0
    for at, to in ((61, 701), (61, 1 << 30), (0, -1), (30, -5), (30, 1 << 30), (59, 100), (61, 1)):
        rs = good.clone()
        rs[at] = to
        got, _ = K_.attn_prompt(q, k, v, rs, max_rows=400)
        assert status() == 1, (at, to)
        if at == 61 and to > 1:
            assert torch.equal(got, want)
    K_.attn_prompt(q, k, v, good, max_rows=399)
    assert status() == 1
    assert torch.equal(K_.attn_prompt(q, k, v, good, max_rows=400)[0], want) and status() == 0


@pytest.mark.parametrize("D,kind", [(64, "f16"), (128, "bf16"), (256, "bf16")])
@pytest.mark.parametrize("gated", [False, True])
def test_many_calls_in_a_row_have_the_same_bits(D, kind, gated):
    """Some 700 blocks a call, two to an SM where they fit, one call behind the other: products of one block wait for those of another, and no wait may take one tile's products for another's."""
    rows = [1000, 251, 501, 751]
    q, k, v = make(rows, 32, 8, D, kind, 31, packed=False)
    g = torch.randn(q.shape, generator=gen(7), device="cuda") if gated else None
    rs = starts(rows)
    got = [K_.attn_prompt(q, k, v, rs, max_rows=1000, gate=g)[0] for _ in range(40)]
    assert status() == 0
    for t in got[1:]:
        assert torch.equal(t, got[0])
    want, tol = prompt64(q, k, v, rows, D ** -0.5, g)
    assert ((got[0].double() - want).abs() <= tol).all()


def test_streams_and_captures():
    rows = [300, 90]
    q, k, v = make(rows, 4, 2, 256, "f16", packed=False)
    rs = starts(rows)
    run = lambda: K_.attn_prompt(q, k, v, rs, max_rows=300)[0]  # noqa: E731
    want = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for i in range(9):
        with torch.cuda.stream(streams[i % 3]):
            got.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = run()
    for r in ([300, 90], [10, 300], [0, 390], [128, 128]):   # other lengths in a captured call: 390 rows are more than it was told
        rs.copy_(starts(r))
        q.normal_(generator=gen(r[0]))
        g.replay()
        torch.cuda.synchronize()
        n = sum(r)
        if max(r) <= 300:
            assert torch.equal(y[:n], run()[:n]) and status() == 0
        else:
            assert status() == 1


def test_prompts_beside_calls_that_hold_all_accumulator_memory():
    st = P.Setup([150, 40], [1500, 700], 2, 256, 64, "i8")
    x = torch.randn((190, 12, 256), generator=gen(1), device="cuda")
    q, k, v = make([500, 100], 8, 2, 128, "bf16")
    paged = lambda: K_.attn_paged(x, st.pool, *st.batch, max_rows=150, max_kv=1500)[0]  # noqa: E731
    prompt = lambda: K_.attn_prompt(q, k, v, starts([500, 100]), max_rows=500)[0]  # noqa: E731
    want = paged(), prompt()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(4)], []
    for i in range(24):
        with torch.cuda.stream(streams[i % 4]):
            got.append((prompt if i % 3 else paged)())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[1 if i % 3 else 0]) for i, g in enumerate(got)) and status() == 0


def test_the_first_call_of_a_process_may_be_captured():
    code = ("import torch\n"
            "from hipster_b200 import kernels as K\n"
            "x = torch.randn((30, 4, 64), device='cuda')\n"
            "rs = torch.tensor([0, 30], dtype=torch.int32, device='cuda')\n"
            "pos = torch.arange(30, dtype=torch.int32, device='cuda')\n"
            "torch.cuda.synchronize()\n"
            "g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g):\n"
            "    rope = K.rope_table(32, 64, 1e4)\n"
            "    q, k, v = K.rope_rows(x[:, :2], x[:, 2:3], x[:, 3:], rope, pos)\n"
            "    y, _ = K.attn_prompt(q, k, v, rs, max_rows=30)\n"
            "g.replay()\n"
            "torch.cuda.synchronize()\n"
            "K.device_status()\n"
            "z, _ = K.attn_prompt(q, k, v, rs, max_rows=30)\n"
            "assert torch.equal(y, z)\n"
            "print('fine')\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_refusals_of_the_python_call(form):
    q, k, v = make([10], 4, 2, 64, "f16", packed=False)
    rs = i32([0, 10])
    f = lambda q=q, k=k, v=v, rs=rs, max_rows=10, **kw: K_.attn_prompt(q, k, v, rs, max_rows, **kw)  # noqa: E731
    f()
    odd = torch.zeros(10 * 4 * 64 + 8, device="cuda", dtype=torch.float16)[1:2561].view(10, 4, 64)
    bad = [lambda: f(q=q.float(), k=k.float(), v=v.float()), lambda: f(k=k.bfloat16()), lambda: f(q=q[:, :3]), lambda: f(k=k[:9]), lambda: f(v=v[:, :1]), lambda: f(v=v[..., :32]), lambda: f(q=q[0]), lambda: f(q=q.cpu()), lambda: f(rs=rs.long()),
           lambda: f(rs=rs.cpu()), lambda: f(rs=rs[:1]), lambda: f(max_rows=0), lambda: f(max_rows=1 << 40), lambda: f(scale=0.0), lambda: f(scale=math.nan), lambda: f(gate=q), lambda: f(gate=q.float()[:, :2]), lambda: f(want_out=False),
           lambda: f(q=odd), lambda: f(q=q[:1].expand(10, -1, -1)), lambda: f(q=q.transpose(1, 2).contiguous().transpose(1, 2)), lambda: f(q=q[:0], k=k[:0], v=v[:0]), lambda: f(q=q[..., :48], k=k[..., :48], v=v[..., :48])]
    for i, g in enumerate(bad):
        with pytest.raises(hb.HipsterError):
            g()
            pytest.fail(f"call {i} was not refused")
    assert status() == 0


def test_a_chat_about_an_image():
    """A prompt with an image and the steps behind it, as a server runs them: the prompt's rows are rotated by time, height and width, attended at full precision and written to a cache in 4 bits; drafts are appended at
    positions that run on behind the image's, verified over the cache, and partly rejected."""
    H, n_kv, D, page, T, steps = 6, 2, 256, 16, 150, 8
    g = gen(11)
    n = T + 3 * steps
    stream = torch.randn((n, H + 2 * n_kv, D), generator=g, device="cuda")
    gates = torch.randn((n, H, D), generator=g, device="cuda")
    qn, kn = ((1 + 0.1 * torch.randn(D, generator=g, device="cuda")).bfloat16() for _ in range(2))
    rope, axes = K_.rope_table(n, 64, 1e7), K_.rope_axes((11, 11, 10), interleaved=True)
    pos = [[], [], []]   # 20 tokens, an image of 10 x 12 patches, text
    for i in range(n):
        j = i - 20
        for a in range(3):
            pos[a].append(i if j < 0 else 20 + (0, j // 12, j % 12)[a] if j < 120 else 32 + j - 120)
    pos = i32(pos)
    table = i32([[3, 0, 5, 1, 4, 9, 10, 11, 2, 6, 7, 8]])
    pool = K_.KVPages.empty(12, n_kv, page, D, dtype="i4")
    rs, ln = i32([0, T]), i32([T])
    x = stream[:T]
    q, k, v = K_.rope_rows(x[:, :H], x[:, H:H + n_kv], x[:, H + n_kv:], rope, pos[:, :T].contiguous(), axes, q_norm=qn, k_norm=kn)
    out, xq = K_.attn_prompt(q, k, v, rs, max_rows=T, gate=gates[:T], want_q8=True)
    K_.kv_append(pool, x[:, H:H + n_kv], x[:, H + n_kv:], table, rs, ln, rope, k_norm=kn, positions=pos[:, :T].contiguous(), axes=axes)
    want, tol = prompt64(q, k, v, [T], D ** -0.5, gates[:T])
    assert ((out.double() - want).abs() <= tol).all() and xq.unpack()[0].shape == (T, H * D) and status() == 0
    # the cache holds the keys that the prompt saw, to a step of 4 bits: S u / 2 and a full one at the ends of a group's range, at most 2 |max - min| / 15
    kb, vb = K_.kv_read(pool, table, rs, ln, R=T)
    for a, b in ((kb, k), (vb, v)):
        lo, hi = b.float().unflatten(-1, (-1, 32)).amin(-1).clamp(max=0), b.float().unflatten(-1, (-1, 32)).amax(-1).clamp(min=0)
        step = (hi - lo).amax(-1, keepdim=True) / 15   # the factor of a group at most one too large: a fifteenth of the largest
        assert ((a.float() - b.float()).unflatten(-1, (-1, 32)).abs() <= ((hi - lo) / 15 + step / 15)[..., None] * 1.01 + 0.01).all()

    import test_four_bits_gpu as F
    at = T
    for i in range(steps):   # three rows, of which one to three are kept
        keep = 1 + i % 3
        x = stream[at:at + 3].clone()
        x[keep:] *= 30
        rs, ln = i32([0, 3]), i32([at + 3])
        q = K_.kv_append(pool, x[:, H:H + n_kv], x[:, H + n_kv:], table, rs, ln, rope, q=x[:, :H], q_norm=qn, k_norm=kn, positions=pos[:, at:at + 3].contiguous(), axes=axes)
        got, _ = K_.attn_paged(q, pool, table, rs, ln, max_rows=3, max_kv=n, gate=gates[at:at + 3])
        st = F.Setup.__new__(F.Setup)
        st.rows, st.lens, st.R, st.D, st.page, st.pool, st.table = [3], [at + 3], 3, D, page, pool, table
        want, tol = P.attn64(st, q, 1 / 16, 0, 0, gates[at:at + 3])
        assert ((got.double() - want).abs() <= tol).all() and status() == 0
        at += keep


def hidden_values(kind, D, gated):
    """Infinite and NaN values of later rows, of the next prompt and behind the last one, in some hundred blocks of three to nine tiles whose references do not move (scores are almost alike), while copies of as much memory as there is keep theirs late: the
    last tile's values may be looked at only when they have come. Bits as without such values, in each of 40 calls."""
    rows, H, n_kv = [500, 384, 640, 300, 513], 24, 4
    R = sum(rows)
    q, k, v = make(rows, H, n_kv, D, kind, 41, tail=100, packed=False)
    q *= 0.01
    rs = starts(rows)
    g = torch.randn(q.shape, generator=gen(9), device="cuda") if gated else None
    run = lambda: K_.attn_prompt(q, k, v, rs, max_rows=640, gate=g)[0]  # noqa: E731
    clean = run()[:R]
    keep = torch.ones(R, dtype=torch.bool, device="cuda")
    at = 0
    for i, T in enumerate(rows):   # the last rows of every other prompt, and what lies behind the last prompt's last row: hidden from the rows in front of them
        if i % 2 == 0:
            bad = at + T - 20
            v[bad:at + T:3] = math.nan
            v[bad + 1:at + T:3] = math.inf
            keep[bad:at + T] = False
        at += T
    v[R:] = math.nan
    big = torch.empty((2, 1 << 28), dtype=torch.uint8, device="cuda")
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(40):
        with torch.cuda.stream(other):
            big[0].copy_(big[1])
        got.append(run()[:R])
    torch.cuda.synchronize()
    assert status() == 0
    for y in got:
        assert torch.equal(y[keep], clean[keep]) and not torch.isfinite(y[~keep]).any()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [128, 256])
def test_hidden_values_of_many_blocks_beside_late_copies(kind, D):
    hidden_values(kind, D, False)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("gated", [False, True])
def test_what_rows_have_of_values_that_are_not_finite(kind, D, gated):
    """Of NaN, or of infinities of both signs, NaN; of infinities of one sign these; by dim, in the block of the key's own row and in later ones, with gates and without, and nothing anywhere else. In int8: the run of 32 dims around it alone."""
    rows, H = [300, 70], 4
    q, k, v = make(rows, H, 2, D, kind, 51, packed=False)
    q *= 0.1   # no weight so small that it is zero in 16 bits
    gate = torch.randn(q.shape, generator=gen(3), device="cuda") if gated else None
    run = lambda **kw: K_.attn_prompt(q, k, v, starts(rows), max_rows=300, gate=gate, **kw)  # noqa: E731
    clean, xc = run(want_q8=True)
    inf, nan = math.inf, math.nan
    put = [(10, 0, inf), (200, 0, -inf), (130, 1, nan), (299, 2, inf), (128, 5, inf), (127, 6, -inf), (250, D - 1, -inf), (369, 3, -inf), (300, 4, nan), (300, 5, inf), (301, 5, -inf)]
    want = torch.zeros((370, D), dtype=torch.float64, device="cuda")   # what is added to the finite part
    for row, d, x in put:
        v[row, 1, d] = x
        want[row:300 if row < 300 else 370, d] += x
    got, _ = run()
    both, xq = run(want_q8=True)
    assert status() == 0 and torch.equal(got.view(torch.int16), both.view(torch.int16)) and torch.equal(got[:, :2], clean[:, :2])
    for h in (2, 3):
        y, w = got[:, h].double(), want
        hit = ~torch.isfinite(w)
        assert torch.equal(y[~hit], clean[:, h].double()[~hit])
        assert torch.equal(torch.isnan(y[hit]), torch.isnan(w[hit])) and torch.equal(y[hit].nan_to_num(7.0, posinf=8.0, neginf=9.0), w[hit].nan_to_num(7.0, posinf=8.0, neginf=9.0))
    runs = torch.cat([torch.zeros_like(want), torch.zeros_like(want), want, want], 1).isfinite().unflatten(1, (-1, 32)).all(-1)
    (c, d, s), (c0, d0, s0) = xq.unpack(), xc.unpack()
    assert torch.equal(d[runs], d0[runs]) and torch.equal(s[runs], s0[runs]) and torch.equal(c.unflatten(1, (-1, 32))[runs], c0.unflatten(1, (-1, 32))[runs])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_hidden_values_of_many_gated_blocks_beside_late_copies(kind, D):
    hidden_values(kind, D, True)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("low", [0, 1, 2])
@pytest.mark.parametrize("e", [24, 25, 26, 27, 28])
def test_references_next_to_larger_scores(kind, D, e, low):
    """Logarithms at 2^e + low steps of 32-bit numbers there (2^(e - 23)), and from the third tile on one step more: the reference moves or the weights reach 2 to that step, which may be more than f16 holds.

    Scores are whole and exact, the factor is 1 (scale = ln 2 in 32 bits, times log2 e, is 1 to 2^-28). Weights are powers of two, so an output has the half step of its type, h, and sums of some 300 weights and products in fp32, together less than 2^-14 of the largest value."""
    step, T = 2.0 ** (e - 23), 300
    q = torch.zeros((T, 1, D), dtype=TYPES[kind], device="cuda")
    k, v = q.clone(), torch.randn((T, 1, D), generator=gen(5), device="cuda").to(TYPES[kind])
    a = 2.0 ** (e // 2)
    q[:, 0, 0], q[:, 0, 1] = a, step
    k[:, 0, 0], k[:, 0, 1] = 2.0 ** e / a, low
    k[128:, 0, 1] = low + 1
    got, _ = K_.attn_prompt(q, k, v, i32([0, T]), max_rows=T, scale=math.log(2))
    w = torch.ones(T, dtype=torch.float64, device="cuda")
    w[128:] = 2.0 ** step
    x = v[:, 0].double() * w[:, None]
    want = x.cumsum(0) / w.cumsum(0)[:, None]
    h = torch.finfo(q.dtype).eps / 2
    assert ((got[:, 0].double() - want).abs() <= h * want.abs() + (2.0 ** -14 + 2.0 ** -24) * v.double().abs().max()).all() and status() == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("far", [24.25, 25.25, 27.0])
def test_many_weak_keys_beside_a_strong_one(D, far):
    """The first key 2^far times as heavy as each of the 20000 behind it, whose values alone are not zero: what they have together is not lost, although a weight of one of them is next to nothing.

    In f16 a weight is off by half a step of it, or of 2^-24 where it is subnormal, and the largest weight is at least 2^6: 2^-31 of the largest one per key. The output is rounded to half a step of f16 or of 2^-24."""
    T = 20001
    q = torch.zeros((T, 1, D), dtype=torch.float16, device="cuda")
    k, v = q.clone(), (torch.rand((T, 1, D), generator=gen(5), device="cuda") + 0.5).half()
    q[:, 0, 0], k[0, 0, 0], v[0] = 1, far, 0
    got, _ = K_.attn_prompt(q, k, v, i32([0, T]), max_rows=T, scale=math.log(2))
    n = torch.arange(T, device="cuda", dtype=torch.float64)[:, None]
    total = v[:, 0].double().cumsum(0)
    want = total * 2.0 ** -far / (1 + n * 2.0 ** -far)
    tol = want * (2 * 2.0 ** -11 + 2.0 ** -15) + 2.0 ** -31 * total + 2.0 ** -25
    assert ((got[:, 0].double() - want).abs() <= tol).all() and status() == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size", [2.5e38, 1e30, 1e-33])
def test_values_of_any_size(D, size):
    """Values in bf16 next to the largest number and to the smallest normal one: outputs are means of them, whatever the sums of weights and values on the way."""
    rows = [700, 90]
    q, k, v = make(rows, 4, 2, D, "bf16", 61, packed=False)
    v = (v.float().clamp(-1, 1) * size).bfloat16()
    v[300:420] = size   # of one sign
    gate = torch.randn(q.shape, generator=gen(3), device="cuda")
    for g in (None, gate):
        got, _ = K_.attn_prompt(q, k, v, starts(rows), max_rows=700, gate=g)
        want, tol = prompt64(q, k, v, rows, D ** -0.5, g)
        assert ((got.double() - want).abs() <= tol).all() and status() == 0


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("rs,there", [([-1, 30, 40, 90], [(1, 30, 40), (2, 40, 90)]), ([0, -5, 40, 90], [(2, 40, 90)]), ([0, 30, 20, 90], [(0, 0, 30)]), ([0, 30, 40, 91], [(0, 0, 30), (1, 30, 40)]), ([0, 30, 1 << 30, 90], [(0, 0, 30)]),
                                      ([-2 ** 31, 30, 40, 2 ** 31 - 1], [(1, 30, 40)])])
def test_prompts_beside_bad_row_starts_are_served(D, rs, there):
    """Rows of a prompt whose two ends fit, as without the others. Of 0, 30, 20, 90 rows 20 to 29 are claimed by two prompts (0 to 29, and 20 on), and are no one's to be compared."""
    q, k, v = make([90], 2, 1, D, "bf16", 3, packed=False)
    got, _ = K_.attn_prompt(q, k, v, i32(rs), max_rows=60)
    assert status() == 1
    for _, a, b in there:
        n = 20 if rs[1:3] == [30, 20] else b - a
        assert torch.equal(got[a:a + n], K_.attn_prompt(q[a:b], k[a:b], v[a:b], i32([0, b - a]), max_rows=60)[0][:n]), (a, b)
    assert status() == 0


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_gated_prompts_over_and_over(kind, D):
    """One wave of blocks whose last ones have few and odd rows, a sync behind each call, outputs in 16 bits and in int8, finite values and others in turn: the same bits every time."""
    rows, H = [1234, 225, 1161, 984, 1135], 6
    q, k, v = make(rows, H, 1, D, kind, 71, packed=False, up=0.2)
    gate = torch.randn(q.shape, generator=gen(3), device="cuda")
    rs, odd = starts(rows), v.clone()
    for i in range(0, sum(rows), 371):
        odd[i, 0, i % D] = (math.nan, math.inf, -math.inf)[i % 3]
    first = {}
    for i in range(200):
        x = (v, odd)[i % 2]
        out, xq = K_.attn_prompt(q, k, x, rs, max_rows=5000, gate=gate, want_q8=True)
        assert status() == 0
        bits = out.view(torch.int16)
        want = first.setdefault(i % 2, (bits, *xq.unpack()))
        assert torch.equal(bits, want[0]) and torch.equal(xq.unpack()[0], want[1])
    hit = torch.cat([torch.where(torch.isfinite(t), 0, t).double().cumsum(0) for t in odd.split(rows)]).isfinite().expand(-1, H, -1)
    assert torch.equal(first[0][0][hit], first[1][0][hit])
