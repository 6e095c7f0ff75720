"""Refusals of the calls for 4 bits, positions of several axes and prompts, and what the host works out for them (no GPU needed)."""
import ctypes

import pytest
import torch

import hipster_b200 as hb
from hipster_b200 import _lib, kernels as K_
from test_paged_cpu import FAKE, append as append8, attn, pages, read, refused
from test_paged_edges_cpu import recorded  # noqa: F401


def more():
    return _lib.more()


def rows(q=(FAKE, 256, 64), qo=(4 * FAKE, 256, 64), n_head=4, k=(FAKE, 128, 64), ko=(2 * FAKE, 128, 64), v=(FAKE, 128, 64), vo=(3 * FAKE, 128, 64), n_kv=2, D=64, kind=1, qn=None, rope=FAKE, n_pos=64, n_rot=64, pos=FAKE, pos_ld=8, axes=bytes(32), n_axes=1, R=4):
    return more().hp_rope_rows(*q, *qo, n_head, *k, *ko, *v, *vo, n_kv, D, kind, qn, None, rope, n_pos, n_rot, 0, pos, pos_ld, axes, n_axes, R, 1e-6, None)


def append(p, pos=FAKE, pos_ld=8, axes=bytes(32), n_axes=1, n_rot=64, n_pos=64, k=(FAKE, 128, 64), rope=FAKE, S=2, R=4):
    return more().hp_kv_append_axes(FAKE, 256, 64, FAKE, 256, 64, 4, *k, FAKE, 128, 64, None, None, rope, n_pos, n_rot, 0, pos, pos_ld, axes, n_axes, FAKE, 4, FAKE, FAKE, S, R, ctypes.addressof(p), 1e-6, None)


def prompt(q=(FAKE, 256, 64), k=(FAKE, 128, 64), v=(FAKE, 128, 64), kind=1, gate=(None, 0, 0), n_head=4, n_kv=2, D=64, rs=FAKE, S=2, R=4, max_rows=4, scale=0.125, out=FAKE, xq=None, sc=None):
    return more().hp_attn_prompt(*q, *k, *v, kind, *gate, n_head, n_kv, D, rs, S, R, max_rows, scale, out, xq, sc, None)


@pytest.mark.parametrize("call", [append8, read, attn])
@pytest.mark.parametrize("bad,word", [(dict(type=3), "type"), (dict(type=5), "type"), (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"), (dict(v=FAKE + 8), "misaligned"), (dict(k_scale=FAKE + 2), "misaligned")])
def test_bad_caches(call, bad, word):
    refused(call(pages(**{"type": 4, **bad})), word)


def test_workspaces_are_those_of_eight_bits():
    L = hb.lib()
    size = lambda kind, **kw: L.hp_attn_paged_workspace_bytes(64, 4, kw.get("R", 8), kw.get("mr", 2), 1000, 4, 0, 0, ctypes.byref(pages(type=kind)))  # noqa: E731
    assert size(4) == size(0) > 0 and size(4, R=300, mr=100) == size(0, R=300, mr=100) > 0


def test_bad_positions():
    p = pages(type=4)
    for f in (lambda **kw: append(p, **kw), rows):
        refused(f(pos=None), "null")
        refused(f(axes=None), "null")
        refused(f(n_axes=0), "positions")
        refused(f(n_axes=5), "positions")
        refused(f(pos=FAKE + 2), "positions")
        refused(f(n_axes=2, pos_ld=-1), "positions")
        refused(f(axes=bytes(31) + b"\1"), "axis 1 of 1")
        refused(f(n_axes=3, axes=bytes(31) + b"\3"), "axis 3 of 3")
        refused(f(n_rot=66, axes=bytes(33)), "n_rot")
        refused(f(n_pos=0), "n_pos")
    refused(append(p, n_rot=0), "n_rot")
    refused(append(p, rope=None), "null")
    refused(append(p, k=(FAKE + 4, 128, 64)), "aligned")
    refused(append(pages(type=2)), "type")
    refused(append(p, R=0), "bad batch")


def test_bad_rows():
    refused(rows(D=96), "head_dim")
    refused(rows(kind=3), "type")
    refused(rows(R=0), "shape")
    refused(rows(n_head=-1), "shape")
    refused(rows(n_rot=3, axes=bytes(32)), "n_rot")
    refused(rows(rope=None), "n_rot")
    refused(rows(rope=FAKE + 4), "n_rot")
    refused(rows(qn=FAKE + 1), "2-byte")
    refused(rows(qo=(None, 256, 64)), "null")
    refused(rows(k=(None, 128, 64)), "null")
    refused(rows(q=(None, 0, 0), qo=(None, 0, 0), k=(None, 0, 0), ko=(None, 0, 0), v=(None, 0, 0), vo=(None, 0, 0)), "no rows")
    refused(rows(n_head=0, n_kv=0), "no rows")
    refused(rows(q=(FAKE + 4, 256, 64)), "aligned")
    refused(rows(q=(FAKE, 258, 64)), "aligned")
    refused(rows(qo=(FAKE, 260, 64)), "aligned")            # 16 bits: multiples of 8
    refused(rows(vo=(3 * FAKE, -128, 64)), "aligned")
    refused(rows(ko=(2 * FAKE, 64, 64)), "over each other")
    refused(rows(q=(FAKE, 256, 64), qo=(FAKE, 256, 64)), "in place")
    refused(rows(kind=0, qo=(FAKE, 320, 64)), "in place")
    refused(rows(qo=(5 * FAKE, 256, 64), ko=(3 * FAKE, 128, 64)), "same")
    refused(rows(kind=0, q=(6 * FAKE, 256, 64), ko=(6 * FAKE, 128, 64)), "another one's input")
    refused(rows(kind=0, qo=(FAKE, 256, 64)), "another one's input")   # q, k and v in one place


def test_bad_prompts():
    refused(prompt(kind=0), "type")
    refused(prompt(kind=3), "type")
    refused(prompt(D=96), "head_dim")
    refused(prompt(n_head=3), "n_head")
    refused(prompt(n_head=0), "n_head")
    refused(prompt(n_kv=0), "n_head")
    for kw in (dict(S=0), dict(R=0), dict(max_rows=0)):
        refused(prompt(**kw), "bad batch")
    refused(prompt(S=65536), "bad batch")
    for kw in (dict(q=(None, 256, 64)), dict(k=(None, 128, 64)), dict(v=(None, 128, 64)), dict(rs=None), dict(out=None)):
        refused(prompt(**kw), "null")
    refused(prompt(xq=FAKE), "both")
    refused(prompt(out=FAKE + 8), "aligned")
    refused(prompt(rs=FAKE + 2), "aligned")
    for t in ((FAKE + 8, 256, 64), (FAKE, 252, 64), (FAKE, 256, 60), (FAKE, 0, 64), (FAKE, 256, 0), (FAKE, -256, 64), (FAKE, 1 << 40, 64)):
        refused(prompt(q=t), "aligned")
    refused(prompt(gate=(FAKE + 4, 256, 64)), "gate")
    refused(prompt(gate=(FAKE, 254, 64)), "gate")
    refused(prompt(gate=(FAKE, 0, 64)), "gate")
    refused(prompt(gate=(FAKE, 256, 0)), "gate")
    refused(prompt(gate=(FAKE, 1 << 38, 64)), "gate")
    refused(prompt(scale=0.0), "scale")
    refused(prompt(scale=float("nan")), "scale")
    there = dict(q=(2 * FAKE, 256, 64), k=(3 * FAKE, 128, 64), v=(4 * FAKE, 128, 64), gate=(5 * FAKE, 256, 64))
    for i in (2, 3, 4, 5):
        refused(prompt(**there, out=i * FAKE), "in place of an input")
        refused(prompt(**there, xq=i * FAKE, sc=6 * FAKE), "in place of an input")
        refused(prompt(**there, xq=6 * FAKE, sc=i * FAKE), "in place of an input")
    for out, xq, sc in ((FAKE, FAKE, 6 * FAKE), (FAKE, 6 * FAKE, FAKE), (None, FAKE, FAKE)):
        refused(prompt(**there, out=out, xq=xq, sc=sc), "same")


def test_axes_of_pairs():
    assert K_.rope_axes((2, 1, 1)) == bytes([0, 0, 1, 2]) and K_.rope_axes([3]) == bytes(3)
    assert K_.rope_axes((11, 11, 10), 64, interleaved=True) == bytes([0, 1, 2] * 10 + [0, 1])
    assert K_.rope_axes((4, 1, 1), interleaved=True) == bytes([0, 1, 2, 0, 0, 0])
    for sections in ((24, 20, 20), (2, 2), (5, 3, 3), (8, 2, 2, 4), (4, 4, 4, 4)):
        for turns in (False, True):
            a = K_.rope_axes(sections, interleaved=turns)
            assert [a.count(i) for i in range(len(sections))][1:] == list(sections)[1:] and len(a) == sum(sections)
    for bad in ((), (1, 1, 1, 1, 1), (2, -1), (0, 0)):
        with pytest.raises(hb.HipsterError):
            K_.rope_axes(bad)
    with pytest.raises(hb.HipsterError):
        K_.rope_axes((2, 2), 6)


def test_pages_of_four_bits():
    for D, page, n_kv in ((64, 16, 1), (128, 32, 3), (256, 1024, 2)):
        p = K_.KVPages.empty(3, n_kv, page, D, dtype="i4", device="cpu")
        assert (p.n_pages, p.n_kv, p.page_size, p.head_dim) == (3, n_kv, page, D) and p._c.type == 4 and p.k.numel() == 3 * n_kv * page * (D // 2 + D // 32)
    u = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    s = torch.zeros((2, 2, 16))
    for bad in ((u(2, 2, 16 * 34 + 1), u(2, 2, 16 * 34 + 1), s, s), (u(2, 2, 16 * 17), u(2, 2, 16 * 17), s, s), (u(2, 2, 16 * 34), u(2, 2, 16 * 68), s, s), (u(2, 2, 16 * 34), u(2, 2, 16 * 34), s, s[..., :8]),
                (u(2, 2, 16 * 34), u(2, 2, 16 * 34), s[0], s[0]), (u(2, 3, 16 * 34), u(2, 3, 16 * 34), s, s), (u(2, 2, 0), u(2, 2, 0), s[..., :0], s[..., :0]), (u(2, 2, 16 * 34).int(), u(2, 2, 16 * 34).int(), s, s)):
        with pytest.raises(hb.HipsterError):
            K_.KVPages(*bad)
    with pytest.raises(hb.HipsterError):
        K_.KVPages.empty(2, 2, 16, 96, dtype="i4", device="cpu")


def test_what_reaches_the_library(recorded, monkeypatch):  # noqa: F811
    """Positions and axes as they are handed over, and the call without them as it was."""
    monkeypatch.setattr(K_, "more", lambda: recorded)
    i = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    pool = K_.KVPages.empty(4, 2, 16, 64, dtype="i4", device="cpu")
    x, rope, pos = torch.zeros((3, 8, 64)), torch.zeros((9, 16, 2)), torch.zeros((3, 5), dtype=torch.int32)[:, :3]
    at = (i([[0, 1]]), i([0, 3]), i([20]))
    K_.kv_append(pool, x[:, 4:6], x[:, 6:], *at, rope, q=x[:, :4])
    K_.kv_append(pool, x[:, 4:6], x[:, 6:], *at, rope, positions=pos, axes=[0, 1, 2, 0] * 4)
    K_.rope_rows(x[:, :4], None, x[:, 4:6], rope, pos[0], dtype=torch.bfloat16)
    K_.rope_rows(None, None, x[:, 4:6])
    (n0, a0), (n1, a1), (n2, a2), (n3, a3) = recorded.calls
    assert n0 == "hp_kv_append" and a0[16:18] == (9, 32)
    assert n1 == "hp_kv_append_axes" and a1[6] == 0 and a1[16:23] == (9, 32, 0, pos.data_ptr(), 5, bytes([0, 1, 2, 0] * 4), 3)
    assert n2 == "hp_rope_rows" and a2[6] == 4 and a2[7] is None and a2[19:22] == (2, 64, 2) and a2[28:32] == (pos.data_ptr(), 0, bytes(16), 1)
    assert n3 == "hp_rope_rows" and a3[24] is None and a3[28] is None and a3[31] == 0


def test_sections_that_turns_do_not_give_are_refused():
    """In turn, an axis has every n-th pair until it has its own; axis 0 has what is left. Sections that come out otherwise are refused, those that fit have all their pairs, axis 0 included."""
    for sections in ((24, 20, 20), (11, 11, 10), (8, 2, 2, 4), (4, 1, 1), (1, 1), (2, 1), (5,), (6, 0, 0), (3, 0, 1)):
        a = K_.rope_axes(sections, interleaved=True)
        assert [a.count(i) for i in range(len(sections))] == list(sections)
    for sections in ((1, 4, 4), (0, 4, 4), (8, 12, 12), (1, 2), (0, 1), (2, 2, 3), (4, 4, 4, 5)):
        with pytest.raises(hb.HipsterError, match="in turn"):
            K_.rope_axes(sections, interleaved=True)
        a = K_.rope_axes(sections)
        assert [a.count(i) for i in range(len(sections))] == list(sections)


def test_axes_that_are_not_a_number_per_pair_are_refused(recorded, monkeypatch):  # noqa: F811
    """A number is not a list of that many zeros, and the bytes of wider integers are not axes. Lists, tuples, bytes and arrays of any integers are taken by value."""
    import numpy as np
    monkeypatch.setattr(K_, "more", lambda: recorded)
    x, rope, pos = torch.zeros((3, 4, 64)), torch.zeros((9, 16, 2)), torch.zeros((3, 3), dtype=torch.int32)
    pool = K_.KVPages.empty(4, 2, 16, 64, dtype="i4", device="cpu")
    i = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    good = [0, 1, 2, 0] * 4
    calls = (lambda axes: K_.rope_rows(x, None, None, rope, pos, axes), lambda axes: K_.kv_append(pool, x[:, :2], x[:, 2:], i([[0, 1]]), i([0, 3]), i([20]), rope, positions=pos, axes=axes))
    for call in calls:
        for axes in (16, np.int64(16), np.zeros(2, dtype=np.int64), np.zeros(4, dtype=np.float32), np.zeros((2, 8), dtype=np.uint8), [0.0] * 16, [0, -1] * 8, [0, 256] * 8, "0" * 16, [True] * 15, torch.zeros(15), None):
            with pytest.raises(hb.HipsterError):
                call(axes)
                pytest.fail(f"{axes!r} was not refused")
        for axes in (good, tuple(good), bytes(good), bytearray(good), np.array(good), np.array(good, dtype=np.uint8), torch.tensor(good), torch.tensor(good, dtype=torch.uint8)):
            call(axes)
            assert recorded.calls[-1][1][30 if recorded.calls[-1][0] == "hp_rope_rows" else 21] == bytes(good)


@pytest.mark.parametrize("R", [2 ** 31 - 1, 2 ** 31 - 128, 2 ** 31 - 256])
def test_rows_whose_tiles_end_beyond_32_bits_are_refused(R):
    """Tiles and blocks reach up to 127 rows beyond the last one, and their numbers are 32-bit."""
    refused(prompt(R=R, max_rows=R, S=1, q=(FAKE, 8, 64), k=(FAKE, 8, 64), v=(FAKE, 8, 64), n_head=1, n_kv=1), "too many rows")
    refused(prompt(R=R, max_rows=1, S=1), "too many rows")
