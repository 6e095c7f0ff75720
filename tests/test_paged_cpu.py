"""Refusals of the paged-cache calls: every bad argument is answered before anything reaches a device (no GPU needed)."""
import ctypes

import pytest
import torch

import hipster_b200 as hb
from hipster_b200 import kernels as K_

FAKE = 1 << 20   # an aligned address that is never read: the calls below are refused


def pages(**kw):
    a = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, type=0, n_pages=8, n_kv=2, page_size=16, head_dim=64)
    a.update(kw)
    return K_._Pages(*a.values())


def refused(rc, word):
    assert rc == 1 and word in hb.lib().hp_last_error().decode(), (rc, hb.lib().hp_last_error())


def batch(**kw):
    a = dict(table=FAKE, table_ld=4, row_start=FAKE, kv_len=FAKE, S=2, R=4)
    a.update(kw)
    return [ctypes.c_void_p(a["table"]), a["table_ld"], ctypes.c_void_p(a["row_start"]), ctypes.c_void_p(a["kv_len"]), a["S"], a["R"]]


def ll(x):
    return ctypes.c_longlong(x)


def append(p, q=(FAKE, 256, 64), qo=(FAKE, 256, 64), n_head=4, k=(FAKE, 128, 64), v=(FAKE, 128, 64), rope=FAKE, n_pos=64, n_rot=64, **b):
    rows = lambda t: [ctypes.c_void_p(t[0]), ll(t[1]), ll(t[2])]  # noqa: E731
    return hb.lib().hp_kv_append(*rows(q), *rows(qo), n_head, *rows(k), *rows(v), None, None, ctypes.c_void_p(rope), n_pos, n_rot, 0, *batch(**b), ctypes.byref(p) if p else None, ctypes.c_float(1e-6), None)


def read(p, ko=FAKE, vo=FAKE, rs=128, hs=64, **b):
    return hb.lib().hp_kv_read(*batch(**b), ctypes.byref(p) if p else None, ctypes.c_void_p(ko), ctypes.c_void_p(vo), ll(rs), ll(hs), None)


def attn(p, q=(FAKE, 256, 64), n_head=4, max_rows=2, max_kv=64, scale=0.125, window=0, n_sink=0, out=FAKE, xq=0, sc=0, ws=FAKE, **b):
    v = ctypes.c_void_p
    return hb.lib().hp_attn_paged(v(q[0]), ll(q[1]), ll(q[2]), None, ll(0), ll(0), n_head, *batch(**b), max_rows, max_kv, ctypes.byref(p) if p else None, ctypes.c_float(scale), window, n_sink, v(out), v(xq), v(sc), v(ws), None)


@pytest.mark.parametrize("call", [append, read, attn])
@pytest.mark.parametrize("bad,word", [
    (dict(type=2), "type"), (dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"), (dict(page_size=2048), "page_size"),
    (dict(n_pages=0), "bad cache"), (dict(n_kv=0), "bad cache"), (dict(n_pages=1 << 30, n_kv=4), "bad cache"), (dict(k=0), "null"), (dict(v_scale=0), "null"), (dict(v=FAKE + 8), "misaligned"), (dict(k_scale=FAKE + 2), "misaligned")])
def test_bad_caches(call, bad, word):
    refused(call(pages(**bad)), word)


@pytest.mark.parametrize("call", [append, read, attn])
@pytest.mark.parametrize("bad,word", [(dict(S=0), "bad batch"), (dict(R=0), "bad batch"), (dict(table_ld=0), "bad cache"), (dict(table_ld=1 << 27), "bad cache"), (dict(table=0), "null"), (dict(row_start=0), "null"),
                                      (dict(kv_len=0), "null"), (dict(kv_len=FAKE + 1), "misaligned")])
def test_bad_batches(call, bad, word):
    refused(call(pages(), **bad), word)
    refused(call(None), "null cache")


def test_bad_rows():
    refused(append(pages(), k=(0, 128, 64)), "null")
    refused(append(pages(), q=(0, 256, 64)), "null")
    refused(append(pages(), rope=0), "null")
    refused(append(pages(), n_rot=66), "n_rot")
    refused(append(pages(), n_rot=3), "n_rot")
    refused(append(pages(), n_pos=0), "n_pos")
    refused(append(pages(), n_head=-1), "null")
    refused(append(pages(), v=(FAKE + 4, 128, 64)), "aligned")
    refused(append(pages(), k=(FAKE, 130, 64)), "aligned")
    refused(append(pages(), qo=(FAKE, 256, 62)), "aligned")
    refused(read(pages(), ko=0), "null")
    refused(read(pages(), vo=FAKE + 8), "aligned")
    refused(read(pages(), rs=132), "aligned")
    for rs, hs in ((0, 64), (128, 0), (64, 64), (96, 64), (64, 248)):   # four rows of two heads of 64
        refused(read(pages(), rs=rs, hs=hs), "over each other")
        refused(append(pages(), qo=(FAKE, rs, hs), n_head=2), "over each other")
    refused(attn(pages(), q=(0, 256, 64)), "null")
    refused(attn(pages(), ws=0), "null")
    refused(attn(pages(), out=0), "null")
    refused(attn(pages(), xq=FAKE), "both")
    refused(attn(pages(), q=(FAKE, 255, 64)), "aligned")
    refused(attn(pages(), ws=FAKE + 4), "aligned")
    refused(attn(pages(), n_head=3), "n_head")
    refused(attn(pages(), n_head=0), "n_head")
    refused(attn(pages(), window=-1), "window")
    refused(attn(pages(), n_sink=4), "window")
    refused(attn(pages(), scale=0.0), "scale")
    refused(attn(pages(), scale=float("nan")), "scale")
    refused(attn(pages(), max_rows=0), "bad batch")
    refused(attn(pages(), max_kv=0), "bad batch")


def test_bad_tables():
    d = ctypes.c_double
    f = lambda n_pos=8, n_rot=64, base=1e4, kind=0, factor=1.0, orig=0, fast=32.0, slow=1.0, m=0.0, at=FAKE: hb.lib().hp_rope_table(ctypes.c_void_p(at), n_pos, n_rot, d(base), kind, d(factor), orig, d(fast), d(slow), d(m), None)  # noqa: E731
    for kw, word in ((dict(at=0), "null"), (dict(n_pos=0), "shape"), (dict(n_rot=63), "shape"), (dict(n_rot=258), "shape"), (dict(base=0.0), "shape"), (dict(kind=3), "scaling"), (dict(kind=1, factor=0.5), "factor"),
                     (dict(kind=2, factor=4.0), "original"), (dict(kind=2, factor=4.0, orig=100, fast=1.0), "original"), (dict(m=-1.0), "attention factor"), (dict(kind=1, factor=float("nan")), "factor")):
        refused(f(**kw), word)


def test_workspace_sizes():
    L = hb.lib()
    L.hp_attn_paged_workspace_bytes.restype = ctypes.c_size_t
    f = lambda p=None, ld=64, S=4, R=8, mr=2, mk=1000, nh=4, w=0, k=0: L.hp_attn_paged_workspace_bytes(ld, S, R, mr, mk, nh, w, k, ctypes.byref(p or pages()))  # noqa: E731
    part = (64 + 2) * 4
    up = lambda n: (n + 127) // 128 * 128  # noqa: E731
    assert f() == up(8 * 4 * 4 * part)                       # four splits of 256 keys
    assert f(ld=1024, mk=1000) == up(8 * 4 * 2 * part)       # two of 512
    assert f(w=200) == up(8 * 4 * 2 * part)                  # a run of up to 201 keys lies in two splits
    assert f(w=200, k=3) == up(8 * 4 * 3 * part)             # and the first tokens in one more
    tiles = lambda mk: 4 * 2 * -(-mk // 64) * 2 * 64 * (64 * 2 + 4)  # noqa: E731
    assert f(R=4000, mr=1000, w=100) == up(4000 * 4 * part) + tiles(1000)   # prompts: keys and values in f16 with their scales; a window in one split
    assert all(f(R=600, mr=300, mk=m) <= f(R=600, mr=300, mk=(m + 1023) // 1024 * 1024) for m in range(1, 5000, 37))
    assert all(f(mk=m) <= f(mk=m + 1) and f(mk=m, w=300, k=5) <= f(mk=m + 1, w=300, k=5) for m in range(1, 1500, 7))
    assert f(p=pages(type=9)) == 0 and f(nh=3) == 0 and f(k=1) == 0


def test_python_refusals():
    c = lambda *s, t=torch.int8: torch.zeros(s, dtype=t)  # noqa: E731
    s = torch.zeros((2, 2, 16))
    for bad in ((c(2, 2, 16, 64), c(2, 2, 16, 32), s, s), (c(2, 2, 16, 64, t=torch.uint8), c(2, 2, 16, 64, t=torch.uint8), s, s), (c(2, 2, 16, 64), c(2, 2, 16, 64), s[..., :8], s),
                (c(2, 2, 16, 64), c(2, 2, 64, 16).transpose(2, 3), s, s), (c(2, 2, 16, 64), c(2, 2, 16, 64, t=torch.float8_e4m3fn), s, s), (c(2, 2, 16, 64), c(2, 2, 16, 64), s, s.double())):
        with pytest.raises(hb.HipsterError):
            K_.KVPages(*bad)
    with pytest.raises(hb.HipsterError):
        K_.rope_table(8, 64, 1e4, scaling="other")
