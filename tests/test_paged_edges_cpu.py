"""Edges of the paged-cache calls that the host decides: sizes of workspaces, refusals, what is handed to the library (no GPU needed)."""
import ctypes

import pytest
import torch

import hipster_b200 as hb
from hipster_b200 import kernels as K_


class Recorded:
    """Stands in for the native entry points: records what they are given, and answers that all is well."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.fixture
def recorded(monkeypatch):
    """The Python form of the calls on tensors of the CPU, up to the library; sizes of what the calls allocate."""
    r, new = Recorded(), torch.Tensor.new_empty
    r.allocated = []
    monkeypatch.setattr(K_, "hot", lambda: r)
    monkeypatch.setattr(K_, "tensors", lambda: None)
    monkeypatch.setattr(K_, "_device", lambda: -1)
    monkeypatch.setattr(K_, "_raw_stream", lambda dev: 0)

    def new_empty(self, *a, **kw):
        t = new(self, *a, **kw)
        r.allocated.append(t)
        return t
    monkeypatch.setattr(torch.Tensor, "new_empty", new_empty, raising=False)
    return r


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def size(pages, ld, S, R, max_rows, max_kv, n_head, window=0, n_sink=0):
    return hb.lib().hp_attn_paged_workspace_bytes(ld, S, R, max_rows, max_kv, n_head, window, n_sink, ctypes.byref(pages._c))


@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("max_kv", [1, 999, 1024, 1025, 4096, 2 ** 31 - 1024, 2 ** 31 - 1023, 2 ** 31 - 1])
def test_the_workspace_holds_what_the_library_asks_for(recorded, rows, max_kv):
    """max_kv up to the largest int, as a caller without a bound gives it."""
    pages = K_.KVPages.empty(70, 2, 16, 64, device="cpu")
    q = torch.zeros((rows, 4, 64))
    K_.attn_paged(q, pages, torch.zeros((1, 64), dtype=torch.int32), i32([0, rows]), i32([rows]), max_rows=rows, max_kv=max_kv)
    (name, a), = recorded.calls
    assert name == "hp_attn_paged" and a[14] == max_kv
    at, need = a[22], size(pages, 64, 1, rows, rows, max_kv, 4)
    ws, = [t for t in recorded.allocated if t.data_ptr() == at]
    assert need > 0 and ws.numel() * ws.element_size() >= need


def test_a_workspace_that_the_library_refuses_ends_the_call(recorded):
    pages = K_.KVPages.empty(70, 2, 16, 64, device="cpu")
    q = torch.zeros((1, 4, 64))
    for kw in (dict(max_rows=0, max_kv=64), dict(max_rows=1, max_kv=0), dict(max_rows=1, max_kv=64, n_sink=1), dict(max_rows=1, max_kv=64, window=-1)):
        for _ in range(2):   # a second time too: no answer is kept
            with pytest.raises(hb.HipsterError, match="bad"):
                K_.attn_paged(q, pages, torch.zeros((1, 64), dtype=torch.int32), i32([0, 1]), i32([1]), **kw)
    assert not recorded.calls


def columns_seen(recorded, monkeypatch, call):
    """(table, table_ld, columns) of the cache and batch that each call hands over."""
    seen = []

    class Reads:
        def __getattr__(self, name):
            at, table = {"hp_kv_append": (25, 19), "hp_kv_read": (6, 0), "hp_attn_paged": (15, 7)}[name]

            def f(*a):
                seen.append((a[table], a[table + 1], K_._Pages.from_address(a[at]).columns))
                return 0
            return f
    monkeypatch.setattr(K_, "hot", lambda: Reads())
    call()
    return seen


def test_a_table_that_is_part_of_a_wider_one_ends_with_its_columns(recorded, monkeypatch):
    """What is handed to the library says where the columns of table[:, a:b] end: what lies beside them is not the caller's to use here."""
    pages = K_.KVPages.empty(70, 2, 16, 64, device="cpu")
    big = torch.zeros((2, 9), dtype=torch.int32)
    x = torch.zeros((2, 2, 64))
    for a, b in ((0, 4), (3, 9), (8, 9), (0, 9)):
        t, rs, kl = big[:, a:b], i32([0, 1, 2]), i32([1, 1])

        def call():
            K_.kv_append(pages, x, x, t, rs, kl)
            K_.kv_read(pages, t, rs, kl, R=2)
            K_.attn_paged(x, pages, t, rs, kl, max_rows=1, max_kv=1000)
        seen = columns_seen(recorded, monkeypatch, call)
        assert len(seen) == 3 and all(at == t.data_ptr() and (cols or ld) == b - a and (cols == 0 or ld == 9) for at, ld, cols in seen)
    one = columns_seen(recorded, monkeypatch, lambda: K_.kv_read(pages, big[1:, 2:5], i32([0, 1]), i32([1]), R=1))
    assert [(cols or ld) for _, ld, cols in one] == [3] and pages._c.columns == 0
    with pytest.raises(hb.HipsterError, match="table"):
        K_.kv_read(pages, big[:, :0], i32([0, 1, 2]), i32([1, 1]), R=2)


def test_columns_of_a_cache():
    L, F = hb.lib(), 1 << 20
    pages = lambda n: K_._Pages(F, F, F, F, 0, 8, 2, 16, 64, n)  # noqa: E731
    v, z = ctypes.c_void_p, ctypes.c_longlong

    def read(n, ld=4):
        return L.hp_kv_read(v(F), ld, v(F), v(F), 2, 4, ctypes.byref(pages(n)), v(F), v(F), z(128), z(8), None)   # refused for its head stride, if not before
    for n, ld in ((5, 4), (-1, 4), (1 << 26, 1 << 27)):
        assert read(n, ld) == 1 and "columns" in L.hp_last_error().decode()
    for n, ld in ((4, 4), (0, 4), (1, 4), (4, 1 << 27)):
        assert read(n, ld) == 1 and "over each other" in L.hp_last_error().decode()
    f = lambda n, ld, mk=10 ** 6: L.hp_attn_paged_workspace_bytes(ld, 4, 8, 2, mk, 4, 0, 0, ctypes.byref(pages(n)))  # noqa: E731
    assert f(64, 5000) == f(0, 64) > 0   # the split of the keys, too, goes by the columns in use


def test_misaligned_outputs_and_weights_are_refused():
    """Before anything reaches a device, where they would be written and read several bytes at a time."""
    L, F = hb.lib(), 1 << 20
    v, z, c = ctypes.c_void_p, ctypes.c_longlong, K_._Pages(F, F, F, F, 0, 8, 2, 16, 64)
    for xq, sc in ((F + 1, F), (F + 4, F), (F + 8, F), (F, F + 2), (F, F + 4)):
        for rows in (2, 20):
            rc = L.hp_attn_paged(v(F), z(256), z(64), None, z(0), z(0), 4, v(F), 4, v(F), v(F), 2, 40, rows, 64, ctypes.byref(c), ctypes.c_float(0.125), 0, 0, v(F), v(xq), v(sc), v(F), None)
            assert rc == 1 and "quantised outputs must be 16-byte aligned" in L.hp_last_error().decode()
    for qn, kn in ((F + 1, F), (F, F + 3)):
        rc = L.hp_kv_append(v(F), z(256), z(64), v(F), z(256), z(64), 4, v(F), z(128), z(64), v(F), z(128), z(64), v(qn), v(kn), None, 0, 0, 0, v(F), 4, v(F), v(F), 2, 4, ctypes.byref(c), ctypes.c_float(1e-6), None)
        assert rc == 1 and "norm weights" in L.hp_last_error().decode()


def test_integers_beyond_32_bits_are_refused(recorded, monkeypatch):
    """They do not arrive as what is left of them in 32 bits: a window of 2^32 + 5 is not one of 5."""
    pages = K_.KVPages.empty(70, 2, 16, 64, device="cpu")
    q = torch.zeros((1, 4, 64))
    good = dict(max_rows=1, max_kv=64, window=5, n_sink=1)
    for name in good:
        for n in (2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1, 2 ** 64 + 5):
            with pytest.raises(hb.HipsterError, match="32 bits"):
                K_.attn_paged(q, pages, torch.zeros((1, 64), dtype=torch.int32), i32([0, 1]), i32([1]), **{**good, name: n})
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: pytest.fail("allocated"))
    for a, kw in (((2 ** 32 + 8, 64), {}), ((8, 2 ** 32 + 2), {}), ((8, 64), dict(scaling="yarn", factor=2.0, orig_ctx=2 ** 32 + 64))):
        with pytest.raises(hb.HipsterError, match="32 bits"):
            K_.rope_table(*a, 1e4, **kw)
    assert not recorded.calls


def test_outputs_that_would_be_written_twice_are_refused():
    L, F = hb.lib(), 1 << 20
    v, z, c = ctypes.c_void_p, ctypes.c_longlong, K_._Pages(F, F, F, F, 0, 8, 2, 16, 64)
    for ld, hs in ((512, 64), (256, 1024), (512, 128)):
        rc = L.hp_kv_append(v(F), z(256), z(64), v(F), z(ld), z(hs), 4, v(F), z(128), z(64), v(F), z(128), z(64), None, None, None, 0, 0, 0, v(F), 4, v(F), v(F), 2, 4, ctypes.byref(c), ctypes.c_float(1e-6), None)
        assert rc == 1 and "in place" in L.hp_last_error().decode()
    assert L.hp_kv_read(v(F), 4, v(F), v(F), 2, 4, ctypes.byref(c), v(F), v(F), z(128), z(64), None) == 1 and "the same" in L.hp_last_error().decode()
