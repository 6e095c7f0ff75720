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
