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
