"""Kernel-level host API: the Python mirror of the reference's free kernel launchers
(engine/kernels/gemv.h, ops.h). Arguments are torch CUDA tensors; every call goes through the C ABI."""
import ctypes
import functools
import operator

import torch

from ._lib import HipsterError, lib, hot, more, tensors, check, ptr

# The calls below are a few microseconds of device work, so what they spend in Python counts: the handle of the current stream
# comes without a Stream object around it, the short calls go through native entry points that take addresses as integers (_lib.hot; to
# a ctypes function an integer would pass as 32 bits, hence the wrapper of _stream), and sizes that depend on shapes alone are computed once (per
# type of the numbers, too: a float or a numpy integer that equals an earlier size is still refused by the library's function).
try:
    _raw_stream, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
except AttributeError:   # torch without CUDA: the package still imports, and a call raises torch's own error
    _raw_stream, _device = (lambda _: torch.cuda.current_stream().cuda_stream), (lambda: 0)


def _stream():
    return ctypes.c_void_p(_raw_stream(_device()))


@functools.lru_cache(maxsize=256, typed=True)
def _xq8_bytes(R, K):
    return lib().hp_xq8_q_bytes(R, K), lib().hp_xq8_sc_bytes(R, K)


@functools.lru_cache(maxsize=256, typed=True)
def _argmax_scratch_bytes(R, n):
    return lib().hp_argmax_scratch_bytes(R, n)


@functools.lru_cache(maxsize=256, typed=True)
def _attn_workspace_bytes(R, n_head, n_kv, max_ctx):
    return lib().hp_attn_workspace_bytes(R, n_head, n_kv, max_ctx)


class XQ8:
    """Quantised activations (reference: struct XQ8, engine/kernels/gemv.h:8) in the library's private layout."""

    def __init__(self, R, K, device="cuda"):
        self.R, self.K = R, K
        nq, ns = _xq8_bytes(R, K)   # nq is a multiple of 512: the scales stay aligned
        self.q, self.sc = torch.zeros(nq + ns, dtype=torch.uint8, device=device).split((nq, ns))

    def unpack(self):
        """-> (q int8 [R][K], d f32 [R][K/32], s f32 [R][K/32]) in the reference's row layout."""
        q = torch.empty((self.R, self.K), dtype=torch.int8, device=self.q.device)
        d = torch.empty((self.R, self.K // 32), dtype=torch.float32, device=self.q.device)
        s = torch.empty_like(d)
        check(lib().hp_xq8_unpack(ptr(self.q), ptr(self.sc), self.R, self.K, ptr(q), ptr(d), ptr(s), _stream()))
        return q, d, s


def quantize_x_q8(x, xq=None):
    """x f32 [R][K] -> XQ8 (reference quantize_x_q8, gemv.h:9)."""
    stride = x.stride()
    assert x.dtype == torch.float32 and len(stride) == 2 and stride[1] == 1
    R, K = x.shape
    xq = xq or XQ8(R, K, x.device)
    check(hot().hp_quantize_x_q8(x.data_ptr(), stride[0], R, K, xq.q.data_ptr(), xq.sc.data_ptr(), _raw_stream(_device())))
    return xq


def dequant_q4k(w, nblk):
    out = torch.empty(nblk * 256, dtype=torch.float32, device=w.device)
    check(lib().hp_dequant_q4k(ptr(w), ctypes.c_size_t(nblk), ptr(out), _stream()))
    return out


def gemv_q4k_q8(w, xq, N, K, y=None):
    """y [R][N] = W . x for Q4_K W [N][K/256 blocks] (uint8 tensor) and quantised x (reference gemv_wmma, gemv.h:33)."""
    R = xq.R
    if y is None:
        y = torch.empty((R, N), dtype=torch.float32, device=w.device)
    check(hot().hp_gemv_q4k_q8(None if w is None else w.data_ptr(), xq.q.data_ptr(), xq.sc.data_ptr(), y.data_ptr(), N, K, R, y.stride(0), _raw_stream(_device())))
    return y


def gemv_q4k_f32(w, x, N, K):
    """f32-activation baseline (reference gemv_q4_K_f32, gemv.h:57)."""
    R = x.shape[0]
    y = torch.empty((R, N), dtype=torch.float32, device=w.device)
    check(lib().hp_gemv_q4k_f32(ptr(w), ptr(x), ptr(y), N, K, R, _stream()))
    return y


def argmax(logits, n=None):
    """Row-wise argmax (max value, lowest index) -> (ids int32 [R], vals f32 [R]) (reference argmax_topk k=1, ops.h:118)."""
    R, ld = logits.shape[0], logits.stride(0)
    n = n or logits.shape[1]
    dev, nb = logits.device, _argmax_scratch_bytes(R, n)
    ids = torch.empty(R, dtype=torch.int32, device=dev)
    vals = torch.empty(R, dtype=torch.float32, device=dev)
    scratch = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    check(hot().hp_argmax(logits.data_ptr(), R, n, ld, ids.data_ptr(), vals.data_ptr(), scratch.data_ptr() if nb else None, _raw_stream(_device())))
    return ids, vals


def argmax_noalloc(logits, n=None):
    """argmax() through the entry point for callers that cannot allocate device memory: it takes only the input and the two
    output tensors (a C caller creates these beforehand), for at most 32 rows of 524288 entries."""
    R, ld = logits.shape[0], logits.stride(0)
    n = n or logits.shape[1]
    ids = torch.empty(R, dtype=torch.int32, device=logits.device)
    vals = torch.empty(R, dtype=torch.float32, device=logits.device)
    check(lib().hp_argmax_noalloc(ptr(logits), R, n, ld, ptr(ids), ptr(vals), _stream()))
    return ids, vals


def accept_greedy(ids, drafts):
    """-> int32 tensor [mm, bonus] on device (reference host loop, engine/bench/spec27b.cpp:92-97)."""
    out = torch.empty(2, dtype=torch.int32, device=ids.device)
    check(hot().hp_accept_greedy(ids.data_ptr(), drafts.data_ptr(), drafts.numel(), out.data_ptr(), _raw_stream(_device())))
    return out


def device_status():
    check(lib().hp_device_status(_stream()))


def attn_decode(qkv, pos0, n_head, n_kv, n_rot, q_norm, k_norm, rope, kc, vc, max_ctx, eps=1e-6, want_q8=True):
    """GQA decode attention of one sequence: qkv f32 [R][ld] (normalised / rotated in place), rows at positions pos0 + r;
    q_norm / k_norm bf16 [256] (int16 tensors), rope f32 [max_ctx][n_rot/2][2], kc / vc f16 [n_kv][max_ctx][256] (updated).
    -> (out f32 [R][n_head*256], XQ8 of it or None). Reference: qk_norm_rope_kv + attn_decode_mq (ops.h:71-72,96)."""
    R, ld = qkv.shape[0], qkv.stride(0)
    ws = torch.empty(_attn_workspace_bytes(R, n_head, n_kv, max_ctx), dtype=torch.uint8, device=qkv.device)
    out = torch.empty((R, n_head * 256), dtype=torch.float32, device=qkv.device)
    xq = XQ8(R, n_head * 256, qkv.device) if want_q8 else None
    check(hot().hp_attn_decode(qkv.data_ptr(), ld, R, int(pos0), n_head, n_kv, n_rot, None if q_norm is None else q_norm.data_ptr(),
                               None if k_norm is None else k_norm.data_ptr(), None if rope is None else rope.data_ptr(), None if kc is None else kc.data_ptr(),
                               None if vc is None else vc.data_ptr(), int(max_ctx), out.data_ptr(), xq.q.data_ptr() if xq else None, xq.sc.data_ptr() if xq else None,
                               eps, ws.data_ptr(), _raw_stream(_device())))
    return out, xq


def repack_tiled(w, N, K, interleave_half=0):
    """ggml Q4_K [N][K/256 blocks] (uint8 tensor) -> the library's tile-major streaming layout (same bytes, permuted)."""
    L = lib()
    L.hp_q4k_tiled_bytes.restype = ctypes.c_size_t
    L.hp_q4k_tiled_bytes.argtypes = [ctypes.c_size_t, ctypes.c_int]
    out = torch.empty(L.hp_q4k_tiled_bytes(N, K), dtype=torch.uint8, device=w.device)
    check(L.hp_q4k_repack_tiled(ptr(w), ptr(out), ctypes.c_size_t(N), K, interleave_half, _stream()))
    return out


def moe_layer(xn, router, exp_gate_up, exp_down, sh_gate_up, sh_down, F, n_expert, k):
    """One mixture-of-experts FFN over the rows of xn f32 [T][E] -> (ids int32 [T][k+1], weights f32 [T][k+1], y f32 [T][E]).
    The expert tensors are given in ggml order and repacked here (an engine does that once at load).
    Reference: Qwen4Exp::moe_layer (qwen4exp.cpp:345-354)."""
    L = lib()
    L.hp_moe_workspace_bytes.restype = ctypes.c_size_t
    T, E = xn.shape
    xq = quantize_x_q8(xn)
    egu = repack_tiled(exp_gate_up, n_expert * 2 * F, E, F); edn = repack_tiled(exp_down, n_expert * E, F, 0)
    sgu = repack_tiled(sh_gate_up, 2 * F, E, F); sdn = repack_tiled(sh_down, E, F, 0)
    ws = torch.empty(L.hp_moe_workspace_bytes(T, E, F, n_expert, k), dtype=torch.uint8, device=xn.device)
    ids = torch.empty((T, k + 1), dtype=torch.int32, device=xn.device)
    w = torch.empty((T, k + 1), dtype=torch.float32, device=xn.device)
    y = torch.empty((T, E), dtype=torch.float32, device=xn.device)
    check(L.hp_moe_layer(ptr(xn), ptr(xq.q), ptr(xq.sc), ptr(router), ptr(egu), ptr(edn), ptr(sgu), ptr(sdn), T, E, F, n_expert, k,
                         ptr(ids), ptr(w), ptr(y), ptr(ws), _stream()))
    return ids, w, y


# ---- a paged cache in 8 bits (no counterpart in the reference)
_F32, _I32, _F16 = torch.float32, torch.int32, torch.float16


class _Pages(ctypes.Structure):   # hp_kv_pages
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p)] + [(n, ctypes.c_int) for n in ("type", "n_pages", "n_kv", "page_size", "head_dim", "columns")]


def _refuse(ok, what):
    if not ok:
        raise HipsterError(1, what)


class KVPages:
    """A pool of pages: k, v [n_pages][n_kv][page_size][head_dim] in int8 or float8_e4m3fn, or 4 bits as uint8 [n_pages][n_kv][page_size * 17 * head_dim / 32] (of a page and head the
    codes of its tokens, head_dim / 2 bytes each, then their groups' bytes, head_dim / 32 each: hipster_b200.h), with k_scale, v_scale f32 [n_pages][n_kv][page_size] (one scale per
    token and head). The tensors are kept, not copied; KVPages.empty() allocates them."""

    def __init__(self, k, v, k_scale, v_scale):
        four = k.dim() == 3 and k.dtype == torch.uint8
        _refuse(four or k.dim() == 4 and k.dtype in (torch.int8, torch.float8_e4m3fn),
                "KVPages: k must be [n_pages][n_kv][page_size][head_dim] in int8 or float8_e4m3fn, or uint8 [n_pages][n_kv][page_size * 17 * head_dim / 32]")
        _refuse(v.dtype == k.dtype and v.shape == k.shape, "KVPages: k and v must be alike")
        _refuse(all(t.dtype == torch.float32 and t.dim() == 3 and t.shape[:2] == k.shape[:2] and (four or t.shape == k.shape[:3]) for t in (k_scale, v_scale)) and k_scale.shape == v_scale.shape,
                "KVPages: scales must be f32 [n_pages][n_kv][page_size]")
        _refuse(all(t.is_contiguous() and t.device == k.device for t in (k, v, k_scale, v_scale)), "KVPages: contiguous tensors of one device")
        if four:
            page = k_scale.shape[2]
            head_dim, rest = divmod(32 * k.shape[2], 17 * page) if page else (0, 1)
            _refuse(rest == 0 and head_dim in (64, 128, 256), "KVPages: 4 bits take page_size * 17 * head_dim / 32 bytes per page and head, with a head_dim of 64, 128 or 256")
            shape = (*k_scale.shape, head_dim)
        else:
            shape = tuple(k.shape)
        self.k, self.v, self.k_scale, self.v_scale, self.device = k, v, k_scale, v_scale, k.device
        self.n_pages, self.n_kv, self.page_size, self.head_dim = shape
        self._c = _Pages(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), 4 if four else int(k.dtype != torch.int8), *shape)
        self._at, self._dev, self._f16 = ctypes.addressof(self._c), k.get_device(), torch.empty(0, dtype=_F16, device=k.device)

    @classmethod
    def empty(cls, n_pages, n_kv, page_size, head_dim, dtype=torch.int8, device="cuda"):
        """dtype: torch.int8, torch.float8_e4m3fn, or "i4" for 4 bits."""
        if dtype == "i4":
            _refuse(head_dim in (64, 128, 256), "KVPages: 4 bits go with a head_dim of 64, 128 or 256")
            codes = [torch.zeros((n_pages, n_kv, page_size * 17 * head_dim // 32), dtype=torch.uint8, device=device) for _ in range(2)]
        else:
            codes = [torch.zeros((n_pages, n_kv, page_size, head_dim), dtype=torch.uint8, device=device).view(dtype) for _ in range(2)]
        return cls(*codes, *(torch.zeros((n_pages, n_kv, page_size), dtype=torch.float32, device=device) for _ in range(2)))


# Calls whose arguments are in order are taken by _lib.tensors(), in C++ (None: not taken). What follows takes the others, says what is wrong with them, and takes all calls
# where that module was not built: it, too, reads each attribute once and makes no message before a test fails.
def _batch(pages, table, row_start, kv_len):
    """Checks what describes a ragged batch; -> number of sequences, the cache as the call sees it (hp_kv_pages: a table that is part of a wider one ends with its own
    columns), and the batch's addresses as the calls take them."""
    dev, S = pages._dev, kv_len.numel()
    (rows, cols), (ld, one) = table.shape, table.stride()
    if dev != _device():
        raise HipsterError(1, f"the pages are on device {dev}, and device {_device()} is current")
    if not (table.dtype is _I32 and row_start.dtype is _I32 and kv_len.dtype is _I32):
        raise HipsterError(1, "table, row_start and kv_len must be int32")
    if not (rows == S and row_start.numel() == S + 1 and one == 1 and cols and (ld >= cols or S == 1) and row_start.is_contiguous() and kv_len.is_contiguous()):
        raise HipsterError(1, "table must be [S][columns], in rows without gaps, row_start [S + 1] and kv_len [S] contiguous")
    if not (table.get_device() == dev and row_start.get_device() == dev and kv_len.get_device() == dev):
        raise HipsterError(1, "table, row_start and kv_len must be on the device of the pages")
    if S == 1:
        ld = cols
    c = pages._c
    if ld != cols:
        c = _Pages.from_buffer_copy(c)
        c.columns = cols
    return S, c, table.data_ptr(), ld, row_start.data_ptr(), kv_len.data_ptr()


def _rows(t, pages, R, heads, what):
    """f32 rows [R][heads][head_dim] -> address, row stride, head stride."""
    ld, hs, one = t.stride()
    if not (t.dtype is _F32 and t.shape == (R, heads, pages.head_dim) and one == 1 and t.get_device() == pages._dev):
        raise HipsterError(1, f"{what} must be f32 [{R}][{heads}][{pages.head_dim}] on the device of the pages")
    return t.data_ptr(), ld, hs


def _ints(what, *numbers):
    """The library takes them as 32 bits; what does not fit would arrive as another number."""
    if not -2 ** 31 <= min(numbers) <= max(numbers) < 2 ** 31:
        raise HipsterError(1, f"{what} must fit 32 bits")


_SCALING = {None: 0, "none": 0, "linear": 1, "yarn": 2}


def rope_table(n_pos, n_rot, base, scaling=None, factor=1.0, orig_ctx=0, beta_fast=32.0, beta_slow=1.0, attn_factor=0.0, device="cuda"):
    """(cos, sin) of pos * base^(-2 i / n_rot), f32 [n_pos][n_rot / 2][2], computed in 64 bits; scaling "linear" divides the frequencies by factor, "yarn"
    by parts: those that turn less than beta_slow times over orig_ctx positions wholly, those over beta_fast times not."""
    if scaling not in _SCALING:
        raise HipsterError(1, f"rope_table: unknown scaling {scaling!r}")
    fast = device == "cuda" and tensors()
    if fast:
        out = fast.rope_table(n_pos, n_rot, base, _SCALING[scaling], factor, orig_ctx, beta_fast, beta_slow, attn_factor)
        if out is not None:
            return out
    _ints("rope_table: n_pos, n_rot and orig_ctx", n_pos, n_rot, orig_ctx)
    if n_pos < 1 or n_rot < 2:
        raise HipsterError(1, f"rope_table: bad shape n_pos={n_pos} n_rot={n_rot}")
    out = torch.empty((n_pos, n_rot // 2, 2), dtype=_F32, device=device)
    if out.get_device() != _device():
        raise HipsterError(1, "rope_table: the device must be the current one")
    check(hot().hp_rope_table(out.data_ptr(), n_pos, n_rot, base, _SCALING[scaling], factor, orig_ctx, beta_fast, beta_slow, attn_factor, _raw_stream(_device())))
    return out


def _norm_weight(w, pages):
    return _norm_weight_on(w, pages.head_dim, pages._dev)


def _norm_weight_on(w, head_dim, dev):
    if w is None:
        return None
    if not (w.dtype in (torch.bfloat16, torch.int16) and w.shape == (head_dim,) and w.is_contiguous() and w.get_device() == dev):
        raise HipsterError(1, "norm weights are bf16 [head_dim]")
    return w.data_ptr()


def rope_axes(sections, n_rot=None, interleaved=False):
    """The axis of each rotated pair of dims, as kv_append and rope_rows take it: sections[a] pairs for axis a, one axis after the other; interleaved: the axes in turn (pair i to axis i mod n)
    until an axis has its pairs, and what is left over to axis 0; sections that do not come out so are refused. n_rot: the dims that are rotated (2 * sum(sections))."""
    n, half = len(sections), sum(sections)
    if not (1 <= n <= 4 and min(sections) >= 0 and half and (n_rot is None or n_rot == 2 * half)):
        raise HipsterError(1, "rope_axes: 1 to 4 sections, which add up to half of the rotated dims")
    if not interleaved:
        return bytes(a for a, m in enumerate(sections) for _ in range(m))
    axes = bytes(i % n if i < n * sections[i % n] else 0 for i in range(half))
    if any(axes.count(a) != m for a, m in enumerate(sections)):
        raise HipsterError(1, f"rope_axes: in turn, {half} pairs cannot be {', '.join(map(str, sections))} of the axes")
    return axes


def _rope_args(who, rope, positions, axes, R, dev):
    """-> table, n_pos, n_rot, and after `interleaved`: positions, their row stride, axes, number of axes."""
    if rope is None:
        if positions is not None or axes is not None:
            raise HipsterError(1, f"{who}: positions and axes go with a rope table")
        return (None, 0, 0), (None, 0, None, 0)
    if not (rope.dtype is _F32 and rope.dim() == 3 and rope.shape[2] == 2 and rope.is_contiguous() and rope.get_device() == dev):
        raise HipsterError(1, f"{who}: rope must be f32 [n_pos][n_rot / 2][2]")
    n_pos, half, _ = rope.shape
    if positions.dim() == 1:
        positions = positions[None]
    if positions.dim() != 2:
        raise HipsterError(1, f"{who}: positions must be int32 [axes][{R}] or [{R}]")
    (n_axes, cols), (ld, one) = positions.shape, positions.stride()
    if not (positions.dtype is _I32 and cols == R and (one == 1 or R == 1) and (n_axes == 1 or ld >= 0) and positions.get_device() == dev):
        raise HipsterError(1, f"{who}: positions must be int32 [axes][{R}], rows without gaps, on the device of the rows")
    if axes is None:
        if n_axes != 1:
            raise HipsterError(1, f"{who}: positions of several axes go with the axis of each pair (rope_axes)")
        axes = bytes(half)
    try:
        if type(axes) is not bytes:
            axes = bytes([operator.index(a) for a in axes])   # bytes() of a number is that many zeros, of an array the bytes of its numbers
    except (ValueError, TypeError):
        raise HipsterError(1, f"{who}: axes are whole numbers below the number of axes, one per rotated pair of dims") from None
    if len(axes) != half:
        raise HipsterError(1, f"{who}: {half} rotated pairs of dims, and {len(axes)} axes")
    return (rope.data_ptr(), n_pos, 2 * half), (positions.data_ptr(), ld if n_axes > 1 else 0, axes, n_axes)


_OUT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def rope_rows(q=None, k=None, v=None, rope=None, positions=None, axes=None, interleaved=False, q_norm=None, k_norm=None, eps=1e-6, dtype=torch.float16):
    """Rows of a prompt, f32 q [R][n_head][head_dim], k and v [R][n_kv][head_dim] (each may be None), as attn_prompt takes them: per head RMSNorm of q and k (q_norm, k_norm bf16 [head_dim], or None),
    rotation by rope f32 [n_pos][n_rot / 2][2] at positions int32 [axes][R] (or [R]), the axis of each pair in axes (rope_axes), rounded to dtype (float16, bfloat16, float32). -> q, k, v"""
    fast = tensors()
    if fast:
        out = fast.rope_rows(q, k, v, rope, positions, axes, interleaved, q_norm, k_norm, eps, _OUT.get(dtype, -1))
        if out is not None:
            return out
    given = [t for t in (q, k, v) if t is not None]
    if not given or dtype not in _OUT or any(t.dim() != 3 for t in given):
        raise HipsterError(1, "rope_rows: q, k and v are [R][heads][head_dim]; outputs are float16, bfloat16 or float32")
    R, _, D = given[0].shape
    dev = given[0].get_device()
    if dev != _device():
        raise HipsterError(1, f"rope_rows: the rows are on device {dev}, and device {_device()} is current")
    if k is not None and v is not None and k.shape[1] != v.shape[1]:
        raise HipsterError(1, "rope_rows: k and v have as many heads")
    if rope is not None and positions is None:
        raise HipsterError(1, "rope_rows: a rope table goes with positions")
    rows, out = [], []
    for t in (q, k, v):
        if t is None:
            rows.append((None, 0, 0, None, 0, 0))
            out.append(None)
            continue
        ld, hs, one = t.stride()
        if not (t.dtype is _F32 and t.shape[0] == R and t.shape[2] == D and one == 1 and t.get_device() == dev):
            raise HipsterError(1, f"rope_rows: rows are f32 [{R}][heads][{D}] on one device")
        o = t.new_empty(t.shape, dtype=dtype)
        rows.append((t.data_ptr(), ld, hs, o.data_ptr(), t.shape[1] * D, D))
        out.append(o)
    table, pos = _rope_args("rope_rows", rope, positions, axes, R, dev)
    n_head, n_kv = 0 if q is None else q.shape[1], k.shape[1] if k is not None else 0 if v is None else v.shape[1]
    check(more().hp_rope_rows(*rows[0], n_head, *rows[1], *rows[2], n_kv, D, _OUT[dtype], _norm_weight_on(q_norm, D, dev), _norm_weight_on(k_norm, D, dev), *table, int(interleaved), *pos, R, eps, _raw_stream(dev)))
    return tuple(out)


def kv_append(pages, k, v, table, row_start, kv_len, rope=None, q=None, q_out=None, interleaved=False, q_norm=None, k_norm=None, eps=1e-6, positions=None, axes=None):
    """Appends rows k, v f32 [R][n_kv][head_dim] of a ragged batch to their sequences' pages, k normalised (k_norm bf16 [head_dim]) and rotated by rope
    f32 [n_pos][n_rot / 2][2]. q [R][n_head][head_dim] is normalised and rotated alike. -> q_out (f32 [R][n_head][head_dim]; None without q).
    Rows row_start[s] .. row_start[s + 1] - 1 are the newest of the kv_len[s] tokens of sequence s. They are rotated by their places in the cache, or by positions int32 [axes][R] (or [R])
    with the axis of each pair in axes (rope_axes)."""
    fast = tensors()
    if fast:
        out = fast.kv_append(pages._at, pages._dev, k, v, table, row_start, kv_len, rope, q, q_out, interleaved, q_norm, k_norm, eps, positions, axes)
        if out is not None:
            return None if out is True else out
    S, c, *at = _batch(pages, table, row_start, kv_len)
    R, n_kv = k.shape[0], pages.n_kv
    qr = qo = (None, 0, 0)
    n_head = n_pos = n_rot = 0
    if q is not None:
        n_head = q.shape[1]
        qr = _rows(q, pages, R, n_head, "q")
        if q_out is None:
            q_out = q.new_empty((R, n_head, pages.head_dim))
        qo = _rows(q_out, pages, R, n_head, "q_out")
    rows = (*qr, *qo, n_head, *_rows(k, pages, R, n_kv, "k"), *_rows(v, pages, R, n_kv, "v"), _norm_weight(q_norm, pages), _norm_weight(k_norm, pages))
    if positions is not None or axes is not None:
        if rope is None or positions is None:
            raise HipsterError(1, "kv_append: positions and axes go with a rope table")
        turn, pos = _rope_args("kv_append", rope, positions, axes, R, pages._dev)
        check(more().hp_kv_append_axes(*rows, *turn, int(interleaved), *pos, *at, S, R, ctypes.addressof(c), eps, _raw_stream(pages._dev)))
        return q_out
    if rope is not None:
        n_pos, n_rot, two = rope.shape
        n_rot *= 2
        if not (rope.dtype is _F32 and two == 2 and rope.is_contiguous() and rope.get_device() == pages._dev):
            raise HipsterError(1, "kv_append: rope must be f32 [n_pos][n_rot / 2][2]")
        rope = rope.data_ptr()
    check(hot().hp_kv_append(*rows, rope, n_pos, n_rot, int(interleaved), *at, S, R, ctypes.addressof(c), eps, _raw_stream(pages._dev)))
    return q_out


def kv_read(pages, table, row_start, kv_len, R=None, k_out=None, v_out=None):
    """The tokens of the rows back as f16 -> k, v [R][n_kv][head_dim]. With kv_len[s] rows for each sequence whole caches; k_out, v_out may be views with other
    strides, as cache.transpose(0, 1) of an f16 [n_kv][max_ctx][256] cache for attn_decode."""
    fast = k_out is None and v_out is None and tensors()
    if fast:
        out = fast.kv_read(pages._at, pages._dev, table, row_start, kv_len, R)
        if out is not None:
            return out
    S, c, *at = _batch(pages, table, row_start, kv_len)
    n_kv, D = pages.n_kv, pages.head_dim
    if k_out is None and v_out is None and R is not None:
        k_out, v_out = pages._f16.new_empty((R, n_kv, D)), pages._f16.new_empty((R, n_kv, D))
        ld, hs = n_kv * D, D
    else:
        if k_out is None or v_out is None:
            raise HipsterError(1, "kv_read: give R, or both outputs")
        R, (ld, hs, one) = k_out.shape[0], k_out.stride()
        if not (k_out.shape == (R, n_kv, D) and v_out.shape == k_out.shape and v_out.stride() == (ld, hs, 1) and one == 1 and k_out.dtype is _F16 and v_out.dtype is _F16 and
                k_out.get_device() == pages._dev and v_out.get_device() == pages._dev):
            raise HipsterError(1, "kv_read: outputs are f16 [R][n_kv][head_dim] with the same strides")
    check(hot().hp_kv_read(*at, S, R, ctypes.addressof(c), k_out.data_ptr(), v_out.data_ptr(), ld, hs, _raw_stream(pages._dev)))
    return k_out, v_out


@functools.lru_cache(maxsize=256, typed=True)
def _attn_paged_workspace_bytes(cols, S, R, max_rows, max_kv, n_head, window, n_sink, kind, n_pages, n_kv, page_size, head_dim):
    nb = lib().hp_attn_paged_workspace_bytes(cols, S, R, max_rows, max_kv, n_head, window, n_sink, ctypes.byref(_Pages(None, None, None, None, kind, n_pages, n_kv, page_size, head_dim)))
    if nb == 0:   # refused: raised from here, so that no answer is kept
        check(1)
    return nb


def attn_paged(q, pages, table, row_start, kv_len, max_rows, max_kv, scale=None, window=0, n_sink=0, gate=None, want_f32=True, want_q8=False):
    """Attention of rows q f32 [R][n_head][head_dim] over their sequences' pages (causal; window > 0: the last `window` tokens and the first n_sink), times sigmoid(gate)
    where a gate [R][n_head][head_dim] is given. scale: 1 / sqrt(head_dim). max_rows, max_kv bound the rows and tokens of a sequence.
    -> (out f32 [R][n_head][head_dim] or None, XQ8 of its rows or None)."""
    fast = want_f32 and not want_q8 and tensors()
    if fast:
        out = fast.attn_paged(pages._at, pages._dev, q, gate, table, row_start, kv_len, max_rows, max_kv, scale, window, n_sink)
        if out is not None:
            return out, None
    _ints("attn_paged: max_rows, max_kv, window and n_sink", max_rows, max_kv, window, n_sink)
    (S, c, *at), (R, n_head, D) = _batch(pages, table, row_start, kv_len), q.shape
    qr = _rows(q, pages, R, n_head, "q")
    gr = (None, 0, 0) if gate is None else _rows(gate, pages, R, n_head, "gate")
    cols = table.shape[1]
    cap = cols * pages.page_size   # as the library bounds max_kv; rounded up, INT_MAX would leave the ints
    nb = _attn_paged_workspace_bytes(cols, S, R, max_rows, min(-(-max_kv // 1024) * 1024, cap), n_head, window, n_sink, c.type, c.n_pages, c.n_kv, c.page_size, c.head_dim)   # grows with max_kv
    ws = q.new_empty(nb // 4 + 4)
    out = q.new_empty((R, n_head, D)) if want_f32 else None
    xq = XQ8(R, n_head * D, pages.device) if want_q8 else None
    check(hot().hp_attn_paged(*qr, *gr, n_head, *at, S, R, max_rows, max_kv, ctypes.addressof(c), D ** -0.5 if scale is None else scale, window, n_sink, None if out is None else out.data_ptr(),
                              xq.q.data_ptr() if xq else None, xq.sc.data_ptr() if xq else None, ws.data_ptr(), _raw_stream(pages._dev)))
    return out, xq


def attn_prompt(q, k, v, row_start, max_rows, scale=None, gate=None, want_out=True, want_q8=False):
    """Causal attention of whole prompts, packed: rows row_start[s] .. row_start[s + 1] - 1 of q [R][n_head][head_dim], k and v [R][n_kv][head_dim] (all float16, or all bfloat16; any strides of rows and
    heads) are prompt s. Times sigmoid(gate) where a gate f32 [R][n_head][head_dim] is given. scale: 1 / sqrt(head_dim). max_rows bounds a prompt's rows.
    -> (out [R][n_head][head_dim] of q's type or None, XQ8 of its rows or None)"""
    fast = want_out and not want_q8 and tensors()
    if fast:
        out = fast.attn_prompt(q, k, v, row_start, max_rows, scale, gate)
        if out is not None:
            return out, None
    if q.dim() != 3 or k.dim() != 3 or q.dtype not in (torch.float16, torch.bfloat16):
        raise HipsterError(1, "attn_prompt: q, k and v are [R][heads][head_dim] in float16 or bfloat16")
    (R, n_head, D), n_kv, dev = q.shape, k.shape[1], q.get_device()
    _ints("attn_prompt: max_rows", max_rows)
    if dev != _device():
        raise HipsterError(1, f"attn_prompt: the rows are on device {dev}, and device {_device()} is current")
    for t, heads, what in ((q, n_head, "q"), (k, n_kv, "k"), (v, n_kv, "v")):
        if not (t.dtype is q.dtype and t.shape == (R, heads, D) and t.stride(2) == 1 and t.get_device() == dev):
            raise HipsterError(1, f"attn_prompt: {what} must be {q.dtype} [{R}][{heads}][{D}] on the device of q")
    if not (row_start.dtype is _I32 and row_start.dim() == 1 and row_start.is_contiguous() and row_start.get_device() == dev):
        raise HipsterError(1, "attn_prompt: row_start must be int32 [S + 1], contiguous, on the device of the rows")
    gr = (None, 0, 0)
    if gate is not None:
        if not (gate.dtype is _F32 and gate.shape == q.shape and gate.stride(2) == 1 and gate.get_device() == dev):
            raise HipsterError(1, f"attn_prompt: gate must be f32 [{R}][{n_head}][{D}] on the device of q")
        gr = (gate.data_ptr(), *gate.stride()[:2])
    out = q.new_empty((R, n_head, D)) if want_out else None
    xq = XQ8(R, n_head * D, q.device) if want_q8 else None
    check(more().hp_attn_prompt(q.data_ptr(), *q.stride()[:2], k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2], _OUT[q.dtype], *gr, n_head, n_kv, D, row_start.data_ptr(), row_start.numel() - 1, R, max_rows,
                                D ** -0.5 if scale is None else scale, None if out is None else out.data_ptr(), xq.q.data_ptr() if xq else None, xq.sc.data_ptr() if xq else None, _raw_stream(dev)))
    return out, xq
