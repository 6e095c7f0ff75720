// extern "C" boundary: argument checks, status codes, last-error string. No exceptions cross it.
#include "hp_common.cuh"
#include "kernels.h"
#include "engine.h"
#include <cstring>
#include "../../include/hipster_b200.h"
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <string>
#include <algorithm>
#include <climits>
#include <exception>

namespace hp {
static thread_local std::string g_last_error;
void set_error(const char* fmt, ...) {
    char buf[512]; va_list ap; va_start(ap, fmt); vsnprintf(buf, sizeof buf, fmt, ap); va_end(ap);
    g_last_error = buf;
}
int cuda_fail(cudaError_t e, const char* what, const char* file, int line) {
    set_error("CUDA error %d (%s) in %s @%s:%d", (int)e, cudaGetErrorString(e), what, file, line);
    return HP_ECUDA;
}
// two status words per device: set by kernels whose bounded waits gave up (kernels that wait look at it), and by kernels that met lengths or indexes that do not fit
static int* g_dev_err[MAX_DEVICES] = {};
int* device_err_flag() {
    const int dev = current_device(); if (dev < 0) return nullptr;
    if (!g_dev_err[dev]) {   // on a stream of its own, and allowed while some stream is capturing: the first call on a device may be a captured one
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
        int* p = nullptr; cudaStream_t s = nullptr;
        const bool ok = cudaMalloc(&p, 2 * sizeof(int)) == cudaSuccess && cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking) == cudaSuccess &&
                        cudaMemsetAsync(p, 0, 2 * sizeof(int), s) == cudaSuccess && cudaStreamSynchronize(s) == cudaSuccess;
        if (s) cudaStreamDestroy(s);
        if (ok) g_dev_err[dev] = p; else if (p) cudaFree(p);
        cudaThreadExchangeStreamCaptureMode(&mode);
    }
    return g_dev_err[dev];
}
int* device_arg_flag() { int* p = device_err_flag(); return p ? p + 1 : nullptr; }
// workspace of the kernel-level GEMV entry point (per device, allocated on first use; the engine owns its own)
static GemvWorkspace g_ws[MAX_DEVICES] = {};
int default_gemv_workspace(GemvWorkspace* out, size_t need) {
    const int dev = current_device();
    HP_REQUIRE(dev >= 0, "no usable current CUDA device");
    GemvWorkspace& ws = g_ws[dev];
    if (need > ws.part_bytes) {
        if (ws.part) HP_CUDA(cudaFree(ws.part));
        ws.part = nullptr; ws.part_bytes = 0;
        HP_CUDA(cudaMalloc(&ws.part, need));
        ws.part_bytes = need;
    }
    ws.err = device_err_flag();
    *out = ws; return HP_OK;
}
}  // namespace hp

#define HP_GUARD_BEGIN try {
#define HP_GUARD_END } catch (const std::exception& e) { hp::set_error("exception: %s", e.what()); return HP_ESTATE; } catch (...) { hp::set_error("unknown exception"); return HP_ESTATE; }

extern "C" {

const char* hp_last_error(void) { return hp::g_last_error.c_str(); }
int hp_version(void) { return 100; }

int hp_device_status(void* stream) {
    HP_GUARD_BEGIN
    int* f = hp::device_err_flag();
    if (!f) { hp::set_error("cannot allocate the device status word"); return HP_ENOMEM; }
    int h[2] = {0, 0};
    HP_CUDA(cudaMemcpyAsync(h, f, sizeof h, cudaMemcpyDeviceToHost, (cudaStream_t)stream));
    HP_CUDA(cudaStreamSynchronize((cudaStream_t)stream));
    if (h[0] || h[1]) HP_CUDA(cudaMemsetAsync(h[0] ? f : f + 1, 0, sizeof(int), (cudaStream_t)stream));   // the one that is reported; the other one by the next call
    if (h[0]) { hp::set_error("a kernel gave up a bounded wait (device status %d)", h[0]); return h[0]; }
    if (h[1]) { hp::set_error("a kernel met a length or an index in device memory that does not fit (device status %d)", h[1]); return h[1]; }
    return HP_OK;
    HP_GUARD_END
}

size_t hp_xq8_q_bytes(int R, int K) { return hp::xq_q_bytes(R, K); }
size_t hp_xq8_sc_bytes(int R, int K) { return hp::xq_sc_floats(R, K) * sizeof(float); }

int hp_quantize_x_q8(const float* x_dev, int ldx, int R, int K, void* xq_q_dev, void* xq_sc_dev, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(x_dev && xq_q_dev && xq_sc_dev, "hp_quantize_x_q8: null pointer");
    return hp::quantize_x_q8(x_dev, ldx, hp::XQ8F{xq_q_dev, xq_sc_dev}, R, K, (cudaStream_t)stream);
    HP_GUARD_END
}
int hp_xq8_unpack(const void* xq_q_dev, const void* xq_sc_dev, int R, int K, int8_t* q_dev, float* d_dev, float* s_dev, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(xq_q_dev && xq_sc_dev && q_dev && d_dev && s_dev, "hp_xq8_unpack: null pointer");
    HP_REQUIRE(R >= 1 && K > 0 && K % 64 == 0, "hp_xq8_unpack: bad shape R=%d K=%d", R, K);
    return hp::xq8_unpack(hp::XQ8F{(void*)xq_q_dev, (void*)xq_sc_dev}, R, K, q_dev, d_dev, s_dev, (cudaStream_t)stream);
    HP_GUARD_END
}
int hp_dequant_q4k(const void* w_dev, size_t nblk, float* out_dev, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(w_dev && out_dev, "hp_dequant_q4k: null pointer");
    return hp::dequant_q4k(w_dev, nblk, out_dev, (cudaStream_t)stream);
    HP_GUARD_END
}
int hp_gemv_q4k_q8(const void* w_dev, const void* xq_q_dev, const void* xq_sc_dev, float* y_dev, int N, int K, int R, int ldy, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(w_dev && xq_q_dev && xq_sc_dev && y_dev, "hp_gemv_q4k_q8: null pointer");
    HP_REQUIRE(((uintptr_t)w_dev & 15) == 0, "hp_gemv_q4k_q8: weights must be 16-byte aligned");
    HP_REQUIRE(N > 0 && K > 0 && K % 256 == 0 && R >= 1 && R <= 32, "hp_gemv_q4k_q8: bad shape N=%d K=%d R=%d", N, K, R);
    hp::GemvWorkspace ws; { const int rc = hp::default_gemv_workspace(&ws, (size_t)4 * R * N * sizeof(float)); if (rc) return rc; }
    static const bool early = getenv("HIPSTER_B200_NO_PDL") == nullptr;
    return hp::gemv_q4k_q8(w_dev, hp::XQ8F{(void*)xq_q_dev, (void*)xq_sc_dev}, y_dev, N, K, R, ldy, ws, (cudaStream_t)stream, early, true);   // launched early, but the caller's weights are read behind the dependency wait
    HP_GUARD_END
}
int hp_gemv_parts(int N, int K) { return (N > 0 && K > 0 && K % 256 == 0) ? hp::gemv_parts(N, K) : 0; }
int hp_gemv_q4k_f32(const void* w_dev, const float* x_dev, float* y_dev, int N, int K, int R, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(w_dev && x_dev && y_dev, "hp_gemv_q4k_f32: null pointer");
    HP_REQUIRE(((uintptr_t)w_dev & 15) == 0, "hp_gemv_q4k_f32: weights must be 16-byte aligned");
    return hp::gemv_q4k_f32(w_dev, x_dev, y_dev, N, K, R, hp::device_err_flag(), (cudaStream_t)stream);
    HP_GUARD_END
}
size_t hp_argmax_scratch_bytes(int R, int n) { return (R < 1 || n < 1) ? 0 : hp::argmax_scratch_bytes(R, n); }
int hp_argmax(const float* logits_dev, int R, int n, int ld, int* ids_dev, float* vals_dev, void* scratch_dev, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(logits_dev && ids_dev, "hp_argmax: null pointer");
    return hp::argmax_rows(logits_dev, R, n, ld, ids_dev, vals_dev, scratch_dev, (cudaStream_t)stream);
    HP_GUARD_END
}
int hp_argmax_noalloc(const float* logits_dev, int R, int n, int ld, int* ids_dev, float* vals_dev, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(logits_dev && ids_dev, "hp_argmax_noalloc: null pointer");
    return hp::argmax_rows_static(logits_dev, R, n, ld, ids_dev, vals_dev, (cudaStream_t)stream);
    HP_GUARD_END
}
int hp_argmax_noalloc_max_rows(void) { return hp::argmax_static_max_rows(); }
int hp_argmax_noalloc_max_n(void) { return hp::argmax_static_max_n(); }
int hp_accept_greedy(const int* ids_dev, const int* drafts_dev, int n_draft, int* out_dev, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(ids_dev && out_dev && (drafts_dev || n_draft == 0), "hp_accept_greedy: null pointer");
    return hp::accept_greedy(ids_dev, drafts_dev, n_draft, out_dev, (cudaStream_t)stream);
    HP_GUARD_END
}

// ------------------------------------------------------------------ layer kernels
int hp_add_rmsnorm_quant(float* x_dev, const float* y_dev, int n_planes, size_t plane_stride, const void* w_bf16_dev, float* xn_dev, void* xq_q_dev, void* xq_sc_dev, int R, int n, float eps, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(x_dev && w_bf16_dev && xq_q_dev && xq_sc_dev && (y_dev || n_planes == 0), "hp_add_rmsnorm_quant: null pointer");
    return hp::add_rmsnorm_quant(x_dev, y_dev, n_planes, plane_stride, n, w_bf16_dev, xn_dev, hp::XQ8F{xq_q_dev, xq_sc_dev}, R, n, eps, (cudaStream_t)stream, false, nullptr, 0, true);
    HP_GUARD_END
}
int hp_silu_mul_quant(const float* gate_up_dev, int ld, int F, void* xq_q_dev, void* xq_sc_dev, int R, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(gate_up_dev && xq_q_dev && xq_sc_dev, "hp_silu_mul_quant: null pointer");
    return hp::silu_mul_quant(gate_up_dev, ld, F, hp::XQ8F{xq_q_dev, xq_sc_dev}, R, (cudaStream_t)stream);
    HP_GUARD_END
}
size_t hp_gdn_conv_state_floats(int n_v) { return (size_t)n_v * 3 * 384; }
size_t hp_gdn_saved_floats(int n_v) { return (size_t)n_v * 8 * 388; }
int hp_gdn_layer(const float* rows_dev, int ld, int T, int n_replay, int n_qk, int n_v, const float* conv_w_dev, const void* dt_bias_bf16_dev, const void* a_neg_bf16_dev,
                 const void* norm_w_bf16_dev, float* state_dev, float* conv_state_dev, float* saved_dev, float* out_dev, void* xq_q_dev, void* xq_sc_dev,
                 float* snap_dev, float eps, int sigmoid_gate, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(T >= 0 && T <= 8 && n_replay >= 0 && n_replay <= 8 && T + n_replay >= 1, "hp_gdn_layer: 0 <= T, n_replay <= 8 and T + n_replay >= 1");
    HP_REQUIRE((rows_dev || T == 0) && conv_w_dev && dt_bias_bf16_dev && a_neg_bf16_dev && norm_w_bf16_dev && state_dev && conv_state_dev && saved_dev, "hp_gdn_layer: null pointer");
    HP_REQUIRE(n_qk >= 1 && n_v >= n_qk && n_v % n_qk == 0 && ld >= (2 * n_qk + 2 * n_v) * 128 + 2 * n_v, "hp_gdn_layer: bad shape");
    hp::GdnParams g; g.rows = rows_dev ? rows_dev : state_dev; g.saved = saved_dev; g.saved_stride = 0; g.ld = ld; g.n_qk = n_qk; g.n_v = n_v;
    g.off_z = (2 * n_qk + n_v) * 128; g.off_b = g.off_z + n_v * 128; g.off_a = g.off_b + n_v;
    g.conv_w = conv_w_dev; g.dt_bias = dt_bias_bf16_dev; g.a_neg = a_neg_bf16_dev; g.norm_w = norm_w_bf16_dev;
    g.state = state_dev; g.conv_state = conv_state_dev; g.state_stride = 0; g.conv_stride = 0; g.seq = nullptr; g.replay_n = nullptr; g.imm_T = T; g.imm_replay = n_replay;   // one sequence, described by value
    g.out = out_dev; g.xq = hp::XQ8F{xq_q_dev, xq_sc_dev}; g.snap = snap_dev; g.snap_row_stride = (size_t)n_v * 128 * 128; g.eps = eps; g.sigmoid_gate = sigmoid_gate; g.late = true;
    return hp::gdn_forward(g, 1, (cudaStream_t)stream);
    HP_GUARD_END
}

size_t hp_attn_workspace_bytes(int R, int n_head, int n_kv, int max_ctx) {
    return (R < 1 || n_kv < 1 || n_head < n_kv || max_ctx < 1) ? 0 : hp::attn_seq_workspace_bytes(R, n_head, n_kv, max_ctx);
}
int hp_attn_decode(float* qkv_dev, int ld, int R, int pos0, int n_head, int n_kv, int n_rot, const void* q_norm_bf16_dev, const void* k_norm_bf16_dev, const float* rope_dev,
                   void* k_cache_dev, void* v_cache_dev, int max_ctx, float* out_dev, void* xq_q_dev, void* xq_sc_dev, float eps, void* workspace_dev, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(qkv_dev && q_norm_bf16_dev && k_norm_bf16_dev && rope_dev && k_cache_dev && v_cache_dev && workspace_dev && (out_dev || xq_q_dev), "hp_attn_decode: null pointer");
    HP_REQUIRE((xq_q_dev == nullptr) == (xq_sc_dev == nullptr), "hp_attn_decode: give both quantised-output buffers or neither");
    HP_REQUIRE(n_rot >= 2 && n_rot % 2 == 0 && n_rot <= 256 && ld % 4 == 0, "hp_attn_decode: bad n_rot / ld");
    return hp::attn_decode_seq(qkv_dev, ld, R, pos0, n_head, n_kv, n_rot, q_norm_bf16_dev, k_norm_bf16_dev, rope_dev, k_cache_dev, v_cache_dev, max_ctx, out_dev,
                               hp::XQ8F{xq_q_dev, xq_sc_dev}, eps, workspace_dev, (cudaStream_t)stream);
    HP_GUARD_END
}
size_t hp_q4k_tiled_bytes(size_t N, int K) { return (N < 1 || K < 256 || K % 256) ? 0 : hp::gemv_tiled_bytes(N, K); }
int hp_q4k_repack_tiled(const void* w_dev, void* w_tiled_dev, size_t N, int K, int interleave_half, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(w_dev && w_tiled_dev, "hp_q4k_repack_tiled: null pointer");
    HP_REQUIRE(((uintptr_t)w_dev & 3) == 0 && ((uintptr_t)w_tiled_dev & 15) == 0, "hp_q4k_repack_tiled: misaligned tensor");
    return hp::gemv_repack_tiled(w_dev, w_tiled_dev, N, K, (cudaStream_t)stream, interleave_half);
    HP_GUARD_END
}
// workspace of hp_moe_layer: router logits | per-pair outputs | ticket counters | quantised activations of the pairs | segments | control words
namespace {
struct MoeWs { size_t logits, cnt, v, q2, sc2, segs, ctl, total; };
MoeWs moe_ws(int T, int E, int F, int n_expert, int k) {
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    const size_t pairs = (size_t)T * (k + 1);
    MoeWs w; size_t o = 0;
    w.logits = o; o += al((size_t)T * (n_expert + 1) * 4);
    w.v = o; o += al(pairs * E * 4);
    w.cnt = o; o += al(32 * 4);   // from here on: cleared at the start of a call
    w.q2 = o; o += al(hp::xq_q_bytes((int)pairs, F));
    w.sc2 = o; o += al(hp::xq_sc_floats((int)pairs, F) * 4);
    w.segs = o; o += al(hp::moe_seg_bytes());
    w.ctl = o; o += 256;
    w.total = o; return w;
}
}
size_t hp_moe_workspace_bytes(int T, int E, int F, int n_expert, int k) { return (T < 1 || E < 1 || F < 1 || n_expert < 1 || k < 1) ? 0 : moe_ws(T, E, F, n_expert, k).total; }
int hp_moe_layer(const float* xn_dev, const void* xq_q_dev, const void* xq_sc_dev, const float* router_dev, const void* exp_gate_up_tiled_dev, const void* exp_down_tiled_dev,
                 const void* sh_gate_up_tiled_dev, const void* sh_down_tiled_dev, int T, int E, int F, int n_expert, int k, int* ids_dev, float* weights_dev, float* y_dev,
                 void* workspace_dev, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(xn_dev && xq_q_dev && xq_sc_dev && router_dev && exp_gate_up_tiled_dev && exp_down_tiled_dev && sh_gate_up_tiled_dev && sh_down_tiled_dev && ids_dev && weights_dev && y_dev && workspace_dev, "hp_moe_layer: null pointer");
    HP_REQUIRE(T >= 1 && T <= 32 && E % 256 == 0 && F % 256 == 0 && n_expert >= k && k >= 1 && k <= 15, "hp_moe_layer: bad shape T=%d E=%d F=%d experts=%d k=%d", T, E, F, n_expert, k);
    cudaStream_t s = (cudaStream_t)stream;
    const MoeWs w = moe_ws(T, E, F, n_expert, k);
    char* ws = (char*)workspace_dev; const int ns = k + 1;
    float* logits = (float*)(ws + w.logits); int* cnt = (int*)(ws + w.cnt); float* v = (float*)(ws + w.v);
    // the router kernel fetches its rows of router_dev in front of its dependency wait: the memset keeps its start behind all that the caller enqueued
    HP_CUDA(cudaMemsetAsync(cnt, 0, w.total - w.cnt, s));
    hp::MoeRouteParams rp; rp.W = router_dev; rp.x = xn_dev; rp.logits = logits; rp.E = n_expert; rp.K = E; rp.k = k; rp.T = T; rp.ids = ids_dev; rp.w = weights_dev; rp.ticket = cnt;
    rp.e_lo = 0; rp.e_hi = n_expert; rp.own_shared = 1; rp.segs = ws + w.segs; rp.ctl = (int*)(ws + w.ctl); rp.err = hp::device_err_flag();
    { const int rc = hp::moe_route_group(rp, s); if (rc) return rc; }
    hp::MoeGroupParams g; g.w_gate_up = exp_gate_up_tiled_dev; g.w_down = exp_down_tiled_dev; g.sh_gate_up = sh_gate_up_tiled_dev; g.sh_down = sh_down_tiled_dev;
    g.E = E; g.F = F; g.nslot = ns; g.T = T; g.e_lo = 0;
    g.xq = hp::XQ8F{(void*)xq_q_dev, (void*)xq_sc_dev}; g.xq2 = hp::XQ8F{ws + w.q2, ws + w.sc2}; g.v = v;
    g.segs = ws + w.segs; g.ctl = (int*)(ws + w.ctl); g.err = hp::device_err_flag();
    { const int rc = hp::moe_experts_grouped(g, s); if (rc) return rc; }
    return hp::moe_combine(v, weights_dev, y_dev, T, ns, E, s);
    HP_GUARD_END
}

// ------------------------------------------------------------------ paged cache in 8 or 4 bits, prompts
namespace {
// columns of the table in use, and the tokens that they hold
int columns_of(const hp_kv_pages* c, int table_ld) { return c->columns ? c->columns : table_ld; }
int capacity(const hp_kv_pages* c, int table_ld) { return columns_of(c, table_ld) * c->page_size; }
int paged_args(const char* who, const hp_kv_pages* c, const int* table, int table_ld, const int* row_start, const int* kv_len, int S, int R, long long max_rows, long long max_kv, hp::PagedPool* p, hp::PagedBatch* b) {
    HP_REQUIRE(c, "%s: null cache", who);
    HP_REQUIRE(c->type == HP_KV_I8 || c->type == HP_KV_E4M3 || c->type == HP_KV_I4, "%s: unknown cache type %d", who, c->type);
    HP_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "%s: head_dim must be 64, 128 or 256, not %d", who, c->head_dim);
    HP_REQUIRE(c->page_size >= 16 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0, "%s: page_size must be a power of two from 16 to 1024, not %d", who, c->page_size);
    const int columns = columns_of(c, table_ld);
    HP_REQUIRE(c->n_pages >= 1 && c->n_kv >= 1 && columns >= 1 && columns <= table_ld && (long long)c->n_pages * c->n_kv < (0xffffffffll / c->page_size) && (long long)columns * c->page_size < (1ll << 30),
               "%s: bad cache n_pages=%d n_kv=%d table_ld=%d columns=%d", who, c->n_pages, c->n_kv, table_ld, c->columns);
    HP_REQUIRE(S >= 1 && R >= 1 && max_rows >= 1 && max_kv >= 1, "%s: bad batch S=%d R=%d max_rows=%lld max_kv=%lld", who, S, R, max_rows, max_kv);
    p->k = (uint8_t*)c->k; p->v = (uint8_t*)c->v; p->k_scale = c->k_scale; p->v_scale = c->v_scale; p->table = table; p->table_ld = table_ld;
    p->kind = c->type; p->n_pages = c->n_pages; p->n_kv = c->n_kv; p->head_dim = c->head_dim; p->lg_page = 0;
    while ((1 << p->lg_page) < c->page_size) ++p->lg_page;
    b->row_start = row_start; b->kv_len = kv_len; b->S = S; b->R = R;
    b->max_rows = (int)(max_rows < R ? max_rows : R); b->max_kv = (int)std::min<long long>(max_kv, capacity(c, table_ld));
    return HP_OK;
}
int paged_ptrs(const char* who, const hp_kv_pages* c, const int* table, const int* row_start, const int* kv_len) {
    HP_REQUIRE(c->k && c->v && c->k_scale && c->v_scale && table && row_start && kv_len, "%s: null pointer", who);
    HP_REQUIRE((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0 && (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale | (uintptr_t)table | (uintptr_t)row_start | (uintptr_t)kv_len) & 3) == 0, "%s: misaligned cache or batch", who);
    return HP_OK;
}
// rows and heads of an output that do not lie over each other: one of the strides spans all that the other one reaches
bool apart(long long R, long long ld, long long heads, long long hs, long long dim) {
    auto nested = [&](long long n, long long inner, long long m, long long outer) { return (n == 1 || inner >= dim) && (m == 1 || (outer >= dim && (outer - dim) / (n > 1 ? n - 1 : 1) >= (n > 1 ? inner : 0))); };
    return nested(heads, hs, R, ld) || nested(R, ld, heads, hs);
}
// positions of several axes: the host's bytes as two bits per pair
int axes_args(const char* who, const int* pos, long long pos_ld, const unsigned char* axes, int n_axes, int n_rot, int R, hp::RopeAxes* o) {
    HP_REQUIRE(pos && axes, "%s: null positions or axes", who);
    HP_REQUIRE(n_axes >= 1 && n_axes <= 4 && ((uintptr_t)pos & 3) == 0 && (n_axes == 1 || pos_ld >= 0), "%s: bad positions n_axes=%d pos_ld=%lld", who, n_axes, pos_ld);
    HP_REQUIRE(n_rot >= 2 && n_rot <= 256, "%s: bad n_rot=%d for positions", who, n_rot);
    o->pos = pos; o->pos_ld = (size_t)pos_ld; o->n_axes = n_axes;
    for (int i = 0; i < 8; ++i) o->axes[i] = 0;
    for (int i = 0; i < n_rot / 2; ++i) {
        HP_REQUIRE(axes[i] < n_axes, "%s: pair %d has axis %d of %d", who, i, (int)axes[i], n_axes);
        o->axes[i >> 4] |= (uint32_t)axes[i] << (2 * (i & 15));
    }
    return HP_OK;
}
bool rows_ok(const void* p, long long ld, long long hs) { return ((uintptr_t)p & 15) == 0 && ld % 4 == 0 && hs % 4 == 0 && ld >= 0 && hs >= 0; }
}
int hp_rope_table(float* table_dev, int n_pos, int n_rot, double base, int scaling, double factor, int orig_ctx, double beta_fast, double beta_slow, double attn_factor, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(table_dev && ((uintptr_t)table_dev & 7) == 0, "hp_rope_table: null or misaligned table");
    HP_REQUIRE(n_pos >= 1 && n_rot >= 2 && n_rot % 2 == 0 && n_rot <= 256 && base > 0, "hp_rope_table: bad shape n_pos=%d n_rot=%d base=%g", n_pos, n_rot, base);
    HP_REQUIRE(scaling == HP_ROPE_NONE || scaling == HP_ROPE_LINEAR || scaling == HP_ROPE_YARN, "hp_rope_table: unknown scaling %d", scaling);
    HP_REQUIRE(scaling == HP_ROPE_NONE || (factor >= 1 && factor < 1e9), "hp_rope_table: factor must be at least 1");
    HP_REQUIRE(scaling != HP_ROPE_YARN || (orig_ctx >= 1 && beta_fast > beta_slow), "hp_rope_table: bad original context or betas");
    HP_REQUIRE(attn_factor >= 0, "hp_rope_table: bad attention factor");
    return hp::rope_table(table_dev, n_pos, n_rot, base, scaling, factor, orig_ctx, beta_fast, beta_slow, attn_factor, (cudaStream_t)stream);
    HP_GUARD_END
}
static int append(const char* who, const hp::RopeAxes& axes, const float* q_dev, long long q_ld, long long q_hs, float* q_out_dev, long long qo_ld, long long qo_hs, int n_head, const float* k_dev, long long k_ld, long long k_hs,
                  const float* v_dev, long long v_ld, long long v_hs, const void* q_norm_bf16_dev, const void* k_norm_bf16_dev, const float* rope_dev, int n_pos, int n_rot, int interleaved,
                  const int* table_dev, int table_ld, const int* row_start_dev, const int* kv_len_dev, int S, int R, const hp_kv_pages* pages, float eps, void* stream) {
    hp::PagedPool pool; hp::PagedBatch b;
    { int rc = paged_args(who, pages, table_dev, table_ld, row_start_dev, kv_len_dev, S, R, R, 1 << 30, &pool, &b); if (!rc) rc = paged_ptrs(who, pages, table_dev, row_start_dev, kv_len_dev); if (rc) return rc; }
    HP_REQUIRE(k_dev && v_dev && n_head >= 0 && (n_head == 0 || (q_dev && q_out_dev)) && (n_rot == 0 || rope_dev), "%s: null pointer", who);
    HP_REQUIRE(n_rot >= 0 && n_rot % 2 == 0 && n_rot <= pool.head_dim && (n_rot == 0 || n_pos >= 1) && ((uintptr_t)rope_dev & 7) == 0, "%s: bad n_rot=%d n_pos=%d or rope table", who, n_rot, n_pos);
    HP_REQUIRE(rows_ok(k_dev, k_ld, k_hs) && rows_ok(v_dev, v_ld, v_hs) && (n_head == 0 || (rows_ok(q_dev, q_ld, q_hs) && rows_ok(q_out_dev, qo_ld, qo_hs))), "%s: rows must be 16-byte aligned, with strides that are multiples of 4", who);
    HP_REQUIRE((((uintptr_t)q_norm_bf16_dev | (uintptr_t)k_norm_bf16_dev) & 1) == 0, "%s: norm weights must be 2-byte aligned", who);
    HP_REQUIRE(n_head == 0 || apart(R, qo_ld, n_head, qo_hs, pool.head_dim), "%s: rows of q_out lie over each other", who);
    HP_REQUIRE(n_head == 0 || q_dev != q_out_dev || ((R == 1 || q_ld == qo_ld) && (n_head == 1 || q_hs == qo_hs)), "%s: q_out in place of q must have its strides", who);
    HP_REQUIRE((long long)R * (n_head + 2 * pool.n_kv) < (1ll << 33), "%s: too many rows", who);
    hp::KvAppendParams p; p.q = q_dev; p.q_ld = q_ld; p.q_hs = q_hs; p.q_out = q_out_dev; p.qo_ld = qo_ld; p.qo_hs = qo_hs; p.n_head = n_head; p.k = k_dev; p.k_ld = k_ld; p.k_hs = k_hs;
    p.v = v_dev; p.v_ld = v_ld; p.v_hs = v_hs; p.q_norm = q_norm_bf16_dev; p.k_norm = k_norm_bf16_dev; p.rope = rope_dev; p.n_pos = n_rot ? n_pos : 1 << 30; p.n_rot = n_rot; p.interleaved = interleaved; p.eps = eps;
    return hp::kv_append(pool, b, p, axes, (cudaStream_t)stream);
}
int hp_kv_append(const float* q_dev, long long q_ld, long long q_hs, float* q_out_dev, long long qo_ld, long long qo_hs, int n_head, const float* k_dev, long long k_ld, long long k_hs,
                 const float* v_dev, long long v_ld, long long v_hs, const void* q_norm_bf16_dev, const void* k_norm_bf16_dev, const float* rope_dev, int n_pos, int n_rot, int interleaved,
                 const int* table_dev, int table_ld, const int* row_start_dev, const int* kv_len_dev, int S, int R, const hp_kv_pages* pages, float eps, void* stream) {
    HP_GUARD_BEGIN
    return append("hp_kv_append", hp::RopeAxes{}, q_dev, q_ld, q_hs, q_out_dev, qo_ld, qo_hs, n_head, k_dev, k_ld, k_hs, v_dev, v_ld, v_hs, q_norm_bf16_dev, k_norm_bf16_dev, rope_dev, n_pos, n_rot, interleaved, table_dev, table_ld,
                  row_start_dev, kv_len_dev, S, R, pages, eps, stream);
    HP_GUARD_END
}
int hp_kv_append_axes(const float* q_dev, long long q_ld, long long q_hs, float* q_out_dev, long long qo_ld, long long qo_hs, int n_head, const float* k_dev, long long k_ld, long long k_hs,
                      const float* v_dev, long long v_ld, long long v_hs, const void* q_norm_bf16_dev, const void* k_norm_bf16_dev, const float* rope_dev, int n_pos, int n_rot, int interleaved,
                      const int* pos_dev, long long pos_ld, const unsigned char* axes_host, int n_axes,
                      const int* table_dev, int table_ld, const int* row_start_dev, const int* kv_len_dev, int S, int R, const hp_kv_pages* pages, float eps, void* stream) {
    HP_GUARD_BEGIN
    hp::RopeAxes axes;
    { const int rc = axes_args("hp_kv_append_axes", pos_dev, pos_ld, axes_host, n_axes, n_rot, R, &axes); if (rc) return rc; }
    return append("hp_kv_append_axes", axes, q_dev, q_ld, q_hs, q_out_dev, qo_ld, qo_hs, n_head, k_dev, k_ld, k_hs, v_dev, v_ld, v_hs, q_norm_bf16_dev, k_norm_bf16_dev, rope_dev, n_pos, n_rot, interleaved, table_dev, table_ld,
                  row_start_dev, kv_len_dev, S, R, pages, eps, stream);
    HP_GUARD_END
}
int hp_rope_rows(const float* q_dev, long long q_ld, long long q_hs, void* q_out_dev, long long qo_ld, long long qo_hs, int n_head, const float* k_dev, long long k_ld, long long k_hs, void* k_out_dev, long long ko_ld, long long ko_hs,
                 const float* v_dev, long long v_ld, long long v_hs, void* v_out_dev, long long vo_ld, long long vo_hs, int n_kv, int head_dim, int out_type, const void* q_norm_bf16_dev, const void* k_norm_bf16_dev,
                 const float* rope_dev, int n_pos, int n_rot, int interleaved, const int* pos_dev, long long pos_ld, const unsigned char* axes_host, int n_axes, int R, float eps, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "hp_rope_rows: head_dim must be 64, 128 or 256, not %d", head_dim);
    HP_REQUIRE(out_type == HP_F32 || out_type == HP_F16 || out_type == HP_BF16, "hp_rope_rows: unknown output type %d", out_type);
    HP_REQUIRE(R >= 1 && n_head >= 0 && n_kv >= 0, "hp_rope_rows: bad shape R=%d n_head=%d n_kv=%d", R, n_head, n_kv);
    HP_REQUIRE(n_rot >= 0 && n_rot % 2 == 0 && n_rot <= head_dim && (n_rot == 0 || (n_pos >= 1 && rope_dev)) && ((uintptr_t)rope_dev & 7) == 0, "hp_rope_rows: bad n_rot=%d n_pos=%d or rope table", n_rot, n_pos);
    HP_REQUIRE((((uintptr_t)q_norm_bf16_dev | (uintptr_t)k_norm_bf16_dev) & 1) == 0, "hp_rope_rows: norm weights must be 2-byte aligned");
    hp::RopeAxes axes{};
    if (n_rot) { const int rc = axes_args("hp_rope_rows", pos_dev, pos_ld, axes_host, n_axes, n_rot, R, &axes); if (rc) return rc; }
    hp::RopeRowsParams p;
    const float* in[3] = {q_dev, k_dev, v_dev}; void* out[3] = {q_out_dev, k_out_dev, v_out_dev};
    const long long ld[3] = {q_ld, k_ld, v_ld}, hs[3] = {q_hs, k_hs, v_hs}, old[3] = {qo_ld, ko_ld, vo_ld}, ohs[3] = {qo_hs, ko_hs, vo_hs};
    int heads = 0;
    for (int i = 0; i < 3; ++i) {
        HP_REQUIRE((in[i] == nullptr) == (out[i] == nullptr), "hp_rope_rows: null pointer");
        const int n = in[i] ? (i ? n_kv : n_head) : 0;
        if (n) {
            HP_REQUIRE(rows_ok(in[i], ld[i], hs[i]) && rows_ok(out[i], old[i], ohs[i]) && (out_type == HP_F32 || ((old[i] | ohs[i]) & 7) == 0), "hp_rope_rows: rows must be 16-byte aligned, with strides that are multiples of 16 bytes");
            HP_REQUIRE(apart(R, old[i], n, ohs[i], head_dim), "hp_rope_rows: rows of an output lie over each other");
            HP_REQUIRE((const void*)in[i] != out[i] || (out_type == HP_F32 && (R == 1 || ld[i] == old[i]) && (n == 1 || hs[i] == ohs[i])), "hp_rope_rows: an output in place of its input must be f32 with its strides");
            for (int j = 0; j < i; ++j) HP_REQUIRE(!p.heads[j] || out[i] != out[j], "hp_rope_rows: two outputs are the same");
        }
        p.in[i] = in[i]; p.out[i] = out[i]; p.in_ld[i] = (size_t)ld[i]; p.in_hs[i] = (size_t)hs[i]; p.out_ld[i] = (size_t)old[i]; p.out_hs[i] = (size_t)ohs[i]; p.heads[i] = n;
        heads += n;
    }
    HP_REQUIRE(heads >= 1, "hp_rope_rows: no rows");
    for (int i = 0; i < 3; ++i)
        for (int j = 0; j < 3; ++j) HP_REQUIRE(i == j || !p.heads[i] || !p.heads[j] || out[i] != (const void*)in[j], "hp_rope_rows: an output in place of another one's input");
    HP_REQUIRE((long long)R * heads < (1ll << 33), "hp_rope_rows: too many rows");
    p.norm[0] = q_norm_bf16_dev; p.norm[1] = k_norm_bf16_dev; p.rope = rope_dev; p.n_pos = n_pos; p.n_rot = n_rot; p.interleaved = interleaved; p.eps = eps; p.R = R; p.head_dim = head_dim; p.type = out_type;
    return hp::rope_rows(p, axes, (cudaStream_t)stream);
    HP_GUARD_END
}
int hp_kv_read(const int* table_dev, int table_ld, const int* row_start_dev, const int* kv_len_dev, int S, int R, const hp_kv_pages* pages, void* k_out_f16_dev, void* v_out_f16_dev, long long row_stride, long long head_stride, void* stream) {
    HP_GUARD_BEGIN
    hp::PagedPool pool; hp::PagedBatch b;
    { int rc = paged_args("hp_kv_read", pages, table_dev, table_ld, row_start_dev, kv_len_dev, S, R, R, 1 << 30, &pool, &b); if (!rc) rc = paged_ptrs("hp_kv_read", pages, table_dev, row_start_dev, kv_len_dev); if (rc) return rc; }
    HP_REQUIRE(k_out_f16_dev && v_out_f16_dev, "hp_kv_read: null pointer");
    HP_REQUIRE((((uintptr_t)k_out_f16_dev | (uintptr_t)v_out_f16_dev) & 15) == 0 && row_stride >= 0 && head_stride >= 0 && row_stride % 8 == 0 && head_stride % 8 == 0, "hp_kv_read: outputs must be 16-byte aligned, with strides that are multiples of 8");
    HP_REQUIRE(apart(R, row_stride, pool.n_kv, head_stride, pool.head_dim), "hp_kv_read: rows of the outputs lie over each other");
    HP_REQUIRE(k_out_f16_dev != v_out_f16_dev, "hp_kv_read: k_out and v_out are the same");
    return hp::kv_read(pool, b, k_out_f16_dev, v_out_f16_dev, (size_t)row_stride, (size_t)head_stride, (cudaStream_t)stream);
    HP_GUARD_END
}
static int attn_paged_check(const char* who, int n_head, int window, int n_sink, const hp::PagedPool& pool) {
    HP_REQUIRE(n_head >= 1 && n_head % pool.n_kv == 0, "%s: n_head=%d must be a multiple of n_kv=%d", who, n_head, pool.n_kv);
    HP_REQUIRE(window >= 0 && n_sink >= 0 && (window > 0 || n_sink == 0), "%s: bad window=%d n_sink=%d (first tokens go with a window)", who, window, n_sink);
    return HP_OK;
}
size_t hp_attn_paged_workspace_bytes(int table_ld, int S, int R, int max_rows, int max_kv, int n_head, int window, int n_sink, const hp_kv_pages* pages) {
    hp::PagedPool pool; hp::PagedBatch b;
    if (paged_args("hp_attn_paged_workspace_bytes", pages, nullptr, table_ld, nullptr, nullptr, S, R, max_rows, max_kv, &pool, &b) || attn_paged_check("hp_attn_paged_workspace_bytes", n_head, window, n_sink, pool)) return 0;
    return hp::attn_paged_workspace_bytes(pool, b, n_head, window > 1 << 30 ? 1 << 30 : window, n_sink > 1 << 30 ? 1 << 30 : n_sink, capacity(pages, table_ld));
}
int hp_attn_paged(const float* q_dev, long long q_ld, long long q_hs, const float* gate_dev, long long g_ld, long long g_hs, int n_head, const int* table_dev, int table_ld, const int* row_start_dev, const int* kv_len_dev,
                  int S, int R, int max_rows, int max_kv, const hp_kv_pages* pages, float scale, int window, int n_sink, float* out_dev, void* xq_q_dev, void* xq_sc_dev, void* workspace_dev, void* stream) {
    HP_GUARD_BEGIN
    hp::PagedPool pool; hp::PagedBatch b;
    { int rc = paged_args("hp_attn_paged", pages, table_dev, table_ld, row_start_dev, kv_len_dev, S, R, max_rows, max_kv, &pool, &b); if (!rc) rc = paged_ptrs("hp_attn_paged", pages, table_dev, row_start_dev, kv_len_dev);
      if (!rc) rc = attn_paged_check("hp_attn_paged", n_head, window, n_sink, pool); if (rc) return rc; }
    HP_REQUIRE(q_dev && workspace_dev && (out_dev || xq_q_dev), "hp_attn_paged: null pointer");
    HP_REQUIRE((xq_q_dev == nullptr) == (xq_sc_dev == nullptr), "hp_attn_paged: give both quantised-output buffers or neither");
    HP_REQUIRE((((uintptr_t)xq_q_dev | (uintptr_t)xq_sc_dev) & 15) == 0, "hp_attn_paged: quantised outputs must be 16-byte aligned");
    HP_REQUIRE(rows_ok(q_dev, q_ld, q_hs) && (!gate_dev || (((uintptr_t)gate_dev & 3) == 0 && g_ld >= 0 && g_hs >= 0)) && ((uintptr_t)workspace_dev & 15) == 0 && ((uintptr_t)out_dev & 3) == 0,
               "hp_attn_paged: rows and workspace must be 16-byte aligned, with strides that are multiples of 4");
    HP_REQUIRE(scale > 0 && scale < 1e30f, "hp_attn_paged: bad scale");
    if (window > 1 << 30) window = 1 << 30;   // longer than any sequence
    if (n_sink > 1 << 30) n_sink = 1 << 30;
    hp::AttnPagedParams p; p.q = q_dev; p.q_ld = q_ld; p.q_hs = q_hs; p.gate = gate_dev; p.g_ld = g_ld; p.g_hs = g_hs; p.n_head = n_head; p.scale = scale; p.window = window; p.n_sink = n_sink; p.cap = capacity(pages, table_ld);
    p.out = out_dev; p.xq = hp::XQ8F{xq_q_dev, xq_sc_dev}; p.workspace = workspace_dev;
    return hp::attn_paged(pool, b, p, (cudaStream_t)stream);
    HP_GUARD_END
}

int hp_attn_prompt(const void* q_dev, long long q_ld, long long q_hs, const void* k_dev, long long k_ld, long long k_hs, const void* v_dev, long long v_ld, long long v_hs, int type, const float* gate_dev, long long g_ld, long long g_hs,
                   int n_head, int n_kv, int head_dim, const int* row_start_dev, int S, int R, int max_rows, float scale, void* out_dev, void* xq_q_dev, void* xq_sc_dev, void* stream) {
    HP_GUARD_BEGIN
    HP_REQUIRE(type == HP_F16 || type == HP_BF16, "hp_attn_prompt: type must be HP_F16 or HP_BF16, not %d", type);
    HP_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "hp_attn_prompt: head_dim must be 64, 128 or 256, not %d", head_dim);
    HP_REQUIRE(n_kv >= 1 && n_head >= 1 && n_head % n_kv == 0, "hp_attn_prompt: n_head=%d must be a multiple of n_kv=%d", n_head, n_kv);
    HP_REQUIRE(S >= 1 && S <= 65535 && R >= 1 && max_rows >= 1, "hp_attn_prompt: bad batch S=%d R=%d max_rows=%d", S, R, max_rows);
    HP_REQUIRE(R < INT_MAX - 256, "hp_attn_prompt: too many rows (%d)", R);   // tiles and blocks end up to 127 rows behind the last
    HP_REQUIRE(q_dev && k_dev && v_dev && row_start_dev && (out_dev || xq_q_dev), "hp_attn_prompt: null pointer");
    HP_REQUIRE((xq_q_dev == nullptr) == (xq_sc_dev == nullptr), "hp_attn_prompt: give both quantised-output buffers or neither");
    HP_REQUIRE((((uintptr_t)out_dev | (uintptr_t)xq_q_dev | (uintptr_t)xq_sc_dev) & 15) == 0 && ((uintptr_t)row_start_dev & 3) == 0, "hp_attn_prompt: outputs must be 16-byte aligned");
    auto fits = [&](const void* p, long long ld, long long hs, int heads) { return rows_ok(p, ld, hs) && ((ld | hs) & 7) == 0 && (R == 1 || (ld > 0 && ld < (1ll << 38))) && (heads == 1 || (hs > 0 && hs < (1ll << 38))); };
    HP_REQUIRE(fits(q_dev, q_ld, q_hs, n_head) && fits(k_dev, k_ld, k_hs, n_kv) && fits(v_dev, v_ld, v_hs, n_kv), "hp_attn_prompt: rows must be 16-byte aligned, with positive strides that are multiples of 8");
    HP_REQUIRE(!gate_dev || (rows_ok(gate_dev, g_ld, g_hs) && (R == 1 || (g_ld > 0 && g_ld < (1ll << 37))) && (n_head == 1 || (g_hs > 0 && g_hs < (1ll << 37)))), "hp_attn_prompt: the gate must be 16-byte aligned, with positive strides that are multiples of 4");
    HP_REQUIRE(scale > 0 && scale < 1e30f, "hp_attn_prompt: bad scale");
    for (const void* o : {(const void*)out_dev, (const void*)xq_q_dev, (const void*)xq_sc_dev})
        HP_REQUIRE(!o || (o != q_dev && o != k_dev && o != v_dev && o != gate_dev), "hp_attn_prompt: an output in place of an input, which other rows still read");
    HP_REQUIRE(!xq_q_dev || (xq_q_dev != xq_sc_dev && out_dev != xq_q_dev && out_dev != xq_sc_dev), "hp_attn_prompt: two outputs are the same");
    hp::AttnPromptParams p; p.q = q_dev; p.q_ld = (size_t)q_ld; p.q_hs = (size_t)q_hs; p.k = k_dev; p.k_ld = (size_t)k_ld; p.k_hs = (size_t)k_hs; p.v = v_dev; p.v_ld = (size_t)v_ld; p.v_hs = (size_t)v_hs; p.type = type;
    p.n_head = n_head; p.n_kv = n_kv; p.head_dim = head_dim; p.gate = gate_dev; p.g_ld = (size_t)g_ld; p.g_hs = (size_t)g_hs; p.row_start = row_start_dev; p.S = S; p.R = R; p.max_rows = max_rows < R ? max_rows : R; p.scale = scale;
    p.out = out_dev; p.xq = hp::XQ8F{xq_q_dev, xq_sc_dev};
    return hp::attn_prompt(p, (cudaStream_t)stream);
    HP_GUARD_END
}

// ------------------------------------------------------------------ engine
struct hp_engine { hp::Engine impl; explicit hp_engine(const hp_model_cfg& c) : impl(c) {} };

int hp_model_preset(const char* preset, hp_model_cfg* o) {
    HP_GUARD_BEGIN
    HP_REQUIRE(preset && o, "hp_model_preset: null pointer");
    memset(o, 0, sizeof *o);
    o->ep_rank = 0; o->ep_world = 1;
    o->rms_eps = 1e-6f; o->rope_base = 1e7f; o->n_rot = 64; o->attn_every = 4; o->has_mtp = 1; o->n_slots = 1;
    if (!strcmp(preset, "qwen35-27b")) {          // struct Qwen35Dims, engine/src/qwen35.h:15-26
        o->n_embd = 5120; o->n_layer = 64; o->n_ff = 17408; o->n_vocab = 248320; o->n_head = 24; o->n_head_kv = 4;
        o->gdn_qk_heads = 16; o->gdn_v_heads = 48; o->max_ctx = 8192; o->seed = 27;
    } else if (!strcmp(preset, "flash-next")) {   // benchmark configuration 4 shape (head geometry from struct FnDims, qwen4exp.h:18-28)
        o->n_embd = 2048; o->n_layer = 48; o->n_ff = 0; o->n_vocab = 248320; o->n_head = 24; o->n_head_kv = 2;
        o->gdn_qk_heads = 16; o->gdn_v_heads = 48; o->max_ctx = 4096; o->n_slots = 8; o->seed = 48;
        o->n_expert = 512; o->n_expert_used = 10; o->expert_ff = 512; o->gdn_sigmoid_gate = 1; o->synth_router_logits = 1;
    } else if (!strcmp(preset, "tiny")) {
        o->n_embd = 512; o->n_layer = 4; o->n_ff = 1024; o->n_vocab = 2048; o->n_head = 4; o->n_head_kv = 2;
        o->gdn_qk_heads = 2; o->gdn_v_heads = 4; o->max_ctx = 512; o->n_slots = 2; o->seed = 7;
    } else if (!strcmp(preset, "tiny-moe")) {
        o->n_embd = 512; o->n_layer = 4; o->n_ff = 0; o->n_vocab = 2048; o->n_head = 4; o->n_head_kv = 2;
        o->gdn_qk_heads = 2; o->gdn_v_heads = 4; o->max_ctx = 512; o->n_slots = 4; o->seed = 9;
        o->n_expert = 16; o->n_expert_used = 4; o->expert_ff = 256; o->gdn_sigmoid_gate = 1;
    } else { hp::set_error("unknown preset '%s'", preset); return HP_EINVAL; }
    return HP_OK;
    HP_GUARD_END
}
int hp_load(const hp_model_cfg* cfg, hp_engine** out) {
    HP_GUARD_BEGIN
    HP_REQUIRE(cfg && out, "hp_load: null pointer");
    hp_engine* e = new hp_engine(*cfg);
    const int rc = e->impl.init();
    if (rc != HP_OK) { delete e; *out = nullptr; return rc; }
    *out = e; return HP_OK;
    HP_GUARD_END
}
int hp_free(hp_engine* e) { delete e; return HP_OK; }
int hp_n_slots(const hp_engine* e) { return e ? e->impl.cfg().n_slots : 0; }
size_t hp_weight_bytes(const hp_engine* e) { return e ? e->impl.weight_bytes() : 0; }
float hp_last_ms(const hp_engine* e) { return e ? e->impl.last_ms() : 0.f; }
#define HP_ENGINE_CALL(expr) HP_GUARD_BEGIN HP_REQUIRE(e, "null engine handle"); return (expr); HP_GUARD_END
int hp_reset(hp_engine* e) { HP_ENGINE_CALL(e->impl.reset()) }
int hp_reset_slot(hp_engine* e, int slot) { HP_ENGINE_CALL(e->impl.reset_slot(slot)) }
int hp_forward(hp_engine* e, const hp_slot_req* reqs, int S, float* ms_out) { HP_ENGINE_CALL(e->impl.forward(reqs, S, ms_out)) }
int hp_accept(hp_engine* e, int slot, int m) { HP_ENGINE_CALL(e->impl.accept(slot, m)) }
int hp_mtp_forward(hp_engine* e, int slot, const int* tokens_host, const float* h_dev, int T, int pos0) { HP_ENGINE_CALL(e->impl.mtp_forward(tokens_host, h_dev, T, pos0, slot, true)) }
int hp_topk(hp_engine* e, int which, int T, int k, int* ids_host, float* vals_host) { HP_ENGINE_CALL(e->impl.topk(which, T, k, ids_host, vals_host)) }
int hp_prefill(hp_engine* e, int slot, const int* tokens_host, int n, int pos0, int with_mtp) { HP_ENGINE_CALL(e->impl.prefill(slot, tokens_host, n, pos0, with_mtp)) }
const float* hp_logits_dev(const hp_engine* e) { return e ? e->impl.logits() : nullptr; }
const float* hp_h_nextn_dev(const hp_engine* e) { return e ? e->impl.h_nextn() : nullptr; }
const float* hp_mtp_logits_dev(const hp_engine* e) { return e ? e->impl.mtp_logits() : nullptr; }
const float* hp_mtp_h_dev(const hp_engine* e) { return e ? e->impl.mtp_h() : nullptr; }
int hp_tensor_dev(const hp_engine* e, int layer, int kind, void** ptr_out, size_t* bytes_out) {
    HP_GUARD_BEGIN HP_REQUIRE(e && ptr_out && bytes_out, "hp_tensor_dev: null pointer"); return e->impl.tensor(layer, kind, ptr_out, bytes_out); HP_GUARD_END
}
int hp_gdn_state_dev(hp_engine* e, int slot, int gdn_layer, float** ptr_out, size_t* bytes_out) {
    HP_GUARD_BEGIN HP_REQUIRE(e && ptr_out && bytes_out, "hp_gdn_state_dev: null pointer"); return e->impl.gdn_state(slot, gdn_layer, ptr_out, bytes_out); HP_GUARD_END
}
int hp_mtp_forward_slots(hp_engine* e, const hp_slot_req* reqs, int S, const float* h_dev) { HP_ENGINE_CALL(e->impl.mtp_forward_reqs(reqs, S, h_dev, true)) }
int hp_ep_unique_id(void* id128_out) { HP_GUARD_BEGIN HP_REQUIRE(id128_out, "hp_ep_unique_id: null pointer"); return hp::Engine::ep_unique_id(id128_out); HP_GUARD_END }
int hp_ep_init(hp_engine* e, const void* id128) { HP_GUARD_BEGIN HP_REQUIRE(e && id128, "hp_ep_init: null pointer"); return e->impl.ep_init(id128); HP_GUARD_END }
int hp_profile_pass(hp_engine* e, int R, int what, int reps, float* ms_out) { HP_ENGINE_CALL(e->impl.profile_pass(R, what, reps, ms_out)) }
int hp_moe_touched(hp_engine* e, unsigned long long* n_out) { HP_ENGINE_CALL(e->impl.moe_touched(n_out)) }
int hp_ep_exchange_us(hp_engine* e, int R, int reps, float* us_out) { HP_ENGINE_CALL(e->impl.ep_exchange_us(R, reps, us_out)) }
int hp_ep_peer(hp_engine* e) { return e && e->impl.ep_peer() ? 1 : 0; }
int hp_ep_owner(int expert, int n_expert, int world) { return hp::ep_owner_of(expert, n_expert, world); }
int hp_ep_wait_probe(const void* flags_dev, int world, int rank, unsigned expect, void* stream) {
    HP_GUARD_BEGIN
    int* f = hp::device_err_flag();
    if (!f) { hp::set_error("cannot allocate the device status word"); return HP_ENOMEM; }
    return hp::ep_wait_probe((const unsigned*)flags_dev, world, rank, expect, f, (cudaStream_t)stream);
    HP_GUARD_END
}
int hp_last_round_kernels(const hp_engine* e) { return e ? e->impl.last_round_kernels() : 0; }
size_t hp_pass_weight_bytes(const hp_engine* e, int mtp, int with_head) { return e ? e->impl.pass_weight_bytes(mtp != 0, with_head != 0) : 0; }
int hp_spec_begin(hp_engine* e, int slot, int id_last, int pos, const float* h_pending_dev) { HP_ENGINE_CALL(e->impl.spec_begin(slot, id_last, pos, h_pending_dev)) }
int hp_spec_round(hp_engine* e, const int* slot_ids_host, int S, int n_draft, const int* subst_host, int* out_tokens_host, int* out_counts_host) {
    HP_ENGINE_CALL(e->impl.spec_round(slot_ids_host, S, n_draft, subst_host, out_tokens_host, out_counts_host))
}
int hp_ep_wait_poll(int (*stream_query)(void*), int (*comm_error)(void*), void* ctx, int limit_ms) {
    HP_GUARD_BEGIN return hp::ep_wait_poll(stream_query, comm_error, ctx, limit_ms); HP_GUARD_END
}

}  // extern "C"
