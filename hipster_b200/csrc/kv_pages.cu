// A cache of 8-bit pages: rotary tables, appending rows with their rotation on the way, and reading tokens back as f16.
//
// k, v: codes [n_pages][n_kv][page][head_dim] in int8 or e4m3, k_scale, v_scale: f32 [n_pages][n_kv][page]: one scale per token and head. A
// scale shared by several tokens would grow with a row that a verify pass writes and then rejects, and kept tokens would be requantised for
// it: the speculative stream would no longer be the plain one. A scale per token costs 4 bytes beside head_dim codes and makes appending a
// plain store: the same token appended again leaves the same bytes.
#include "paged.cuh"
#include <algorithm>
#include <cuda_fp8.h>

namespace hp {
namespace {

// ---- rotary table: [n_pos][n_rot / 2] (cos, sin) of pos * f_i, f_i = base^(-2 i / n_rot) and scaled. Linear: f_i / factor. By parts (YaRN, Peng et
// al. 2023, eq. 17 to 20 and 22): with r = orig_ctx * f_i / 2 pi turns over the original context and g = clamp((r - slow) / (fast - slow), 0, 1), f_i *
// (g + (1 - g) / factor), and cos and sin times `mul`. Angles and functions in 64 bits, one rounding at the end.
__global__ void __launch_bounds__(256) k_rope_table(float2* __restrict__ table, int n_pos, int half, double base, int scaling, double factor, double orig_ctx, double fast, double slow, double mul) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ double f[128];
    if (threadIdx.x < half) {
        const int i = threadIdx.x;
        double x = pow(base, -2.0 * i / (2.0 * half));
        if (scaling == 1) x = x / factor;
        if (scaling == 2) {
            double g = (orig_ctx * x / 6.283185307179586476925 - slow) / (fast - slow);
            g = fmin(1.0, fmax(0.0, g));
            x = x * (g + (1.0 - g) / factor);
        }
        f[i] = x;
    }
    __syncthreads();
    const size_t n = (size_t)n_pos * half;
    for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (size_t)gridDim.x * 256) {
        double s, c;
        sincos((double)(e / half) * f[e % half], &s, &c);
        table[e] = make_float2((float)(c * mul), (float)(s * mul));
    }
}

// NE codes of one lane from its quotients
template <int KIND> __device__ __forceinline__ uint32_t kv_code(float x) {
    if constexpr (KIND == KV_I8) return (uint32_t)min(127, max(-127, __float2int_rn(x))) & 0xffu;
    else return (uint32_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
// One warp per row and head (n_head query heads, then n_kv key heads, then n_kv value heads). A lane holds D / 32 elements, in groups of four
// neighbours; the row goes through shared memory once, where each element finds the other one of its pair in either layout.
template <int D, int KIND>
__global__ void __launch_bounds__(256) k_kv_append(PagedPool pool, PagedBatch b, KvAppendParams p, int* err) {
    constexpr int NV = D >= 128 ? 4 : 2, NG = D / 32 / NV;   // neighbours of a group, groups of a lane
    __shared__ __align__(16) float buf[8][D];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = p.n_head + 2 * pool.n_kv;
    const long long item = (long long)blockIdx.x * 8 + warp;
    const int r = (int)(item / heads), h = (int)(item % heads);
    if (r >= b.R) return;
    const PagedSeq q = paged_find(b, r, lane, err);
    if (q.s < 0) return;
    const int pos = q.len - q.T + r - q.row0;
    if (pos < 0 || pos >= p.n_pos) { paged_bad(err); return; }
    const int kind = h < p.n_head ? 0 : h < p.n_head + pool.n_kv ? 1 : 2, hh = kind == 0 ? h : kind == 1 ? h - p.n_head : h - p.n_head - pool.n_kv;
    const float* x = kind == 0 ? p.q + (size_t)r * p.q_ld + hh * p.q_hs : kind == 1 ? p.k + (size_t)r * p.k_ld + hh * p.k_hs : p.v + (size_t)r * p.v_ld + hh * p.v_hs;
    float y[NG][NV];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const float* s = x + (g * 32 + lane) * NV;
        if constexpr (NV == 4) { const float4 t = *reinterpret_cast<const float4*>(s); y[g][0] = t.x; y[g][1] = t.y; y[g][2] = t.z; y[g][3] = t.w; }
        else { const float2 t = *reinterpret_cast<const float2*>(s); y[g][0] = t.x; y[g][1] = t.y; }
    }
    const uint16_t* nw = (const uint16_t*)(kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr);
    if (nw) {
        float ss = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int j = 0; j < NV; ++j) ss = fmaf(y[g][j], y[g][j], ss);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) ss = ss + __shfl_xor_sync(0xffffffffu, ss, off);
        const float inv = 1.0f / sqrtf(ss / (float)D + p.eps);
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int j = 0; j < NV; ++j) y[g][j] = (y[g][j] * inv) * bf2f(nw[(g * 32 + lane) * NV + j]);
    }
    if (kind < 2 && p.n_rot) {
        float* row = buf[warp];
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int j = 0; j < NV; ++j) row[(g * 32 + lane) * NV + j] = y[g][j];
        __syncwarp();
        const int half = p.n_rot / 2;
        const float2* cs = reinterpret_cast<const float2*>(p.rope) + (size_t)pos * half;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int d = (g * 32 + lane) * NV + j;
                if (d < p.n_rot) {
                    const int i = p.interleaved ? d >> 1 : d < half ? d : d - half;
                    const bool first = p.interleaved ? !(d & 1) : d < half;
                    const float x0 = row[p.interleaved ? 2 * i : i], x1 = row[p.interleaved ? 2 * i + 1 : i + half];
                    const float2 t = cs[i];
                    y[g][j] = first ? fmaf(-x1, t.y, x0 * t.x) : fmaf(x1, t.x, x0 * t.y);
                }
            }
    }
    if (kind == 0) {
        float* o = p.q_out + (size_t)r * p.qo_ld + hh * p.qo_hs;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float* t = o + (g * 32 + lane) * NV;
            if constexpr (NV == 4) *reinterpret_cast<float4*>(t) = make_float4(y[g][0], y[g][1], y[g][2], y[g][3]);
            else *reinterpret_cast<float2*>(t) = make_float2(y[g][0], y[g][1]);
        }
        return;
    }
    // largest magnitude, over the bit patterns: an infinity or a NaN wins, and the token is then marked by a NaN scale over codes of zero
    uint32_t m = 0;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int j = 0; j < NV; ++j) m = max(m, __float_as_uint(y[g][j]) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    const bool finite = m < 0x7f800000u;
    const float scale = finite ? __fdiv_rn(__uint_as_float(m), KIND == KV_I8 ? 127.f : 448.f) : __uint_as_float(0x7fc00000u);
    const bool live = finite && scale > 0.f;
    const uint32_t base = paged_row(pool, q.s, pos >> pool.lg_page, hh, err);
    if (base == 0xffffffffu) return;
    const size_t at = (size_t)base + (pos & ((1 << pool.lg_page) - 1));
    uint8_t* o = (kind == 1 ? pool.k : pool.v) + at * D;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) w |= (live ? kv_code<KIND>(__fdiv_rn(y[g][j], scale)) : 0u) << (8 * j);
        if constexpr (NV == 4) reinterpret_cast<uint32_t*>(o)[g * 32 + lane] = w;
        else reinterpret_cast<uint16_t*>(o)[g * 32 + lane] = (uint16_t)w;
    }
    if (lane == 0) (kind == 1 ? pool.k_scale : pool.v_scale)[at] = scale;
}

// code times scale, rounded to f16 once; the e4m3 patterns 0x7f and 0xff, which the quantiser does not write, read as 480 and -480
template <int KIND> __device__ __forceinline__ float kv_value(uint32_t code) {
    if constexpr (KIND == KV_I8) return (float)(int8_t)code;
    else { const uint32_t h = ((code & 0x80u) << 8) | ((code & 0x7fu) << 7); return h2f((uint16_t)h) * 256.f; }
}
// 8 rows per block; thread = 16 neighbouring codes of a row, a head and k or v
template <int KIND>
__global__ void __launch_bounds__(256) k_kv_read(PagedPool pool, PagedBatch b, __half* __restrict__ ko, __half* __restrict__ vo, size_t row_stride, size_t head_stride, int* err) {
    __shared__ uint32_t base[8];   // of head 0
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r0 = blockIdx.x * 8, D = pool.head_dim, cpr = D / 16;
    const int page = 1 << pool.lg_page;
    {
        const int r = r0 + warp;
        uint32_t at = 0xffffffffu;
        if (r < b.R) {
            const PagedSeq q = paged_find(b, r, lane, err);
            const int pos = q.len - q.T + r - q.row0;
            if (q.s >= 0 && pos < 0) paged_bad(err);
            if (q.s >= 0 && pos >= 0) { at = paged_row(pool, q.s, pos >> pool.lg_page, 0, err); if (at != 0xffffffffu) at += pos & (page - 1); }
        }
        if (lane == 0) base[warp] = at;
    }
    __syncthreads();
    const int n = 2 * pool.n_kv * 8 * cpr;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int c = i % cpr, t = i / cpr % 8, hv = i / (8 * cpr), h = hv >> 1;
        if (base[t] == 0xffffffffu) continue;
        const size_t at = (size_t)base[t] + ((size_t)h << pool.lg_page);
        const uint4 w = *reinterpret_cast<const uint4*>((hv & 1 ? pool.v : pool.k) + at * D + c * 16);
        const float s = (hv & 1 ? pool.v_scale : pool.k_scale)[at];
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t u = ws[j / 2] >> (16 * (j & 1));
            const __half2 v = __floats2half2_rn(kv_value<KIND>(u & 0xffu) * s, kv_value<KIND>((u >> 8) & 0xffu) * s);
            o[j] = *reinterpret_cast<const uint32_t*>(&v);
        }
        uint4* dst = reinterpret_cast<uint4*>((hv & 1 ? vo : ko) + (size_t)(r0 + t) * row_stride + (size_t)h * head_stride + c * 16);
        dst[0] = make_uint4(o[0], o[1], o[2], o[3]); dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
}

template <int KIND> int launch_append(const PagedPool& pool, const PagedBatch& b, const KvAppendParams& p, cudaStream_t s) {
    const long long items = (long long)b.R * (p.n_head + 2 * pool.n_kv);
    const dim3 grid((unsigned)((items + 7) / 8));
    int* err = device_arg_flag();
    HP_CUDA(pool.head_dim == 256 ? launch_pdl<4>(k_kv_append<256, KIND>, grid, dim3(256), 0, s, pool, b, p, err)
            : pool.head_dim == 128 ? launch_pdl<4>(k_kv_append<128, KIND>, grid, dim3(256), 0, s, pool, b, p, err)
                                   : launch_pdl<4>(k_kv_append<64, KIND>, grid, dim3(256), 0, s, pool, b, p, err));
    return HP_OK;
}

}  // namespace

int rope_table(float* table, int n_pos, int n_rot, double base, int scaling, double factor, int orig_ctx, double beta_fast, double beta_slow, double attn_factor, cudaStream_t s) {
    const double mul = scaling == 2 ? (attn_factor > 0 ? attn_factor : 0.1 * log(factor) + 1.0) : (attn_factor > 0 ? attn_factor : 1.0);
    const size_t n = (size_t)n_pos * (n_rot / 2);
    HP_CUDA(launch_pdl<4>(k_rope_table, dim3((unsigned)std::min<size_t>((n + 255) / 256, 148 * 8)), dim3(256), 0, s, (float2*)table, n_pos, n_rot / 2, base, scaling, factor, (double)orig_ctx, beta_fast, beta_slow, mul));
    return HP_OK;
}
int kv_append(const PagedPool& pool, const PagedBatch& b, const KvAppendParams& p, cudaStream_t s) {
    return pool.kind == KV_I8 ? launch_append<KV_I8>(pool, b, p, s) : launch_append<KV_E4M3>(pool, b, p, s);
}
int kv_read(const PagedPool& pool, const PagedBatch& b, void* k_out, void* v_out, size_t row_stride, size_t head_stride, cudaStream_t s) {
    const dim3 grid((b.R + 7) / 8);
    int* err = device_arg_flag();
    HP_CUDA(pool.kind == KV_I8 ? launch_pdl<4>(k_kv_read<KV_I8>, grid, dim3(256), 0, s, pool, b, (__half*)k_out, (__half*)v_out, row_stride, head_stride, err)
                               : launch_pdl<4>(k_kv_read<KV_E4M3>, grid, dim3(256), 0, s, pool, b, (__half*)k_out, (__half*)v_out, row_stride, head_stride, err));
    return HP_OK;
}

}  // namespace hp
