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
struct RopeArgs { float2* table; int n_pos, half; double base; int scaling; double factor, orig_ctx, fast, slow, mul; };
__device__ __forceinline__ double rope_freq(const RopeArgs& a, int i) {
    double x = pow(a.base, -2.0 * i / (2.0 * a.half));
    if (a.scaling == 1) x = x / a.factor;
    if (a.scaling == 2) {
        double g = (a.orig_ctx * x / 6.283185307179586476925 - a.slow) / (a.fast - a.slow);
        g = fmin(1.0, fmax(0.0, g));
        x = x * (g + (1.0 - g) / a.factor);
    }
    return x;
}
// one sine and cosine per entry
__global__ void __launch_bounds__(256) k_rope_table(const RopeArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ double f[128];
    if (threadIdx.x < a.half) f[threadIdx.x] = rope_freq(a, threadIdx.x);
    __syncthreads();
    const size_t n = (size_t)a.n_pos * a.half;
    for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (size_t)gridDim.x * 256) {
        double s, c;
        sincos((double)(e / a.half) * f[e % a.half], &s, &c);
        a.table[e] = make_float2((float)(c * a.mul), (float)(s * a.mul));
    }
}
// Large tables: position 32 h + k by the addition theorems from 32 h and k, in 64 bits: four products instead of some 80 operations per entry, which left
// the 64-bit pipe the bound (262144 x 64 entries: 69 us; the bytes alone 20). A block holds the functions of k < 32 and of its `groups` values of h.
constexpr int ROPE_GROUP = 32;
__global__ void __launch_bounds__(256) k_rope_table_sums(const RopeArgs a, int groups) {
    extern __shared__ __align__(16) double2 rope_sm[];
    __shared__ double f[128];
    pdl_launch_dependents();
    pdl_wait();
    if (threadIdx.x < a.half) f[threadIdx.x] = rope_freq(a, threadIdx.x);
    __syncthreads();
    double2* const near = rope_sm; double2* const far = rope_sm + ROPE_GROUP * a.half;   // (cos, sin), far ones times mul
    const int h0 = blockIdx.x * groups;
    for (int e = threadIdx.x; e < (ROPE_GROUP + groups) * a.half; e += 256) {
        const int k = e / a.half;
        double s, c;
        sincos((k < ROPE_GROUP ? (double)k : (double)(h0 + k - ROPE_GROUP) * ROPE_GROUP) * f[e % a.half], &s, &c);
        rope_sm[e] = k < ROPE_GROUP ? make_double2(c, s) : make_double2(c * a.mul, s * a.mul);
    }
    __syncthreads();
    const int n = ROPE_GROUP * a.half;
    for (int h = 0; h < groups; ++h) {
        const size_t p0 = (size_t)(h0 + h) * ROPE_GROUP;
        if (p0 >= (size_t)a.n_pos) break;
        const int live = min(n, (int)min((size_t)n, ((size_t)a.n_pos - p0) * a.half));
        int i = threadIdx.x % a.half;
        const int step = 256 % a.half;
        for (int e = threadIdx.x; e < live; e += 256) {
            const double2 u = far[h * a.half + i], v = near[e];
            a.table[p0 * a.half + e] = make_float2((float)(u.x * v.x - u.y * v.y), (float)(u.y * v.x + u.x * v.y));
            i += step; if (i >= a.half) i -= a.half;
        }
    }
}

// NE codes of one lane from its quotients
template <int KIND> __device__ __forceinline__ uint32_t kv_code(float x) {
    if constexpr (KIND == KV_I8) return (uint32_t)min(127, max(-127, __float2int_rn(x))) & 0xffu;
    else return (uint32_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
// A warp takes HPW neighbouring heads of a row (n_head query heads, then n_kv key heads, then n_kv value heads), whose loads are all in flight before the row's
// place is known. A lane holds D / 32 elements of a head, in groups of four neighbours; a head goes through shared memory once, where each element finds the
// other one of its pair in either layout; the angles are the row's, read once.
template <int D, int KIND, int HPW>
__global__ void __launch_bounds__(256) k_kv_append(PagedPool pool, PagedBatch b, KvAppendParams p, int* err) {
    constexpr int NV = D >= 128 ? 4 : 2, NG = D / 32 / NV;   // neighbours of a group, groups of a lane
    __shared__ __align__(16) float buf[8][D];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = p.n_head + 2 * pool.n_kv, parts = (heads + HPW - 1) / HPW;
    const long long item = (long long)blockIdx.x * 8 + warp;
    const int r = (int)(item / parts), h0 = (int)(item % parts) * HPW;
    if (r >= b.R) return;
    float y[HPW][NG][NV];
#pragma unroll
    for (int i = 0; i < HPW; ++i) {
        const int h = h0 + i;
        if (h < heads) {
            const float* x = h < p.n_head ? p.q + (size_t)r * p.q_ld + h * p.q_hs : h < p.n_head + pool.n_kv ? p.k + (size_t)r * p.k_ld + (h - p.n_head) * p.k_hs : p.v + (size_t)r * p.v_ld + (h - p.n_head - pool.n_kv) * p.v_hs;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float* s = x + (g * 32 + lane) * NV;
                if constexpr (NV == 4) { const float4 t = *reinterpret_cast<const float4*>(s); y[i][g][0] = t.x; y[i][g][1] = t.y; y[i][g][2] = t.z; y[i][g][3] = t.w; }
                else { const float2 t = *reinterpret_cast<const float2*>(s); y[i][g][0] = t.x; y[i][g][1] = t.y; }
            }
        }
    }
    const PagedSeq q = paged_find(b, r, lane, err);
    if (q.s < 0) return;
    const int pos = q.len - q.T + r - q.row0;
    if (pos < 0 || pos >= p.n_pos) { paged_bad(err); return; }
    const uint32_t page = h0 + HPW > p.n_head ? paged_row(pool, q.s, pos >> pool.lg_page, 0, err) : 0u;
    const int half = p.n_rot / 2;
    float2 cs[NG][NV];
    if (p.n_rot && h0 < p.n_head + pool.n_kv) {
        const float2* t = reinterpret_cast<const float2*>(p.rope) + (size_t)pos * half;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int d = (g * 32 + lane) * NV + j;
                if (d < p.n_rot) cs[g][j] = t[p.interleaved ? d >> 1 : d < half ? d : d - half];
            }
    }
#pragma unroll
    for (int i = 0; i < HPW; ++i) {
        const int h = h0 + i;
        if (h >= heads) return;
        const int kind = h < p.n_head ? 0 : h < p.n_head + pool.n_kv ? 1 : 2, hh = kind == 0 ? h : kind == 1 ? h - p.n_head : h - p.n_head - pool.n_kv;
        float (&x)[NG][NV] = y[i];
        const uint16_t* nw = (const uint16_t*)(kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr);
        if (nw) {
            float ss = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int j = 0; j < NV; ++j) ss = fmaf(x[g][j], x[g][j], ss);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) ss = ss + __shfl_xor_sync(0xffffffffu, ss, off);
            const float inv = 1.0f / sqrtf(ss / (float)D + p.eps);
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int j = 0; j < NV; ++j) x[g][j] = (x[g][j] * inv) * bf2f(nw[(g * 32 + lane) * NV + j]);
        }
        if (kind < 2 && p.n_rot) {
            float* row = buf[warp];
            if (HPW > 1) __syncwarp();
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float* t = row + (g * 32 + lane) * NV;
                if constexpr (NV == 4) *reinterpret_cast<float4*>(t) = make_float4(x[g][0], x[g][1], x[g][2], x[g][3]);
                else *reinterpret_cast<float2*>(t) = make_float2(x[g][0], x[g][1]);
            }
            __syncwarp();
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int d = (g * 32 + lane) * NV + j;
                    if (d < p.n_rot) {
                        const bool first = p.interleaved ? !(d & 1) : d < half;
                        const float other = row[p.interleaved ? d ^ 1 : first ? d + half : d - half];
                        const float2 t = cs[g][j];
                        x[g][j] = first ? fmaf(-other, t.y, x[g][j] * t.x) : fmaf(x[g][j], t.x, other * t.y);
                    }
                }
        }
        if (kind == 0) {
            float* o = p.q_out + (size_t)r * p.qo_ld + hh * p.qo_hs;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float* t = o + (g * 32 + lane) * NV;
                if constexpr (NV == 4) *reinterpret_cast<float4*>(t) = make_float4(x[g][0], x[g][1], x[g][2], x[g][3]);
                else *reinterpret_cast<float2*>(t) = make_float2(x[g][0], x[g][1]);
            }
            continue;
        }
        if (page == 0xffffffffu) continue;
        // largest magnitude, over the bit patterns: an infinity or a NaN wins, and the token is then marked by a NaN scale over codes of zero
        uint32_t m = 0;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int j = 0; j < NV; ++j) m = max(m, __float_as_uint(x[g][j]) & 0x7fffffffu);
        m = __reduce_max_sync(0xffffffffu, m);
        const bool finite = m < 0x7f800000u;
        const float scale = finite ? __fdiv_rn(__uint_as_float(m), KIND == KV_I8 ? 127.f : 448.f) : __uint_as_float(0x7fc00000u);
        const bool live = finite && scale > 0.f;
        const size_t at = (size_t)page + ((size_t)hh << pool.lg_page) + (pos & ((1 << pool.lg_page) - 1));
        uint8_t* o = (kind == 1 ? pool.k : pool.v) + at * D;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < NV; ++j) w |= (live ? kv_code<KIND>(__fdiv_rn(x[g][j], scale)) : 0u) << (8 * j);
            if constexpr (NV == 4) reinterpret_cast<uint32_t*>(o)[g * 32 + lane] = w;
            else reinterpret_cast<uint16_t*>(o)[g * 32 + lane] = (uint16_t)w;
        }
        if (lane == 0) (kind == 1 ? pool.k_scale : pool.v_scale)[at] = scale;
    }
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
    for (int i0 = threadIdx.x; i0 < n; i0 += 4 * 256) {   // four pieces of a thread in flight
        uint4 w[4]; float sc[4]; size_t to[4]; bool live[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * 256, c = i % cpr, t = i / cpr % 8, hv = i / (8 * cpr), h = hv >> 1;
            live[u] = i < n && base[t] != 0xffffffffu;
            if (live[u]) {
                const size_t at = (size_t)base[t] + ((size_t)h << pool.lg_page);
                w[u] = *reinterpret_cast<const uint4*>((hv & 1 ? pool.v : pool.k) + at * D + c * 16);
                sc[u] = (hv & 1 ? pool.v_scale : pool.k_scale)[at];
                to[u] = (size_t)(r0 + t) * row_stride + (size_t)h * head_stride + c * 16;
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (!live[u]) continue;
            const int hv = (i0 + u * 256) / (8 * cpr);
            const uint32_t ws[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t v = ws[j / 2] >> (16 * (j & 1));
                const __half2 x = __floats2half2_rn(kv_value<KIND>(v & 0xffu) * sc[u], kv_value<KIND>((v >> 8) & 0xffu) * sc[u]);
                o[j] = *reinterpret_cast<const uint32_t*>(&x);
            }
            uint4* dst = reinterpret_cast<uint4*>((hv & 1 ? vo : ko) + to[u]);
            dst[0] = make_uint4(o[0], o[1], o[2], o[3]); dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
    }
}

template <int D, int KIND> int launch_append(const PagedPool& pool, const PagedBatch& b, const KvAppendParams& p, cudaStream_t s) {
    const int heads = p.n_head + 2 * pool.n_kv;
    int* err = device_arg_flag();
    // one head per warp while all of them fit on the GPU at once; four beyond
    const bool few = (long long)b.R * heads <= 148 * 64;
    const long long items = (long long)b.R * (few ? heads : (heads + 3) / 4);
    const dim3 grid((unsigned)((items + 7) / 8));
    HP_CUDA(few ? launch_pdl<4>(k_kv_append<D, KIND, 1>, grid, dim3(256), 0, s, pool, b, p, err) : launch_pdl<4>(k_kv_append<D, KIND, 4>, grid, dim3(256), 0, s, pool, b, p, err));
    return HP_OK;
}
template <int KIND> int launch_append(const PagedPool& pool, const PagedBatch& b, const KvAppendParams& p, cudaStream_t s) {
    return pool.head_dim == 256 ? launch_append<256, KIND>(pool, b, p, s) : pool.head_dim == 128 ? launch_append<128, KIND>(pool, b, p, s) : launch_append<64, KIND>(pool, b, p, s);
}

}  // namespace

int rope_table(float* table, int n_pos, int n_rot, double base, int scaling, double factor, int orig_ctx, double beta_fast, double beta_slow, double attn_factor, cudaStream_t s) {
    const double mul = scaling == 2 ? (attn_factor > 0 ? attn_factor : 0.1 * log(factor) + 1.0) : (attn_factor > 0 ? attn_factor : 1.0);
    RopeArgs a; a.table = (float2*)table; a.n_pos = n_pos; a.half = n_rot / 2; a.base = base; a.scaling = scaling; a.factor = factor; a.orig_ctx = orig_ctx; a.fast = beta_fast; a.slow = beta_slow; a.mul = mul;
    const size_t n = (size_t)n_pos * a.half;
    const int total = (n_pos + ROPE_GROUP - 1) / ROPE_GROUP;
    int groups = (total + 2 * 148 - 1) / (2 * 148);   // two blocks per SM
    if (groups > ROPE_GROUP) groups = ROPE_GROUP;
    if (groups < 4) {   // fewer groups share too little: see k_rope_table_sums
        HP_CUDA(launch_pdl<4>(k_rope_table, dim3((unsigned)std::min<size_t>((n + 255) / 256, 148 * 8)), dim3(256), 0, s, a));
        return HP_OK;
    }
    static bool attr[MAX_DEVICES] = {};
    const int dev = current_device(); if (dev < 0) return HP_ECUDA;
    if (!attr[dev]) { HP_CUDA(cudaFuncSetAttribute(k_rope_table_sums, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * ROPE_GROUP * 128 * 16)); attr[dev] = true; }
    HP_CUDA(launch_pdl<4>(k_rope_table_sums, dim3((unsigned)((total + groups - 1) / groups)), dim3(256), (size_t)(ROPE_GROUP + groups) * a.half * 16, s, a, groups));
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
