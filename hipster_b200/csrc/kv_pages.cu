// A cache of 8-bit pages: rotary tables, appending rows with their rotation on the way, and reading tokens back as f16.
//
// k, v: codes [n_pages][n_kv][page][head_dim] in int8 or e4m3, k_scale, v_scale: f32 [n_pages][n_kv][page]: one scale per token and head. A
// scale shared by several tokens would grow with a row that a verify pass writes and then rejects, and kept tokens would be requantised for
// it: the speculative stream would no longer be the plain one. A scale per token costs 4 bytes beside head_dim codes and makes appending a
// plain store: the same token appended again leaves the same bytes.
#include "paged.cuh"
#include <algorithm>
#include <cuda_fp8.h>
#include <type_traits>

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
// the 64-bit pipe the bound (262144 x 64 entries: 69 us, now 28; the bytes alone 20). A block holds the functions of k < 32 and of its `groups` values of h; blocks of
// 1024 threads (of 256: 35), one per SM at a time by registers and shared memory, in two waves. Issue slots 72 %, the 64-bit pipe 26 %: instructions, and the functions at a block's start, during which nothing is written.
constexpr int ROPE_GROUP = 32;
__global__ void __launch_bounds__(1024) k_rope_table_sums(const RopeArgs a, int groups) {
    extern __shared__ __align__(16) double2 rope_sm[];
    __shared__ double f[128];
    pdl_launch_dependents();
    pdl_wait();
    if (threadIdx.x < a.half) f[threadIdx.x] = rope_freq(a, threadIdx.x);
    __syncthreads();
    double2* const near = rope_sm; double2* const far = rope_sm + ROPE_GROUP * a.half;   // (cos, sin), far ones times mul
    const int h0 = blockIdx.x * groups;
    for (int e = threadIdx.x; e < (ROPE_GROUP + groups) * a.half; e += 1024) {
        const int k = e / a.half;
        double s, c;
        sincos((k < ROPE_GROUP ? (double)k : (double)(h0 + k - ROPE_GROUP) * ROPE_GROUP) * f[e % a.half], &s, &c);
        rope_sm[e] = k < ROPE_GROUP ? make_double2(c, s) : make_double2(c * a.mul, s * a.mul);
    }
    __syncthreads();
    // a thread keeps k and i, and goes through the values of h: one read of shared memory per entry
    const int n = ROPE_GROUP * a.half;
    const size_t end = (size_t)a.n_pos * a.half;
    for (int e = threadIdx.x; e < n; e += 1024) {
        const double2 v = near[e];
        const double2* u = far + e % a.half;
        size_t at = (size_t)h0 * n + e;
#pragma unroll 4
        for (int h = 0; h < groups; ++h, at += n, u += a.half)
            if (at < end) a.table[at] = make_float2((float)(u->x * v.x - u->y * v.y), (float)(u->y * v.x + u->x * v.y));
    }
}

// NE codes of one lane from its quotients
template <int KIND> __device__ __forceinline__ uint32_t kv_code(float x) {
    if constexpr (KIND == KV_I8) return (uint32_t)min(127, max(-127, __float2int_rn(x))) & 0xffu;
    else return (uint32_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
// D / 8 lanes take a head of a row, eight neighbouring elements each, so that a warp has 1, 2 or 4 heads side by side; it takes hpw such sets of neighbouring
// heads (n_head query heads, then n_kv key heads, then n_kv value heads) in a loop that fetches a set ahead. The row's place and angles are found once. Four prompts of
// up to 1000 rows of 48 heads of 128: 22.5 us, 73 MB, 95 instructions per head (with a warp per head and the loop unrolled four times 220, which did not fit the instruction cache). Neither issue
// slots (56 %) nor memory (3.3 TB/s) are used up: the warps, 43 % of what an SM holds, wait for their next set of heads (4.6 of them at a time). One row of 32 heads of 256 3.3 us, latency.
template <int D, int KIND>
__global__ void __launch_bounds__(256, 4) k_kv_append(PagedPool pool, PagedBatch b, KvAppendParams p, int hpw, int* err) {
    constexpr int LPH = D / 8, HPS = 32 / LPH;   // lanes of a head, heads of a set
    __shared__ __align__(16) float buf[8][32 * 8];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LPH, d0 = (lane % LPH) * 8, heads = p.n_head + 2 * pool.n_kv, parts = (heads + hpw * HPS - 1) / (hpw * HPS);
    const unsigned mask = LPH == 32 ? 0xffffffffu : ((1u << (LPH & 31)) - 1u) << (sub * LPH);
    const long long item = (long long)blockIdx.x * 8 + warp;
    const int r = (int)(item / parts), h0 = (int)(item % parts) * hpw * HPS + sub, h1 = min(heads, h0 - sub + hpw * HPS);
    if (r >= b.R) return;
    float4 next[2];
    auto fetch = [&](int h) {
        const float* from = h < p.n_head ? p.q + (size_t)r * p.q_ld + (size_t)h * p.q_hs : h < p.n_head + pool.n_kv ? p.k + (size_t)r * p.k_ld + (size_t)(h - p.n_head) * p.k_hs
                                                                                            : p.v + (size_t)r * p.v_ld + (size_t)(h - p.n_head - pool.n_kv) * p.v_hs;
        next[0] = reinterpret_cast<const float4*>(from + d0)[0]; next[1] = reinterpret_cast<const float4*>(from + d0)[1];
    };
    const PagedSeq q = paged_find(b, r, lane, err);
    if (q.s < 0) return;
    if (h0 < h1) fetch(h0);   // a row of a sequence, and no other, is read
    const int pos = paged_place(q, r);
    if ((unsigned)pos >= (unsigned)min(b.max_kv, p.n_pos)) { paged_bad(err); return; }
    const uint32_t page = h1 > p.n_head ? paged_row(pool, q.s, pos >> pool.lg_page, 0, err) : 0u;
    const int half = p.n_rot / 2;
    // angles of the lane's elements; interleaved: of its four pairs
    float2 cs[8];
    const bool turns = d0 < p.n_rot;
    if (turns) {
        const float2* t = reinterpret_cast<const float2*>(p.rope) + (size_t)pos * half;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int d = d0 + j;
            if (d < p.n_rot && (!p.interleaved || !(j & 1))) cs[j] = t[p.interleaved ? d >> 1 : d < half ? d : d - half];
        }
    }
#pragma unroll 1
    for (int h = h0; h < h1; h += HPS) {
        float x[8] = {next[0].x, next[0].y, next[0].z, next[0].w, next[1].x, next[1].y, next[1].z, next[1].w};
        if (h + HPS < h1) fetch(h + HPS);
        const int kind = h < p.n_head ? 0 : h < p.n_head + pool.n_kv ? 1 : 2, hh = kind == 0 ? h : kind == 1 ? h - p.n_head : h - p.n_head - pool.n_kv;
        const uint16_t* nw = (const uint16_t*)(kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr);
        if (nw) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
            for (int off = LPH / 2; off > 0; off >>= 1) ss = ss + __shfl_xor_sync(mask, ss, off);
            const float inv = 1.0f / sqrtf(ss / (float)D + p.eps);
            const uint16_t* w = nw + d0;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (x[j] * inv) * bf2f(w[j]);
        }
        if (kind < 2 && p.n_rot) {
            if (p.interleaved) {   // the other one of a pair is the lane's own
#pragma unroll
                for (int j = 0; j < 8; j += 2)
                    if (d0 + j < p.n_rot) {
                        const float x0 = x[j], x1 = x[j + 1];
                        x[j] = fmaf(-x1, cs[j].y, x0 * cs[j].x); x[j + 1] = fmaf(x1, cs[j].x, x0 * cs[j].y);
                    }
            } else {
                float* row = buf[warp] + sub * D;
                __syncwarp(mask);
                reinterpret_cast<float4*>(row + d0)[0] = make_float4(x[0], x[1], x[2], x[3]); reinterpret_cast<float4*>(row + d0)[1] = make_float4(x[4], x[5], x[6], x[7]);
                __syncwarp(mask);
                if (turns) {
                    if (half % 8 == 0) {   // the lane's elements are all first or all second ones
                        const float* t = row + (d0 < half ? d0 + half : d0 - half);
                        const float4 u = reinterpret_cast<const float4*>(t)[0], v = reinterpret_cast<const float4*>(t)[1];
                        const float o[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w}, sign = d0 < half ? -1.f : 1.f;
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] = d0 < half ? fmaf(sign * o[j], cs[j].y, x[j] * cs[j].x) : fmaf(x[j], cs[j].x, o[j] * cs[j].y);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int d = d0 + j;
                            if (d < half) x[j] = fmaf(-row[d + half], cs[j].y, x[j] * cs[j].x); else if (d < p.n_rot) x[j] = fmaf(x[j], cs[j].x, row[d - half] * cs[j].y);
                        }
                    }
                }
            }
        }
        if (kind == 0) {
            float4* o = reinterpret_cast<float4*>(p.q_out + (size_t)r * p.qo_ld + (size_t)hh * p.qo_hs + d0);
            o[0] = make_float4(x[0], x[1], x[2], x[3]); o[1] = make_float4(x[4], x[5], x[6], x[7]);
            continue;
        }
        // largest magnitude, over the bit patterns: an infinity or a NaN wins, and the token is then marked by a NaN scale over codes of zero
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
        for (int off = LPH / 2; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(mask, m, off));
        if (page == 0xffffffffu) continue;
        const bool finite = m < 0x7f800000u;
        const float scale = finite ? __fdiv_rn(__uint_as_float(m), KIND == KV_I8 ? 127.f : 448.f) : __uint_as_float(0x7fc00000u);
        const bool live = finite && scale > 0.f;
        const float inv = live ? __fdiv_rn(1.f, scale) : 0.f;
        const size_t at = (size_t)page + ((size_t)hh << pool.lg_page) + (pos & ((1 << pool.lg_page) - 1));
        uint32_t w[2] = {0u, 0u};
        if (live) {
            if (inv < INFINITY) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j >> 2] |= kv_code<KIND>(x[j] * inv) << (8 * (j & 3));
            } else {   // a scale below 2^-128 has no reciprocal in 32 bits
                for (int j = 0; j < 8; ++j) w[j >> 2] |= kv_code<KIND>(__fdiv_rn(x[j], scale)) << (8 * (j & 3));
            }
        }
        *reinterpret_cast<uint2*>((kind == 1 ? pool.k : pool.v) + at * D + d0) = make_uint2(w[0], w[1]);
        if (d0 == 0) (kind == 1 ? pool.k_scale : pool.v_scale)[at] = scale;
    }
}

// RB rows per block, RB / 8 of them found by each warp; thread = 16 neighbouring codes of a row, a head and k or v, times the scale, rounded to f16 once. The e4m3
// patterns 0x7f and 0xff, which the quantiser does not write, read as 480 and -480. Bound by memory: 16 caches of up to 5000 tokens of 8 x 128 67 us (322 MB, 4.8 TB/s; pages of 16
// tokens are runs of 2 KB), with one piece in flight per thread 88; 4096 tokens of 4 x 256 7.4 us.
template <int D, int KIND, int RB>
__global__ void __launch_bounds__(256) k_kv_read(PagedPool pool, PagedBatch b, __half* __restrict__ ko, __half* __restrict__ vo, size_t row_stride, size_t head_stride, int* err) {
    constexpr int CPR = D / 16, PER = RB / 8;
    __shared__ uint32_t base[RB];   // of head 0
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r0 = blockIdx.x * RB;
    {
        int s = -1, pos = -1;   // of row `lane` of the warp's
        PagedSeq q{-1, 0, 0, 0, 0};
#pragma unroll 1
        for (int i = 0; i < PER; ++i) {
            const int r = r0 + warp * PER + i;
            if (r >= b.R) break;
            if (q.s < 0 || r >= q.row0 + q.T) q = paged_find(b, r, lane, err);   // neighbours mostly belong to one sequence
            if (q.s >= 0 && lane == i) { s = q.s; pos = paged_place(q, r); }
        }
        uint32_t at = 0xffffffffu;
        const bool fits = (unsigned)pos < (unsigned)b.max_kv;
        if (s >= 0 && !fits) paged_bad(err);
        if (s >= 0 && fits) { at = paged_row(pool, s, pos >> pool.lg_page, 0, err); if (at != 0xffffffffu) at += pos & ((1 << pool.lg_page) - 1); }
        if (lane < PER) base[warp * PER + lane] = at;
    }
    __syncthreads();
    const int n = 2 * pool.n_kv * RB * CPR;
    for (int i0 = threadIdx.x; i0 < n; i0 += 4 * 256) {   // four pieces of a thread in flight
        uint4 w[4]; float sc[4]; uint32_t row[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * 256, hv = i / (RB * CPR), c = i % CPR;
            row[u] = i < n ? base[i / CPR % RB] : 0xffffffffu;
            if (row[u] != 0xffffffffu) {
                const size_t at = (size_t)row[u] + ((size_t)(hv >> 1) << pool.lg_page);
                w[u] = *reinterpret_cast<const uint4*>((hv & 1 ? pool.v : pool.k) + at * D + c * 16);
                sc[u] = (hv & 1 ? pool.v_scale : pool.k_scale)[at];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (row[u] == 0xffffffffu) continue;
            const int i = i0 + u * 256, hv = i / (RB * CPR), c = i % CPR;
            const float s = KIND == KV_I8 ? sc[u] : sc[u] * 256.f;   // code_pair gives e4m3 codes times 2^-8
            const uint32_t ws[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t pr = j & 1 ? code_pair<KIND, 2>(ws[j / 2]) : code_pair<KIND, 0>(ws[j / 2]);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pr));
                o[j] = h2_bits(__floats2half2_rn(f.x * s, f.y * s));
            }
            uint4* dst = reinterpret_cast<uint4*>((hv & 1 ? vo : ko) + (size_t)(r0 + i / CPR % RB) * row_stride + (size_t)(hv >> 1) * head_stride + c * 16);
            dst[0] = make_uint4(o[0], o[1], o[2], o[3]); dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
    }
}

template <int D, int KIND> int launch_append(const PagedPool& pool, const PagedBatch& b, const KvAppendParams& p, cudaStream_t s) {
    const int heads = p.n_head + 2 * pool.n_kv;
    int* err = device_arg_flag();
    // One set of heads per warp while all of them fit on the GPU at once; six beyond. One and six, us: 256 rows of 48 heads of 128 6.7 and 7.9, 512 10.3 and 10.5, 1024 17.5 and 12.0, 4096 63 and 40; of 32
    // heads of 256 512 rows 12.5 and 13.0, 1024 21.9 and 20.8; of 24 heads of 64 1024 rows 6.7 and 8.0, 4096 17.5 and 13.0
    constexpr int HPS = 32 / (D / 8);
    const int hpw = (long long)b.R * heads <= 148 * 64 * HPS ? 1 : 6;
    const long long items = (long long)b.R * ((heads + hpw * HPS - 1) / (hpw * HPS));
    HP_CUDA(launch_pdl<4>(k_kv_append<D, KIND>, dim3((unsigned)((items + 7) / 8)), dim3(256), 0, s, pool, b, p, hpw, err));
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
    const int total = (int)(((long long)n_pos + ROPE_GROUP - 1) / ROPE_GROUP);
    int groups = (total + 2 * 148 - 1) / (2 * 148);   // two blocks per SM
    if (groups > ROPE_GROUP) groups = ROPE_GROUP;
    if (groups < 4) {   // fewer groups share too little: see k_rope_table_sums
        HP_CUDA(launch_pdl<4>(k_rope_table, dim3((unsigned)std::min<size_t>((n + 255) / 256, 148 * 8)), dim3(256), 0, s, a));
        return HP_OK;
    }
    static bool attr[MAX_DEVICES] = {};
    const int dev = current_device(); if (dev < 0) return HP_ECUDA;
    if (!attr[dev]) { HP_CUDA(cudaFuncSetAttribute(k_rope_table_sums, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * ROPE_GROUP * 128 * 16)); attr[dev] = true; }
    HP_CUDA(launch_pdl<4>(k_rope_table_sums, dim3((unsigned)((total + groups - 1) / groups)), dim3(1024), (size_t)(ROPE_GROUP + groups) * a.half * 16, s, a, groups));
    return HP_OK;
}
int kv_append(const PagedPool& pool, const PagedBatch& b, const KvAppendParams& p, cudaStream_t s) {
    return pool.kind == KV_I8 ? launch_append<KV_I8>(pool, b, p, s) : launch_append<KV_E4M3>(pool, b, p, s);
}
int kv_read(const PagedPool& pool, const PagedBatch& b, void* k_out, void* v_out, size_t row_stride, size_t head_stride, cudaStream_t s) {
    // 8 rows per block until there are several blocks for every SM; 32 beyond, where finding the rows bounds a block of 8. Eight and 32, us, 16 caches in pages of 16: 250 tokens each of 1 x 64 2.9 and 3.1, of 4 x 256 7.5
    // and 9.4; 5000 tokens of 1 x 64 24 and 12, of 1 x 256 43 and 28, of 4 x 64 44 and 29, of 8 x 128 98 and 100. Between, wide rows would do better with 8: 1000 tokens of 8 x 128 21 and 30, of 1 x 64 6.7 and 4.2
    const bool many = b.R > 148 * 32;
    int* err = device_arg_flag();
    auto go = [&](auto kernel, int rb) { return launch_pdl<4>(kernel, dim3((b.R + rb - 1) / rb), dim3(256), 0, s, pool, b, (__half*)k_out, (__half*)v_out, row_stride, head_stride, err); };
    auto type = [&](auto kind) {
        constexpr int KIND = decltype(kind)::value;
        return pool.head_dim == 256 ? (many ? go(k_kv_read<256, KIND, 32>, 32) : go(k_kv_read<256, KIND, 8>, 8)) : pool.head_dim == 128 ? (many ? go(k_kv_read<128, KIND, 32>, 32) : go(k_kv_read<128, KIND, 8>, 8))
                                                                                                                          : (many ? go(k_kv_read<64, KIND, 32>, 32) : go(k_kv_read<64, KIND, 8>, 8));
    };
    HP_CUDA(pool.kind == KV_I8 ? type(std::integral_constant<int, KV_I8>()) : type(std::integral_constant<int, KV_E4M3>()));
    return HP_OK;
}

}  // namespace hp
