// A cache of pages in 8 or 4 bits: rotary tables, appending rows with their rotation on the way (at the row's place, or at positions of several axes), reading tokens back as f16; and the same norm and
// rotation for rows that stay rows.
//
// k, v: codes [n_pages][n_kv][page][head_dim] in int8 or e4m3, k_scale, v_scale: f32 [n_pages][n_kv][page]: one scale per token and head. A
// scale shared by several tokens would grow with a row that a verify pass writes and then rejects, and kept tokens would be requantised for
// it: the speculative stream would no longer be the plain one. A scale per token costs 4 bytes beside head_dim codes and makes appending a
// plain store: the same token appended again leaves the same bytes. 4 bits (i4_row in paged.cuh) hold to that: the scale, the factors and the zeros of a head's groups are a token's own.
#include "paged.cuh"
#include <algorithm>
#include <cuda_bf16.h>
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
__device__ __forceinline__ float max_nan(float a, float b) { float y; asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b)); return y; }
__device__ __forceinline__ float min_nan(float a, float b) { float y; asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b)); return y; }
// A lane's 8 norm weights, in bf16: one load where they are aligned
__device__ __forceinline__ uint4 norm_words(const void* norm, int d0) {
    const uint16_t* const w = (const uint16_t*)norm + d0;
    if (((uintptr_t)w & 15) == 0) return *reinterpret_cast<const uint4*>(w);
    return make_uint4(w[0] | (uint32_t)w[1] << 16, w[2] | (uint32_t)w[3] << 16, w[4] | (uint32_t)w[5] << 16, w[6] | (uint32_t)w[7] << 16);
}
// A head's norm (weights `norm`, nullptr: none; HELD: fetched before) and rotation (n_rot = 0: none) where D / 8 lanes hold 8 neighbouring dims each; cs: angles of the lane's elements, interleaved of its four pairs; row: D floats of
// shared memory of these lanes
template <int D, bool HELD>
__device__ __forceinline__ void turn_head(float (&x)[8], const void* norm, uint4 held, int n_rot, int interleaved, float eps, const float2 (&cs)[8], int d0, unsigned mask, float* row) {
    constexpr int LPH = D / 8;
    const int half = n_rot / 2;
    const bool turns = d0 < n_rot;
    if (norm) {
        const uint4 nw = HELD ? held : norm_words(norm, d0);
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
        for (int off = LPH / 2; off > 0; off >>= 1) ss = ss + __shfl_xor_sync(mask, ss, off);
        const float inv = 1.0f / sqrtf(ss / (float)D + eps);
        const uint32_t w[4] = {nw.x, nw.y, nw.z, nw.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (x[j] * inv) * __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
    }
    if (!n_rot) return;
    if (interleaved) {   // the other one of a pair is the lane's own
#pragma unroll
        for (int j = 0; j < 8; j += 2)
            if (d0 + j < n_rot) {
                const float x0 = x[j], x1 = x[j + 1];
                x[j] = fmaf(-x1, cs[j].y, x0 * cs[j].x); x[j + 1] = fmaf(x1, cs[j].x, x0 * cs[j].y);
            }
        return;
    }
    __syncwarp(mask);
    reinterpret_cast<float4*>(row + d0)[0] = make_float4(x[0], x[1], x[2], x[3]); reinterpret_cast<float4*>(row + d0)[1] = make_float4(x[4], x[5], x[6], x[7]);
    __syncwarp(mask);
    if (!turns) return;
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
            if (d < half) x[j] = fmaf(-row[d + half], cs[j].y, x[j] * cs[j].x); else if (d < n_rot) x[j] = fmaf(x[j], cs[j].x, row[d - half] * cs[j].y);
        }
    }
}
// angles of the lane's elements (interleaved: of its four pairs) at one position
__device__ __forceinline__ void angles(float2 (&cs)[8], const float* rope, int pos, int n_rot, int interleaved, int d0) {
    const int half = n_rot / 2;
    const float2* t = reinterpret_cast<const float2*>(rope) + (size_t)pos * half;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int d = d0 + j;
        if (d < n_rot && (!interleaved || !(j & 1))) cs[j] = t[interleaved ? d >> 1 : d < half ? d : d - half];
    }
}
// Positions of a row, one per axis; false where one lies outside of the table
struct RowPos { int at[4]; };
__device__ __forceinline__ bool row_pos(RowPos& p, const RopeAxes& a, int r, int n_pos) {
    bool ok = true;
#pragma unroll
    for (int k = 0; k < 4; ++k) { p.at[k] = k < a.n_axes ? a.pos[(size_t)k * a.pos_ld + r] : 0; ok &= (unsigned)p.at[k] < (unsigned)n_pos; }
    return ok;
}
// position on axis k, chosen without a branch: lanes have different axes (four prompts of up to 1000 rows in 4 bits 31.6 -> 30.5 us, 8 x 3 rows 4.4 -> 3.75)
__device__ __forceinline__ int pick(const RowPos& p, uint32_t k) {
    int o;
    asm("{\n.reg .pred a, b;\n.reg .b32 t, u, v;\nand.b32 t, %5, 1;\nsetp.ne.u32 a, t, 0;\nand.b32 t, %5, 2;\nsetp.ne.u32 b, t, 0;\nselp.b32 u, %2, %1, a;\nselp.b32 v, %4, %3, a;\nselp.b32 %0, v, u, b;\n}"
        : "=r"(o) : "r"(p.at[0]), "r"(p.at[1]), "r"(p.at[2]), "r"(p.at[3]), "r"(k));
    return o;
}
__device__ __forceinline__ uint32_t axis_word(const RopeAxes& a, int w) {   // selected, not indexed: the words are kernel arguments
    uint32_t v = a.axes[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) v = w == i ? a.axes[i] : v;
    return v;
}
// the same angles where each pair has an axis of its own
__device__ __forceinline__ void angles(float2 (&cs)[8], const float* rope, const RowPos& p, const RopeAxes& a, int n_rot, int interleaved, int d0) {
    const int half = n_rot / 2;
    const float2* t = reinterpret_cast<const float2*>(rope);
    auto pair_of = [&](int d) { return interleaved ? d >> 1 : d < half ? d : d - half; };
    const bool run = interleaved || half % 8 == 0;   // the lane's pairs are 4 or 8 neighbours in one word
    uint32_t w = run ? axis_word(a, pair_of(d0) >> 4) : 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int d = d0 + j, i = pair_of(d);
        if (d >= n_rot || (interleaved && (j & 1))) continue;
        if (!run) w = axis_word(a, i >> 4);
        const uint32_t k = w >> (2 * (i & 15)) & 3u;
        cs[j] = t[(size_t)pick(p, k) * half + i];
    }
}
// D / 8 lanes take a head of a row, eight neighbouring elements each, so that a warp has 1, 2 or 4 heads side by side; it takes hpw such sets of neighbouring
// heads (n_head query heads, then n_kv key heads, then n_kv value heads) in a loop that fetches a set ahead. The row's place and angles are found once. Four prompts of
// up to 1000 rows of 48 heads of 128, normalised: 26 us, 73 MB of DRAM traffic, 95 instructions per head (with a warp per head and the loop unrolled four times 220, which did not fit the instruction cache). Neither issue
// slots (56 %) nor memory (3.3 TB/s) are used up: the warps, 43 % of what an SM holds, wait for their next set of heads (4.6 of them at a time). One row of 32 heads of 256 3.3 us, latency.
// AXES: positions of several axes. 4 bits: four lanes share a group; its range takes four exchanges, the largest range of the head the others. The same four prompts of 48 heads of 128 with three axes 28.3 us, to 4 bits 30.5 to 31, at the rows' places 29.2;
// 160 instructions per head, issue slots 58 %, otherwise waiting for exchanges and rows, in 1.6 waves of blocks. 8 x 3 rows of 24 + 4 heads of 256 3.75, latency.
template <int D, int KIND, bool AXES>
__global__ void __launch_bounds__(256, 4) k_kv_append(PagedPool pool, PagedBatch b, KvAppendParams p, RopeAxes axes, int hpw, int* err) {
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
    RowPos at;
    float2 cs[8];
    bool placed = true;
    if constexpr (AXES) {   // under way while the sequence is looked up
        placed = row_pos(at, axes, r, p.n_pos);
        if (placed && d0 < p.n_rot) angles(cs, p.rope, at, axes, p.n_rot, p.interleaved, d0);
    }
    const PagedSeq q = paged_find(b, r, lane, err);
    if (q.s < 0) return;
    if (h0 < h1) fetch(h0);   // a row of a sequence, and no other, is read
    const int pos = paged_place(q, r);
    if (!placed || (unsigned)pos >= (unsigned)(AXES ? b.max_kv : min(b.max_kv, p.n_pos))) { paged_bad(err); return; }
    const uint32_t page = h1 > p.n_head ? paged_row(pool, q.s, pos >> pool.lg_page, 0, err) : 0u;
    if (!AXES && d0 < p.n_rot) angles(cs, p.rope, pos, p.n_rot, p.interleaved, d0);
    // Norm weights are kept from head to head, and fetched again where k's follow q's: four prompts of up to 1000 rows in 8 bits 27.6 -> 26.0 us. With axes they would spill others (4 bits 31.6 -> 33.1)
    constexpr bool HELD = !AXES;
    int held = -1;
    uint4 nw = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
    for (int h = h0; h < h1; h += HPS) {
        float x[8] = {next[0].x, next[0].y, next[0].z, next[0].w, next[1].x, next[1].y, next[1].z, next[1].w};
        if (h + HPS < h1) fetch(h + HPS);
        const int kind = h < p.n_head ? 0 : h < p.n_head + pool.n_kv ? 1 : 2, hh = kind == 0 ? h : kind == 1 ? h - p.n_head : h - p.n_head - pool.n_kv;
        const void* const norm = kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr;
        if constexpr (HELD) if (norm && held != kind) { held = kind; nw = norm_words(norm, d0); }
        turn_head<D, HELD>(x, norm, nw, kind < 2 ? p.n_rot : 0, p.interleaved, p.eps, cs, d0, mask, buf[warp] + sub * D);
        if (kind == 0) {
            float4* o = reinterpret_cast<float4*>(p.q_out + (size_t)r * p.qo_ld + (size_t)hh * p.qo_hs + d0);
            o[0] = make_float4(x[0], x[1], x[2], x[3]); o[1] = make_float4(x[4], x[5], x[6], x[7]);
            continue;
        }
        if constexpr (KIND == KV_I4) {
            // A group spans lo to hi, zero among them, in 15 steps of scale * u; halves, since hi - lo may pass the largest number. The largest span of the head has u = 15. Infinities and NaN stay in spans, and
            // the token is then marked by a NaN scale over codes of zero
            float lo = 0.f, hi = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) { lo = min_nan(lo, x[j]); hi = max_nan(hi, x[j]); }
#pragma unroll
            for (int off = 1; off < 4; off <<= 1) { lo = min_nan(lo, __shfl_xor_sync(mask, lo, off)); hi = max_nan(hi, __shfl_xor_sync(mask, hi, off)); }
            const float span = 0.5f * hi - 0.5f * lo;
            float most = span;
#pragma unroll
            for (int off = LPH / 2; off >= 4; off >>= 1) most = max_nan(most, __shfl_xor_sync(mask, most, off));
            if (page == 0xffffffffu) continue;
            const bool finite = most < INFINITY;
            const float scale = finite ? __fdiv_rn(most, 112.5f) : __uint_as_float(0x7fc00000u);
            uint32_t w = 0, group = 0;
            if (finite && scale > 0.f) {
                const float f = most > 1e37f ? 0.0625f : 1.f, ratio = fminf(ceilf(__fdiv_rn(15.f * (span * f), most * f)), 15.f);   // u
                const float step = scale * ratio;
                if (step > 0.f) {
                    const float inv = __fdiv_rn(1.f, step);
                    int z;
                    if (inv < INFINITY) {   // rounded by adding 1.5 * 2^23: the whole number is in the low bits, as a difference of bit patterns
                        constexpr float BIG = 12582912.f;
                        const int unit = __float_as_int(BIG);
                        z = min(15, __float_as_int(-lo * inv + BIG) - unit);
#pragma unroll
                        for (int j = 0; j < 8; ++j) w += (uint32_t)max(0, min(15, __float_as_int(x[j] * inv + BIG) + (z - unit))) << (4 * j);
                    } else {   // a step below 2^-128 has no reciprocal in 32 bits
                        z = (int)fminf(rintf(__fdiv_rn(-lo, step)), 15.f);
#pragma unroll 1
                        for (int j = 0; j < 8; ++j) {
                            float y = 0.f;
#pragma unroll
                            for (int e = 0; e < 8; ++e) if (e == j) y = x[e];
                            w |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(y, step)) + (float)z, 0.f), 15.f) << (4 * j);
                        }
                    }
                    group = (uint32_t)z | (uint32_t)ratio << 4;
                }
            }
            const size_t at_row = (size_t)page + ((size_t)hh << pool.lg_page) + (pos & ((1 << pool.lg_page) - 1));
            const I4Row to = i4_row((uint32_t)at_row, pool.lg_page, D);
            uint8_t* const base = kind == 1 ? pool.k : pool.v;
            *reinterpret_cast<uint32_t*>(base + to.codes + d0 / 2) = w;
            if (d0 % 32 == 0) base[to.groups + d0 / 32] = (uint8_t)group;
            if (d0 == 0) (kind == 1 ? pool.k_scale : pool.v_scale)[at_row] = scale;
        } else {
            // largest magnitude, over the bit patterns: an infinity or a NaN wins, and the token is then marked by a NaN scale over codes of zero
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
            for (int off = LPH / 2; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(mask, m, off));
            if (page == 0xffffffffu) continue;
            const bool finite = m < 0x7f800000u;
            const size_t at_row = (size_t)page + ((size_t)hh << pool.lg_page) + (pos & ((1 << pool.lg_page) - 1));
            const float scale = finite ? __fdiv_rn(__uint_as_float(m), KIND == KV_I8 ? 127.f : 448.f) : __uint_as_float(0x7fc00000u);
            const bool live = finite && scale > 0.f;
            const float inv = live ? __fdiv_rn(1.f, scale) : 0.f;
            uint32_t w[2] = {0u, 0u};
            if (live) {
                if (inv < INFINITY) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j >> 2] |= kv_code<KIND>(x[j] * inv) << (8 * (j & 3));
                } else {   // a scale below 2^-128 has no reciprocal in 32 bits
                    for (int j = 0; j < 8; ++j) w[j >> 2] |= kv_code<KIND>(__fdiv_rn(x[j], scale)) << (8 * (j & 3));
                }
            }
            *reinterpret_cast<uint2*>((kind == 1 ? pool.k : pool.v) + at_row * D + d0) = make_uint2(w[0], w[1]);
            if (d0 == 0) (kind == 1 ? pool.k_scale : pool.v_scale)[at_row] = scale;
        }
    }
}

// RB rows per block, RB / 8 of them found by each warp; thread = 16 neighbouring codes of a row, a head and k or v, times the scale, rounded to f16 once. The e4m3
// patterns 0x7f and 0xff, which the quantiser does not write, read as 480 and -480. Bound by memory: 16 caches of up to 5000 tokens of 8 x 128 66 us (322 MB, 4.9 TB/s; pages of 16
// tokens are runs of 2 KB), with one piece in flight per thread 88; 4096 tokens of 4 x 256 7.4 us. 4 bits: a word of 8 codes per piece, eight pieces in flight; bound by instructions (issue slots 78 %, 214 MB of it written or read):
// the same caches 61 us, 4096 tokens 7.2. Where a row's codes lie, looked up once per row in shared memory: 63.8.
template <int D, int KIND, int RB>
__global__ void __launch_bounds__(256) k_kv_read(PagedPool pool, PagedBatch b, __half* __restrict__ ko, __half* __restrict__ vo, size_t row_stride, size_t head_stride, int* err) {
    constexpr int PIECE = KIND == KV_I4 ? 8 : 16, CPR = D / PIECE, PER = RB / 8;   // codes of a thread's piece
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
    constexpr int FLY = KIND == KV_I4 ? 8 : 4;   // pieces of a thread in flight
    for (int i0 = threadIdx.x; i0 < n; i0 += FLY * 256) {
        uint4 w[FLY]; float sc[FLY]; uint32_t row[FLY], group[FLY];
#pragma unroll
        for (int u = 0; u < FLY; ++u) {
            const int i = i0 + u * 256, hv = i / (RB * CPR), c = i % CPR;
            row[u] = i < n ? base[i / CPR % RB] : 0xffffffffu;
            if (row[u] != 0xffffffffu) {
                const size_t at = (size_t)row[u] + ((size_t)(hv >> 1) << pool.lg_page);
                const uint8_t* const from = hv & 1 ? pool.v : pool.k;
                if constexpr (KIND == KV_I4) {   // a word of codes: 16 bytes of the output per lane
                    const I4Row at4 = i4_row((uint32_t)at, pool.lg_page, D);
                    w[u].x = *reinterpret_cast<const uint32_t*>(from + at4.codes + c * 4);
                    group[u] = from[at4.groups + c / 4];
                } else w[u] = *reinterpret_cast<const uint4*>(from + at * D + c * 16);
                sc[u] = (hv & 1 ? pool.v_scale : pool.k_scale)[at];
            }
        }
#pragma unroll
        for (int u = 0; u < FLY; ++u) {
            if (row[u] == 0xffffffffu) continue;
            const int i = i0 + u * 256, hv = i / (RB * CPR), c = i % CPR;
            auto place = [&] { return reinterpret_cast<uint4*>((hv & 1 ? vo : ko) + (size_t)(r0 + i / CPR % RB) * row_stride + (size_t)(hv >> 1) * head_stride + c * PIECE); };
            constexpr bool EARLY = KIND == KV_E4M3 && D == 128;   // what is worked out in front of the products the compiler has in registers with the loads. 16 caches, us, in front and behind: of up to 5000 tokens of 8 x 128 e4m3 72.4 and
                                                                  // 75.5, int8 85.4 and 73.7, 4 bits 63.2 and 62.3; of 5000 of 4 x 256 e4m3 116.9 and 114.5, 4 bits 88.7 and 87.1; of 4 x 64 int8 29.7 and 28.1
            uint4* dst = nullptr;
            if constexpr (EARLY) dst = place();
            // code_pair gives e4m3 codes times 2^-8, i4_word 4 bits times 1 / I4_UNIT. A scale that is too large for that factor: what is not zero becomes infinite in f16 with a smaller one too
            const float s = KIND == KV_E4M3 ? sc[u] * 256.f : KIND == KV_I4 ? (sc[u] > 8e34f && sc[u] < INFINITY ? 8e34f : sc[u]) * I4_UNIT : sc[u];
            constexpr int N = PIECE / 2;
            uint32_t o[N];
            if constexpr (KIND == KV_I4) { const uint4 t = i4_word(w[u].x, i4_group(__byte_perm(group[u], 0x64u, 0x4040))); o[0] = t.x; o[1] = t.y; o[2] = t.z; o[3] = t.w; }
            const uint32_t ws[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
            for (int j = 0; j < N; ++j) {
                uint32_t pr;
                if constexpr (KIND == KV_I4) pr = o[j]; else pr = j & 1 ? code_pair<KIND, 2>(ws[j / 2]) : code_pair<KIND, 0>(ws[j / 2]);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pr));
                o[j] = h2_bits(__floats2half2_rn(f.x * s, f.y * s));
            }
            if constexpr (!EARLY) dst = place();
            dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
            if constexpr (N == 8) dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
    }
}

// Rows of q, k and v, each head's norm and rotation, to outputs of another type: what k_kv_append does for rows that stay rows. The same lanes, sets of heads and loop. Bound by memory: 8403 rows of 48 heads of 128 with
// three axes to bf16 58.7 us, 310 MB (5.3 TB/s; copies 6.5); the rows' own start, behind their positions, hides under other warps' heads. To f32 11 % more. 48 rows of 32 heads of 256 3.6 us, latency.
template <int D, typename T>
__global__ void __launch_bounds__(256, 4) k_rope_rows(RopeRowsParams p, RopeAxes axes, int hpw, int* err) {
    constexpr int LPH = D / 8, HPS = 32 / LPH;
    __shared__ __align__(16) float buf[8][32 * 8];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LPH, d0 = (lane % LPH) * 8, heads = p.heads[0] + p.heads[1] + p.heads[2], parts = (heads + hpw * HPS - 1) / (hpw * HPS);
    const unsigned mask = LPH == 32 ? 0xffffffffu : ((1u << (LPH & 31)) - 1u) << (sub * LPH);
    const long long item = (long long)blockIdx.x * 8 + warp;
    const int r = (int)(item / parts), h0 = (int)(item % parts) * hpw * HPS + sub, h1 = min(heads, h0 - sub + hpw * HPS);
    if (r >= p.R) return;
    // which of q, k and v a head belongs to, and its number there
    auto which = [&](int& h) { int w = 0; if (h >= p.heads[0]) { h -= p.heads[0]; w = 1; if (h >= p.heads[1]) { h -= p.heads[1]; w = 2; } } return w; };
    float4 next[2];
    auto fetch = [&](int h) {
        const int w = which(h);
        const float* from = (w == 0 ? p.in[0] : w == 1 ? p.in[1] : p.in[2]) + (size_t)r * (w == 0 ? p.in_ld[0] : w == 1 ? p.in_ld[1] : p.in_ld[2]) + (size_t)h * (w == 0 ? p.in_hs[0] : w == 1 ? p.in_hs[1] : p.in_hs[2]) + d0;
        next[0] = reinterpret_cast<const float4*>(from)[0]; next[1] = reinterpret_cast<const float4*>(from)[1];
    };
    if (h0 < h1) fetch(h0);
    RowPos at;
    float2 cs[8];
    if (p.n_rot) {
        if (!row_pos(at, axes, r, p.n_pos)) { paged_bad(err); return; }   // a row without a place stays as it was
        if (d0 < p.n_rot) angles(cs, p.rope, at, axes, p.n_rot, p.interleaved, d0);
    }
#pragma unroll 1
    for (int h = h0; h < h1; h += HPS) {
        float x[8] = {next[0].x, next[0].y, next[0].z, next[0].w, next[1].x, next[1].y, next[1].z, next[1].w};
        if (h + HPS < h1) fetch(h + HPS);
        int hh = h;
        const int w = which(hh);
        const void* const norm = w == 0 ? p.norm[0] : w == 1 ? p.norm[1] : nullptr;
        turn_head<D, false>(x, norm, make_uint4(0u, 0u, 0u, 0u), w < 2 ? p.n_rot : 0, p.interleaved, p.eps, cs, d0, mask, buf[warp] + sub * D);
        T* to = (T*)(w == 0 ? p.out[0] : w == 1 ? p.out[1] : p.out[2]) + (size_t)r * (w == 0 ? p.out_ld[0] : w == 1 ? p.out_ld[1] : p.out_ld[2]) + (size_t)hh * (w == 0 ? p.out_hs[0] : w == 1 ? p.out_hs[1] : p.out_hs[2]) + d0;
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(to)[0] = make_float4(x[0], x[1], x[2], x[3]); reinterpret_cast<float4*>(to)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (std::is_same<T, __half>::value) o[j] = h2_bits(__floats2half2_rn(x[2 * j], x[2 * j + 1]));
                else { const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]); o[j] = *reinterpret_cast<const uint32_t*>(&b); }
            }
            *reinterpret_cast<uint4*>(to) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// Sets of heads per warp. What a warp does once per row (its sequence, its place, its angles) takes as long as one or two sets; 4736 warps run at once. So a number of sets costs the warps' mean length for each full wave of them, and the longest one
// (two fifths of it, however few) for what is left; least wins. Us with one set, with six, with eight (rows that stay rows: all) and so: int8, 2000 rows of 32 heads of 64 11.1, 7.7, 12.0 and 8.0, 1500 rows of 32 heads of
// 128 17.2, 10.6, 14.7 and 10.4, four prompts of up to 1000 rows of 48 40.6, 28.3, 25.7 and 25.7; the same to 4 bits with axes 54.5, 33.9, 31.1 and 31.1; 8403 rows of 48 heads of 128 that stay rows, at positions as they come, 144, 77, 72.4 and 72.5. Over 696 shapes of 300 to 12000 rows the best of all numbers is 1 % faster on average, where it was 13 %.
struct Cut { int hpw; unsigned blocks; };
Cut cut_heads(long long R, int heads, int D) {
    constexpr long long WARPS = 148 * 32;
    const int HPS = 32 / (D / 8), sets = (heads + HPS - 1) / HPS;
    int hpw = 1;
    if (R * sets > WARPS) {
        double least = 0;
        for (int h = 1; h <= std::min(sets, 24); ++h) {
            const int parts = (sets + h - 1) / h;
            const long long n = R * parts, full = n / WARPS, left = n % WARPS;
            const double cost = full * (1.5 + (double)sets / parts) + (left ? (1.5 + h) * (full ? 0.4 + 0.6 * left / WARPS : 1.0) : 0.0);
            if (h == 1 || cost < least) { least = cost; hpw = h; }
        }
    }
    return Cut{hpw, (unsigned)((R * ((heads + hpw * HPS - 1) / (hpw * HPS)) + 7) / 8)};
}
template <int D, int KIND> int launch_append(const PagedPool& pool, const PagedBatch& b, const KvAppendParams& p, const RopeAxes& axes, cudaStream_t s) {
    int* err = device_arg_flag();
    const Cut c = cut_heads(b.R, p.n_head + 2 * pool.n_kv, D);
    HP_CUDA(launch_pdl<4>(axes.pos ? k_kv_append<D, KIND, true> : k_kv_append<D, KIND, false>, dim3(c.blocks), dim3(256), 0, s, pool, b, p, axes, c.hpw, err));
    return HP_OK;
}
template <int KIND> int launch_append(const PagedPool& pool, const PagedBatch& b, const KvAppendParams& p, const RopeAxes& axes, cudaStream_t s) {
    return pool.head_dim == 256 ? launch_append<256, KIND>(pool, b, p, axes, s) : pool.head_dim == 128 ? launch_append<128, KIND>(pool, b, p, axes, s) : launch_append<64, KIND>(pool, b, p, axes, s);
}
template <typename T> int launch_rows(const RopeRowsParams& p, const RopeAxes& axes, cudaStream_t s) {
    int* err = device_arg_flag();
    const Cut c = cut_heads(p.R, p.heads[0] + p.heads[1] + p.heads[2], p.head_dim);
    HP_CUDA(launch_pdl<4>(p.head_dim == 256 ? k_rope_rows<256, T> : p.head_dim == 128 ? k_rope_rows<128, T> : k_rope_rows<64, T>, dim3(c.blocks), dim3(256), 0, s, p, axes, c.hpw, err));
    return HP_OK;
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
int kv_append(const PagedPool& pool, const PagedBatch& b, const KvAppendParams& p, const RopeAxes& axes, cudaStream_t s) {
    return pool.kind == KV_I8 ? launch_append<KV_I8>(pool, b, p, axes, s) : pool.kind == KV_E4M3 ? launch_append<KV_E4M3>(pool, b, p, axes, s) : launch_append<KV_I4>(pool, b, p, axes, s);
}
int rope_rows(const RopeRowsParams& p, const RopeAxes& axes, cudaStream_t s) {
    return p.type == OUT_F32 ? launch_rows<float>(p, axes, s) : p.type == OUT_F16 ? launch_rows<__half>(p, axes, s) : launch_rows<__nv_bfloat16>(p, axes, s);
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
    HP_CUDA(pool.kind == KV_I8 ? type(std::integral_constant<int, KV_I8>()) : pool.kind == KV_E4M3 ? type(std::integral_constant<int, KV_E4M3>()) : type(std::integral_constant<int, KV_I4>()));
    return HP_OK;
}

}  // namespace hp
