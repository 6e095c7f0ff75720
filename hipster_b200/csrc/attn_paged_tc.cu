// Attention over pages in 8 or 4 bits for prompts: calls of many rows per sequence. The formulas, the exact splits of q and of the weights, and the merge are those of
// attn_paged.cu; here the products run on tcgen05, and the codes are turned into f16 once per call instead of once per block of rows.
//
// k_paged_f16 writes each visible tile of 64 tokens of a kv head as the picture that shared memory holds: rows of 64 dims (128 bytes) per token, 128-byte
// swizzle, one group of 64 dims behind the other, and the tile's scales behind k and v. A row of a picture is read as the K-major operand of the scores and as the N-major one of
// the outputs.
//
// The 128 rows of tcgen05.mma are pairs (row of the batch, query head) of a kv head. A CTA holds a block of 128 pairs and the keys of one split, in tiles of 64:
//   S[128 pairs][64 keys] = q_rest K^T + q K^T,   O[128 pairs][dims] = w_rest V + w V   (rests first: what they add up to is not yet rounded at the size of the whole)
// with q as values in accumulator memory and its rests in shared memory, and the weights in accumulator memory: the products read no more of shared memory than they have time for
// (S 1280 clocks at 256 dims, 512 of them the rests of q beyond the products' own time; O 1024). Warps:
//   copies (a warp for k, one for v), two pictures each ahead
//   products (one thread; issuing them takes as long as they take): scores of a tile in front of the outputs of the one before
//   weights (eight warps, a thread per pair and half of the keys): S -> w, in its place. The mask, the sum and the rescaling are a thread's own; two warps tell each other whether a reference moves
//   sums (eight warps, a thread per pair and half of the dims): O of the tile into registers, while the scores of the next but one are formed
// Measured: 509 rows of 24 heads of 256 over 4 behind 4096 tokens 148 us, of these the pictures 8, the merge 15; operations alone 33, and 65 as they are done, q and weights as two f16 each. A tile takes
// 3200 clocks, 2400 of them products: an output waits for its weights (700 clocks to read the scores and see whether a reference moves, 300 for the other half's
// answer, 1200 for the weights), and each hand-over between products and warps for some 200. A CTA starts in 11000 clocks, 6500 of them q, and writes its sums in 5500. Keys and dims as the 128
// rows, with pairs as columns (48 a block) and tiles of 128 keys: 225 us, since a thread then needs all other warps to know whether a reference moves, and the
// operands pass shared memory twice as often. Weights of a tile by one of two groups in turn: 210, by four warps with all keys of a pair: 255 (199
// as now, before the arithmetic was packed). Hand-over of the halves by mbarrier under the exponentials instead of the named barrier: 151 -> 163.
// 32 to 68 bytes a thread are spilled.
#include "paged.cuh"
#include "tc.cuh"
#include <algorithm>

namespace hp {
namespace {

constexpr int TK = 64, MB = PAGED_TC_PAIRS;   // keys of a tile, pairs of a block
static_assert(MB == 128, "rows of the products");

// Shared memory of a CTA, operands on 1024-byte boundaries. 64 dims of a key or of a pair are a row of 128 bytes. Accumulator memory: columns of O, of q's values, and two tiles of S, which w replaces.
template <int D> struct PagedGeo {
    static constexpr int W_ACC = 8, W_MMA = 16, W_V = 18, WARPS = 20;
    static constexpr int PICTURE = TK * D * 2, SCALES = 2 * TK * 4, TILE = 2 * PICTURE + SCALES;   // bytes of a tile of k or v, of its scales, of all
    static constexpr int OFF_Q = 0, OFF_K = MB * D * 2, OFF_V = OFF_K + 2 * PICTURE, OFF_S = OFF_V + 2 * PICTURE, OFF_X = OFF_S + 4 * SCALES;
    static constexpr int X_BYTES = 8192, SMEM = OFF_X + X_BYTES + 1024;                             // 1024 for the alignment
    static constexpr int T_O = 0, T_Q = 256, T_S = 384, TMEM = 512;
    static constexpr int DW = D / 2, STRIDE = DW + 4;                                               // dims of a warp that sums; its outputs pass through shared memory at the end
    static_assert(8 * 32 * STRIDE * 4 <= OFF_S && 2 * PICTURE == MB * D * 2 && SMEM <= 226 * 1024, "");
};

__device__ __forceinline__ float warp_max(float x) { float y; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x)); return y; }
// 128-byte swizzle, groups of 8 rows 1024 bytes apart. K-major: a row holds 64 elements along K. M- or N-major: a row is one step along K and holds 64 elements
// along M or N, the next 64 lie `next` bytes behind.
__device__ __forceinline__ uint64_t desc128(uint32_t addr, uint32_t next) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(next >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int add) {   // D = A * B (+ D)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void mma_f16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, int add) {   // A in accumulator memory: a row per lane, two elements per column
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
// 16 columns of this warp's 32 lanes; there behind ld_wait
__device__ __forceinline__ void ld16(float* a, uint32_t col) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=f"(a[0]), "=f"(a[1]), "=f"(a[2]), "=f"(a[3]), "=f"(a[4]), "=f"(a[5]), "=f"(a[6]), "=f"(a[7]), "=f"(a[8]), "=f"(a[9]), "=f"(a[10]), "=f"(a[11]), "=f"(a[12]), "=f"(a[13]), "=f"(a[14]), "=f"(a[15])
                 : "r"(col) : "memory");
}
__device__ __forceinline__ void st8(uint32_t col, const uint32_t (&a)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "r"(col), "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(a[4]), "r"(a[5]), "r"(a[6]), "r"(a[7]) : "memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ld_there(float* a) {   // orders the use of the registers behind the wait
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+f"(a[i]));
}
// Registers: 640 threads start with 96 each, 61440; eight warps with 152, eight with 72 and four with 32 take all of them (160 and 64: 157 us where this took 151).
// A share holds what is compiled here; a library function with registers of its own (printf) must not be called behind these
template <int N> __device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void pair_sync(int qt) { asm volatile("bar.sync %0, 64;" ::"r"(qt + 1) : "memory"); }
// a wait that is over already takes a test, not the 250 clocks of an attempt that may suspend
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err) { return __all_sync(0xffffffffu, mbar_test(bar, parity) || tc_wait(bar, parity, err)); }
__device__ __forceinline__ void warp_arrive(uint32_t bar, int lane) { __syncwarp(); if (lane == 0) mbar_arrive(bar); }

// grid (splits, n_kv, blocks). DIRECT: the only split there is writes the outputs itself
template <int D, int KIND, bool DIRECT>
__global__ void __launch_bounds__(PagedGeo<D>::WARPS * 32, 1) k_paged_prompt(const PagedArgs a) {
    using Geo = PagedGeo<D>;
    extern __shared__ uint8_t sm_raw[];
    __shared__ uint32_t tmem_ptr;
    uint8_t* const sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    struct Shared {
        uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], sc_full[4], s_full[2], p_full[2], pv_done, o_empty, l_there[4], fin;
        float c[MB], alpha[4][MB];   // factor of a pair's scores; rescaling by tile
        float top[2][MB];            // by half of the keys: a pair's largest logarithm where a reference may move
        float end[MB];               // sums of the weights of the second halves; direct: of all keys
        long long from[MB];          // a pair's row of q, -1: none
        int pos[MB], at[MB];         // its position, -1: none; row * n_head + head, -1: nothing to write (direct: rows without a key are zeros)
        int moved[4][4];             // by tile and warp: the tile's number + 1 where a reference moves, and alpha holds
    };
    static_assert(sizeof(Shared) <= Geo::X_BYTES, "");
    Shared& x = *reinterpret_cast<Shared*>(sm + Geo::OFF_X);
    pdl_wait();
    pdl_launch_dependents();   // behind the wait: what was enqueued in front of this kernel is complete when the merge starts
    const Block blk = find_block(a.b, a.G, MB, gridDim.z - 1 - blockIdx.z, lane, a.arg_err);   // the last rows see most: first
    if (blk.q.s < 0) return;
    const PagedSeq& sq = blk.q;
    const int kh = blockIdx.y, np = blk.np;
    const Span sp = span_of(a, blk);
    const int lo = sp.lo, sink = sp.sink;
    if (sp.u0 >= sp.kend) {   // no row of the block has a key
        if constexpr (DIRECT)
            for (int e = tid; e < np * (D / 4); e += Geo::WARPS * 32) {
                const int p = blk.p0 + e / (D / 4), t = p / a.G;
                put(make_float4(0.f, 0.f, 0.f, 0.f), 0.f, sq.row0 + t, kh * a.G + p - t * a.G, e % (D / 4) * 4, D, a);
            }
        return;
    }
    const int t_end = (int)((sp.u1 + TK - 1) / TK);
    auto first_from = [&](int t) { return t * TK >= sink && t * TK + TK <= lo ? lo / TK : t; };   // first visible tile at or behind t
    const int t_first = first_from((int)(sp.u0 / TK));
    if (t_first >= t_end) return;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&x.k_full[i]), 1); mbar_init(smem_u32(&x.k_empty[i]), 1); mbar_init(smem_u32(&x.v_full[i]), 1); mbar_init(smem_u32(&x.v_empty[i]), 1); }
        for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&x.sc_full[i]), 1);
        for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&x.l_there[i]), 1);
        for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&x.s_full[i]), 1); mbar_init(smem_u32(&x.p_full[i]), 8); }
        mbar_init(smem_u32(&x.pv_done), 1); mbar_init(smem_u32(&x.o_empty), 8); mbar_init(smem_u32(&x.fin), 1);
        fence_barrier_init();
    }
    if (tid < 16) x.moved[tid >> 2][tid & 3] = 0;
    if (warp == Geo::W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_ptr)), "n"(Geo::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid < MB) {
        const int p = blk.p0 + tid, t = p / a.G, head = kh * a.G + p - t * a.G, pos = tid < np ? max(-1, sq.len - sq.T + t) : -1;
        x.from[tid] = tid < np ? (long long)((size_t)(sq.row0 + t) * a.q_ld + (size_t)head * a.q_hs) : -1;
        x.pos[tid] = pos; x.at[tid] = (DIRECT ? tid < np : pos >= 0) ? (sq.row0 + t) * a.n_head + head : -1;
    }
    __syncthreads();
    // q: a warp per pair, 8 dims per lane, a warp's pairs all in flight; rests to their place, values to that of k, on their way to accumulator memory
    if (warp < 16) {
        float4 v[MB / 16][2];
#pragma unroll
        for (int u = 0; u < MB / 16; ++u) {
            const long long from = x.from[warp + u * 16];
            v[u][0] = v[u][1] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (from >= 0 && lane < D / 8) {
                const float4* src = reinterpret_cast<const float4*>(a.q + from) + 2 * lane;
                v[u][0] = src[0]; v[u][1] = src[1];
            }
        }
#pragma unroll
        for (int u = 0; u < MB / 16; ++u) {
            const int i = warp + u * 16;
            const float y[8] = {v[u][0].x, v[u][0].y, v[u][0].z, v[u][0].w, v[u][1].x, v[u][1].y, v[u][1].z, v[u][1].w};
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(y[j]) & 0x7fffffffu);
            m = __reduce_max_sync(0xffffffffu, m);
            const int e = q_exponent(m);
            const float up = __uint_as_float((uint32_t)(e + 127) << 23);
            if (lane < D / 8) {
                uint32_t h[4], r[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float y0 = y[2 * j] * up, y1 = y[2 * j + 1] * up;
                    const __half2 hh = __floats2half2_rn(y0, y1);
                    const float2 f = __half22float2(hh);
                    h[j] = h2_bits(hh); r[j] = h2_bits(__floats2half2_rn(y0 - f.x, y1 - f.y));
                }
                const int at = (lane >> 3) * (MB * 128) + i * 128 + (((lane & 7) ^ (i & 7)) << 4);
                *reinterpret_cast<uint4*>(sm + Geo::OFF_K + at) = make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4*>(sm + Geo::OFF_Q + at) = make_uint4(r[0], r[1], r[2], r[3]);
            }
            if (lane == 0) x.c[i] = a.scale2 * __uint_as_float((uint32_t)(127 - e) << 23);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_ptr;
    if (warp < 4) {
#pragma unroll 4
        for (int i = 0; i < D / 16; ++i) {   // 16 dims
            uint32_t w[8];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int ch = 2 * i + c;
                const uint4 h = *reinterpret_cast<const uint4*>(sm + Geo::OFF_K + (ch >> 3) * (MB * 128) + tid * 128 + (((ch & 7) ^ (tid & 7)) << 4));
                w[4 * c] = h.x; w[4 * c + 1] = h.y; w[4 * c + 2] = h.z; w[4 * c + 3] = h.w;
            }
            st8(tmem + ((uint32_t)warp << 21) + Geo::T_Q + 8 * i, w);
        }
        st_wait();
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    bool ok = true;

    if (warp < 8) {   // ---- weights: two warps share 32 pairs, a thread has half of the keys of one
        regs_less<72>();
        const int half = warp >> 2, qt = warp & 3, row = tid & (MB - 1);
        const uint32_t sw = tmem + ((uint32_t)qt << 21) + Geo::T_S + half * 32;
        const bool idle = 32 * qt >= np;   // rows of the products hang on nothing but themselves
        const float c = x.c[row]; const float2 c2 = make_float2(c, c);
        const int all_hi = sp.pos_lo, all_lo = a.window ? sp.pos_hi - a.window : -1;   // positions between which a tile is visible to all pairs
        float mu = MU_NONE;
        float2 l2 = make_float2(0.f, 0.f);
        int n = 0;
        // A wait that gave up does not end the loop, which is as long for the two warps of a pair: their barrier is not bounded, so both have to come to it
#pragma unroll 1
        for (int t = t_first; t < t_end; t = first_from(t + 1), ++n) {
            const float* const ks = reinterpret_cast<const float*>(sm + Geo::OFF_S + (n & 3) * Geo::SCALES) + half * 32; const float* const vs = ks + TK;
            ok = ok && warp_wait(smem_u32(&x.sc_full[n & 3]), (n >> 2) & 1, a.err) && warp_wait(smem_u32(&x.s_full[n & 1]), (n >> 1) & 1, a.err);
            tc_fence_after();
            if (idle) {
                if (lane == 0) mbar_arrive(smem_u32(&x.p_full[n & 1]));
                continue;
            }
            const uint32_t at = sw + (n & 1) * TK;
            const int j0 = t * TK + 32 * half;
            const bool whole = j0 + 31 <= all_hi && (j0 > all_lo || j0 + 32 <= sink);
            uint32_t see = ~0u;   // a bit per key
            if (!whole) {
                auto below = [&](int j) -> uint32_t { const int k = j - j0; return k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1; };   // keys below j
                const int pos = x.pos[row];
                see = below(pos + 1) & (a.window ? ~below(max(pos - a.window + 1, 0)) | below(sink) : ~0u);
            }
            const float lv = scale_lg2(warp_max(vs[lane]));
            float d[32];
            auto measure = [&] {   // distances of the logarithms from their reference
                ld16(d, at); ld16(d + 16, at + 16);
                ld_wait(); ld_there(d); ld_there(d + 16);
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 k = *reinterpret_cast<const float4*>(ks + e);
                    float2 a = make_float2(-mu, -mu), b = a;
                    fma2(a, make_float2(d[e], d[e + 1]), mul2(make_float2(k.x, k.y), c2)); fma2(b, make_float2(d[e + 2], d[e + 3]), mul2(make_float2(k.z, k.w), c2));
                    d[e] = a.x; d[e + 1] = a.y; d[e + 2] = b.x; d[e + 3] = b.y;
                }
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) if (!(see >> e & 1)) d[e] = -INFINITY;
                }
            };
            measure();
            float top = d[0];
#pragma unroll
            for (int e = 1; e < 32; ++e) top = fmaxf(top, d[e]);
            // Looked at from 2^-6 below the limit: this sum and the logarithms below are rounded apart by less than that (up to logarithms of 2^17), so a pair that would move is always looked at, whatever its neighbours do
            if (__any_sync(0xffffffffu, top + lv > MU_LIMIT - 0.015625f) && lane == 0) x.moved[n & 3][qt] = n + 1;
            pair_sync(qt);
            if (x.moved[n & 3][qt] == n + 1) {   // rare behind the first tiles. A pair moves by its own keys alone
                float exact = -INFINITY;
#pragma unroll 1
                for (int i = 0; i < 32; i += 16) {
                    float y[16];
                    ld16(y, at + i); ld_wait(); ld_there(y);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float z = y[e] * (ks[i + e] * c) + scale_lg2(vs[i + e]);
                        exact = fmaxf(exact, see >> (i + e) & 1 ? z : -INFINITY);
                    }
                }
                x.top[half][row] = exact;
                pair_sync(qt);
                exact = fmaxf(exact, x.top[half ^ 1][row]);
                float al = 1.f;
                if (exact - mu > MU_LIMIT) { const float next = mu_next(mu, exact); al = pow2i(mu - next); l2 = make_float2(add_scaled(0.f, l2.x, al, mu - next), add_scaled(0.f, l2.y, al, mu - next)); mu = next; }
                if (half == 0) x.alpha[n & 3][row] = al;
                measure();
                if (fabsf(mu) >= 67108864.f) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) d[e] = cut_off(d[e], lv);
                }
            }
#pragma unroll
            for (int i = 0; i < 32; i += 16) {
                uint32_t h[8], r[8];
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(vs + i + e);
                    float* const y = d + i + e;
#pragma unroll
                    for (int u = 0; u < 4; ++u) y[u] = ex2(y[u]);
                    l2 = add2(l2, add2(make_float2(y[0], y[1]), make_float2(y[2], y[3])));
                    const float2 a = mul2(make_float2(y[0], y[1]), make_float2(v.x, v.y)), b = mul2(make_float2(y[2], y[3]), make_float2(v.z, v.w));
                    y[0] = a.x; y[1] = a.y; y[2] = b.x; y[3] = b.y;
                    if (!whole) {   // a masked key's scale may be anything
#pragma unroll
                        for (int u = 0; u < 4; ++u) if (!(see >> (i + e + u) & 1)) y[u] = 0.f;
                    }
#pragma unroll
                    for (int u = 0; u < 4; u += 2) {
                        const __half2 hh = __floats2half2_rn(y[u], y[u + 1]);
                        const float2 f = __half22float2(hh);
                        float2 w = make_float2(y[u], y[u + 1]); fma2(w, f, make_float2(-1.f, -1.f));
                        h[(e + u) / 2] = h2_bits(hh); r[(e + u) / 2] = h2_bits(__floats2half2_rn(w.x, w.y));
                    }
                }
                st8(at + i, h); st8(at + i + 8, r);   // in place of these keys' scores
            }
            st_wait();
            tc_fence_before();
            warp_arrive(smem_u32(&x.p_full[n & 1]), lane);
        }
        if (!idle) {
            const float l = l2.x + l2.y;
            if (half) x.end[row] = l;
            pair_sync(qt);
            if (DIRECT && half == 0) { x.end[row] = l + x.end[row]; warp_arrive(smem_u32(&x.l_there[qt]), lane); }
            else if (ok && half == 0 && x.at[row] >= 0) a.pml[(size_t)x.at[row] * (a.ns + a.nwin) + blockIdx.x] = make_float2(mu, l + x.end[row]);
        }
    } else if (warp < Geo::W_MMA) {   // ---- sums
        regs_more<152>();
        constexpr int DW = Geo::DW;
        const int qt = warp & 3, d0 = (warp - Geo::W_ACC) / 4 * DW;
        const uint32_t ob = tmem + ((uint32_t)qt << 21) + Geo::T_O + d0;
        const bool idle = 32 * qt >= np;
        float O[DW];
#pragma unroll
        for (int i = 0; i < DW; ++i) O[i] = 0.f;
        int n = 0;
#pragma unroll 1
        for (int t = t_first; t < t_end && ok; t = first_from(t + 1), ++n) {
            ok = warp_wait(smem_u32(&x.pv_done), n & 1, a.err);
            if (!ok) break;
            tc_fence_after();
            if (!idle) {
                if (x.moved[n & 3][qt] == n + 1) {
                    const float al = x.alpha[n & 3][32 * qt + lane];
#pragma unroll
                    for (int i = 0; i < DW; i += 2) { const float2 u = mul2(make_float2(O[i], O[i + 1]), make_float2(al, al)); O[i] = u.x; O[i + 1] = u.y; }
                }
#pragma unroll
                for (int i = 0; i < DW; i += 16) {
                    float f[16];
                    ld16(f, ob + i); ld_wait(); ld_there(f);
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float2 u = add2(make_float2(O[i + e], O[i + e + 1]), make_float2(f[e], f[e + 1]));
                        O[i + e] = u.x; O[i + e + 1] = u.y;
                    }
                }
            }
            tc_fence_before();
            warp_arrive(smem_u32(&x.o_empty), lane);
        }
        if (ok && !idle) {   // rows through shared memory, which nothing reads or writes behind the last outputs
            float* const w = reinterpret_cast<float*>(sm) + (warp - Geo::W_ACC) * 32 * Geo::STRIDE;
#pragma unroll
            for (int i = 0; i < DW; i += 4) *reinterpret_cast<float4*>(w + lane * Geo::STRIDE + i) = make_float4(O[i], O[i + 1], O[i + 2], O[i + 3]);
            __syncwarp();
            if constexpr (DIRECT) ok = warp_wait(smem_u32(&x.l_there[qt]), 0, a.err);
            constexpr int LPR = DW / 4, RPI = 32 / LPR;   // lanes of a row, rows at a time
#pragma unroll 4
            for (int r = lane / LPR; r < 32; r += RPI) {
                const int at = x.at[32 * qt + r], d = lane % LPR * 4;
                if (at < 0) continue;
                const float4 o = *reinterpret_cast<const float4*>(w + r * Geo::STRIDE + d);
                if constexpr (DIRECT) put(o, x.end[32 * qt + r], at / a.n_head, at % a.n_head, d0 + d, D, a);
                else *reinterpret_cast<float4*>(a.pO + ((size_t)at * (a.ns + a.nwin) + blockIdx.x) * D + d0 + d) = o;
            }
        }
    } else {
        regs_less<32>();
        if (warp == Geo::W_MMA) {   // ---- products
            if (tc_elect()) {
                const uint32_t base = smem_u32(sm);
                constexpr uint32_t ID = (1u << 4) | (8u << 24), ID_S = ID | ((uint32_t)(TK >> 3) << 17), ID_O = ID | ((uint32_t)(D >> 3) << 17) | (1u << 16);   // f32 = f16 x f16, M = 128; O: V is N-major
                auto wait = [&](uint64_t& bar, uint32_t parity) { return mbar_test(smem_u32(&bar), parity) || tc_wait(smem_u32(&bar), parity, a.err); };
                int n = 0;
#pragma unroll 1
                for (int t = t_first;; ++n) {   // scores of tile n, outputs of tile n - 1
                    const bool more = t < t_end;
                    if (more) {
                        if (!wait(x.k_full[n & 1], (n >> 1) & 1) || (n > 1 && !wait(x.pv_done, n & 1))) break;   // the weights of n - 2 are read
                        tc_fence_after();
                        const uint32_t kb = base + Geo::OFF_K + (n & 1) * Geo::PICTURE, st = tmem + Geo::T_S + (n & 1) * TK;
#pragma unroll 4
                        for (int i = 0; i < D / 16; ++i)   // 16 dims
                            mma_f16(st, desc128(base + Geo::OFF_Q + (i >> 2) * (MB * 128) + (i & 3) * 32, 16), desc128(kb + (i >> 2) * (TK * 128) + (i & 3) * 32, 16), ID_S, i != 0);
#pragma unroll 4
                        for (int i = 0; i < D / 16; ++i) mma_f16_ta(st, tmem + Geo::T_Q + 8 * i, desc128(kb + (i >> 2) * (TK * 128) + (i & 3) * 32, 16), ID_S, 1);
                        tc_commit(smem_u32(&x.s_full[n & 1]));
                        tc_commit(smem_u32(&x.k_empty[n & 1]));
                        t = first_from(t + 1);
                    }
                    if (n) {
                        const int m = n - 1;
                        if (!wait(x.v_full[m & 1], (m >> 1) & 1) || !wait(x.o_empty, (m & 1) ^ 1) || !wait(x.p_full[m & 1], (m >> 1) & 1)) break;
                        tc_fence_after();
                        const uint32_t vb = base + Geo::OFF_V + (m & 1) * Geo::PICTURE, wt = tmem + Geo::T_S + (m & 1) * TK;
#pragma unroll
                        for (int i = 0; i < TK / 16; ++i) mma_f16_ta(tmem + Geo::T_O, wt + 16 * i + 8, desc128(vb + i * 2048, TK * 128), ID_O, i != 0);   // 16 keys
#pragma unroll
                        for (int i = 0; i < TK / 16; ++i) mma_f16_ta(tmem + Geo::T_O, wt + 16 * i, desc128(vb + i * 2048, TK * 128), ID_O, 1);
                        tc_commit(smem_u32(&x.pv_done));
                        tc_commit(smem_u32(&x.v_empty[m & 1]));
                    }
                    if (!more) break;
                }
                tc_commit(smem_u32(&x.fin));
                tc_wait(smem_u32(&x.fin), 0, a.err);   // nothing in flight when the accumulator memory is given back
            }
            __syncwarp();
        } else if (warp < Geo::WARPS - 1) {   // ---- copies: k of tile n and all its scales when the scores of tile n - 2 are there, v when the outputs are
            // A tile's scales have their place from tile n - 4, whose outputs were there before the scores of n - 2 were begun.
            const int kv = warp == Geo::W_V;
            const uint8_t* src = a.f16 + ((size_t)sq.s * a.pool.n_kv + kh) * a.tiles * Geo::TILE + kv * Geo::PICTURE;
            const uint32_t dst = smem_u32(sm) + (kv ? Geo::OFF_V : Geo::OFF_K);
            int n = 0;
            for (int t = t_first; t < t_end && ok; t = first_from(t + 1)) {
                const uint32_t full = smem_u32(kv ? &x.v_full[n & 1] : &x.k_full[n & 1]), empty = smem_u32(kv ? &x.v_empty[n & 1] : &x.k_empty[n & 1]);
                ok = warp_wait(empty, ((n >> 1) & 1) ^ 1, a.err);
                if (!ok) break;
                if (tc_elect()) {
                    mbar_expect_tx(full, Geo::PICTURE);
#pragma unroll
                    for (int i = 0; i < D / 64; ++i) bulk_g2s(dst + (n & 1) * Geo::PICTURE + i * (TK * 128), src + (size_t)t * Geo::TILE + i * (TK * 128), TK * 128, full);
                    if (!kv) {
                        const uint32_t sf = smem_u32(&x.sc_full[n & 3]);
                        mbar_expect_tx(sf, Geo::SCALES);
                        bulk_g2s(smem_u32(sm) + Geo::OFF_S + (n & 3) * Geo::SCALES, src + (size_t)t * Geo::TILE + 2 * Geo::PICTURE, Geo::SCALES, sf);
                    }
                }
                __syncwarp();
                ++n;
            }
            for (int m = max(0, n - 2); m < n; ++m) {   // no copy outlives the CTA
                tc_wait(smem_u32(kv ? &x.v_full[m & 1] : &x.k_full[m & 1]), (m >> 1) & 1, a.err);
                if (!kv) tc_wait(smem_u32(&x.sc_full[m & 3]), (m >> 2) & 1, a.err);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == Geo::W_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Geo::TMEM) : "memory");
}

// The pictures: grid (tiles, 2 n_kv, sequences); a thread turns 16 codes into two pieces of 16 bytes. Tokens that no row sees are zeros in a tile of which others are seen;
// tiles without a visible token are not written, nor read. The tile's scales of k or v (unseen tokens: 0) lie behind both pictures.
template <int KIND>
__global__ void __launch_bounds__(256) k_paged_f16(const PagedArgs a) {
    const int lane = threadIdx.x & 31, t = blockIdx.x, h = blockIdx.y >> 1, kv = blockIdx.y & 1, D = a.pool.head_dim, cpr = D / 16, lg = a.pool.lg_page, pmask = (1 << lg) - 1;
    __shared__ uint32_t rows[TK / 16];   // the pool's rows of the tile's runs of 16 tokens
    pdl_wait();
    pdl_launch_dependents();   // behind the wait: what was enqueued in front of this kernel is complete when the attention starts
    const PagedSeq q = paged_seq(a.b, blockIdx.z, a.arg_err);
    const int pos_lo = max(q.len - q.T, 0), lo = a.window ? max(0, pos_lo - a.window + 1) : 0, sink = a.window ? a.n_sink : 0;
    if (q.T == 0 || t * TK >= q.len || (t * TK >= sink && t * TK + TK <= lo)) return;
    if (threadIdx.x < TK / 16) {
        const int j = t * TK + 16 * lane, k = j & ~pmask;
        uint32_t r = 0xffffffffu;
        if (j < q.len && (k < sink || k + pmask >= lo)) { r = paged_row(a.pool, q.s, j >> lg, h, a.arg_err); if (r != 0xffffffffu) r += j & pmask; }
        rows[lane] = r;
    }
    __syncthreads();
    const size_t picture = (size_t)TK * D * 2;
    uint8_t* const tile = a.f16 + (((size_t)blockIdx.z * a.pool.n_kv + h) * a.tiles + t) * (2 * picture + 2 * TK * 4); uint8_t* const dst = tile + kv * picture;
    if (threadIdx.x < TK) {
        const uint32_t r = rows[threadIdx.x >> 4];
        reinterpret_cast<float*>(tile + 2 * picture)[kv * TK + threadIdx.x] = r != 0xffffffffu && t * TK + (int)threadIdx.x < q.len ? (kv ? a.pool.v_scale : a.pool.k_scale)[(size_t)r + (threadIdx.x & 15)] : 0.f;
    }
    const uint8_t* src = kv ? a.pool.v : a.pool.k;
    for (int e0 = threadIdx.x; e0 < TK * cpr; e0 += 4 * 256) {
        uint4 w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int e = e0 + u * 256, row = e / cpr, part = e % cpr;
            w[u] = make_uint4(0, 0, 0, 0);   // codes of zero; 4 bits: two words of codes, and a factor of zero
            if (e < TK * cpr && rows[row >> 4] != 0xffffffffu && t * TK + row < q.len) {
                if constexpr (KIND == KV_I4) {
                    const I4Row at = i4_row(rows[row >> 4] + (row & 15), lg, D);
                    const uint2 c = *reinterpret_cast<const uint2*>(src + at.codes + part * 8);
                    w[u] = make_uint4(c.x, c.y, src[at.groups + (part >> 1)], 0u);
                } else w[u] = *reinterpret_cast<const uint4*>(src + ((size_t)rows[row >> 4] + (row & 15)) * D + part * 16);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int e = e0 + u * 256, row = e / cpr, part = e % cpr;
            if (e >= TK * cpr) break;
            uint8_t* o = dst + (part >> 2) * (TK * 128) + row * 128;
            const int ch = (part & 3) * 2;
            if constexpr (KIND == KV_I4) {
                const I4Group g = i4_group(__byte_perm(w[u].z, 0x64u, 0x4040));
                *reinterpret_cast<uint4*>(o + ((ch ^ (row & 7)) << 4)) = i4_word(w[u].x, g);
                *reinterpret_cast<uint4*>(o + (((ch + 1) ^ (row & 7)) << 4)) = i4_word(w[u].y, g);
            } else {
                *reinterpret_cast<uint4*>(o + ((ch ^ (row & 7)) << 4)) = make_uint4(code_pair<KIND, 0>(w[u].x), code_pair<KIND, 2>(w[u].x), code_pair<KIND, 0>(w[u].y), code_pair<KIND, 2>(w[u].y));
                *reinterpret_cast<uint4*>(o + (((ch + 1) ^ (row & 7)) << 4)) = make_uint4(code_pair<KIND, 0>(w[u].z), code_pair<KIND, 2>(w[u].z), code_pair<KIND, 0>(w[u].w), code_pair<KIND, 2>(w[u].w));
            }
        }
    }
}

template <int D, int KIND, bool DIRECT> int launch_split(const PagedArgs& a, dim3 grid, cudaStream_t s) {
    using Geo = PagedGeo<D>;
    static bool attr[MAX_DEVICES] = {};   // per device: the opt-in belongs to the device's copy of the kernel
    const int dev = current_device(); if (dev < 0) return HP_ECUDA;
    if (!attr[dev]) { HP_CUDA(cudaFuncSetAttribute(k_paged_prompt<D, KIND, DIRECT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo::SMEM)); attr[dev] = true; }
    HP_CUDA(launch_pdl<4>(a.pool.kind == KV_I4 ? k_paged_f16<KV_I4> : k_paged_f16<KIND>, dim3(a.tiles, 2 * a.pool.n_kv, a.b.S), dim3(256), 0, s, a));
    HP_CUDA(launch_pdl<4>(k_paged_prompt<D, KIND, DIRECT>, grid, dim3(Geo::WARPS * 32), Geo::SMEM, s, a));
    return HP_OK;
}
template <int D, int KIND> int launch_split(const PagedArgs& a, dim3 grid, cudaStream_t s) { return a.direct ? launch_split<D, KIND, true>(a, grid, s) : launch_split<D, KIND, false>(a, grid, s); }
template <int KIND> int launch_split(const PagedArgs& a, dim3 grid, cudaStream_t s) {
    return a.pool.head_dim == 256 ? launch_split<256, KIND>(a, grid, s) : a.pool.head_dim == 128 ? launch_split<128, KIND>(a, grid, s) : launch_split<64, KIND>(a, grid, s);
}

}  // namespace

size_t attn_paged_tc_bytes(const PagedPool& pool, const PagedBatch& b) { return (size_t)b.S * pool.n_kv * ((b.max_kv + TK - 1) / TK) * (2 * TK) * (2 * pool.head_dim + 4); }
int attn_paged_tc(PagedArgs& a, dim3 grid, cudaStream_t s) {
    a.tiles = (a.b.max_kv + TK - 1) / TK;
    HP_REQUIRE(a.b.S <= 65535 && 2 * a.pool.n_kv <= 65535, "attn_paged: too many sequences (%d) or heads for a prompt", a.b.S);
    return a.pool.kind == KV_E4M3 ? launch_split<KV_E4M3>(a, grid, s) : launch_split<KV_I8>(a, grid, s);   // behind the pictures 4 bits are whole numbers as int8 is
}

}  // namespace hp
