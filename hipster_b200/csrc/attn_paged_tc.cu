// Attention over 8-bit pages for prompts: calls of many rows per sequence. The formulas, the exact splits of q and of the weights, and the merge are those of
// attn_paged.cu; here the products run on tcgen05, and the codes are turned into f16 once per call instead of once per block of rows.
//
// k_paged_f16 writes each visible tile of 128 tokens of a kv head as the picture that shared memory holds: rows of 64 dims (128 bytes) per token, 128-byte
// swizzle, one group of 64 dims behind the other. A row of it is read as the K-major operand of the scores and as the M-major one of the outputs. Converting in the
// attention kernel itself (from a ring of codes, four warps) took 11000 clocks per tile of 32 pairs: the conversion's instructions, and
// 3600 clocks of shared memory for codes in, codes out, f16 in and operands out.
//
// Both products stand on their heads: keys, then dims, are the 128 rows of tcgen05.mma, and its columns are the pairs (row of the batch, query head) of a
// kv head, each twice: column i its values, column MB + i what is left of them. So a thread that reads a row of the accumulator has value and rest of every pair
// at hand, needs one scale of k and of v, and adds up its own keys' weights without another thread until the end. A CTA holds a block of 48 pairs
// and the keys of one split, in tiles of 128 keys:
//   copies (a warp for k, one for v: in one warp a copy of k waits behind the outputs that a copy of v waits for, 6600 clocks per tile): pictures into shared memory
//   products (one thread; its warp does nothing else, since issuing them takes as long as they take): S[128 keys][pairs] = K q^T, and O[128 dims][pairs] = V^T w, one tile
//     of scores ahead
//   weights (two groups of four warps, a thread per key, a group takes every second set of eight pairs): S -> w in shared memory (N-major operand)
//   sums (four warps per 128 dims, a thread per dim): O of the tile into registers
// Bound by shared memory: a tile's pictures go in (1024 clocks at 256 dims) and, as operands with q and the weights, out again (1800), against 1536 clocks of products.
#include "paged.cuh"
#include "tc.cuh"
#include <algorithm>

namespace hp {
namespace {

constexpr int TK = 128;   // keys of a tile

// Shared memory of a CTA, operands on 1024-byte boundaries. 64 dims of a key (or of a pair of q, 64 columns of the weights of a key) are a row of 128 bytes.
template <int D, int MB> struct PagedGeo {
    static constexpr int N = 2 * MB, NB = D > 128 ? 2 : 1, ACC = 4 * NB;                 // columns, blocks of 128 dims, warps that sum
    static constexpr int W_ACC = 8, W_MMA = W_ACC + ACC, W_K = W_MMA + 1, W_V = W_K + 1, WARPS = W_V + 1;
    static constexpr int PICTURE = TK * D * 2;                                            // bytes of a tile of k or v
    static constexpr int OFF_Q = 0, OFF_K = N * D * 2, OFF_V = OFF_K + PICTURE, OFF_P = OFF_V + PICTURE, OFF_X = OFF_P + (N + 63) / 64 * TK * 128;
    static constexpr int X_BYTES = 4096, SMEM = OFF_X + X_BYTES + 1024;                   // 1024 for the alignment
    static constexpr int TMEM = 512;
    static_assert(OFF_K % 1024 == 0 && NB * N + 2 * N + MB <= TMEM && SMEM <= 226 * 1024, "");
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
// eight columns of this warp's 32 lanes; there behind ld_wait
__device__ __forceinline__ void ld8(float (&a)[8], uint32_t col) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(a[0]), "=f"(a[1]), "=f"(a[2]), "=f"(a[3]), "=f"(a[4]), "=f"(a[5]), "=f"(a[6]), "=f"(a[7]) : "r"(col) : "memory");
}
__device__ __forceinline__ void st8(uint32_t col, const float (&a)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "r"(col), "f"(a[0]), "f"(a[1]), "f"(a[2]), "f"(a[3]), "f"(a[4]), "f"(a[5]), "f"(a[6]), "f"(a[7]) : "memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ld_there(float (&a)[8]) {   // orders the use of the registers behind the wait
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+f"(a[i]));
}
__device__ __forceinline__ void group_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory"); }
// a wait that is over already takes a test, not the 250 clocks of an attempt that may suspend
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err) { return __all_sync(0xffffffffu, mbar_test(bar, parity) || tc_wait(bar, parity, err)); }
__device__ __forceinline__ void warp_arrive(uint32_t bar, int lane) { __syncwarp(); if (lane == 0) mbar_arrive(bar); }

// grid (splits, n_kv, blocks)
template <int D, int KIND, int MB>
__global__ void __launch_bounds__(PagedGeo<D, MB>::WARPS * 32, 1) k_paged_prompt(const PagedArgs a) {
    using Geo = PagedGeo<D, MB>;
    constexpr int N = Geo::N, NB = Geo::NB, NC = MB / 16;
    extern __shared__ uint8_t sm_raw[];
    __shared__ uint32_t tmem_ptr;
    uint8_t* const sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    struct Shared {
        uint64_t k_full, k_empty, v_full, s_full[2], s_empty[2], p_full, pv_done, o_empty, fin;
        alignas(16) float c[MB]; float mu[8][8 * NC], alpha[4][MB], top[2][4][8 * NC], l[2][4][8 * NC];   // factor of a pair's scores, references (a copy of each warp's own); rescaling by tile; largest logarithms by group, warp
        int2 see[MB]; int at[MB];   // a pair's position and the last key in front of its window; row * n_head + head, -1: nothing to write
        int moved[4][2];            // by tile and group: the tile's number + 1 where references move, and alpha holds
    };
    static_assert(sizeof(Shared) <= Geo::X_BYTES, "");
    Shared& x = *reinterpret_cast<Shared*>(sm + Geo::OFF_X);
    pdl_wait();
    pdl_launch_dependents();   // behind the wait: what was enqueued in front of this kernel is complete when the merge starts
    const Block blk = find_block(a.b, a.G, MB, blockIdx.z, lane, a.arg_err);
    if (blk.q.s < 0) return;
    const PagedSeq& sq = blk.q;
    const int kh = blockIdx.y, np = blk.np;
    const Span sp = span_of(a, blk);
    const int pos_lo = sp.pos_lo, pos_hi = sp.pos_hi, kend = sp.kend, lo = sp.lo, sink = sp.sink;
    if (sp.u0 >= kend) return;
    const int t_end = (int)((sp.u1 + TK - 1) / TK);
    auto first_from = [&](int t) { return t * TK >= sink && t * TK + TK <= lo ? lo / TK : t; };   // first visible tile at or behind t
    const int t_first = first_from((int)(sp.u0 / TK));
    if (t_first >= t_end) return;
    const int lg = a.pool.lg_page, pmask = (1 << lg) - 1;

    if (tid == 0) {
        mbar_init(smem_u32(&x.k_full), 1); mbar_init(smem_u32(&x.k_empty), 1); mbar_init(smem_u32(&x.v_full), 1);
        for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&x.s_full[i]), 1); mbar_init(smem_u32(&x.s_empty[i]), 8); }
        mbar_init(smem_u32(&x.p_full), 8); mbar_init(smem_u32(&x.pv_done), 1); mbar_init(smem_u32(&x.o_empty), Geo::ACC); mbar_init(smem_u32(&x.fin), 1);
        fence_barrier_init();
    }
    if (tid < 8) x.moved[tid >> 1][tid & 1] = 0;
    if (warp < 8 && lane < 8 * NC) x.mu[warp][lane] = MU_NONE;
    if (warp == Geo::W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_ptr)), "n"(Geo::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // q: a warp per pair, 8 dims per lane, as values (row i) and rests (row MB + i)
    for (int i = warp; i < MB; i += Geo::WARPS) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        uint32_t m = 0;
        const bool live = i < np;
        const int p = blk.p0 + i, t = live ? p / a.G : 0;
        if (live && lane < D / 8) {
            const float4* src = reinterpret_cast<const float4*>(a.q + (size_t)(sq.row0 + t) * a.q_ld + (size_t)(kh * a.G + p - t * a.G) * a.q_hs) + 2 * lane;
            const float4 v0 = src[0], v1 = src[1];
            v[0] = v0.x; v[1] = v0.y; v[2] = v0.z; v[3] = v0.w; v[4] = v1.x; v[5] = v1.y; v[6] = v1.z; v[7] = v1.w;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
        }
        m = __reduce_max_sync(0xffffffffu, m);
        const int e = q_exponent(m);
        const float up = __uint_as_float((uint32_t)(e + 127) << 23);
        if (lane < D / 8) {
            uint32_t h[4], r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float y0 = v[2 * j] * up, y1 = v[2 * j + 1] * up;
                const __half2 hh = __floats2half2_rn(y0, y1);
                const float2 f = __half22float2(hh);
                h[j] = h2_bits(hh); r[j] = h2_bits(__floats2half2_rn(y0 - f.x, y1 - f.y));
            }
            uint8_t* dst = sm + Geo::OFF_Q + (lane >> 3) * (N * 128);
            const int ch = lane & 7;
            *reinterpret_cast<uint4*>(dst + i * 128 + ((ch ^ (i & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(dst + (MB + i) * 128 + ((ch ^ (i & 7)) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
        }
        if (lane == 0) {
            const int pos = live ? max(-1, sq.len - sq.T + t) : -1;
            x.c[i] = a.scale2 * __uint_as_float((uint32_t)(127 - e) << 23);
            x.see[i] = make_int2(pos, a.window ? pos - a.window : -1);
            x.at[i] = pos >= 0 ? (sq.row0 + t) * a.n_head + kh * a.G + p - t * a.G : -1;
        }
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_ptr;
    bool ok = true;

    if (warp < 8) {   // ---- weights
        // The loops over the sets of eight pairs are not unrolled, and the sums of the weights wait in accumulator memory: with everything in registers and unrolled the
        // roles' loops did not fit the instruction cache (some 10 clocks per instruction; 8400 clocks per tile). A wait that gave up does not end the loop, which is as long for
        // all warps of a group: their barrier is not bounded, so all of them have to come to it.
        const int grp = warp >> 2, qt = warp & 3, key = qt * 32 + lane, nc = (np - 8 * grp + 15) / 16;   // sets of this group: pairs 8 (2 i + grp) ..
        const uint32_t tlane = tmem + ((uint32_t)qt << 21), lcol = tlane + 2 * N + NB * N + 8 * grp;
        uint8_t* const pw = sm + Geo::OFF_P + key * 128;
        {
            const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int i = 0; i < nc; ++i) st8(lcol + 16 * i, zero);
            st_wait();
        }
        // positions between which a tile is visible to all pairs
        const int all_hi = pos_lo, all_lo = a.window ? pos_hi - a.window : -1;
        // scales of this thread's key, a tile ahead, and its page, two tiles ahead
        float ks = 0.f, vs = 0.f;
        auto id_of = [&](int t) -> int {   // its check waits for it: a tile ahead of its use
            const int j = t * TK + key, k = j & ~pmask;
            return t < t_end && j < kend && (k < sink || k + pmask >= lo) ? paged_id(a.pool, sq.s, j >> lg) : -1;
        };
        auto row_of = [&](int t, int id) -> uint32_t {
            const int j = t * TK + key, k = j & ~pmask;
            return t < t_end && j < kend && (k < sink || k + pmask >= lo) ? paged_row_of(a.pool, id, kh, a.arg_err) : 0xffffffffu;
        };
        uint32_t page = row_of(t_first, id_of(t_first));
        auto scales = [&](int t, float& k, float& v) {
            k = v = 0.f;
            if (t < t_end && page != 0xffffffffu) { const size_t at = (size_t)page + ((t * TK + key) & pmask); k = a.pool.k_scale[at]; v = a.pool.v_scale[at]; }
        };
        scales(t_first, ks, vs);
        int t1 = first_from(t_first + 1), id = id_of(t1);
        int n = 0;
        for (int t = t_first; t < t_end; t = t1, ++n) {
            float ks1, vs1;
            t1 = first_from(t + 1);
            page = row_of(t1, id);
            scales(t1, ks1, vs1);
            id = id_of(first_from(t1 + 1));
            const uint32_t sb = tlane + (n & 1) * N + 8 * grp;
            ok = ok && warp_wait(smem_u32(&x.s_full[n & 1]), (n >> 1) & 1, a.err);
            tc_fence_after();
            const float lv = lg2(fmaxf(vs, 8.0779357e-28f));   // 2^-90: the weights' sum cannot overflow
            const int j = t * TK + key;
            const bool whole = t * TK + TK - 1 <= all_hi && (t * TK > all_lo || t * TK + TK <= sink);
            uint32_t hide = 0;   // a bit per pair
            if (!whole) {
#pragma unroll 1
                for (int i = 0; i < nc; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) { const int2 v = x.see[8 * (2 * i + grp) + e]; if (!(j <= v.x && (j > v.y || j < sink))) hide |= 1u << (8 * i + e); }
            }
            auto scores = [&](float (&s)[8], int i) {
                float r[8];
                ld8(s, sb + 16 * i); ld8(r, sb + MB + 16 * i);
                ld_wait(); ld_there(s); ld_there(r);
#pragma unroll
                for (int e = 0; e < 8; ++e) s[e] = s[e] + r[e];
            };
            // distances of the logarithms from their references
            auto measure = [&](float (&d)[8], int i) {
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const float4 c = *reinterpret_cast<const float4*>(&x.c[8 * (2 * i + grp) + e]), m = *reinterpret_cast<const float4*>(&x.mu[warp][8 * i + e]);
                    d[e] = fmaf(d[e], ks * c.x, -m.x); d[e + 1] = fmaf(d[e + 1], ks * c.y, -m.y); d[e + 2] = fmaf(d[e + 2], ks * c.z, -m.z); d[e + 3] = fmaf(d[e + 3], ks * c.w, -m.w);
                }
                if (hide) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) if (hide >> (8 * i + e) & 1) d[e] = -INFINITY;
                }
            };
            // a full block: the distances of all sets stay in registers, their loads in flight together
            const bool full = nc == NC;
            float da[NC][8];
            auto measure_all = [&] {
                float r[NC][8];
#pragma unroll
                for (int i = 0; i < NC; ++i) { ld8(da[i], sb + 16 * i); ld8(r[i], sb + MB + 16 * i); }
                ld_wait();
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    ld_there(da[i]); ld_there(r[i]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) da[i][e] = da[i][e] + r[i][e];
                }
#pragma unroll
                for (int i = 0; i < NC; ++i) measure(da[i], i);
            };
            float top = -INFINITY;
            if (full) {
                measure_all();
#pragma unroll
                for (int i = 0; i < NC; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, da[i][e]);
            } else {
#pragma unroll 1
                for (int i = 0; i < nc; ++i) {
                    float d[8];
                    scores(d, i); measure(d, i);
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, d[e]);
                }
            }
            if (__any_sync(0xffffffffu, top + lv > MU_LIMIT) && lane == 0) x.moved[n & 3][grp] = n + 1;
            group_sync(grp);
            if (x.moved[n & 3][grp] == n + 1) {   // rare behind the first tiles. A pair moves by its own keys alone
                float mine = -INFINITY;
#pragma unroll 1
                for (int i = 0; i < nc; ++i) {
                    float d[8];
                    scores(d, i);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float m = warp_max(hide >> (8 * i + e) & 1 ? -INFINITY : d[e] * (ks * x.c[8 * (2 * i + grp) + e]) + lv);
                        if (lane == 8 * i + e) mine = m;
                    }
                }
                if (lane < 8 * NC) x.top[grp][qt][lane] = mine;
                group_sync(grp);
                float al = 1.f;
                if (lane < 8 * NC) {
                    const float m = fmaxf(fmaxf(x.top[grp][0][lane], x.top[grp][1][lane]), fmaxf(x.top[grp][2][lane], x.top[grp][3][lane])), mu = x.mu[warp][lane], next = ceilf(m) - MU_TOP;
                    if (m - mu > MU_LIMIT) { al = pow2i(mu - next); x.mu[warp][lane] = next; }
                    if (qt == 0) x.alpha[n & 3][8 * (2 * (lane >> 3) + grp) + (lane & 7)] = al;
                }
#pragma unroll 1
                for (int i = 0; i < nc; ++i) {
                    float l[8];
                    ld8(l, lcol + 16 * i); ld_wait(); ld_there(l);
#pragma unroll
                    for (int e = 0; e < 8; ++e) l[e] = l[e] * __shfl_sync(0xffffffffu, al, 8 * i + e);
                    st8(lcol + 16 * i, l); st_wait();
                }
                __syncwarp();
                if (full) measure_all();
            }
            ok = ok && warp_wait(smem_u32(&x.pv_done), (n & 1) ^ 1, a.err);   // the weights of the tile before are read
            auto weigh = [&](float (&d)[8], float (&l)[8], int i) {
                uint32_t h[4], r[4];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float p0 = ex2(d[e]), p1 = ex2(d[e + 1]);
                    l[e] = l[e] + p0; l[e + 1] = l[e + 1] + p1;
                    float y0 = p0 * vs, y1 = p1 * vs;
                    if (hide) { y0 = hide >> (8 * i + e) & 1 ? 0.f : y0; y1 = hide >> (8 * i + e + 1) & 1 ? 0.f : y1; }   // a masked key's scale may be anything
                    const __half2 hh = __floats2half2_rn(y0, y1);
                    const float2 f = __half22float2(hh);
                    h[e / 2] = h2_bits(hh); r[e / 2] = h2_bits(__floats2half2_rn(y0 - f.x, y1 - f.y));
                }
                st8(lcol + 16 * i, l);
                const int ch = 2 * i + grp, cr = MB / 8 + ch;   // eights of columns; 64 columns of all keys lie one behind the other
                *reinterpret_cast<uint4*>(pw + (ch >> 3) * (TK * 128) + (((ch & 7) ^ (key & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4*>(pw + (cr >> 3) * (TK * 128) + (((cr & 7) ^ (key & 7)) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
            };
            if (full) {
                float l[NC][8];
#pragma unroll
                for (int i = 0; i < NC; ++i) ld8(l[i], lcol + 16 * i);
                ld_wait();
#pragma unroll
                for (int i = 0; i < NC; ++i) ld_there(l[i]);
#pragma unroll
                for (int i = 0; i < NC; ++i) weigh(da[i], l[i], i);
            } else {
#pragma unroll 1
                for (int i = 0; i < nc; ++i) {
                    float d[8], l[8];
                    ld8(l, lcol + 16 * i);
                    scores(d, i);
                    ld_there(l);
                    measure(d, i);
                    weigh(d, l, i);
                }
            }
            st_wait();
            tc_fence_before();
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) { mbar_arrive(smem_u32(&x.s_empty[n & 1])); mbar_arrive(smem_u32(&x.p_full)); }
            ks = ks1; vs = vs1;
        }
        // weights' sums: the 32 keys of a warp in a tree, then the warps in order
#pragma unroll 1
        for (int i = 0; i < nc; ++i) {
            float l[8];
            ld8(l, lcol + 16 * i); ld_wait(); ld_there(l);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float v = l[e];
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) v = v + __shfl_xor_sync(0xffffffffu, v, off);
                if (lane == 0) x.l[grp][qt][8 * i + e] = v;
            }
        }
        group_sync(grp);
        if (ok && qt == 0 && lane < 8 * NC) {
            const int pair = 8 * (2 * (lane >> 3) + grp) + (lane & 7);
            if (pair < np && x.at[pair] >= 0)
                a.pml[(size_t)x.at[pair] * (a.ns + a.nwin) + blockIdx.x] = make_float2(x.mu[warp][lane], ((x.l[grp][0][lane] + x.l[grp][1][lane]) + x.l[grp][2][lane]) + x.l[grp][3][lane]);
        }
    } else if (warp < Geo::W_MMA) {   // ---- sums
        const int b = (warp - Geo::W_ACC) >> 2, qt = warp & 3, dim = 128 * b + 32 * qt + lane;
        const uint32_t ob = tmem + ((uint32_t)qt << 21) + 2 * N + b * N;
        float O[MB];
#pragma unroll
        for (int i = 0; i < MB; ++i) O[i] = 0.f;
        int n = 0;
#pragma unroll 1
        for (int t = t_first; t < t_end && ok; t = first_from(t + 1), ++n) {
            ok = warp_wait(smem_u32(&x.pv_done), n & 1, a.err);
            if (!ok) break;
            tc_fence_after();
            const int moved[2] = {x.moved[n & 3][0], x.moved[n & 3][1]};
#pragma unroll
            for (int c0 = 0; c0 < MB / 8; c0 += 2) {
                if (8 * c0 < np) {
                    float f[2][8], g[2][8];
#pragma unroll
                    for (int c = 0; c < 2; ++c) { ld8(f[c], ob + 8 * (c0 + c)); ld8(g[c], ob + MB + 8 * (c0 + c)); }
                    ld_wait();
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        ld_there(f[c]); ld_there(g[c]);
                        float* o = O + 8 * (c0 + c);
                        if (moved[c] == n + 1) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) o[e] = o[e] * x.alpha[n & 3][8 * (c0 + c) + e];
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] = o[e] + (f[c][e] + g[c][e]);
                    }
                }
            }
            tc_fence_before();
            warp_arrive(smem_u32(&x.o_empty), lane);
        }
        if (ok && dim < D) {
#pragma unroll
            for (int i = 0; i < MB; ++i)
                if (i < np && x.at[i] >= 0) a.pO[((size_t)x.at[i] * (a.ns + a.nwin) + blockIdx.x) * D + dim] = O[i];
        }
    } else if (warp == Geo::W_MMA) {   // ---- products
        const uint32_t base = smem_u32(sm);
        constexpr uint32_t ID_S = (1u << 4) | ((uint32_t)(N >> 3) << 17) | (8u << 24), ID_O = ID_S | (1u << 15) | (1u << 16);   // f32 = f16 x f16, M = 128; O: both operands M- / N-major
        int n = 0;
#pragma unroll 1
        for (int t = t_first; ok; ++n) {   // scores of tile n, outputs of tile n - 1
            const bool more = t < t_end;
            if (more) {
                ok = warp_wait(smem_u32(&x.k_full), n & 1, a.err) && warp_wait(smem_u32(&x.s_empty[n & 1]), ((n >> 1) & 1) ^ 1, a.err);
                if (!ok) break;
                tc_fence_after();
                if (tc_elect()) {
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)   // 16 dims
                        mma_f16(tmem + (n & 1) * N, desc128(base + Geo::OFF_K + (i >> 2) * (TK * 128) + (i & 3) * 32, 16), desc128(base + Geo::OFF_Q + (i >> 2) * (N * 128) + (i & 3) * 32, 16), ID_S, i != 0);
                    tc_commit(smem_u32(&x.s_full[n & 1]));
                    tc_commit(smem_u32(&x.k_empty));
                }
                __syncwarp();
                t = first_from(t + 1);
            }
            if (n) {
                const int m = n - 1;
                ok = warp_wait(smem_u32(&x.p_full), m & 1, a.err) && warp_wait(smem_u32(&x.v_full), m & 1, a.err) && warp_wait(smem_u32(&x.o_empty), (m & 1) ^ 1, a.err);
                if (!ok) break;
                tc_fence_after();
                if (tc_elect()) {
#pragma unroll
                    for (int d = 0; d < NB; ++d)
#pragma unroll
                        for (int i = 0; i < TK / 16; ++i)   // 16 keys
                            mma_f16(tmem + 2 * N + d * N, desc128(base + Geo::OFF_V + d * 2 * (TK * 128) + i * 2048, TK * 128), desc128(base + Geo::OFF_P + i * 2048, TK * 128), ID_O, i != 0);
                    tc_commit(smem_u32(&x.pv_done));
                }
                __syncwarp();
            }
            if (!more) break;
        }
        if (tc_elect()) tc_commit(smem_u32(&x.fin));
        __syncwarp();
        tc_wait(smem_u32(&x.fin), 0, a.err);   // nothing in flight when the accumulator memory is given back
    } else {   // ---- copies: k of tile n when the scores of tile n - 1 are there, v when the outputs are
        const int kv = warp == Geo::W_V;
        const uint8_t* src = a.f16 + (((size_t)sq.s * a.pool.n_kv + kh) * a.tiles * 2 + kv) * Geo::PICTURE;
        const uint32_t full = smem_u32(kv ? &x.v_full : &x.k_full), empty = smem_u32(kv ? &x.pv_done : &x.k_empty), dst = smem_u32(sm) + (kv ? Geo::OFF_V : Geo::OFF_K);
        int n = 0;
        for (int t = t_first; t < t_end && ok; t = first_from(t + 1)) {
            ok = warp_wait(empty, (n & 1) ^ 1, a.err);
            if (!ok) break;
            if (tc_elect()) {
                mbar_expect_tx(full, Geo::PICTURE);
#pragma unroll
                for (int i = 0; i < D / 64; ++i) bulk_g2s(dst + i * (TK * 128), src + (size_t)t * (2 * Geo::PICTURE) + i * (TK * 128), TK * 128, full);
            }
            __syncwarp();
            ++n;
        }
        if (n) tc_wait(full, (n - 1) & 1, a.err);   // no copy outlives the CTA
    }
    tc_fence_before();
    __syncthreads();
    if (warp == Geo::W_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Geo::TMEM) : "memory");
}

// The pictures: grid (tiles, 2 n_kv, sequences); a thread turns 16 codes into two pieces of 16 bytes. Tokens that no row sees are zeros in a tile of which others are seen;
// tiles without a visible token are not written, nor read.
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
    uint8_t* const dst = a.f16 + ((((size_t)blockIdx.z * a.pool.n_kv + h) * a.tiles + t) * 2 + kv) * ((size_t)TK * D * 2);
    const uint8_t* src = kv ? a.pool.v : a.pool.k;
    for (int e0 = threadIdx.x; e0 < TK * cpr; e0 += 4 * 256) {
        uint4 w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int e = e0 + u * 256, row = e / cpr, part = e % cpr;
            w[u] = make_uint4(0, 0, 0, 0);   // codes of zero
            if (e < TK * cpr && rows[row >> 4] != 0xffffffffu && t * TK + row < q.len) w[u] = *reinterpret_cast<const uint4*>(src + ((size_t)rows[row >> 4] + (row & 15)) * D + part * 16);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int e = e0 + u * 256, row = e / cpr, part = e % cpr;
            if (e >= TK * cpr) break;
            uint8_t* o = dst + (part >> 2) * (TK * 128) + row * 128;
            const int ch = (part & 3) * 2;
            *reinterpret_cast<uint4*>(o + ((ch ^ (row & 7)) << 4)) = make_uint4(code_pair<KIND, 0>(w[u].x), code_pair<KIND, 2>(w[u].x), code_pair<KIND, 0>(w[u].y), code_pair<KIND, 2>(w[u].y));
            *reinterpret_cast<uint4*>(o + (((ch + 1) ^ (row & 7)) << 4)) = make_uint4(code_pair<KIND, 0>(w[u].z), code_pair<KIND, 2>(w[u].z), code_pair<KIND, 0>(w[u].w), code_pair<KIND, 2>(w[u].w));
        }
    }
}

template <int D, int KIND, int MB> int launch_split(const PagedArgs& a, dim3 grid, cudaStream_t s) {
    using Geo = PagedGeo<D, MB>;
    static bool attr[MAX_DEVICES] = {};   // per device: the opt-in belongs to the device's copy of the kernel
    const int dev = current_device(); if (dev < 0) return HP_ECUDA;
    if (!attr[dev]) { HP_CUDA(cudaFuncSetAttribute(k_paged_prompt<D, KIND, MB>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo::SMEM)); attr[dev] = true; }
    HP_CUDA(launch_pdl<4>(k_paged_f16<KIND>, dim3(a.tiles, 2 * a.pool.n_kv, a.b.S), dim3(256), 0, s, a));
    HP_CUDA(launch_pdl<4>(k_paged_prompt<D, KIND, MB>, grid, dim3(Geo::WARPS * 32), Geo::SMEM, s, a));
    return HP_OK;
}
template <int KIND> int launch_split(const PagedArgs& a, dim3 grid, cudaStream_t s) {
    return a.pool.head_dim == 256 ? launch_split<256, KIND, PAGED_TC_PAIRS>(a, grid, s) : a.pool.head_dim == 128 ? launch_split<128, KIND, PAGED_TC_PAIRS>(a, grid, s) : launch_split<64, KIND, PAGED_TC_PAIRS>(a, grid, s);
}

}  // namespace

size_t attn_paged_tc_bytes(const PagedPool& pool, const PagedBatch& b) { return (size_t)b.S * pool.n_kv * ((b.max_kv + TK - 1) / TK) * (2 * TK * 2) * pool.head_dim; }
int attn_paged_tc(PagedArgs& a, dim3 grid, cudaStream_t s) {
    a.tiles = (a.b.max_kv + TK - 1) / TK;
    HP_REQUIRE(a.b.S <= 65535 && 2 * a.pool.n_kv <= 65535, "attn_paged: too many sequences (%d) or heads for a prompt", a.b.S);
    return a.pool.kind == KV_I8 ? launch_split<KV_I8>(a, grid, s) : launch_split<KV_E4M3>(a, grid, s);
}

}  // namespace hp
