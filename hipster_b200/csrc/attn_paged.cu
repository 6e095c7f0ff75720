// Attention of a ragged batch of rows over a cache of 8-bit pages (kv_pages.cu), with a window and first tokens that stay visible.
//
// Row r at position p of its sequence: o = sum_j w_j v_j / sum_j w_j over the keys j <= p with j > p - window or j < n_sink (no window: all), w_j =
// 2^(s_j - mu), s_j = (q . k_j) * scale * log2 e, times sigmoid(gate). No key: zeros.
//
// fp32 results from the f16 tensor pipe: codes of int8 and of e4m3 (times 2^-8) are exact in f16, a token's scale multiplies its score or its weight in
// fp32, and q and the weights (times the scale of v) go in as two f16 each, the value and what is left of it: 22 bits. q is brought to [2^14, 2^15) by a
// power of two per row, the weights by the reference mu: whole, at least the largest of s_j + log2(scale of v_j) - 14, so that a weight times
// its scale stays below 2^15 and every rescaling is by a power of two, exact. The tensor pipe adds 16 keys (or head_dim products) at a time; these sums
// are added to the running ones in fp32.
//
// The pairs (row, head) of a sequence and kv head, row by row, are cut into blocks of up to 32; a CTA holds one block and the keys of one split, in tiles of
// 64 keys through a ring of asynchronous copies. Four warps share 16 pairs, a quarter of each tile each, scores, weights and outputs in
// registers from end to end. Splits lie at fixed positions and a warp's sums at fixed keys: a row's bits depend neither on the other rows of the call
// nor on the other sequences.
#include "paged.cuh"
#include <algorithm>

namespace hp {
namespace {

constexpr int TK = 64, KW = 4, KPW = TK / KW, KPAD = 32, VPAD = 16;   // keys of a tile, warps that share it, keys of a warp in it; bytes behind a row of k / v in shared memory: 64-bit reads of 4 rows x 4 lanes from distinct banks
constexpr int MAX_TILES_M = 2;                           // 16-pair tiles of a CTA

__host__ __device__ constexpr int out_stride(int D) { return D + 4; }
struct PagedArgs {
    PagedPool pool; PagedBatch b;
    const float* q; size_t q_ld, q_hs; int n_head, G; float scale2;   // scale2 = scale * log2 e (times 256 for e4m3)
    int window, n_sink;
    int U, ns, nwin, stages;    // keys of a split, splits of the first tokens, splits behind them, stages of the ring
    float* pO; float2* pml;     // partials [row][head][ns + nwin] (x head_dim): sums, (mu, sum of weights)
    int* err;
};

__host__ __device__ constexpr int stage_bytes(int D) { return TK * (2 * D + KPAD + VPAD) + 2 * TK * 4; }
__host__ __device__ constexpr int q_bytes(int D, int m) { return m * D * 64; }   // per 16 pairs and 16 dims: two fragments (value, rest) of 32 lanes x 16 bytes

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float lg2(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float pow2i(float d) { return d < -126.f ? 0.f : __uint_as_float((uint32_t)((int)d + 127) << 23); }   // 2^d, d whole and <= 0
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// Four codes as they are loaded -> what `pair` takes; bytes LO and LO + 1 of it as two f16. int8: the code plus 128 becomes the low bits of 1024 + code + 128,
// and 1152 is subtracted, exactly. e4m3: its bits are those of the f16 2^-8 times as large, subnormals included (so 0x7f, which the quantiser does
// not write, reads as 480 and not as NaN: bytes of absent tokens are harmless).
template <int KIND> __device__ __forceinline__ uint32_t prepare4(uint32_t w) { return KIND == KV_I8 ? w ^ 0x80808080u : w; }
template <int KIND, int LO> __device__ __forceinline__ uint32_t pair(uint32_t w) {
    if constexpr (KIND == KV_I8) {
        const uint32_t h = prmt(w, 0x64646464u, LO == 0 ? 0x4140 : 0x4342);
        return h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&h), __floats2half2_rn(1152.f, 1152.f)));
    } else {
        const uint32_t h = prmt(w, 0u, LO == 0 ? 0x1404 : 0x3424);
        return (h & 0x80008000u) | ((h >> 1) & 0x3f803f80u);
    }
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void cp_async4_u(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait(int left) {
    switch (left) {
        case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
        case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
        case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
        default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    }
}
template <typename T> __device__ __forceinline__ T at_smem(const uint8_t* p) { return *reinterpret_cast<const T*>(p); }

// The block of pairs that blockIdx.z stands for: sequences in order, each with ceil(T * G / MB) blocks.
struct Block { PagedSeq q; int p0, np; };
__device__ __forceinline__ Block find_block(const PagedBatch& b, int G, int MB, int blk, int lane, int* err) {
    Block o; o.q.s = -1; o.p0 = o.np = 0;
    int acc = 0;
    for (int s0 = 0; s0 < b.S; s0 += 32) {
        PagedSeq q{-1, 0, 0, 0};
        if (s0 + lane < b.S) q = paged_seq(b, s0 + lane, err);
        const int n = (q.T * G + MB - 1) / MB;
        int incl = n;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) { const int t = __shfl_up_sync(0xffffffffu, incl, off); if (lane >= off) incl += t; }
        const unsigned hit = __ballot_sync(0xffffffffu, acc + incl > blk);
        if (hit) {
            const int l = __ffs(hit) - 1;
            o.q.s = s0 + l; o.q.row0 = __shfl_sync(0xffffffffu, q.row0, l); o.q.T = __shfl_sync(0xffffffffu, q.T, l); o.q.len = __shfl_sync(0xffffffffu, q.len, l);
            o.p0 = (blk - acc - __shfl_sync(0xffffffffu, incl - n, l)) * MB;
            o.np = min(MB, o.q.T * G - o.p0);
            return o;
        }
        acc += __shfl_sync(0xffffffffu, incl, 31);
    }
    return o;
}

// grid (splits, n_kv, blocks), 128 threads per 16 pairs
template <int D, int KIND>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2) k_paged_split(PagedArgs a) {
    constexpr int KS = D + KPAD, VS = D + VPAD, CPR = D / 16, NT = KPW / 8, XS = out_stride(D);   // row strides in shared memory, 16-byte pieces of a row, 8-key tiles of a warp
    static_assert(NT == 2, "the weights of a warp are one fragment");
    extern __shared__ __align__(16) uint8_t sm[];
    const int tid = threadIdx.x, nthr = blockDim.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q4 = lane & 3;
    const int MT = nthr / (32 * KW), MB = MT * 16, mw = warp / KW, kw = warp % KW;
    uint8_t* const sQ = sm;
    float* const sC = reinterpret_cast<float*>(sm + q_bytes(D, MT));        // [MB] factor of a pair's scores
    int* const sPos = reinterpret_cast<int*>(sC + MB);                      // [MB] position of a pair's row, -1: no pair
    uint8_t* const ring = reinterpret_cast<uint8_t*>(sPos + MB);
    const uint32_t ring_u = smem_u32(ring);
    pdl_launch_dependents();
    pdl_wait();
    const Block blk = find_block(a.b, a.G, MB, blockIdx.z, lane, a.err);
    if (blk.q.s < 0) return;
    const PagedSeq& sq = blk.q;
    const int kh = blockIdx.y;
    const int pos_lo = sq.len - sq.T + blk.p0 / a.G, pos_hi = sq.len - sq.T + (blk.p0 + blk.np - 1) / a.G;
    const int kend = pos_hi + 1, lo = a.window ? max(0, pos_lo - a.window + 1) : 0, sink = a.window ? a.n_sink : 0;   // keys [0, sink) and [lo, kend)
    int split = blockIdx.x;
    if (split >= a.ns) {   // the split of the window whose number leaves this remainder
        const int w0 = max(a.ns, lo / a.U), m = (w0 - a.ns) % a.nwin, j = split - a.ns - m;
        split = w0 + (j < 0 ? j + a.nwin : j);
    }
    const long long u0 = (long long)split * a.U;
    if (u0 >= kend) return;
    const int t_end = (int)((min(u0 + a.U, (long long)kend) + TK - 1) / TK);
    auto first_from = [&](int t) { return t * TK >= sink && t * TK + TK <= lo ? lo / TK : t; };   // first visible tile at or behind t
    int lt = first_from((int)(u0 / TK));   // next tile to fetch
    if (lt >= t_end) return;

    // ---- fetching: a lane holds the page of 16-token pieces of the tile; key rows go round the threads
    const int lg = a.pool.lg_page, pmask = (1 << lg) - 1, row_step = nthr / CPR, row_of = tid / CPR, col = (tid % CPR) * 16;
    auto page_of = [&](int t) -> uint32_t {   // of the tile's page number `lane`
        const int c = ((t * TK) >> lg) + lane;
        uint32_t p = 0;
        const long long k = (long long)c << lg;   // a page without a visible key is not looked up: page 0 stands for it, and for a number out of range
        if (t < t_end && lane < max(1, TK >> lg) && k < kend && (k < sink || k + pmask >= lo)) p = paged_row(a.pool, sq.s, c, kh, a.err);
        return p == 0xffffffffu ? 0u : p;
    };
    uint32_t pages = page_of(lt);
    auto fetch = [&](int slot) {
        if (lt < t_end) {
            const int k0 = lt * TK, c0 = k0 >> lg;
            const uint32_t st = ring_u + slot * stage_bytes(D);
#pragma unroll 4
            for (int r0 = 0; r0 < TK; r0 += row_step) {   // the same number of steps for every lane
                const int r = r0 + row_of, key = k0 + r;
                const size_t at = (size_t)__shfl_sync(0xffffffffu, pages, (key >> lg) - c0) + (key & pmask);
                if (r < TK && key < kend) {
                    cp_async16(st + r * KS + col, a.pool.k + at * D + col);
                    cp_async16(st + TK * KS + r * VS + col, a.pool.v + at * D + col);
                }
            }
            for (int i = warp * 32; i < 2 * TK; i += nthr) {
                const int r = (i + lane) & (TK - 1), key = k0 + r;
                const size_t at = (size_t)__shfl_sync(0xffffffffu, pages, (key >> lg) - c0) + (key & pmask);
                if (key < kend) cp_async4_u(st + TK * (KS + VS) + (i + lane) * 4, (i < TK ? a.pool.k_scale : a.pool.v_scale) + at);
            }
            lt = first_from(lt + 1);
            pages = page_of(lt);
        }
        cp_commit();
    };
    int ct = lt;   // tile to compute
    for (int i = 0; i + 1 < a.stages; ++i) fetch(i);

    // ---- q: a warp per pair; its 8 dims of a lane are one fragment word of two steps of 16 dims each, for the values and for the rests
    for (int i = warp; i < MB; i += nthr >> 5) {
        float x[8];
        uint32_t m = 0;
        const bool live = i < blk.np;
        const int p = blk.p0 + i, t = live ? p / a.G : 0;
        if (lane < D / 8) {
            float4 x0 = make_float4(0.f, 0.f, 0.f, 0.f), x1 = x0;
            if (live) {
                const float4* src = reinterpret_cast<const float4*>(a.q + (size_t)(sq.row0 + t) * a.q_ld + (size_t)(kh * a.G + p - t * a.G) * a.q_hs) + 2 * lane;
                x0 = src[0]; x1 = src[1];
            }
            x[0] = x0.x; x[1] = x0.y; x[2] = x0.z; x[3] = x0.w; x[4] = x1.x; x[5] = x1.y; x[6] = x1.z; x[7] = x1.w;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
        }
        m = __reduce_max_sync(0xffffffffu, m);
        const int e = m == 0 || m >= 0x7f800000u ? 0 : min(100, 14 - ((int)(m >> 23) - 127));
        const float up = __uint_as_float((uint32_t)(e + 127) << 23);
        if (lane < D / 8) {
            uint32_t* dst = reinterpret_cast<uint32_t*>(sQ + (size_t)(i >> 4) * D * 64 + (lane >> 2) * 2048) + ((i & 7) * 4 + (lane & 3)) * 4 + ((i >> 3) & 1);
#pragma unroll
            for (int j = 0; j < 4; ++j) {   // dims 2 j, 2 j + 1: step j / 2, words 0 and 2 (rows 8 and more: 1 and 3)
                const float y0 = x[2 * j] * up, y1 = x[2 * j + 1] * up;
                const __half2 h = __floats2half2_rn(y0, y1);
                const float2 f = __half22float2(h);
                const __half2 l = __floats2half2_rn(y0 - f.x, y1 - f.y);
                dst[(j >> 1) * 256 + (j & 1) * 2] = h2_bits(h);
                dst[(j >> 1) * 256 + 128 + (j & 1) * 2] = h2_bits(l);
            }
        }
        if (lane == 0) { sC[i] = a.scale2 * __uint_as_float((uint32_t)(127 - e) << 23); sPos[i] = live ? max(-1, sq.len - sq.T + t) : -1; }
    }
    __syncthreads();
    const int i0 = mw * 16 + g, i1 = i0 + 8;   // this lane's pairs
    const float c0 = sC[i0], c1 = sC[i1];
    const int p0 = sPos[i0], p1 = sPos[i1];
    const int w0 = a.window ? p0 - a.window : -1, w1 = a.window ? p1 - a.window : -1;   // keys behind these, or in front of `sink`
    const int mpos = (int)__reduce_max_sync(0xffffffffu, (unsigned)(max(p0, p1) + 1)) - 1;   // last position of the 16 pairs
    // tiles between these positions are visible to all 16 (an absent pair counts as nothing)
    const int all_hi = (int)__reduce_min_sync(0xffffffffu, (unsigned)min(p0 < 0 ? 0x7fffffff : p0, p1 < 0 ? 0x7fffffff : p1));
    const int all_lo = a.window ? mpos - a.window : -1;
    const uint8_t* const qf = sQ + mw * D * 64 + lane * 16;

    float O[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) { O[i][0] = O[i][1] = O[i][2] = O[i][3] = 0.f; }
    float mu0 = -1e30f, mu1 = -1e30f, l0 = 0.f, l1 = 0.f;

    for (int slot = 0; ct < t_end; ct = first_from(ct + 1), slot = slot + 1 == a.stages ? 0 : slot + 1) {
        cp_wait(a.stages - 2);
        __syncthreads();
        fetch(slot == 0 ? a.stages - 1 : slot - 1);
        const int kb = ct * TK + kw * KPW;
        if (kb > mpos) continue;   // nothing of this half is visible to these pairs
        const uint8_t* const st = ring + slot * stage_bytes(D);
        // ---- scores of 16 pairs x 16 keys
        float s[NT][4], sl[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[n][c] = sl[n][c] = 0.f;
        {
            const uint8_t* kr = st + (kw * KPW + g) * KS + q4 * 8;
#pragma unroll
            for (int x = 0; x < D / 32; ++x) {
                const uint4 h0 = at_smem<uint4>(qf + x * 2048), r0 = at_smem<uint4>(qf + x * 2048 + 512), h1 = at_smem<uint4>(qf + x * 2048 + 1024), r1 = at_smem<uint4>(qf + x * 2048 + 1536);
                uint32_t b[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint2 kk = at_smem<uint2>(kr + n * 8 * KS + x * 32);
                    const uint32_t w0 = prepare4<KIND>(kk.x), w1 = prepare4<KIND>(kk.y);
                    b[n][0] = pair<KIND, 0>(w0); b[n][1] = pair<KIND, 2>(w0); b[n][2] = pair<KIND, 0>(w1); b[n][3] = pair<KIND, 2>(w1);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) { mma_f16(s[n], h0, b[n][0], b[n][1]); mma_f16(sl[n], r0, b[n][0], b[n][1]); }
#pragma unroll
                for (int n = 0; n < NT; ++n) { mma_f16(s[n], h1, b[n][2], b[n][3]); mma_f16(sl[n], r1, b[n][2], b[n][3]); }
            }
        }
        // ---- weights
        const uint8_t* sc = st + TK * (KS + VS) + (kw * KPW + 2 * q4) * 4;
        float2 vs[NT];
        float t0 = -INFINITY, t1 = -INFINITY;
        const bool whole = kb + KPW - 1 <= all_hi && (kb > all_lo || kb + KPW <= sink);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float2 ks = at_smem<float2>(sc + n * 32);
            vs[n] = at_smem<float2>(sc + TK * 4 + n * 32);
            s[n][0] = (s[n][0] + sl[n][0]) * (ks.x * c0); s[n][1] = (s[n][1] + sl[n][1]) * (ks.y * c0);
            s[n][2] = (s[n][2] + sl[n][2]) * (ks.x * c1); s[n][3] = (s[n][3] + sl[n][3]) * (ks.y * c1);
        }
        float wv[NT][4];   // the scale of v that a weight takes
#pragma unroll
        for (int n = 0; n < NT; ++n) { wv[n][0] = wv[n][2] = vs[n].x; wv[n][1] = wv[n][3] = vs[n].y; }
        if (!whole) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int key = kb + n * 8 + 2 * q4 + (c & 1);
                    const bool see = key <= (c < 2 ? p0 : p1) && (key > (c < 2 ? w0 : w1) || key < sink);
                    if (!see) { s[n][c] = -INFINITY; wv[n][c] = 0.f; }
                }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float lx = lg2(fmaxf(vs[n].x, 8.0779357e-28f)), ly = lg2(fmaxf(vs[n].y, 8.0779357e-28f));   // 2^-90: the weights' sum cannot overflow
            t0 = fmaxf(t0, fmaxf(s[n][0] + lx, s[n][1] + ly));
            t1 = fmaxf(t1, fmaxf(s[n][2] + lx, s[n][3] + ly));
        }
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1)); t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2)); t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
        const float n0 = fmaxf(mu0, ceilf(t0) - 14.f), n1 = fmaxf(mu1, ceilf(t1) - 14.f);
        const float al0 = pow2i(mu0 - n0), al1 = pow2i(mu1 - n1);
        mu0 = n0; mu1 = n1; l0 = l0 * al0; l1 = l1 * al1;
        uint4 ph, pr;   // A fragment of the 16 keys: weights times scales, values and rests
        {
            uint32_t h[NT][2], r[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int c = 0; c < 4; c += 2) {
                    const float m = c ? mu1 : mu0, e0 = ex2(s[n][c] - m), e1 = ex2(s[n][c + 1] - m);
                    if (c) l1 = (l1 + e0) + e1; else l0 = (l0 + e0) + e1;
                    const float y0 = e0 * wv[n][c], y1 = e1 * wv[n][c + 1];
                    const __half2 hh = __floats2half2_rn(y0, y1);
                    const float2 f = __half22float2(hh);
                    h[n][c / 2] = h2_bits(hh); r[n][c / 2] = h2_bits(__floats2half2_rn(y0 - f.x, y1 - f.y));
                }
            }
            ph = make_uint4(h[0][0], h[0][1], h[1][0], h[1][1]); pr = make_uint4(r[0][0], r[0][1], r[1][0], r[1][1]);
        }
        // ---- outputs: 64 dims at a time, lane group g holds 8 neighbouring ones of the rows of its keys
        const uint8_t* vr = st + TK * KS + (kw * KPW + 2 * q4) * VS + g * 8;
#pragma unroll
        for (int y = 0; y < D / 64; ++y) {
            const uint2 v0 = at_smem<uint2>(vr + y * 64), v1 = at_smem<uint2>(vr + VS + y * 64), v2 = at_smem<uint2>(vr + 8 * VS + y * 64), v3 = at_smem<uint2>(vr + 9 * VS + y * 64);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint32_t a0 = prepare4<KIND>(w ? v0.y : v0.x), a1 = prepare4<KIND>(w ? v1.y : v1.x), a2 = prepare4<KIND>(w ? v2.y : v2.x), a3 = prepare4<KIND>(w ? v3.y : v3.x);
                const uint32_t u0 = prmt(a0, a1, 0x5140), u1 = prmt(a0, a1, 0x7362), u2 = prmt(a2, a3, 0x5140), u3 = prmt(a2, a3, 0x7362);
                const uint32_t b0[4] = {pair<KIND, 0>(u0), pair<KIND, 2>(u0), pair<KIND, 0>(u1), pair<KIND, 2>(u1)};
                const uint32_t b1[4] = {pair<KIND, 0>(u2), pair<KIND, 2>(u2), pair<KIND, 0>(u3), pair<KIND, 2>(u3)};
                float f[4][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) { f[j][0] = f[j][1] = f[j][2] = f[j][3] = 0.f; mma_f16(f[j], pr, b0[j], b1[j]); }
#pragma unroll
                for (int j = 0; j < 4; ++j) mma_f16(f[j], ph, b0[j], b1[j]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float (&o)[4] = O[y * 8 + w * 4 + j];
                    o[0] = fmaf(o[0], al0, f[j][0]); o[1] = fmaf(o[1], al0, f[j][1]); o[2] = fmaf(o[2], al1, f[j][2]); o[3] = fmaf(o[3], al1, f[j][3]);
                }
            }
        }
    }
    l0 = l0 + __shfl_xor_sync(0xffffffffu, l0, 1); l1 = l1 + __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 = l0 + __shfl_xor_sync(0xffffffffu, l0, 2); l1 = l1 + __shfl_xor_sync(0xffffffffu, l1, 2);

    // ---- the warps that share the tiles meet, in order. Thread (g, q4) holds dims 64 y + 16 q4 + 0..15 of rows g and g + 8
    cp_wait(0);
    __syncthreads();   // the ring and q are free
    float* const xo = reinterpret_cast<float*>(sm);   // [warp][16][XS]: D sums, mu, sum of weights
    {
        float* dst = xo + (size_t)(warp * 16 + g) * XS + 16 * q4;
#pragma unroll
        for (int y = 0; y < D / 64; ++y)
#pragma unroll
            for (int j = 0; j < 8; j += 4)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *reinterpret_cast<float4*>(dst + (c >> 1) * 8 * XS + 64 * y + 8 * (c & 1) + j) = make_float4(O[y * 8 + j][c], O[y * 8 + j + 1][c], O[y * 8 + j + 2][c], O[y * 8 + j + 3][c]);
        if (q4 == 0) {
            float* e = xo + (size_t)(warp * 16 + g) * XS + D;
            e[0] = mu0; e[1] = l0; e[8 * XS] = mu1; e[8 * XS + 1] = l1;
        }
    }
    __syncthreads();
    for (int i = warp; i < blk.np; i += nthr >> 5) {   // a warp per pair
        const int p = blk.p0 + i, t = p / a.G;
        if (sq.len - sq.T + t < 0) continue;
        const float* src = xo + (size_t)((i >> 4) * KW * 16 + (i & 15)) * XS;
        float m[KW], w[KW], mu = -INFINITY, l = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) { m[k] = src[k * 16 * XS + D]; mu = fmaxf(mu, m[k]); }
#pragma unroll
        for (int k = 0; k < KW; ++k) { w[k] = pow2i(m[k] - mu); l = fmaf(src[k * 16 * XS + D + 1], w[k], l); }
        const size_t at = ((size_t)(sq.row0 + t) * a.n_head + kh * a.G + p - t * a.G) * (a.ns + a.nwin) + blockIdx.x;
        for (int d = 2 * lane; d < D; d += 64) {
            float2 o = make_float2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < KW; ++k) { const float2 v = *reinterpret_cast<const float2*>(src + k * 16 * XS + d); o.x = fmaf(v.x, w[k], o.x); o.y = fmaf(v.y, w[k], o.y); }
            *reinterpret_cast<float2*>(a.pO + at * D + d) = o;
        }
        if (lane == 0) a.pml[at] = make_float2(mu, l);
    }
}

// Splits of a row in order, gate, f32 and q8 outputs. One block of head_dim threads per row and head.
struct MergeArgs {
    PagedBatch b; const float* pO; const float2* pml; const float* gate; size_t g_ld, g_hs; int n_head, D, window, n_sink, U, ns, nwin; float mul;
    float* out; int8_t* oq; float* osc; int* err;
};
__global__ void __launch_bounds__(256) k_paged_merge(MergeArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int r = blockIdx.x / a.n_head, head = blockIdx.x % a.n_head, d = threadIdx.x, lane = d & 31;
    const PagedSeq q = paged_find(a.b, r, lane, a.err);
    if (q.s < 0) return;
    const int pos = q.len - q.T + r - q.row0;
    float v = 0.f;
    if (pos >= 0) {
        const int lo = a.window ? max(0, pos - a.window + 1) : 0, w0 = max(a.ns, lo / a.U), w1 = pos / a.U;
        const int s1 = a.ns ? (min(a.n_sink, pos + 1) + a.U - 1) / a.U : 0;   // splits [0, s1) and [w0, w1]
        const int n = s1 + max(0, w1 - w0 + 1);
        const size_t base = ((size_t)r * a.n_head + head) * (a.ns + a.nwin);
        auto slot = [&](int i) { return base + (i < s1 ? i : a.ns + (w0 + i - s1 - a.ns) % a.nwin); };
        float mu = -INFINITY;
        for (int i = lane; i < n; i += 32) mu = fmaxf(mu, a.pml[slot(i)].x);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) mu = fmaxf(mu, __shfl_xor_sync(0xffffffffu, mu, off));
        float o = 0.f, l = 0.f;
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const size_t at = slot(i);
            const float2 ml = a.pml[at];
            const float w = pow2i(ml.x - mu);
            o = fmaf(w, a.pO[at * a.D + d], o); l = fmaf(w, ml.y, l);
        }
        v = l == 0.f ? 0.f : o * a.mul / l;
        if (a.gate) v = v * sigmoid_det(a.gate[(size_t)r * a.g_ld + (size_t)head * a.g_hs + d]);
    }
    if (a.out) a.out[((size_t)r * a.n_head + head) * a.D + d] = v;
    if (a.oq) warp_quant32_store(v, r, (head * a.D + d) >> 5, a.n_head * a.D, a.oq, a.osc, lane);
}

struct Plan { int U, ns, nwin, MT; long long blocks; };
// Splits lie at multiples of U, a number that the cache's capacity and the window alone decide, so that a row's sums do not hang on what else is in the
// call. Calls of more than 8 rows per sequence (prompts) have blocks enough and take a row's keys as one split.
Plan plan_of(const PagedPool& pool, const PagedBatch& b, int n_head, int window, int n_sink) {
    Plan p;
    const int G = n_head / pool.n_kv, cap = pool.table_ld << pool.lg_page;
    const long long eff = window ? std::min<long long>(cap, (long long)window + n_sink) : cap;
    const long long pairs = (long long)b.max_rows * G, nb = (pairs + 16 * MAX_TILES_M - 1) / (16 * MAX_TILES_M);
    p.MT = (int)std::min<long long>(MAX_TILES_M, ((pairs + nb - 1) / nb + 15) / 16);
    const int MB = p.MT * 16;
    p.blocks = std::min<long long>((long long)b.S * ((pairs + MB - 1) / MB), (long long)b.R * G / MB + b.S);
    if (b.max_rows > 8) { p.U = 1 << 30; p.ns = 0; p.nwin = 1; return p; }
    p.U = eff <= 8192 ? 256 : eff <= 32768 ? 512 : 1024;
    const int total = (b.max_kv + p.U - 1) / p.U;   // splits of the longest sequence
    p.ns = window ? std::min((n_sink + p.U - 1) / p.U, total) : 0;
    p.nwin = std::max(1, total);
    if (window) {   // a block's rows see at most this many keys in a run
        const long long rows = std::min<long long>(b.max_rows, (MB - 1) / G + 2), run = (long long)window + rows - 1;
        p.nwin = (int)std::min<long long>(p.nwin, run < 2 ? 1 : (run - 2) / p.U + 2);
    }
    return p;
}
size_t partials(const Plan& p, const PagedBatch& b, int n_head) { return (size_t)b.R * n_head * (p.ns + p.nwin); }

template <int D, int KIND> int launch_split(const PagedArgs& a, dim3 grid, int MT, cudaStream_t s) {
    static bool attr[MAX_DEVICES] = {};   // per device: the opt-in belongs to the device's copy of the kernel
    const int dev = current_device(); if (dev < 0) return HP_ECUDA;
    if (!attr[dev]) { HP_CUDA(cudaFuncSetAttribute(k_paged_split<D, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024)); attr[dev] = true; }
    // the outputs of the tiles' halves pass through the same memory at the end
    const size_t smem = std::max<size_t>(q_bytes(D, MT) + MT * 16 * 8 + (size_t)a.stages * stage_bytes(D), (size_t)KW * MT * 16 * out_stride(D) * 4);
    HP_CUDA(launch_pdl<4>(k_paged_split<D, KIND>, grid, dim3(32 * KW * MT), smem, s, a));
    return HP_OK;
}

}  // namespace

size_t attn_paged_workspace_bytes(const PagedPool& pool, const PagedBatch& b, int n_head, int window, int n_sink) {
    const Plan p = plan_of(pool, b, n_head, window, n_sink);
    return partials(p, b, n_head) * (pool.head_dim + 2) * sizeof(float);
}

int attn_paged(const PagedPool& pool, const PagedBatch& b, const AttnPagedParams& p, cudaStream_t s) {
    const Plan pl = plan_of(pool, b, p.n_head, p.window, p.n_sink);
    HP_REQUIRE(pl.blocks <= 65535 && (long long)b.R * p.n_head < (1ll << 31), "attn_paged: too many rows (%d) for one call", b.R);
    PagedArgs a; a.pool = pool; a.b = b; a.q = p.q; a.q_ld = p.q_ld; a.q_hs = p.q_hs; a.n_head = p.n_head; a.G = p.n_head / pool.n_kv;
    a.scale2 = (float)((double)p.scale * 1.4426950408889634074 * (pool.kind == KV_E4M3 ? 256.0 : 1.0)); a.window = p.window; a.n_sink = p.n_sink;
    a.U = pl.U; a.ns = pl.ns; a.nwin = pl.nwin; a.stages = pool.head_dim == 256 ? (pl.MT == 1 ? 2 : 4) : 3;
    a.pO = (float*)p.workspace; a.pml = (float2*)(a.pO + partials(pl, b, p.n_head) * pool.head_dim); a.err = device_arg_flag();
    const dim3 grid(pl.ns + pl.nwin, pool.n_kv, (unsigned)pl.blocks);
    int rc;
    if (pool.kind == KV_I8) rc = pool.head_dim == 256 ? launch_split<256, KV_I8>(a, grid, pl.MT, s) : pool.head_dim == 128 ? launch_split<128, KV_I8>(a, grid, pl.MT, s) : launch_split<64, KV_I8>(a, grid, pl.MT, s);
    else rc = pool.head_dim == 256 ? launch_split<256, KV_E4M3>(a, grid, pl.MT, s) : pool.head_dim == 128 ? launch_split<128, KV_E4M3>(a, grid, pl.MT, s) : launch_split<64, KV_E4M3>(a, grid, pl.MT, s);
    if (rc != HP_OK) return rc;
    MergeArgs m; m.b = b; m.pO = a.pO; m.pml = a.pml; m.gate = p.gate; m.g_ld = p.g_ld; m.g_hs = p.g_hs; m.n_head = p.n_head; m.D = pool.head_dim; m.window = p.window; m.n_sink = p.n_sink;
    m.U = pl.U; m.ns = pl.ns; m.nwin = pl.nwin; m.mul = pool.kind == KV_E4M3 ? 256.f : 1.f; m.out = p.out; m.oq = (int8_t*)p.xq.q; m.osc = (float*)p.xq.sc; m.err = a.err;
    HP_CUDA(launch_pdl<4>(k_paged_merge, dim3((unsigned)(b.R * p.n_head)), dim3(pool.head_dim), 0, s, m));
    return HP_OK;
}

}  // namespace hp
