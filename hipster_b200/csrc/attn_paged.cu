// Attention of a ragged batch of rows over a cache of pages in 8 or 4 bits (kv_pages.cu), with a window and first tokens that stay visible: calls of up to
// 16 rows per sequence (decode steps, drafts, verify passes), the merge of the splits, and the plan. Prompts: attn_paged_tc.cu.
//
// Row r at position p of its sequence: o = sum_j w_j v_j / sum_j w_j over the keys j <= p with j > p - window or j < n_sink (no window: all), w_j =
// 2^(s_j - mu), s_j = (q . k_j) * scale * log2 e, times sigmoid(gate). No key: zeros.
//
// fp32 results from the f16 tensor pipe: codes of int8, of e4m3 (times 2^-8) and of 4 bits (u (c - z), times 2^-12) are exact in f16, a token's scale multiplies its score or its weight in
// fp32, and q and the weights (times the scale of v) go in as two f16 each, the value and what is left of it: 22 bits. q is brought to [2^14, 2^15) by a
// power of two per row, the weights by the reference mu, which is whole: every rescaling is by a power of two, exact (MU_TOP in paged.cuh). The tensor pipe adds up
// head_dim / 2 products for a score, in three sums, and 16 keys for an output; these are added to the running sums in fp32 (4 bits: by the tensor pipe itself).
//
// Keys, and dims, are the 16 rows of mma.sync, the pairs (row of the batch, query head) of a kv head its 8 columns: few pairs waste nothing. A warp has 16 keys at a
// time, every fourth such slice of its CTA's split, in a ring of three slots of its own (k, v, k, ...), so that no warp waits for another; 16 keys of a head
// lie in one page, one run of memory. The weights change from rows of keys to columns of pairs by movmatrix. Splits lie at fixed positions and a
// slice's keys at fixed lanes and warps: a row's bits depend neither on the other rows of the call nor on the other sequences.
//
// A warp looks up the pages of all its slices at once, a lane each, and fetches a slice's scales with its keys; hidden keys are masked in the slices that have some.
//
// Measured (captured, us): one token of 24 heads of 256 over 4 at 4097 11.9 (bytes alone 1.3): start, four slices per warp and merge one after the other. 48 such sequences of up to
// 8192 108 to 114 by card (80), 118 to 121 with the page looked up per slice, every slice masked, and blocks looked for where each sequence has one: issue slots 58 %, a third of the instructions turning codes into f16. 8 x 3 rows over 2 kv heads at 2051 21.3 (2.0); 32 x 2
// rows of 32 heads of 128, window 1000, 32.5 (11): half of the instructions are starts and ends of the CTAs. Pairs as the 16 rows of the products: 260 for the 48 sequences; eight warps per CTA: 128.
// 4 bits: one token at 4097 11.5 (0.7), the 48 sequences 100 (43), 64 of 32 heads of 128 over 8 at up to 12001 211 (86): issue slots 57 to 66 %; a slice takes 464 instructions at 128 dims, 675 at 256,
// a warp and split some 850 and 1050 around them. Two dims become f16 by one mask and one fma; by two masks and conversions 129 for the 48. Products of tcgen05 with the pictures of attn_paged_tc.cu: 15.9 for one token, 180 for the 48;
// a head's dims split over the warps, 64 keys shared by them: 13.1, 110.
// Two sets of pairs spill up to 56 bytes a thread (4 bits, 64 dims; 8 bits 40), 256 dims and one set none.
#include "paged.cuh"
#include <algorithm>
#include <type_traits>

namespace hp {
namespace {

constexpr int KW = 4, KS = 16, SLOTS = 3;   // warps that share a split, keys of a slice, slots of a warp's ring
__host__ __device__ constexpr int out_stride(int D) { return D + 4; }
__host__ __device__ constexpr int row_bytes(int D, int KIND) { return KIND == KV_I4 ? D / 2 : D; }                       // codes of a row
__host__ __device__ constexpr int code_bytes(int D, int KIND) { return KS * (row_bytes(D, KIND) + (KIND == KV_I4 ? D / 32 : 0)); }   // of a slice; 4 bits: codes, then the bytes of the groups
__host__ __device__ constexpr int slot_bytes(int D, int KIND) { return code_bytes(D, KIND) + 2 * KS * 4; }                            // and, beside a slice's k, its scales of k and of v
__host__ __device__ constexpr int smem_bytes(int D, int KIND, int NT) {   // fragments of q | rings; the outputs of the warps pass through the same memory at the end
    const int run = NT * D * 32 + KW * SLOTS * slot_bytes(D, KIND), end = KW * NT * 8 * out_stride(D) * 4;
    return run > end ? run : end;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {   // c = a * b: no zeros to be put into registers
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) { uint32_t r; asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v)); return r; }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
template <typename T> __device__ __forceinline__ T at_smem(const uint8_t* p) { return *reinterpret_cast<const T*>(p); }
// Where 16-byte piece c of row r of a slot lies. k is read as 8 bytes of four neighbouring rows and four neighbouring places, v of every second row: each
// of these has to hit 16 different pairs of banks, so neighbours (v: every second) shift by two pieces. 64 dims: two rows share 128 bytes, and
// rows 4 to 7 swap halves.
template <int D, bool V> __device__ __forceinline__ int place(int r, int c) {
    if constexpr (D == 64) return (r >> 1) * 128 + (((r & 1) ^ ((r >> 2) & 1)) << 6) + ((c ^ (((r >> 1) & 1) << 1)) << 4);
    else return r * D + ((c ^ (((V ? r >> 1 : r) & 3) << 1)) << 4);
}
// The same for 4 bits, rows of D / 2 bytes. A lane reads a group of k (16 bytes) of rows g, and of v D / 8 dims (16, 8 or 4 bytes) of every second row. 256 dims: rows are 128 bytes, and neighbours (v: every
// second) shift. 128 dims: v as above for rows of 64 bytes; k, and 64 dims' k, hit distinct banks as they lie. 64 dims, v: four rows share 128 bytes, rows 4 to 7 swap neighbours.
template <int D, bool V> __device__ __forceinline__ int place4(int r, int c) {
    if constexpr (D == 256) return r * 128 + ((c ^ (V ? ((r >> 1) & 3) << 1 : (r & 1) << 2)) << 4);
    else if constexpr (D == 128) return V ? place<64, true>(r, c) : r * 64 + (c << 4);
    else return V ? (r >> 2) * 128 + ((r & 3) ^ ((r >> 2) & 1)) * 32 + (c << 4) : r * 32 + (c << 4);
}
template <int D, int KIND, bool V> __device__ __forceinline__ int place_of(int r, int c) { if constexpr (KIND == KV_I4) return place4<D, V>(r, c); else return place<D, V>(r, c); }

// grid (splits, n_kv, blocks), four warps; NT sets of 8 pairs. DIRECT: the only split there is writes the outputs itself
template <int D, int KIND, int NT, bool DIRECT>
__global__ void __launch_bounds__(32 * KW, NT == 2 ? (D == 256 ? 2 : D == 128 ? 3 : 4) : (D == 256 ? 3 : 4)) k_paged_split(const PagedArgs a) {
    constexpr int RB = row_bytes(D, KIND), SLOT = slot_bytes(D, KIND), SCALES = code_bytes(D, KIND), CPR = RB / 16, MB = 8 * NT, XS = out_stride(D);   // 16-byte pieces of a row
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ float s_c[MB];   // factor of a pair's scores
    __shared__ int s_pos[MB];   // position of a pair's row, -1: none
    __shared__ float s_mu[KW][MB], s_l[KW][MB];
    __shared__ float* s_out[MB];
    __shared__ int s_row[MB];   // direct: row of a pair
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q4 = lane & 3;
    pdl_wait();
    pdl_launch_dependents();   // behind the wait: what was enqueued in front of this kernel is complete when the merge starts
    const Block blk = a.single ? only_block(a.b, a.G, blockIdx.z, a.arg_err) : find_block(a.b, a.G, MB, blockIdx.z, lane, a.arg_err);
    if (blk.q.s < 0) return;
    const PagedSeq& sq = blk.q;
    const Span sp = span_of(a, blk);
    const int kh = blockIdx.y;
    if (sp.u0 >= sp.kend && !DIRECT) return;   // direct: rows without a key are zeros
    // slices of 16 keys [i * 16, i * 16 + 16): those of this warp leave remainder `warp`. Visible are those in front of the end of the first tokens and those from the window's first key on: two runs, na
    // slices from ia and the others from ib. A split has 1024 keys at most: 16 slices per warp
    const int i_end = (int)((sp.u1 + KS - 1) / KS), i_lo = sp.lo / KS, i_first = (int)(sp.u0 / KS);
    {   // is any slice of the split visible?
        if ((i_first * KS >= sp.sink && i_first < i_lo ? i_lo : i_first) >= i_end && !DIRECT) return;
    }
    const int ia = i_first + ((warp - i_first) & (KW - 1)), a_end = min(i_end, sp.sink / KS + (sp.sink % KS != 0)), na = max(0, (a_end - ia + KW - 1) / KW);
    int ib = max(ia + na * KW, i_lo);
    ib += (warp - ib) & (KW - 1);
    const int n_slices = na + max(0, (i_end - ib + KW - 1) / KW);
    auto slice = [&](int t) { return t < na ? ia + t * KW : ib + (t - na) * KW; };
    // q: a warp per pair, 8 dims per lane; under way while the pages are looked up
    constexpr int QP = MB / KW;
    float4 qv[QP][2];
#pragma unroll
    for (int u = 0; u < QP; ++u) {
        const int i = warp + KW * u, p = blk.p0 + i, t = p / a.G;
        qv[u][0] = qv[u][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < blk.np && lane < D / 8) {
            const float4* src = reinterpret_cast<const float4*>(a.q + (size_t)(sq.row0 + t) * a.q_ld + (size_t)(kh * a.G + p - t * a.G) * a.q_hs) + 2 * lane;
            qv[u][0] = src[0]; qv[u][1] = src[1];
        }
    }
    const int lg = a.pool.lg_page, pmask = (1 << lg) - 1;
    // the pool's rows of the warp's slices' first keys, a slice per lane; 0 for a page number out of range (told by the status word)
    uint32_t where = 0;
    if (lane < n_slices) {
        const int i = slice(lane);
        const uint32_t r = paged_row(a.pool, sq.s, (i * KS) >> lg, kh, a.arg_err);
        where = r == 0xffffffffu ? 0u : r + (uint32_t)((i * KS) & pmask);
    }
    uint8_t* const ring = sm + NT * D * 32 + warp * (SLOTS * SLOT);
    const uint32_t ring_u = smem_u32(ring);
    // A slot's 16 rows are one run of memory; piece e = 32 i + lane of it goes to place(e / CPR, e % CPR), which is 512 i and a part that repeats after two (k) or four (v) i
    int kput[2], vput[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = 32 * i + lane;
        if (i < 2) kput[i] = place_of<D, KIND, false>(e / CPR, e % CPR) - 512 * i;
        vput[i] = place_of<D, KIND, true>(e / CPR, e % CPR) - 512 * i;
    }
    const uint8_t* const kbase = a.pool.k + lane * 16; const uint8_t* const vbase = a.pool.v + lane * 16;
    // slice t's k and scales, its v
    const float* const sbase = (lane < 16 ? a.pool.k_scale : a.pool.v_scale) + (lane & 15);   // scales of k in lanes 0 to 15, of v in the others
    auto fetch_k = [&](int slot, int t) {
        const uint32_t row = __shfl_sync(0xffffffffu, where, t & 31);
        if (t < n_slices) {
            const uint8_t* src;
            cp_async4(ring + slot * SLOT + SCALES + lane * 4, sbase + row);
            if constexpr (KIND == KV_I4) {
                const I4Row at = i4_row(row, lg, D);
                src = kbase + at.codes;
                if (lane < D / 32) cp_async16(ring_u + slot * SLOT + KS * RB + lane * 16, kbase + at.groups);
            } else src = kbase + (size_t)row * D;
            const uint32_t d0 = ring_u + slot * SLOT + kput[0], d1 = ring_u + slot * SLOT + kput[1];
#pragma unroll
            for (int i = 0; i < KS * CPR / 32; ++i) cp_async16((i & 1 ? d1 : d0) + 512 * i, src + 512 * i);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto fetch_v = [&](int slot, int t) {
        const uint32_t row = __shfl_sync(0xffffffffu, where, t & 31);
        if (t < n_slices) {
            const uint32_t at = ring_u + slot * SLOT, d[4] = {at + vput[0], at + vput[1], at + vput[2], at + vput[3]};
            const uint8_t* src;
            if constexpr (KIND == KV_I4) {
                const I4Row from = i4_row(row, lg, D);
                src = vbase + from.codes;
                if (lane < D / 32) cp_async16(at + KS * RB + lane * 16, vbase + from.groups);
            } else src = vbase + (size_t)row * D;
#pragma unroll
            for (int i = 0; i < KS * CPR / 32; ++i) cp_async16(d[i & 3] + 512 * i, src + 512 * i);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int m = 0; m < SLOTS; ++m) { if (m & 1) fetch_v(m, m / 2); else fetch_k(m, m / 2); }   // k and v in turn

    // the 8 dims of a lane are its words of two steps of 16 dims, values and rests; 4 bits: dims i and i + 4 side by side, at the step and the four lanes that the word of codes falls to
#pragma unroll
    for (int u = 0; u < QP; ++u) {
        const int i = warp + KW * u, t = (blk.p0 + i) / a.G;
        const float x[8] = {qv[u][0].x, qv[u][0].y, qv[u][0].z, qv[u][0].w, qv[u][1].x, qv[u][1].y, qv[u][1].z, qv[u][1].w};
        const bool live = i < blk.np;
        const int step = KIND != KV_I4 ? lane >> 2 : D == 64 ? lane & 1 : (lane >> 4) * 4 + (lane & 3), four = KIND != KV_I4 ? lane & 3 : D == 64 ? lane >> 1 : (lane >> 2) & 3;
        uint4* const dst = reinterpret_cast<uint4*>(sm + (i >> 3) * D * 32 + step * 1024) + (i & 7) * 4 + four;
        if (!live) {   // the warp's: zeros
            if (lane < D / 8) dst[0] = dst[32] = make_uint4(0u, 0u, 0u, 0u);
            if (lane == 0) { s_c[i] = a.scale2; s_pos[i] = -1; }
            continue;
        }
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
        m = __reduce_max_sync(0xffffffffu, m);
        const int e = q_exponent(m);
        const float up = __uint_as_float((uint32_t)(e + 127) << 23);
        if (lane < D / 8) {
            uint32_t h[4], r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float y0 = x[KIND == KV_I4 ? j : 2 * j] * up, y1 = x[KIND == KV_I4 ? j + 4 : 2 * j + 1] * up;
                const __half2 hh = __floats2half2_rn(y0, y1);
                const float2 f = __half22float2(hh);
                h[j] = h2_bits(hh); r[j] = h2_bits(__floats2half2_rn(y0 - f.x, y1 - f.y));
            }
            dst[0] = make_uint4(h[0], h[1], h[2], h[3]);
            dst[32] = make_uint4(r[0], r[1], r[2], r[3]);
        }
        if (lane == 0) { s_c[i] = a.scale2 * __uint_as_float((uint32_t)(127 - e) << 23); s_pos[i] = max(-1, sq.len - sq.T + t); }
    }
    __syncthreads();
    float cf[NT][2], mu[NT][2], l[NT][2];
    int pos[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) { cf[n][c] = s_c[8 * n + 2 * q4 + c]; pos[n][c] = s_pos[8 * n + 2 * q4 + c]; mu[n][c] = MU_NONE; l[n][c] = 0.f; }
    const int win = a.window ? a.window : 1 << 30;
    // slices between these positions are visible to all pairs
    const int all_hi = sp.pos_lo, all_lo = a.window ? sp.pos_hi - a.window : -1;
    const uint8_t* const qf = sm + lane * 16;

    float O[D / 16][NT][4];   // dims (tile m of 64 y: 64 y + 8 g + 2 m, and the next one; 4 bits: D / 8 * g + 8 y + 2 m) x pairs (2 q4, 2 q4 + 1)
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) { O[i][n][0] = O[i][n][1] = O[i][n][2] = O[i][n][3] = 0.f; }

    // where a lane's 8 bytes lie: rows g and g + 8 of k (these shift alike), the 32 dims x; rows 2 q4 and 2 q4 + 1 (+ 8) of v, the 64 dims y
    int kofs[4], vofs[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) kofs[i] = KIND == KV_I4 ? (i < D / 128 ? place4<D, false>(g, q4 + 4 * i) : place4<D, false>(g, q4 >> 1) + (q4 & 1) * 8) : i < D / 32 ? place<D, false>(g, 2 * i + (q4 >> 1)) + (q4 & 1) * 8 : 0;   // 4 bits: groups q4 and q4 + 4; 64 dims: half of one
#pragma unroll
    for (int i = 0; i < 4; ++i) vofs[i >> 1][i & 1] = KIND == KV_I4 ? place4<D, true>(2 * q4 + (i >> 1), g / (256 / D)) + g % (256 / D) * (D / 16) : (i & 1) < D / 64 ? place<D, true>(2 * q4 + (i >> 1), 4 * (i & 1) + (g >> 1)) + (g & 1) * 8 : 0;   // 4 bits: D / 8 dims from D / 8 * g on
    int slot = 0;
    constexpr int AHEAD = SLOTS / 2;   // slices of v; k is fetched one further
#pragma unroll 1
    for (int t = 0; t < n_slices; ++t) {
        const int i0 = slice(t);
        asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 1) : "memory");
        __syncwarp();
        const float* const sc = reinterpret_cast<const float*>(ring + slot * SLOT + SCALES);
        const float k0 = sc[g], k1 = sc[g + 8], v0 = sc[g + 16], v1 = sc[g + 24];
        // ---- scores of 16 keys
        float s[NT][4];
        {
            float sh[NT][2][4], sl[NT][4];
            const uint8_t* kr = ring + slot * SLOT;
            auto products = [&](int x, const uint32_t (&a0)[4], const uint32_t (&a1)[4]) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint4 h = at_smem<uint4>(qf + n * D * 32 + x * 1024), r = at_smem<uint4>(qf + n * D * 32 + x * 1024 + 512);
                    if (x == 0) { mma_f16_first(sh[n][0], a0, h.x, h.y); mma_f16_first(sl[n], a0, r.x, r.y); mma_f16_first(sh[n][1], a1, h.z, h.w); }
                    else { mma_f16(sh[n][0], a0, h.x, h.y); mma_f16(sl[n], a0, r.x, r.y); mma_f16(sh[n][1], a1, h.z, h.w); }
                    mma_f16(sl[n], a1, r.z, r.w);
                }
            };
            if constexpr (KIND == KV_I4) {
                constexpr int PER = D == 64 ? 2 : 4;   // words of a lane that lie together, in one group
#pragma unroll
                for (int y = 0; y < D / 32 / PER; ++y) {
                    const uint8_t *kx = kr + kofs[y], *gx = kr + KS * RB + g * (D / 32) + (D == 64 ? q4 >> 1 : q4 + 4 * y);
                    const I4Group ga = i4_group(__byte_perm(gx[0], 0x64u, 0x4040)), gb = i4_group(__byte_perm(gx[8 * (D / 32)], 0x64u, 0x4040));
                    uint32_t ka[PER], kb[PER];
                    if constexpr (PER == 4) {
                        const uint4 u = at_smem<uint4>(kx), v = at_smem<uint4>(kx + 8 * RB);
                        ka[0] = u.x; ka[1] = u.y; ka[2] = u.z; ka[3] = u.w; kb[0] = v.x; kb[1] = v.y; kb[2] = v.z; kb[3] = v.w;
                    } else {
                        const uint2 u = at_smem<uint2>(kx), v = at_smem<uint2>(kx + 8 * RB);
                        ka[0] = u.x; ka[1] = u.y; kb[0] = v.x; kb[1] = v.y;
                    }
#pragma unroll
                    for (int i = 0; i < PER; ++i) {
                        const uint32_t a0[4] = {i4_low(ka[i], ga), i4_low(kb[i], gb), i4_high(ka[i], ga), i4_high(kb[i], gb)};
                        const uint32_t a1[4] = {i4_low(ka[i] >> 8, ga), i4_low(kb[i] >> 8, gb), i4_high(ka[i] >> 8, ga), i4_high(kb[i] >> 8, gb)};
                        products(y * PER + i, a0, a1);
                    }
                }
            } else {
#pragma unroll
                for (int x = 0; x < D / 32; ++x) {
                    const uint8_t* kx = kr + kofs[x & 3] + (x >> 2) * 128;
                    const uint2 ka = at_smem<uint2>(kx), kb = at_smem<uint2>(kx + 8 * D);
                    const uint32_t a0[4] = {code_pair<KIND, 0>(ka.x), code_pair<KIND, 0>(kb.x), code_pair<KIND, 2>(ka.x), code_pair<KIND, 2>(kb.x)};
                    const uint32_t a1[4] = {code_pair<KIND, 0>(ka.y), code_pair<KIND, 0>(kb.y), code_pair<KIND, 2>(ka.y), code_pair<KIND, 2>(kb.y)};
                    products(x, a0, a1);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[n][c] = (sh[n][0][c] + sh[n][1][c]) + sl[n][c];
        }
        __syncwarp();
        fetch_v(slot, t + AHEAD);
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
        // ---- weights
        const float lv0 = scale_lg2(v0), lv1 = scale_lg2(v1);
        const int j = i0 * KS + g;
        const bool whole = i0 * KS + KS - 1 <= all_hi && (i0 * KS > all_lo || i0 * KS + KS <= sp.sink);
        uint32_t hidden = 0;   // a bit per score; most slices have none
        if (!whole) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) { const int key = c < 2 ? j : j + 8, p = pos[n][c & 1]; hidden |= (uint32_t)!(key <= p && (key > p - win || key < sp.sink)) << (4 * n + c); }
        }
        float d[NT][4], top = -INFINITY;
        auto distance = [&](int n, int c) { return fmaf(s[n][c], (c < 2 ? k0 : k1) * cf[n][c & 1], -mu[n][c & 1]); };
        auto hide = [&](float none) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) if (hidden >> (4 * n + c) & 1) d[n][c] = none;
        };
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) d[n][c] = distance(n, c);
        if (!whole) hide(-INFINITY);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) top = fmaxf(top, d[n][c] + (c < 2 ? lv0 : lv1));
        if (__any_sync(0xffffffffu, top > MU_LIMIT)) {   // rare behind the first slices. A pair moves by its own keys alone, and by the very sums that brought the warp here: others, rounded elsewhere, would move it only beside a pair that moves
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float t = fmaxf(d[n][c] + lv0 > MU_LIMIT ? s[n][c] * (k0 * cf[n][c]) + lv0 : -INFINITY, d[n][c + 2] + lv1 > MU_LIMIT ? s[n][c + 2] * (k1 * cf[n][c]) + lv1 : -INFINITY);
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4)); t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8)); t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                    if (t > -INFINITY) {
                        const float next = mu_next(mu[n][c], t), al = pow2i(mu[n][c] - next);
                        l[n][c] = add_scaled(0.f, l[n][c], al, mu[n][c] - next); mu[n][c] = next;
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) { O[i][n][c] = O[i][n][c] * al; O[i][n][c + 2] = O[i][n][c + 2] * al; }
                    }
                }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) d[n][c] = cut_off(distance(n, c), c < 2 ? lv0 : lv1);
            if (!whole) hide(-INFINITY);
        }
        uint32_t bh[NT][2], br[NT][2];   // weights times scales of v as columns of pairs: values and rests
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float e0 = ex2(d[n][c]), e1 = ex2(d[n][c + 2]);
                l[n][c] = l[n][c] + (e0 + e1);
                d[n][c] = e0 * v0; d[n][c + 2] = e1 * v1;
            }
        if (!whole) hide(0.f);   // a masked key's scale may be anything
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const __half2 hh = __floats2half2_rn(d[n][2 * c], d[n][2 * c + 1]);
                const float2 f = __half22float2(hh);
                bh[n][c] = transpose8(h2_bits(hh)); br[n][c] = transpose8(h2_bits(__floats2half2_rn(d[n][2 * c] - f.x, d[n][2 * c + 1] - f.y)));
            }
        asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 1) : "memory");
        __syncwarp();
        // ---- outputs: 64 dims at a time; the 8 dims of a lane group are four tiles of 16 rows
        {
            const uint8_t* vr = ring + slot * SLOT;
            auto products = [&](float (&o)[NT][4], const uint32_t (&af)[4]) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (KIND == KV_I4) {   // into the running sums: two products, a step of 2^-23 of them each, 2^-22 per slice at most, 2^-18 in a split (16 slices of a warp); the 48 sequences of the head of this file 107 us so, 114 with adds of their own
                        mma_f16(o[n], af, br[n][0], br[n][1]);
                        mma_f16(o[n], af, bh[n][0], bh[n][1]);
                        continue;
                    }
                    float f[4];
                    mma_f16_first(f, af, br[n][0], br[n][1]);
                    mma_f16(f, af, bh[n][0], bh[n][1]);
                    const float2 u = add2(make_float2(o[n][0], o[n][1]), make_float2(f[0], f[1])), t = add2(make_float2(o[n][2], o[n][3]), make_float2(f[2], f[3]));
                    o[n][0] = u.x; o[n][1] = u.y; o[n][2] = t.x; o[n][3] = t.y;
                }
            };
            if constexpr (KIND == KV_I4) {   // D / 64 words of a lane group, of one group of 32 dims; a word is four tiles
                constexpr int W = D / 64;
                uint32_t v[4][W];   // keys 2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint8_t* vx = vr + vofs[i & 1][0] + (i >> 1) * 8 * RB;
                    if constexpr (W == 4) { const uint4 u = at_smem<uint4>(vx); v[i][0] = u.x; v[i][1] = u.y; v[i][2] = u.z; v[i][3] = u.w; }
                    else if constexpr (W == 2) { const uint2 u = at_smem<uint2>(vx); v[i][0] = u.x; v[i][1] = u.y; }
                    else v[i][0] = at_smem<uint32_t>(vx);
                }
                const uint8_t* gx = vr + KS * RB + 2 * q4 * (D / 32) + g / (256 / D);
                const I4Group ga = i4_group(gx[0] | (uint32_t)gx[D / 32] << 16 | 0x64006400u), gb = i4_group(gx[8 * (D / 32)] | (uint32_t)gx[9 * (D / 32)] << 16 | 0x64006400u);
#pragma unroll
                for (int w = 0; w < W; ++w)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t lo = __byte_perm(v[0][w], v[1][w], h ? 0x7632 : 0x5410), hi = __byte_perm(v[2][w], v[3][w], h ? 0x7632 : 0x5410);   // four dims of two keys
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t af[4] = {i4_low(lo >> (8 * k), ga), i4_high(lo >> (8 * k), ga), i4_low(hi >> (8 * k), gb), i4_high(hi >> (8 * k), gb)};
                            products(O[w * 4 + h * 2 + k], af);
                        }
                    }
            } else {
#pragma unroll
                for (int y = 0; y < D / 64; ++y) {
                    uint2 v[4];   // keys 2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = at_smem<uint2>(vr + vofs[i & 1][y & 1] + (y >> 1) * 128 + (i >> 1) * 8 * D);
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const uint32_t x0 = w ? v[0].y : v[0].x, x1 = w ? v[1].y : v[1].x, x2 = w ? v[2].y : v[2].x, x3 = w ? v[3].y : v[3].x;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t lo2 = __byte_perm(x0, x1, h ? 0x7362 : 0x5140), hi2 = __byte_perm(x2, x3, h ? 0x7362 : 0x5140);
                            const uint32_t af[4] = {code_pair<KIND, 0>(lo2), code_pair<KIND, 2>(lo2), code_pair<KIND, 0>(hi2), code_pair<KIND, 2>(hi2)};
                            products(O[y * 4 + w * 2 + h], af);
                        }
                    }
                }
            }
        }
        __syncwarp();
        fetch_k(slot, t + AHEAD + 1);
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) l[n][c] = l[n][c] + __shfl_xor_sync(0xffffffffu, l[n][c], off);

    // ---- the warps meet, in order
    cp_async_wait_all();
    __syncthreads();   // rings and q are free
    float* const xo = reinterpret_cast<float*>(sm);   // [warp][pair][XS]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float* dst = xo + (size_t)(warp * MB + 8 * n + 2 * q4 + c) * XS + (KIND == KV_I4 ? D / 8 : 8) * g;
#pragma unroll
            for (int y = 0; y < D / 64; ++y)
#pragma unroll
                for (int m = 0; m < 4; m += 2)
                    *reinterpret_cast<float4*>(dst + (KIND == KV_I4 ? 8 : 64) * y + 2 * m) = make_float4(O[y * 4 + m][n][c], O[y * 4 + m][n][c + 2], O[y * 4 + m + 1][n][c], O[y * 4 + m + 1][n][c + 2]);
            if (g == 0) { s_mu[warp][8 * n + 2 * q4 + c] = mu[n][c]; s_l[warp][8 * n + 2 * q4 + c] = l[n][c]; }
        }
    __syncthreads();
    if (tid < blk.np) {   // a thread per pair: the warps' factors, the weights' sum, and where the sums go
        const int p = blk.p0 + tid, t = p / a.G;
        float m = -INFINITY, ls = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) m = fmaxf(m, s_mu[k][tid]);
#pragma unroll
        for (int k = 0; k < KW; ++k) { const float d = s_mu[k][tid] - m, w = pow2i(d); s_mu[k][tid] = w; ls = add_scaled(ls, s_l[k][tid], w, d); }
        if (DIRECT) { s_l[0][tid] = ls; s_row[tid] = sq.row0 + t; s_pos[tid] = kh * a.G + p - t * a.G; }   // its head in place of its position
        else {
            const bool live = s_pos[tid] >= 0;
            const size_t at = ((size_t)(sq.row0 + t) * a.n_head + kh * a.G + p - t * a.G) * (a.ns + a.nwin) + blockIdx.x;
            s_out[tid] = live ? a.pO + at * D : nullptr;
            if (live) a.pml[at] = make_float2(m, ls);
        }
    }
    __syncthreads();
#pragma unroll 4
    for (int e = tid; e < blk.np * (D / 4); e += 32 * KW) {
        const int i = e / (D / 4), d = e % (D / 4) * 4;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < KW; ++k) {
            const float4 v = *reinterpret_cast<const float4*>(xo + (size_t)(k * MB + i) * XS + d); const float w = s_mu[k][i];
            o.x = fmaf(v.x, w, o.x); o.y = fmaf(v.y, w, o.y); o.z = fmaf(v.z, w, o.z); o.w = fmaf(v.w, w, o.w);
        }
        if constexpr (DIRECT) put(o, s_l[0][i], s_row[i], s_pos[i], d, D, a);
        else if (s_out[i]) *reinterpret_cast<float4*>(s_out[i] + d) = o;
    }
}

// Splits of a row, gate, f32 and q8 outputs; more than eight splits, or gates and outputs at odd addresses. A block per row and head: D / 4 threads hold four dims each, and 1024 / D sets of them take every such
// split in order; the sets are added in order. Bound by latency: the row, its place and gate are read ahead of the dependency wait (the kernel of the splits
// releases this one once its predecessors are complete), the partials of up to four splits of each set are in flight.
struct MergeArgs {
    PagedBatch b; const float* pO; const float2* pml; const float* gate; size_t g_ld, g_hs; int n_head, window, n_sink, U, ns, nwin; float mul;
    float* out; int8_t* oq; float* osc; int* err;
};
template <int D>
__global__ void __launch_bounds__(256) k_paged_merge(const MergeArgs a) {
    constexpr int TD = D / 4, SETS = 256 / TD, PF = 4;
    __shared__ float4 s_o[SETS][TD]; __shared__ float s_l[SETS];
    const int r = blockIdx.x / a.n_head, head = blockIdx.x % a.n_head, set = threadIdx.x / TD, d4 = threadIdx.x % TD, lane = threadIdx.x & 31;
    const PagedSeq q = paged_find(a.b, r, lane, a.err);
    const int pos = q.len - q.T + r - q.row0;
    float gate = 0.f;
    if (a.gate && q.s >= 0 && threadIdx.x < D) gate = a.gate[(size_t)r * a.g_ld + (size_t)head * a.g_hs + threadIdx.x];
    pdl_wait();
    pdl_launch_dependents();
    if (q.s < 0) return;
    const int lo = a.window ? max(0, pos - a.window + 1) : 0, w0 = max(a.ns, lo / a.U), w1 = max(pos, 0) / a.U;
    const int s1 = a.ns ? (min(a.n_sink, pos + 1) + a.U - 1) / a.U : 0;   // splits [0, s1) and [w0, w1]
    const int n = pos < 0 ? 0 : s1 + max(0, w1 - w0 + 1);
    const size_t base = ((size_t)r * a.n_head + head) * (a.ns + a.nwin);
    auto slot = [&](int i) { return base + (i < s1 ? i : a.ns + (w0 + i - s1 - a.ns) % a.nwin); };
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f); float l = 0.f, mu = -INFINITY;
    bool far = false;
    float4 v[PF];
#pragma unroll
    for (int i = 0; i < PF; ++i) if (set + i * SETS < n) v[i] = reinterpret_cast<const float4*>(a.pO + slot(set + i * SETS) * D)[d4];
    for (int i = lane; i < n; i += 32) mu = fmaxf(mu, a.pml[slot(i)].x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mu = fmaxf(mu, __shfl_xor_sync(0xffffffffu, mu, off));
    for (int i0 = set; i0 < n; i0 += PF * SETS) {
#pragma unroll
        for (int j = 0; j < PF; ++j) {
            const int i = i0 + j * SETS;
            if (i < n) {
                const float2 ml = a.pml[slot(i)];
                const float w = pow2i(ml.x - mu);
                o.x = fmaf(w, v[j].x, o.x); o.y = fmaf(w, v[j].y, o.y); o.z = fmaf(w, v[j].z, o.z); o.w = fmaf(w, v[j].w, o.w); l = fmaf(w, ml.y, l); far |= ml.x - mu < -126.f;
                if (i + PF * SETS < n) v[j] = reinterpret_cast<const float4*>(a.pO + slot(i + PF * SETS) * D)[d4];
            }
        }
    }
    if (far) {   // rare, so apart from the loop (8 x 3 rows over 2 kv heads at 2051: 22.3 us with it inside, 21.8)
        l = 0.f;
        for (int i = set; i < n; i += SETS) { const float2 ml = a.pml[slot(i)]; const float d = ml.x - mu; l = add_scaled(l, ml.y, pow2i(d), d); }
    }
    s_o[set][d4] = o;
    if (d4 == 0) s_l[set] = l;
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= D) return;
    float x = 0.f; l = 0.f;
#pragma unroll
    for (int i = 0; i < SETS; ++i) { x = x + reinterpret_cast<const float*>(&s_o[i][0])[d]; l = l + s_l[i]; }
    x = l == 0.f ? 0.f : x * a.mul / l;
    if (a.gate) x = x * sigmoid_det(gate);
    if (a.out) a.out[((size_t)r * a.n_head + head) * D + d] = x;
    if (a.oq) warp_quant32_store(x, r, (head * D + d) >> 5, a.n_head * D, a.oq, a.osc, lane);
}

// The same sums, bit for bit, where a row has at most eight splits: a thread for four dims over all splits, 1024 dims of a row's heads per block. k_paged_merge's blocks, a head each,
// are bound by their instructions and start-up once there are thousands of them. 509 rows of 24 heads in three splits (cold, us): 51 there, 27 here. At 256 dims five
// blocks per SM, with 48 registers a thread and 140 bytes spilled, take less than two with the 95 that 64 and 128 dims have (the call 146 us, 151); squeezed like that, 128 dims take more (32 x 2 rows of 32 heads
// behind a window: 41 us, 34).
constexpr int FEW = 8;
template <int D>
__global__ void __launch_bounds__(256, D == 256 ? 5 : 1) k_paged_merge_few(const MergeArgs a) {
    constexpr int HEADS = 1024 / D, SETS = 1024 / D < FEW ? 1024 / D : FEW;   // sums of k_paged_merge's sets
    const int per = (a.n_head + HEADS - 1) / HEADS, r = blockIdx.x / per, h = (blockIdx.x - r * per) * HEADS + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4, lane = threadIdx.x & 31;
    const PagedSeq q = paged_find(a.b, r, lane, a.err);
    const bool live = q.s >= 0 && h < a.n_head;
    float4 gate = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.gate && live) gate = *reinterpret_cast<const float4*>(a.gate + (size_t)r * a.g_ld + (size_t)h * a.g_hs + d);
    pdl_wait();
    pdl_launch_dependents();
    if (!__any_sync(0xffffffffu, live)) return;   // 64 dims: a warp has two heads
    const int pos = live ? q.len - q.T + r - q.row0 : -1;
    const int lo = a.window ? max(0, pos - a.window + 1) : 0, w0 = max(a.ns, lo / a.U), w1 = max(pos, 0) / a.U;
    const int s1 = a.ns ? (min(a.n_sink, pos + 1) + a.U - 1) / a.U : 0;   // splits [0, s1) and [w0, w1]
    const int n = pos < 0 ? 0 : s1 + max(0, w1 - w0 + 1), first = (w0 - a.ns) % a.nwin;
    const size_t base = ((size_t)r * a.n_head + h) * (a.ns + a.nwin);
    auto slot = [&](int i) { const int k = first + i - s1; return base + (i < s1 ? i : a.ns + (k < a.nwin ? k : k - a.nwin)); };
    float2 ml[FEW];
    float mu = -INFINITY;
#pragma unroll
    for (int i = 0; i < FEW; ++i) if (i < n) { ml[i] = a.pml[slot(i)]; mu = fmaxf(mu, ml[i].x); }
    float4 o[SETS]; float l[SETS];
#pragma unroll
    for (int i = 0; i < SETS; ++i) { o[i] = make_float4(0.f, 0.f, 0.f, 0.f); l[i] = 0.f; }
#pragma unroll
    for (int i0 = 0; i0 < FEW; i0 += 4) {
        if (i0 >= n) break;
        float4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) if (i0 + j < n) v[j] = *reinterpret_cast<const float4*>(a.pO + slot(i0 + j) * D + d);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j < n) {
                const float w = pow2i(ml[i0 + j].x - mu);
                float4& t = o[(i0 + j) % SETS];
                t.x = fmaf(w, v[j].x, t.x); t.y = fmaf(w, v[j].y, t.y); t.z = fmaf(w, v[j].z, t.z); t.w = fmaf(w, v[j].w, t.w); l[(i0 + j) % SETS] = add_scaled(l[(i0 + j) % SETS], ml[i0 + j].y, w, ml[i0 + j].x - mu);
            }
    }
    float x[4] = {0.f, 0.f, 0.f, 0.f}, ls = 0.f;
#pragma unroll
    for (int i = 0; i < SETS; ++i) { x[0] = x[0] + o[i].x; x[1] = x[1] + o[i].y; x[2] = x[2] + o[i].z; x[3] = x[3] + o[i].w; ls = ls + l[i]; }
    const float g[4] = {gate.x, gate.y, gate.z, gate.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = ls == 0.f ? 0.f : x[e] * a.mul / ls;
        if (a.gate) x[e] = x[e] * sigmoid_det(g[e]);
    }
    if (a.out && live) *reinterpret_cast<float4*>(a.out + ((size_t)r * a.n_head + h) * D + d) = make_float4(x[0], x[1], x[2], x[3]);
    if (a.oq) {   // runs of 32 dims lie in eight lanes: a run at a time to all lanes
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int from = 8 * b + (lane >> 2), at = __shfl_sync(0xffffffffu, live ? h * D + d : -1, 8 * b);
            if (at < 0) continue;
            const float y0 = __shfl_sync(0xffffffffu, x[0], from), y1 = __shfl_sync(0xffffffffu, x[1], from), y2 = __shfl_sync(0xffffffffu, x[2], from), y3 = __shfl_sync(0xffffffffu, x[3], from);
            warp_quant32_store((lane & 2) ? (lane & 1 ? y3 : y2) : (lane & 1 ? y1 : y0), r, at >> 5, a.n_head * D, a.oq, a.osc, lane);
        }
    }
}

struct Plan { int U, ns, nwin, MB; long long blocks; };
// Splits lie at multiples of U, which the cache's capacity and the window alone decide (16 to 32 splits and more of a full sequence), so that a row's sums do not hang on what
// else is in the call. Captured, us: 1 token of 24 heads at 4097, U = 128 12.8, 256 12.6, 512 16.9, 1024 26.6; 48 sequences of up to 8192, 187, 139, 118, 116.
// Prompts have blocks of rows: their keys are split as the launch fills the GPU best, a split costing the start of a CTA, some six tiles, and several of them
// the merge (without it in the sum 1000 rows of 24 heads 91 us, now 80). Sixteen splits at most (eight: 64 rows of 24 heads at 16000 104 us, now 91).
// Behind a window a block has all its keys in one split, however few the blocks: 17 rows of 24 heads over 4 at 8000 take 174 us with a window of 4000, 83 of 1000, 46 without one.
// A table for 131072 tokens has splits of 1024: one token at 4097 27.8 us there, 12.8 with a table of its own length; at 131072 both 79.
Plan plan_of(const PagedPool& pool, const PagedBatch& b, int n_head, int window, int n_sink, int cap) {
    Plan p;
    const int G = n_head / pool.n_kv;
    const long long eff = window ? std::min<long long>(cap, (long long)window + n_sink) : cap;
    const long long pairs = (long long)b.max_rows * G;
    const bool prompt = b.max_rows > PAGED_DECODE_ROWS;
    p.MB = prompt ? PAGED_TC_PAIRS : pairs <= 8 ? 8 : 16;
    p.blocks = std::min<long long>((long long)b.S * ((pairs + p.MB - 1) / p.MB), (long long)b.R * G / p.MB + b.S);
    p.U = eff < 8192 ? 256 : eff < 32768 ? 512 : 1024;
    if (prompt) {
        const long long ctas = p.blocks * pool.n_kv, band = (b.max_kv + 1023) / 1024 * 16, tiles = (b.max_kv + 63) / 64;   // of 64 keys; as many splits for all max_kv up to the next 1024: the workspace grows with max_kv
        long long best = 0; int n = 1;
        for (int i = 1; i <= 16; ++i) {
            const long long cost = (ctas * i + 147) / 148 * ((band + i - 1) / i + 6) + (i == 1 ? 0 : 2 + ((long long)b.R * n_head * pool.head_dim * (i + 1) * 8 >> 20) / 12);   // and the merge, 12 MB in the time of a tile
            if (i == 1 || cost < best) { best = cost; n = i; }
        }
        if (n == 1 || window) { p.U = 1 << 30; p.ns = 0; p.nwin = 1; }
        else { p.U = (int)((tiles + n - 1) / n * 64); p.ns = 0; p.nwin = n; }
        return p;
    }
    const int total = (b.max_kv + p.U - 1) / p.U;   // splits of the longest sequence
    p.ns = window ? std::min((n_sink + p.U - 1) / p.U, total) : 0;
    p.nwin = std::max(1, total);
    if (window) {   // a block's rows see at most this many keys in a run
        const long long rows = std::min<long long>(b.max_rows, (p.MB - 1) / G + 2), run = (long long)window + rows - 1;
        p.nwin = (int)std::min<long long>(p.nwin, run < 2 ? 1 : (run - 2) / p.U + 2);
    }
    return p;
}
size_t partials(const Plan& p, const PagedBatch& b, int n_head) { return (size_t)b.R * n_head * (p.ns + p.nwin); }

template <int D, int KIND, int NT, bool DIRECT> int launch_split(const PagedArgs& a, dim3 grid, cudaStream_t s) {
    constexpr int smem = smem_bytes(D, KIND, NT);
    static bool attr[MAX_DEVICES] = {};   // per device: the opt-in belongs to the device's copy of the kernel
    const int dev = current_device(); if (dev < 0) return HP_ECUDA;
    if (!attr[dev]) { HP_CUDA(cudaFuncSetAttribute(k_paged_split<D, KIND, NT, DIRECT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)); attr[dev] = true; }
    HP_CUDA(launch_pdl<4>(k_paged_split<D, KIND, NT, DIRECT>, grid, dim3(32 * KW), smem, s, a));
    return HP_OK;
}
template <int D, int KIND> int launch_split(const PagedArgs& a, dim3 grid, int MB, cudaStream_t s) {
    if (a.direct) return MB == 8 ? launch_split<D, KIND, 1, true>(a, grid, s) : launch_split<D, KIND, 2, true>(a, grid, s);
    return MB == 8 ? launch_split<D, KIND, 1, false>(a, grid, s) : launch_split<D, KIND, 2, false>(a, grid, s);
}
template <int KIND> int launch_split(const PagedArgs& a, dim3 grid, int MB, cudaStream_t s) {
    return a.pool.head_dim == 256 ? launch_split<256, KIND>(a, grid, MB, s) : a.pool.head_dim == 128 ? launch_split<128, KIND>(a, grid, MB, s) : launch_split<64, KIND>(a, grid, MB, s);
}

}  // namespace

size_t attn_paged_workspace_bytes(const PagedPool& pool, const PagedBatch& b, int n_head, int window, int n_sink, int cap) {
    const Plan p = plan_of(pool, b, n_head, window, n_sink, cap);
    return (partials(p, b, n_head) * (pool.head_dim + 2) * sizeof(float) + 127) / 128 * 128 + (b.max_rows > PAGED_DECODE_ROWS ? attn_paged_tc_bytes(pool, b) : 0);
}

int attn_paged(const PagedPool& pool, const PagedBatch& b, const AttnPagedParams& p, cudaStream_t s) {
    const Plan pl = plan_of(pool, b, p.n_head, p.window, p.n_sink, p.cap);
    HP_REQUIRE(pl.blocks <= 65535 && pool.n_kv <= 65535 && (long long)b.R * p.n_head < (1ll << 31), "attn_paged: too many rows (%d) or heads for one call", b.R);
    PagedArgs a; a.pool = pool; a.b = b; a.q = p.q; a.q_ld = p.q_ld; a.q_hs = p.q_hs; a.n_head = p.n_head; a.G = p.n_head / pool.n_kv;
    a.scale2 = (float)((double)p.scale * 1.4426950408889634074 * (pool.kind == KV_E4M3 ? 256.0 : pool.kind == KV_I4 ? (double)I4_UNIT : 1.0)); a.window = p.window; a.n_sink = p.n_sink;
    a.U = pl.U; a.ns = pl.ns; a.nwin = pl.nwin; a.single = (long long)b.max_rows * a.G <= pl.MB;
    a.pO = (float*)p.workspace; a.pml = (float2*)(a.pO + partials(pl, b, p.n_head) * pool.head_dim); a.err = device_err_flag(); a.arg_err = device_arg_flag();
    a.f16 = (uint8_t*)p.workspace + (partials(pl, b, p.n_head) * (pool.head_dim + 2) * sizeof(float) + 127) / 128 * 128; a.tiles = 0;
    a.gate = p.gate; a.g_ld = p.g_ld; a.g_hs = p.g_hs; a.mul = pool.kind == KV_E4M3 ? 256.f : pool.kind == KV_I4 ? I4_UNIT : 1.f; a.out = p.out; a.oq = (int8_t*)p.xq.q; a.osc = (float*)p.xq.sc;
    const bool wide = (((uintptr_t)p.gate | (uintptr_t)p.out) & 15) == 0 && (!p.gate || ((p.g_ld | p.g_hs) & 3) == 0);   // four dims of gate and output at a time
    // One split: its kernel writes the outputs, for the price of a merge's launch (captured and host's time of 32 tokens of 32 heads over 8 at 256 tokens 14.6 and 9.9 us, now 8.6 and 7.3)
    a.direct = wide && pl.ns + pl.nwin == 1;
    const dim3 grid(pl.ns + pl.nwin, pool.n_kv, (unsigned)pl.blocks);
    const int rc = b.max_rows > PAGED_DECODE_ROWS ? attn_paged_tc(a, grid, s) : pool.kind == KV_I8 ? launch_split<KV_I8>(a, grid, pl.MB, s) : pool.kind == KV_E4M3 ? launch_split<KV_E4M3>(a, grid, pl.MB, s) : launch_split<KV_I4>(a, grid, pl.MB, s);
    if (rc != HP_OK || a.direct) return rc;
    MergeArgs m; m.b = b; m.pO = a.pO; m.pml = a.pml; m.gate = p.gate; m.g_ld = p.g_ld; m.g_hs = p.g_hs; m.n_head = p.n_head; m.window = p.window; m.n_sink = p.n_sink;
    m.U = pl.U; m.ns = pl.ns; m.nwin = pl.nwin; m.mul = a.mul; m.out = p.out; m.oq = (int8_t*)p.xq.q; m.osc = (float*)p.xq.sc; m.err = a.arg_err;
    auto merge = [&](auto dims) {
        constexpr int D = decltype(dims)::value, HPB = 1024 / D;
        if (pl.ns + pl.nwin <= FEW && wide) return launch_pdl<4>(k_paged_merge_few<D>, dim3((unsigned)(b.R * ((p.n_head + HPB - 1) / HPB))), dim3(256), 0, s, m);
        return launch_pdl<4>(k_paged_merge<D>, dim3((unsigned)(b.R * p.n_head)), dim3(256), 0, s, m);
    };
    HP_CUDA(pool.head_dim == 256 ? merge(std::integral_constant<int, 256>()) : pool.head_dim == 128 ? merge(std::integral_constant<int, 128>()) : merge(std::integral_constant<int, 64>()));
    return HP_OK;
}

}  // namespace hp
