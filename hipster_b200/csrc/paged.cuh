// What the operators of the paged 8-bit cache share: the description of a cache and of a ragged batch, and where a row belongs.
#pragma once
#include "hp_common.cuh"
#include "kernels.h"
#include <climits>

namespace hp {

// Rows of a batch as the kernels see them. Lengths come from device memory, so nothing they hold is trusted: rows stay inside [0, R), a
// sequence's tokens inside its columns of the table, page numbers inside the pool; what does not is left out and told by the status word.
struct PagedSeq { int s, row0, T, len, base; };   // sequence, its first row, rows, tokens with these rows (s < 0: none); what a row's number lacks to its position

__device__ __forceinline__ void paged_bad(int* err) { if (err) *err = HP_EINVAL; }
// rows and tokens of sequence s
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, int s, int* err) {
    const int a = b.row_start[s], e = b.row_start[s + 1], n = b.kv_len[s];
    PagedSeq q; q.s = s; q.base = n < 0 ? INT_MIN : (int)((unsigned)n - (unsigned)e);   // of the numbers as given: what does not fit shifts no other row
    q.row0 = min(max(a, 0), b.R); q.T = min(max(min(max(e, 0), b.R) - q.row0, 0), b.max_rows); q.len = min(max(n, 0), b.max_kv);   // no row from e on, whatever a is: these belong to others
    if (q.row0 != a || q.row0 + q.T != e || q.len != n) paged_bad(err);
    return q;
}
// Position of one of its rows; beyond max_kv (as an unsigned number) where it has no place
__device__ __forceinline__ int paged_place(const PagedSeq& q, int r) { return (int)((unsigned)q.base + (unsigned)r); }
// The sequence of row r, by one warp: the number of sequences that end at or in front of it. Rows behind the last one: s = -1.
__device__ __forceinline__ PagedSeq paged_find(const PagedBatch& b, int r, int lane, int* err) {
    int s = 0;
    for (int s0 = 0; s0 < b.S; s0 += 32) {
        const bool behind = s0 + lane < b.S && b.row_start[s0 + lane + 1] <= r;
        const int n = __popc(__ballot_sync(0xffffffffu, behind));
        s += n;
        if (n < 32) break;
    }
    if (s >= b.S) return PagedSeq{-1, 0, 0, 0, 0};
    PagedSeq q = paged_seq(b, s, err);
    if (r < q.row0 || r >= q.row0 + q.T) q.s = -1;
    return q;
}
// First row of a page for one head, counted over the pool's rows of head_dim codes: ((page * n_kv + head) << log2 page_size); 0xffffffff for a number out of
// range. The number is fetched apart: its check waits for it, so a loop fetches the next page's number while it works on this one's.
__device__ __forceinline__ int paged_id(const PagedPool& p, int s, int column) { return p.table[(size_t)s * p.table_ld + column]; }
__device__ __forceinline__ uint32_t paged_row_of(const PagedPool& p, int id, int head, int* err) {
    if ((unsigned)id >= (unsigned)p.n_pages) { paged_bad(err); return 0xffffffffu; }
    return ((uint32_t)id * (uint32_t)p.n_kv + (uint32_t)head) << p.lg_page;
}
__device__ __forceinline__ uint32_t paged_row(const PagedPool& p, int s, int column, int head, int* err) { return paged_row_of(p, paged_id(p, s, column), head, err); }

// ---- attention: what its two kernels (attn_paged.cu, attn_paged_tc.cu) share
struct PagedArgs {
    PagedPool pool; PagedBatch b;
    const float* q; size_t q_ld, q_hs; int n_head, G; float scale2;   // scale2 = scale * log2 e (times 256 for e4m3)
    int window, n_sink;
    int U, ns, nwin;            // keys of a split, splits of the first tokens, splits behind them
    float* pO; float2* pml;     // partials [row][head][ns + nwin] (x head_dim): sums, (mu, sum of weights)
    uint8_t* f16; int tiles;    // prompts: tiles of 64 tokens in f16, [sequence][kv head][tiles][k, v, scales]
    // outputs of the rows: written by the merge, or by the only split there is (direct)
    const float* gate; size_t g_ld, g_hs; float mul; float* out; int8_t* oq; float* osc; int direct;
    int* err; int* arg_err;
};

// Prompts, calls of more than PAGED_DECODE_ROWS rows per sequence: blocks of PAGED_TC_PAIRS pairs, and the bytes of their f16 tiles
constexpr int PAGED_DECODE_ROWS = 16, PAGED_TC_PAIRS = 128;
size_t attn_paged_tc_bytes(const PagedPool& pool, const PagedBatch& b);
int attn_paged_tc(PagedArgs& a, dim3 grid, cudaStream_t s);

// The reference mu of a pair's weights is whole. It moves when a logarithm passes mu + MU_LIMIT, to MU_TOP below the largest of the keys at hand: weights times scales stay
// below 2^15 (f16 ends at 65504), the largest is above 2^7 (f16 ends in steps of 2^-24), and almost all keys take no maximum at all.
constexpr float MU_TOP = 8.f, MU_LIMIT = 15.f, MU_NONE = -3.4028235e38f;
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float lg2(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// logarithm of a scale of v, at least 2^-90: the weights' sum cannot overflow. NaN counts as that; infinity as the largest number, so that a reference stays finite and the rows that see it become NaN
__device__ __forceinline__ float scale_lg2(float v) { return lg2(fminf(fmaxf(v, 8.0779357e-28f), 3.4028235e38f)); }
__device__ __forceinline__ float pow2i(float d) { return d < -126.f ? 0.f : __uint_as_float((uint32_t)((int)d + 127) << 23); }   // 2^d, d whole and <= 0
// The reference for a largest logarithm t, never below the one there is. Logarithms from 2^26 on lie in steps of 8 and more: these take a reference some steps lower, and what passes the
// limit behind a move all the same, a distance being rounded less than t, is cut off there (cut_off), so that finite scores of any size have finite weights. NaN stays, and an infinite t becomes one.
__device__ __forceinline__ float mu_next(float mu, float t) {
    const float a = fabsf(t), next = ceilf(a >= 67108864.f ? fmaf(a, -2.3841858e-7f, t) : t) - MU_TOP;
    float o; asm("max.NaN.f32 %0, %1, %2;" : "=f"(o) : "f"(mu), "f"(next)); return o;
}
__device__ __forceinline__ float cut_off(float d, float lv) { float o; asm("min.NaN.f32 %0, %1, %2;" : "=f"(o) : "f"(d), "f"(MU_LIMIT + 0.5f - lv)); return o; }   // half a power beyond: what the limit let pass stays as it is
// l + y * 2^d, w = pow2i(d), for sums of weights. Sums of outputs scaled down by more than 2^-126 are nothing beside what they are added to; sums of weights are not: logarithms of scales
// span 218, so the weights of tokens with tiny values may be as large as 2^105, and count in full behind a reference that has moved by twice as much. Hence two factors, the second mostly 1
__device__ __forceinline__ float add_scaled(float l, float y, float w, float d) { return fmaf(y * pow2i(fminf(d + 126.f, 0.f)), d < -126.f ? 1.17549435e-38f : w, l); }
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// Two of four codes as two f16. int8: the code plus 128 becomes the low bits of 1024 + code + 128, and 1152 is subtracted, exactly. e4m3: its bits
// are those of the f16 2^-8 times as large, subnormals included (so 0x7f, which the quantiser does not write, reads as 480 and not as NaN: what lies in
// slots of absent tokens is harmless).
template <int KIND, int LO> __device__ __forceinline__ uint32_t code_pair(uint32_t w) {
    if constexpr (KIND == KV_I8) {
        const uint32_t h = __byte_perm(w ^ 0x80808080u, 0x64646464u, LO == 0 ? 0x4140 : 0x4342);
        return h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&h), __floats2half2_rn(1152.f, 1152.f)));
    } else {
        const uint32_t h = __byte_perm(w, 0u, LO == 0 ? 0x1404 : 0x3424);
        return (h & 0x80008000u) | ((h >> 1) & 0x3f803f80u);
    }
}
// The block of pairs that blockIdx.z stands for: sequences in order, each with ceil(T * G / MB) blocks.
struct Block { PagedSeq q; int p0, np; };
__device__ __forceinline__ Block find_block(const PagedBatch& b, int G, int MB, int blk, int lane, int* err) {
    Block o; o.q.s = -1; o.p0 = o.np = 0;
    int acc = 0;
    for (int s0 = 0; s0 < b.S; s0 += 32) {
        PagedSeq q{-1, 0, 0, 0, 0};
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

// What a CTA of a block has to look at: keys [0, sink) and [lo, kend), of these its split's.
struct Span { int kend, lo, sink, pos_lo, pos_hi; long long u0, u1; };
__device__ __forceinline__ Span span_of(const PagedArgs& a, const Block& blk) {
    Span v;
    v.pos_lo = blk.q.len - blk.q.T + blk.p0 / a.G; v.pos_hi = blk.q.len - blk.q.T + (blk.p0 + blk.np - 1) / a.G;
    v.kend = v.pos_hi + 1; v.lo = a.window ? max(0, v.pos_lo - a.window + 1) : 0; v.sink = a.window ? a.n_sink : 0;
    int split = blockIdx.x;
    if (split >= a.ns) {   // the split of the window whose number leaves this remainder
        const int w0 = max(a.ns, v.lo / a.U), m = (w0 - a.ns) % a.nwin, j = split - a.ns - m;
        split = w0 + (j < 0 ? j + a.nwin : j);
    }
    v.u0 = (long long)split * a.U; v.u1 = min(v.u0 + a.U, (long long)v.kend);
    return v;
}
// sums of a row to its output: quotient and gate
__device__ __forceinline__ void finish(float4& o, float l, float4 g, const PagedArgs& a) {
    float x[4] = {0.f + o.x, 0.f + o.y, 0.f + o.z, 0.f + o.w}; const float y[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = l == 0.f ? 0.f : x[e] * a.mul / l;
        if (a.gate) x[e] = x[e] * sigmoid_det(y[e]);
    }
    o = make_float4(x[0], x[1], x[2], x[3]);
}
// warp_quant32_store for four dims at k per lane: groups of eight lanes, which are there together, have 32 dims each
__device__ __forceinline__ void quant_four(float4 x, int r, int k, int K, int8_t* q, float* sc) {
    const unsigned mask = 0xffu << (threadIdx.x & 24);
    float amax = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, off));
    const float dd = amax / 127.f, id = amax > 0.f ? 127.f / amax : 0.f;
    const int q0 = __float2int_rn(x.x * id), q1 = __float2int_rn(x.y * id), q2 = __float2int_rn(x.z * id), q3 = __float2int_rn(x.w * id);
    int sum = (q0 + q1) + (q2 + q3);
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) sum += __shfl_xor_sync(mask, sum, off);
    *reinterpret_cast<uint32_t*>(q + xq_q_index(r, k, K)) = (q0 & 0xff) | (q1 & 0xff) << 8 | (q2 & 0xff) << 16 | (uint32_t)q3 << 24;   // four bytes of one lane's eight
    if ((threadIdx.x & 7) == 0) { const size_t di = xq_d_index(r, k >> 5, K); sc[di] = dd; sc[di + 2] = dd * (float)sum; }
}
// four dims at d of a row and head, as the merge would write them from one split, bit for bit; eight neighbouring lanes hold 32 dims
__device__ __forceinline__ void put(float4 o, float l, int r, int h, int d, int D, const PagedArgs& a) {
    float4 gate = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.gate) gate = *reinterpret_cast<const float4*>(a.gate + (size_t)r * a.g_ld + (size_t)h * a.g_hs + d);
    finish(o, l, gate, a);
    if (a.out) *reinterpret_cast<float4*>(a.out + ((size_t)r * a.n_head + h) * D + d) = o;
    if (a.oq) quant_four(o, r, h * D + d, a.n_head * D, a.oq, a.osc);
}
// power of two that brings the largest magnitude (its bits) to [2^14, 2^15)
__device__ __forceinline__ int q_exponent(uint32_t m) { return m == 0 || m >= 0x7f800000u ? 0 : min(100, 14 - ((int)(m >> 23) - 127)); }

}  // namespace hp
