// Causal attention of whole prompts, packed one behind the other, with grouped heads, in f16 or bf16: o_i = sum_{j <= i} w_ij v_j / sum_{j <= i} w_ij, w_ij =
// 2^(q_i . k_j * scale * log2 e - mu_i), times sigmoid(gate). No cache: a prompt sees its own keys and values as they are, not what a cache of few bits makes of them.
//
// A CTA has 128 rows of one sequence and query head, and goes through its keys in tiles of 128, the tile of its own rows last: the only one with hidden keys. Warps:
//   weights (four warps, a thread per row): S of a tile into registers, the row's largest score, weights in 16 bits in place of the scores, the outputs at the end
//   products (one thread): S[128 rows][128 keys] = Q K^T with both from shared memory, O[128 rows][dims] += W V with W from accumulator memory
//   copies (one thread): K in parts of 64 dims, V in parts of 32 keys, each of them fetched again as soon as its products are through
// Up to 128 dims take half of the accumulator memory and of shared memory: two CTAs per SM, one's weights under the other's products. 256 dims take an SM, with two tiles of scores.
// A row's reference mu moves when a logarithm passes it by more than MU_STEP, so the sums are rescaled rarely (by the row's own thread); weights reach 2^MU_STEP at most. Sums of weights are fp32 of the
// weights before they are rounded to 16 bits: that rounding is at most half a step of the outputs' own type per weight.
//
// A value that is infinite or NaN must not reach the rows in front of it through a weight of zero. Hidden keys lie in the last tile alone: its values are looked at there, such elements are taken out
// (and noted), and the rows that see them get their weight times that element at the end.
#include "paged.cuh"
#include "tc.cuh"
#include <algorithm>
#include <cuda.h>
#include <cuda_bf16.h>
#include <type_traits>

namespace hp {
namespace {

constexpr int TQ = 128, TK = 128;   // rows of a CTA, keys of a tile
constexpr float MU_STEP = 8.f;

struct PromptArgs {
    const int* row_start; int S, R, max_rows, n_head, n_kv, G; float scale2;   // scale * log2 e
    const void *q, *k, *v; size_t q_ld, q_hs, k_ld, k_hs, v_ld, v_hs;          // as the tensor maps have them
    const float* gate; size_t g_ld, g_hs; void* out; int8_t* oq; float* osc; int* err; int* arg_err;
};

template <int D> struct Geo {
    static constexpr int PARTS = D / 64, VP = 4, VROWS = TK / VP;              // parts of K (64 dims), of V (32 keys)
    static constexpr int K_PART = TK * 128, V_PART = VROWS * D * 2;
    static constexpr int OFF_Q = 0, OFF_K = TQ * D * 2, OFF_V = OFF_K + TK * D * 2, SMEM = OFF_V + TK * D * 2 + 1024;   // 1024 for the alignment
    static constexpr int NS = D == 256 ? 2 : 1;                                // tiles of scores
    static constexpr int T_O = 0, T_S = D, TMEM = D == 256 ? 512 : 256;
    static constexpr int CTAS = D == 256 ? 1 : 2, THREADS = 192;
    static_assert(T_S + NS * TK <= TMEM && CTAS * SMEM <= 227 * 1024, "");
};

// 128-byte swizzle, groups of 8 rows 1024 bytes apart; N-major: the next 64 elements lie `next` bytes behind
__device__ __forceinline__ uint64_t desc128(uint32_t addr, uint32_t next) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(next >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, int add) {   // A in accumulator memory
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void tma3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
#define HP_R8(a, i) "=f"(a[i]), "=f"(a[i + 1]), "=f"(a[i + 2]), "=f"(a[i + 3]), "=f"(a[i + 4]), "=f"(a[i + 5]), "=f"(a[i + 6]), "=f"(a[i + 7])
__device__ __forceinline__ void ld32(float* a, uint32_t col) {   // 32 columns of this warp's lanes; there behind ld_wait
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : HP_R8(a, 0), HP_R8(a, 8), HP_R8(a, 16), HP_R8(a, 24) : "r"(col) : "memory");
}
#undef HP_R8
#define HP_R8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])
__device__ __forceinline__ void st8(uint32_t col, const uint32_t* a) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(col), HP_R8(a, 0) : "memory");
}
__device__ __forceinline__ void st32(uint32_t col, const uint32_t* a) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 ::"r"(col), HP_R8(a, 0), HP_R8(a, 8), HP_R8(a, 16), HP_R8(a, 24) : "memory");
}
#undef HP_R8
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N> __device__ __forceinline__ void ld_wait(float* a) {   // orders the use of the registers behind the wait
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(a[i]));
}
__device__ __forceinline__ bool one_wait(uint32_t bar, uint32_t parity, int* err) { return mbar_test(bar, parity) || tc_wait(bar, parity, err); }
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err) { return __all_sync(0xffffffffu, one_wait(bar, parity, err)); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (std::is_same<T, __half>::value) return h2_bits(__floats2half2_rn(x, y));
    else { const __nv_bfloat162 b = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t*>(&b); }
}
template <typename T> __device__ __forceinline__ float to_f32(uint16_t b) { if constexpr (std::is_same<T, __half>::value) return h2f(b); else return bf2f(b); }
template <typename T> __device__ __forceinline__ bool odd16(uint32_t b) { constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u; return (b & E) == E; }   // infinite or NaN
// the top bits of both halves: set where the half is infinite or NaN, its exponent plus one
template <typename T> __device__ __forceinline__ uint32_t odd_pair(uint32_t w) { constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u, ONE = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u; return (w & E) + ONE; }

// The block of 128 rows that number `blk` stands for: those with most keys first, whatever sequence they belong to. Blocks i of a sequence (rows from 128 i on): F(i) = sum_s max(0, n_s - i) blocks have number
// i or more in a sequence of n_s; the largest i with F(i) > blk is the block's, and blk - F(i + 1) counts the sequences that have an i-th one.
struct QBlock { int s, row0, T, i; };
__device__ __forceinline__ QBlock find_rows(const PromptArgs& a, int blk, int lane) {
    auto seq = [&](int s, int& row0) {   // rows of sequence s, within what the call says
        const int b = a.row_start[s], e = a.row_start[s + 1];
        row0 = min(max(b, 0), a.R);
        const int T = min(max(min(max(e, 0), a.R) - row0, 0), a.max_rows);
        if (row0 != b || row0 + T != e) paged_bad(a.arg_err);
        return T;
    };
    QBlock o{-1, 0, 0, 0};
    if (a.S == 1) { o.T = seq(0, o.row0); o.i = (o.T + TQ - 1) / TQ - 1 - blk; o.s = o.i < 0 ? -1 : 0; return o; }
    auto from = [&](int i) {   // F(i)
        int n = 0, r;
        for (int s = lane; s < a.S; s += 32) n += max(0, (seq(s, r) + TQ - 1) / TQ - i);
        return __reduce_add_sync(0xffffffffu, n);
    };
    int lo = 0, hi = (a.max_rows + TQ - 1) / TQ;   // F(lo) > blk >= F(hi)
    if (from(0) <= blk) return o;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (from(mid) > blk) lo = mid; else hi = mid; }
    int k = blk - from(lo + 1);
    for (int s0 = 0; s0 < a.S; s0 += 32) {
        int row0 = 0, T = 0;
        if (s0 + lane < a.S) T = seq(s0 + lane, row0);
        const unsigned has = __ballot_sync(0xffffffffu, (T + TQ - 1) / TQ > lo);
        const int n = __popc(has);
        if (k < n) {
            const int l = __ffs(__ballot_sync(0xffffffffu, (has >> lane & 1) && __popc(has & ((1u << lane) - 1)) == k)) - 1;
            o.s = s0 + l; o.row0 = __shfl_sync(0xffffffffu, row0, l); o.T = __shfl_sync(0xffffffffu, T, l); o.i = lo;
            return o;
        }
        k -= n;
    }
    return o;
}

template <int D, typename T>
__global__ void __launch_bounds__(Geo<D>::THREADS, Geo<D>::CTAS) k_attn_prompt(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const PromptArgs a) {
    using G = Geo<D>;
    extern __shared__ uint8_t sm_raw[];
    struct Shared {
        uint64_t q_full, k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[2], p_full[2], pv_done, fin;
        uint32_t tmem, odd[TK / 32];   // keys of the last tile with an infinite or NaN value
    };
    __shared__ Shared x;
    uint8_t* const sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_launch_dependents();
    const int head = blockIdx.x % a.n_head;
    const QBlock b = find_rows(a, blockIdx.x / a.n_head, lane);
    if (b.s < 0) return;
    const int kh = head / a.G, tiles = b.i + 1, q0 = b.i * TQ;   // first row of the block in its sequence
    const uint32_t base = smem_u32(sm);
    if (tid == 0) {
        mbar_init(smem_u32(&x.q_full), 1);
        for (int i = 0; i < 4; ++i) { mbar_init(smem_u32(&x.k_full[i]), 1); mbar_init(smem_u32(&x.k_empty[i]), 1); mbar_init(smem_u32(&x.v_full[i]), 1); mbar_init(smem_u32(&x.v_empty[i]), 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&x.s_full[i]), 1); mbar_init(smem_u32(&x.p_full[i]), 4); }
        mbar_init(smem_u32(&x.pv_done), 1); mbar_init(smem_u32(&x.fin), 1);
        for (int i = 0; i < TK / 32; ++i) x.odd[i] = 0;
        fence_barrier_init();
    }
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&x.tmem)), "n"(G::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = x.tmem;
    bool ok = true;

    if (warp < 4) {   // ---- weights
        const int row = tid;                              // of the block
        const uint32_t at = tmem + ((uint32_t)warp << 21);
        const float c = a.scale2;
        float mu = MU_NONE, l = 0.f;
#pragma unroll 1
        for (int n = 0; n < tiles; ++n) {
            const uint32_t sc = at + G::T_S + n % G::NS * TK;
            ok = ok && warp_wait(smem_u32(&x.s_full[n % G::NS]), n / G::NS & 1, a.err);
            if (!ok) break;
            tc_fence_after();
            float s[TK];
#pragma unroll
            for (int i = 0; i < TK; i += 32) ld32(s + i, sc + i);
            ld_wait<TK>(s);
            const bool last = n == tiles - 1;
            if (last) {
#pragma unroll
                for (int i = 0; i < TK; ++i) if (i > row) s[i] = -INFINITY;
            }
            float t[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < TK; i += 4) { t[0] = fmaxf(t[0], s[i]); t[1] = fmaxf(t[1], s[i + 1]); t[2] = fmaxf(t[2], s[i + 2]); t[3] = fmaxf(t[3], s[i + 3]); }
            const float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) * c;
            if (__any_sync(0xffffffffu, top > mu + MU_STEP)) {   // a row moves by its own scores alone
                float al = 1.f;
                if (top > mu + MU_STEP) { al = ex2(mu - top); mu = top; l = l * al; }   // the first reference: 0
                if (n) {
                    ok = warp_wait(smem_u32(&x.pv_done), (n - 1) & 1, a.err);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int i = 0; i < D; i += 32) {
                        float o[32];
                        ld32(o, at + G::T_O + i); ld_wait<32>(o);
                        uint32_t u[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(o[e] * al);
                        st32(at + G::T_O + i, u);
                    }
                    st_wait();
                }
            }
            // distances from the reference. Logarithms from 2^26 on lie in steps of 8: there the product is rounded as it was for the reference
            if (__any_sync(0xffffffffu, fabsf(mu) >= 67108864.f && mu != MU_NONE)) {
#pragma unroll
                for (int i = 0; i < TK; ++i) s[i] = s[i] * c - mu;
            } else {
#pragma unroll
                for (int i = 0; i < TK; i += 2) { float2 d = make_float2(-mu, -mu); fma2(d, make_float2(s[i], s[i + 1]), make_float2(c, c)); s[i] = d.x; s[i + 1] = d.y; }
            }
            float2 l2 = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < TK; i += 16) {
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const float2 y = make_float2(ex2(s[i + e]), ex2(s[i + e + 1]));
                    l2 = add2(l2, y);
                    w[e / 2] = pack2<T>(y.x, y.y);
                }
                st8(sc + i, w);   // 16 keys in the first half of their scores' columns
            }
            l = l + (l2.x + l2.y);
            if (last) {   // a key per thread: its values
                const int part = warp;   // 32 keys
                ok = warp_wait(smem_u32(&x.v_full[part]), n & 1, a.err);
                if (!ok) break;
                uint8_t* const vr = sm + G::OFF_V + part * G::V_PART + lane * 128;
                uint32_t any = 0;
#pragma unroll 4
                for (int i = 0; i < D / 8; ++i) {
                    const uint4 u = *reinterpret_cast<const uint4*>(vr + (i >> 3) * (G::VROWS * 128) + (((i & 7) ^ (lane & 7)) << 4));
                    any |= odd_pair<T>(u.x) | odd_pair<T>(u.y) | odd_pair<T>(u.z) | odd_pair<T>(u.w);
                }
                any &= 0x80008000u;
                if (any) {
                    for (int i = 0; i < D; ++i) {
                        uint16_t* const e = reinterpret_cast<uint16_t*>(vr + (i >> 6) * (G::VROWS * 128) + (((i >> 3 & 7) ^ (lane & 7)) << 4)) + (i & 7);
                        if (odd16<T>(*e)) *e = 0;
                    }
                    fence_proxy_async();
                }
                const unsigned bad = __ballot_sync(0xffffffffu, any != 0);
                if (lane == 0) x.odd[part] = bad;
            }
            st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&x.p_full[n % G::NS]));
        }
        // ---- outputs
        ok = ok && warp_wait(smem_u32(&x.pv_done), (tiles - 1) & 1, a.err);
        tc_fence_after();
        asm volatile("bar.sync 1, 128;" ::: "memory");   // odd[] of all four warps, which all come here
        const int r = b.row0 + q0 + row;
        const bool mine = ok && q0 + row < b.T;
        if (ok) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const bool odd = (x.odd[0] | x.odd[1] | x.odd[2] | x.odd[3]) != 0;
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
                float o[32];
                ld32(o, at + G::T_O + i); ld_wait<32>(o);
                if (!mine) continue;
                if (odd) {
                    const uint16_t* const qr = (const uint16_t*)a.q + (size_t)r * a.q_ld + (size_t)head * a.q_hs;
                    for (int j = 0; j <= row; ++j) {
                        if (!(x.odd[j >> 5] >> (j & 31) & 1)) continue;
                        const uint16_t* const kr = (const uint16_t*)a.k + (size_t)(b.row0 + q0 + j) * a.k_ld + (size_t)kh * a.k_hs;
                        const uint16_t* const vr = (const uint16_t*)a.v + (size_t)(b.row0 + q0 + j) * a.v_ld + (size_t)kh * a.v_hs + i;
                        float dot = 0.f;
                        for (int d = 0; d < D; ++d) dot = fmaf(to_f32<T>(qr[d]), to_f32<T>(kr[d]), dot);
                        const float w = ex2(fminf(dot * c - mu, 2.f * MU_STEP));   // summed in another order than S: not beyond what a weight can be
#pragma unroll
                        for (int e = 0; e < 32; ++e) if (odd16<T>(vr[e])) o[e] = o[e] + w * to_f32<T>(vr[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = o[e] * inv;
                if (a.gate) {
                    const float4* const g = reinterpret_cast<const float4*>(a.gate + (size_t)r * a.g_ld + (size_t)head * a.g_hs + i);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float4 y = g[e];
                        o[4 * e] = o[4 * e] * sigmoid_det(y.x); o[4 * e + 1] = o[4 * e + 1] * sigmoid_det(y.y); o[4 * e + 2] = o[4 * e + 2] * sigmoid_det(y.z); o[4 * e + 3] = o[4 * e + 3] * sigmoid_det(y.w);
                    }
                }
                if (a.out) {
                    uint4* const to = reinterpret_cast<uint4*>((T*)a.out + ((size_t)r * a.n_head + head) * D + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[e] = make_uint4(pack2<T>(o[8 * e], o[8 * e + 1]), pack2<T>(o[8 * e + 2], o[8 * e + 3]), pack2<T>(o[8 * e + 4], o[8 * e + 5]), pack2<T>(o[8 * e + 6], o[8 * e + 7]));
                }
                if (a.oq) {   // as warp_quant32_store has it, 32 dims in one thread
                    const int K = a.n_head * D, k = head * D + i;
                    float amax = 0.f;
#pragma unroll
                    for (int e = 0; e < 32; ++e) amax = fmaxf(amax, fabsf(o[e]));
                    const float dd = amax / 127.f, id = amax > 0.f ? 127.f / amax : 0.f;
                    int sum = 0;
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint32_t w[2] = {0u, 0u};
#pragma unroll
                        for (int j = 0; j < 8; ++j) { const int qi = __float2int_rn(o[e + j] * id); sum += qi; w[j >> 2] |= (uint32_t)(qi & 0xff) << (8 * (j & 3)); }
                        *reinterpret_cast<uint2*>(a.oq + xq_q_index(r, k + e, K)) = make_uint2(w[0], w[1]);
                    }
                    const size_t di = xq_d_index(r, k >> 5, K);
                    a.osc[di] = dd; a.osc[di + 2] = dd * (float)sum;
                }
            }
        }
    } else if (warp == 4) {
        if (tc_elect()) {   // ---- products
            constexpr uint32_t TYPE = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
            constexpr uint32_t ID = (1u << 4) | TYPE | ((uint32_t)(TQ >> 4) << 24), ID_S = ID | ((uint32_t)(TK >> 3) << 17), ID_O = ID | ((uint32_t)(D >> 3) << 17) | (1u << 16);   // O: V is N-major
            auto scores = [&](int n) {
                if (n >= G::NS && !one_wait(smem_u32(&x.pv_done), (n - G::NS) & 1, a.err)) return false;   // the weights in its place are read
                const uint32_t st = tmem + G::T_S + n % G::NS * TK;
#pragma unroll
                for (int p = 0; p < G::PARTS; ++p) {
                    if (!one_wait(smem_u32(&x.k_full[p]), n & 1, a.err)) return false;
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < 4; ++i) mma_ss(st, desc128(base + G::OFF_Q + p * (TQ * 128) + i * 32, 16), desc128(base + G::OFF_K + p * G::K_PART + i * 32, 16), ID_S, p | i);
                    tc_commit(smem_u32(&x.k_empty[p]));
                }
                tc_commit(smem_u32(&x.s_full[n % G::NS]));
                return true;
            };
            auto outputs = [&](int n) {
                const uint32_t wt = tmem + G::T_S + n % G::NS * TK;
                if (!one_wait(smem_u32(&x.p_full[n % G::NS]), n / G::NS & 1, a.err)) return false;
#pragma unroll
                for (int p = 0; p < G::VP; ++p) {
                    if (!one_wait(smem_u32(&x.v_full[p]), n & 1, a.err)) return false;
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < G::VROWS / 16; ++i) mma_ts(tmem + G::T_O, wt + (p * (G::VROWS / 16) + i) * 16, desc128(base + G::OFF_V + p * G::V_PART + i * 2048, G::VROWS * 128), ID_O, n | p | i);
                    tc_commit(smem_u32(&x.v_empty[p]));
                }
                tc_commit(smem_u32(&x.pv_done));
                return true;
            };
            ok = one_wait(smem_u32(&x.q_full), 0, a.err) && scores(0);
            for (int n = 0; n < tiles && ok; ++n) {
                if (G::NS == 2 && n + 1 < tiles) ok = scores(n + 1);
                ok = ok && outputs(n);
                if (G::NS == 1 && n + 1 < tiles && ok) ok = scores(n + 1);
            }
            tc_commit(smem_u32(&x.fin));
            tc_wait(smem_u32(&x.fin), 0, a.err);   // nothing in flight when the accumulator memory is given back
        }
    } else if (tc_elect()) {   // ---- copies: whichever part is free next
        mbar_expect_tx(smem_u32(&x.q_full), TQ * D * 2);
#pragma unroll
        for (int i = 0; i < G::PARTS; ++i) tma3(base + G::OFF_Q + i * (TQ * 128), &mq, i * 64, head, b.row0 + q0, smem_u32(&x.q_full));
        int nk = 0, nv = 0, pk = 0, pv = 0;   // tile and part next to be fetched
        uint32_t idle = 0;
        while ((nk < tiles || nv < tiles) && idle < (1u << 24)) {
            ++idle;
            if (nk < tiles && mbar_test(smem_u32(&x.k_empty[pk]), (nk & 1) ^ 1)) {
                const uint32_t bar = smem_u32(&x.k_full[pk]);
                mbar_expect_tx(bar, G::K_PART);
                tma3(base + G::OFF_K + pk * G::K_PART, &mk, pk * 64, kh, b.row0 + nk * TK, bar);
                if (++pk == G::PARTS) { pk = 0; ++nk; }
                idle = 0;
            }
            if (nv < tiles && mbar_test(smem_u32(&x.v_empty[pv]), (nv & 1) ^ 1)) {
                const uint32_t bar = smem_u32(&x.v_full[pv]);
                mbar_expect_tx(bar, G::V_PART);
#pragma unroll
                for (int i = 0; i < G::PARTS; ++i) tma3(base + G::OFF_V + pv * G::V_PART + i * (G::VROWS * 128), &mv, i * 64, kh, b.row0 + nv * TK + pv * G::VROWS, bar);
                if (++pv == G::VP) { pv = 0; ++nv; }
                idle = 0;
            }
            if (idle > 16) __nanosleep(20);
        }
        if (nk < tiles || nv < tiles) {   // gave up: no copy outlives the CTA
            if (a.err) atomicExch(a.err, HP_ETIMEOUT);
            for (int i = 0; i < G::PARTS; ++i) { const int n = i < pk ? nk : nk - 1; if (n >= 0) tc_wait(smem_u32(&x.k_full[i]), n & 1, a.err); }
            for (int i = 0; i < G::VP; ++i) { const int n = i < pv ? nv : nv - 1; if (n >= 0) tc_wait(smem_u32(&x.v_full[i]), n & 1, a.err); }
            tc_wait(smem_u32(&x.q_full), 0, a.err);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(G::TMEM) : "memory");
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// [R][heads][D] in boxes of `rows` x 64 dims of one head. Rows behind the tensor read as zeros
int encode(EncodeFn f, CUtensorMap* m, const void* p, size_t ld, size_t hs, int R, int heads, int D, int rows, int type) {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)R}, strides[2] = {heads == 1 ? (cuuint64_t)D * 2 : hs * 2, R == 1 ? (cuuint64_t)D * 2 : ld * 2};
    const cuuint32_t box[3] = {64, 1, (cuuint32_t)rows}, step[3] = {1, 1, 1};
    const CUresult r = f(m, type == OUT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    HP_REQUIRE(r == CUDA_SUCCESS, "attn_prompt: rows that a tensor map cannot describe (%d): ld=%zu hs=%zu", (int)r, ld, hs);
    return HP_OK;
}
template <int D, typename T> int launch(const CUtensorMap (&m)[3], const PromptArgs& a, long long blocks, cudaStream_t s) {
    static bool attr[MAX_DEVICES] = {};   // per device: the opt-in belongs to the device's copy of the kernel
    const int dev = current_device(); if (dev < 0) return HP_ECUDA;
    if (!attr[dev]) { HP_CUDA(cudaFuncSetAttribute(k_attn_prompt<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<D>::SMEM)); attr[dev] = true; }
    HP_CUDA(launch_pdl<4>(k_attn_prompt<D, T>, dim3((unsigned)(blocks * a.n_head)), dim3(Geo<D>::THREADS), Geo<D>::SMEM, s, m[0], m[1], m[2], a));
    return HP_OK;
}
template <typename T> int launch(const CUtensorMap (&m)[3], const PromptArgs& a, long long blocks, int D, cudaStream_t s) {
    return D == 256 ? launch<256, T>(m, a, blocks, s) : D == 128 ? launch<128, T>(m, a, blocks, s) : launch<64, T>(m, a, blocks, s);
}

}  // namespace

int attn_prompt(const AttnPromptParams& p, cudaStream_t s) {
    static const EncodeFn f = [] {
        void* at = nullptr; cudaDriverEntryPointQueryResult found;
        return cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &at, 12000, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess ? (EncodeFn)at : nullptr;
    }();
    if (!f) { set_error("attn_prompt: the driver has no tensor maps"); return HP_ECUDA; }
    const long long per = (p.max_rows + TQ - 1) / TQ, blocks = std::min<long long>((long long)p.S * per, (long long)p.R / TQ + p.S);
    HP_REQUIRE(blocks * p.n_head < (1ll << 31), "attn_prompt: too many rows (%d) or heads for one call", p.R);
    CUtensorMap m[3];
    int rc = encode(f, &m[0], p.q, p.q_ld, p.q_hs, p.R, p.n_head, p.head_dim, TQ, p.type);
    if (!rc) rc = encode(f, &m[1], p.k, p.k_ld, p.k_hs, p.R, p.n_kv, p.head_dim, TK, p.type);
    if (!rc) rc = encode(f, &m[2], p.v, p.v_ld, p.v_hs, p.R, p.n_kv, p.head_dim, TK / 4, p.type);
    if (rc) return rc;
    PromptArgs a; a.row_start = p.row_start; a.S = p.S; a.R = p.R; a.max_rows = p.max_rows; a.n_head = p.n_head; a.n_kv = p.n_kv; a.G = p.n_head / p.n_kv; a.scale2 = (float)((double)p.scale * 1.4426950408889634074);
    a.q = p.q; a.k = p.k; a.v = p.v; a.q_ld = p.q_ld; a.q_hs = p.q_hs; a.k_ld = p.k_ld; a.k_hs = p.k_hs; a.v_ld = p.v_ld; a.v_hs = p.v_hs;
    a.gate = p.gate; a.g_ld = p.g_ld; a.g_hs = p.g_hs; a.out = p.out; a.oq = (int8_t*)p.xq.q; a.osc = (float*)p.xq.sc; a.err = device_err_flag(); a.arg_err = device_arg_flag();
    return p.type == OUT_F16 ? launch<__half>(m, a, blocks, p.head_dim, s) : launch<__nv_bfloat16>(m, a, blocks, p.head_dim, s);
}

}  // namespace hp
