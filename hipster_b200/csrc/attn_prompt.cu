// Causal attention of whole prompts, packed one behind the other, with grouped heads, in f16 or bf16: o_i = sum_{j <= i} w_ij v_j / sum_{j <= i} w_ij, w_ij =
// 2^(q_i . k_j * scale * log2 e - mu_i), times sigmoid(gate). No cache: a prompt sees its own keys and values as they are, not what a cache of few bits makes of them.
//
// A CTA has 128 rows of one sequence and query head and goes through their keys in tiles of 64 (256 dims: 128), its own rows' last: hidden keys lie in these alone. Warps:
//   weights (four warps, a thread per row): S of a tile into registers, the row's largest score, weights in 16 bits in place of the scores, the outputs at the end
//   scores (one thread): S[128 rows][keys] = Q K^T from shared memory, a tile ahead of the weights; K's copies (tensor maps; 64 dims of 128 bytes to a row, 128-byte swizzle)
//   outputs (one thread): O[128 rows][dims] += W V with W from accumulator memory; V's copies (256 dims: a warp of their own has all copies)
// Up to 128 dims take half of the accumulator memory and of shared memory: two CTAs per SM. 256 dims take an SM; K is fetched in parts of 64 dims and V in parts of 32 keys, each again as soon as its products are through.
// A row's reference mu moves to TOP below a logarithm that passes it by more than LIMIT, so the sums are rescaled rarely (by the row's own thread). Sums of weights are fp32 of the weights before they are rounded to 16 bits: that
// rounding is half a step of the outputs' own type per weight. f16 has steps of 2^-24 below 2^-14 as well: the largest weight is at least 2^6 there, so that a key loses 2^-31 of it at most, and 2^18 weak keys beside a strong
// one lose less than half a step together; none is above 2^15 (f16 ends at 65504). bf16 has weights of 2^-10 at most: sums of 1000 of the largest values, or of 2^18 where scores do not rise, stay finite, and products of
// values down to 2^-108 are normal numbers (subnormal ones keep the bits that an output has down to 2^-121).
//
// A value that is infinite or NaN must not reach the rows in front of it through a weight of zero: in the tiles with hidden keys such elements are taken out of shared memory before the products. A weight being positive, a row has
// NaN, infinity or minus infinity of all that it sees, so the first key of each kind is noted per dim, and outputs from that row on get it added on their way out.
//
// Measured (captured; cuBLAS' burst rate is 1655 TFLOP/s, its sustained one 1402): 8190 rows of 24 heads of 256 605 to 630 us in threes, 1.31 to 1.36 PFLOP/s; 715 to 740 one behind the other for longer, 1.12 to 1.16, at some
// 1.44 GHz under the power limit. 16384 rows of 16 heads of 256 1526 us (1.44 PFLOP/s), of 128 946 (1.16), of 64 803 (0.68). Bounds: 256 dims shared memory (320 KB per tile of 128 keys of 2048 clocks of products) and power; 128
// and 64 the weights' warps, two per scheduler, some 1300 clocks per 64 keys each. Seven prompts of up to 3001 rows of 32 heads of 128 250 to 300 us (by card and power): of a CTA's 37000 clocks 6000 pass before its first scores are
// there, 2700 with its outputs. Five gated prompts of up to 77 rows of 24 heads of 256 11.1 us: 400 KB of a CTA at some 64 bytes a clock, and latency. Gates come in place of q and k while the last weights are formed, each warp's by its own threads,
// and at 256 dims all eight warps write outputs: with gates fetched into registers by the four weights' warps, a step ahead, 13.3, and 8 x 600 rows of 16 heads 92.7 instead of 74; without gates four warps, or eight, take the same.
// Int8 outputs go 32 dims at a time through exchanges of eight lanes, row by row: 8 x 600 rows of 16 heads of 256 159 us, in 16 bits 55.
// Tried: one warp for both products 1119 us at 128 dims where two take 1080 (a wait that is over still takes 250 clocks, and an output waited behind the next scores'); waits that ask without a pause in those warps: they take the
// issue slots of the weights' warp beside them (2360 -> 3440 clocks per tile); a quarter, a half of the exponentials as polynomials on the fp32 pipe: 1732 -> 1762, 1802 us at 256 dims, 819 -> 827, 892 at 64 (instructions, not the
// special functions, bound them); outputs unrolled over a row: 14800 clocks instead of 5800, cold instructions.
#include "paged.cuh"
#include "tc.cuh"
#include <algorithm>
#include <cuda.h>
#include <cuda_bf16.h>
#include <type_traits>

namespace hp {
namespace {

constexpr int TQ = 128;   // rows of a CTA
template <typename T> struct Ref { static constexpr float TOP = -18.f, LIMIT = -10.f; };
template <> struct Ref<__half> { static constexpr float TOP = 6.f, LIMIT = 14.f; };
constexpr float FAR = 16777216.f;   // 2^24: references from here on
constexpr int PASS = 68;            // floats of a row of 64 outputs on their way out: 16-byte pieces of 8 rows hit distinct banks

struct PromptArgs {
    const int* row_start; int S, R, max_rows, order, n_head, G; float scale2;   // scale * log2 e
    const float* gate; size_t g_ld, g_hs; void* out; int8_t* oq; float* osc; int* err; int* arg_err;
};

// Tiles of TK keys in ST stages; a stage's K comes in KP parts of 64 dims or as one, its V in VP parts of 32 keys or as one. Two tiles of scores: one is formed while the other is weighed.
template <int D, bool GATE = false> struct Geo {
    static constexpr int TK = D == 256 ? 128 : 64, ST = D == 256 ? 1 : 2, PARTS = D / 64, KP = D == 256 ? PARTS : 1, VP = D == 256 ? 4 : 1, VROWS = TK / VP;
    static constexpr int HAND = 2;                                             // hand-overs of a tile's weights
    static constexpr int K_GROUP = TK * 128, K_PART = PARTS / KP * K_GROUP, V_PART = VROWS * D * 2, TILE = TK * D * 2;
    static constexpr int OFF_Q = 0, OFF_K = TQ * D * 2, OFF_V = OFF_K + ST * TILE;
    static constexpr int OUT_WARPS = D == 256 && GATE ? 8 : 4;   // warps that write outputs: two per quarter of the accumulator memory's lanes, or the weights' warps alone
    static constexpr int PASSES = OUT_WARPS * 32 * PASS * 4, SMEM = OFF_V + (ST * TILE > PASSES ? ST * TILE : PASSES) + 1024;   // 1024 for the alignment. At the end gates in place of q and k, outputs on their way in place of v
    static constexpr int T_O = 0, T_S = D, TMEM = D == 256 ? 512 : 256;
    static constexpr int CTAS = D == 256 ? 1 : 2;
    // 256 dims: a warp of its own fetches whichever part is free next (copies by the products' warps: 1.76 -> 1.95 ms for 16384 rows of 16 heads). Two CTAs per SM: 224 threads would leave 128 registers each, with spills (1.04 -> 1.08 ms)
    static constexpr bool COPIER = D == 256;
    static constexpr int THREADS = !COPIER ? 192 : GATE ? 256 : 224;
    static_assert(T_S + 2 * TK <= TMEM && CTAS * SMEM <= 227 * 1024 && OFF_V == TQ * D * 4, "");
};

// Operands in shared memory: 128-byte swizzle, groups of 8 rows 1024 bytes apart; N-major: the next 64 elements lie `next` bytes behind. The lower half of a descriptor, to which offsets / 16 are added; the upper one is
// the same for all. Few instructions per product: the products' warp shares its instruction cache with the weights' long loops
constexpr uint32_t DESC_HIGH = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t next) { return (addr >> 4) | ((next >> 4) << 16); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int add) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 a, {%1, %5};\nmov.b64 b, {%2, %5};\ntcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(DESC_HIGH) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int add) {   // A in accumulator memory
    asm volatile("{\n.reg .pred p;\n.reg .b64 b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 b, {%2, %5};\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(DESC_HIGH) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
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
// Bounded waits that keep asking, some half a second: a wait that may park its warp sees a hand-over some 300 clocks later, and a tile has four in a row
__device__ __forceinline__ bool one_wait(uint32_t bar, uint32_t parity, int* err) {
#pragma unroll 1
    for (uint32_t i = 0; i < (1u << 24); ++i) if (mbar_test(bar, parity)) return true;
    if (err) atomicExch(err, HP_ETIMEOUT);
    return false;
}
// of the products' warps: where two CTAs share an SM, one's wait costs less than its questions
template <int D> __device__ __forceinline__ bool mma_wait(uint32_t bar, uint32_t parity, int* err) { return D == 256 ? one_wait(bar, parity, err) : mbar_test(bar, parity) || tc_wait(bar, parity, err); }
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err) { return __all_sync(0xffffffffu, one_wait(bar, parity, err)); }
__device__ __forceinline__ float max3(float a, float b, float c) { float y; asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c)); return y; }
template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (std::is_same<T, __half>::value) return h2_bits(__floats2half2_rn(x, y));
    else { const __nv_bfloat162 b = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t*>(&b); }
}
// to 2^-21: outputs have 16 bits or 8
__device__ __forceinline__ float sigmoid16(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + ex2(x * -1.4426950408889634f))); return y; }
template <typename T> __device__ __forceinline__ float to_f32(uint16_t b) { if constexpr (std::is_same<T, __half>::value) return h2f(b); else return bf2f(b); }
template <typename T> __device__ __forceinline__ bool odd16(uint32_t b) { constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u; return (b & E) == E; }   // infinite or NaN
// the top bits of both halves: set where the half is infinite or NaN, its exponent plus one
template <typename T> __device__ __forceinline__ uint32_t odd_pair(uint32_t w) { constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u, ONE = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u; return (w & E) + ONE; }

// The block of 128 rows that number `blk` stands for, in one of three ways (the rule stands at the launch):
//   GRID: i-th blocks of all sequences (rows from 128 i on) behind the later ones of all. Nothing to look for, and a number per sequence and i, most of them for nothing where lengths differ
//   SORTED: the same order without gaps. F(i) = sum_s max(0, n_s - i) blocks have number i or more in a sequence of n_s; the largest i with F(i) > blk is the block's, and blk - F(i + 1) counts the sequences that have an i-th one
//   ALONG: one sequence behind the other. Sequence s has the numbers from row_start[s] / 128 + s on, which is room enough for its blocks; s by 32 questions at a time. The first CTA sees whether all sequences are as they should be
enum : int { GRID, SORTED, ALONG };
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
    if (a.order == GRID) {
        const int per = (a.max_rows + TQ - 1) / TQ, s = blk % a.S;
        o.T = seq(s, o.row0); o.i = per - 1 - blk / a.S;
        if (o.i * TQ < o.T) o.s = s;
        return o;
    }
    if (a.order == ALONG) {
        auto first = [&](int s) { return min(max(a.row_start[s], 0), a.R) / TQ + s; };
        int s = 0, n = a.S;   // the last one of s .. s + n - 1 with first(s) <= blk
        while (n > 1) {
            const int step = (n + 31) / 32, at = s + lane * step;
            const int k = __popc(__ballot_sync(0xffffffffu, lane * step < n && first(at) <= blk)) - 1;
            if (k < 0) return o;
            s += k * step; n = min(step, n - k * step);
        }
        if (blockIdx.x == 0) for (int i = lane, r; i < a.S; i += 32) seq(i, r);
        o.T = seq(s, o.row0); o.i = (o.T + TQ - 1) / TQ - 1 - (blk - first(s));
        if (o.i >= 0 && blk >= first(s)) o.s = s;
        return o;
    }
    int row0 = 0, T = 0;   // of sequence `lane`: 32 at most
    if (lane < a.S) T = seq(lane, row0);
    const int n = (T + TQ - 1) / TQ;
    auto from = [&](int i) { return __reduce_add_sync(0xffffffffu, max(0, n - i)); };   // F(i)
    int lo = 0, hi = (a.max_rows + TQ - 1) / TQ;   // F(lo) > blk >= F(hi)
    if (from(0) <= blk) return o;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (from(mid) > blk) lo = mid; else hi = mid; }
    const unsigned has = __ballot_sync(0xffffffffu, n > lo);
    const int k = blk - from(lo + 1), l = __ffs(__ballot_sync(0xffffffffu, (has >> lane & 1) && __popc(has & ((1u << lane) - 1)) == k)) - 1;
    o.s = l; o.row0 = __shfl_sync(0xffffffffu, row0, l); o.T = __shfl_sync(0xffffffffu, T, l); o.i = lo;
    return o;
}

// Infinite and NaN values of a tile that has hidden keys are taken out of the tile in shared memory, before its products, and noted in `first`: the first key with NaN, infinity, minus infinity at a dim, counted in the block's rows
// (k0: the tile's first). A thread has a key, or half of its dims
template <int D> struct Odd { int any, first[3 * D]; };
template <int D, typename T>
__device__ bool take_out(uint8_t* v, uint64_t* v_full, Odd<D>& odd, int k0, uint32_t parity, int tid, int* err) {
    using G = Geo<D>;
    constexpr int SHARE = 128 / G::TK, N = D / 8 / SHARE;   // 16-byte pieces of a thread
    const int key = tid % G::TK, i0 = tid / G::TK * N, part = key / G::VROWS, in = key % G::VROWS;
    const bool ok = warp_wait(smem_u32(&v_full[part]), parity, err);
    if (!ok) return false;
    uint8_t* const vr = v + part * G::V_PART + in * 128;
    uint32_t any = 0;
#pragma unroll 8
    for (int i = i0; i < i0 + N; ++i) {
        const uint4 u = *reinterpret_cast<const uint4*>(vr + (i >> 3) * (G::VROWS * 128) + (((i & 7) ^ (in & 7)) << 4));
        any |= odd_pair<T>(u.x) | odd_pair<T>(u.y) | odd_pair<T>(u.z) | odd_pair<T>(u.w);
    }
    if (any & 0x80008000u) {
#pragma unroll 1
        for (int i = i0 * 8; i < (i0 + N) * 8; ++i) {
            uint16_t* const e = reinterpret_cast<uint16_t*>(vr + (i >> 6) * (G::VROWS * 128) + (((i >> 3 & 7) ^ (in & 7)) << 4)) + (i & 7);
            if (!odd16<T>(*e)) continue;
            const float x = to_f32<T>(*e);
            atomicMin(&odd.first[(x != x ? 0 : x > 0.f ? 1 : 2) * D + i], k0 + key);
            *e = 0;
        }
        odd.any = 1;
        fence_proxy_async();
    }
    __syncwarp();
    return true;
}
// and what a row of the block has of them at dim d; 0: it sees none
template <int D> __device__ __forceinline__ float put_in(const Odd<D>& odd, int row, int d) {
    const bool nan = row >= odd.first[d], up = row >= odd.first[D + d], down = row >= odd.first[2 * D + d];
    return nan || (up && down) ? __uint_as_float(0x7fc00000u) : up ? INFINITY : down ? -INFINITY : 0.f;
}

template <int D, typename T, bool GATE>
__global__ void __launch_bounds__(Geo<D, GATE>::THREADS, Geo<D, GATE>::CTAS) k_attn_prompt(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const PromptArgs a) {
    using G = Geo<D, GATE>;
    extern __shared__ uint8_t sm_raw[];
    struct Shared {
        uint64_t q_full, k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[2], p_full[2][G::HAND], pv_done[2], fin[2];   // parts: stage * (KP or VP) + part. pv_done: of even and of odd tiles. Who waits for a tile's may be a tile ahead or behind, and a phase's bit tells only neighbours apart
        float inv[TQ];   // of a row's sum of weights
        int failed;
        uint32_t tmem;
        Odd<D> odd;   // infinite and NaN values of the block's own rows
    };
    __shared__ Shared x;
    uint8_t* const sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = smem_u32(sm);
    for (int i = tid; i < 3 * D; i += G::THREADS) x.odd.first[i] = TQ;
    if (tid == 0) {
        mbar_init(smem_u32(&x.q_full), 1);
        for (int i = 0; i < 4; ++i) { mbar_init(smem_u32(&x.k_full[i]), 1); mbar_init(smem_u32(&x.k_empty[i]), 1); mbar_init(smem_u32(&x.v_full[i]), 1); mbar_init(smem_u32(&x.v_empty[i]), 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&x.s_full[i]), 1); mbar_init(smem_u32(&x.pv_done[i]), 1); mbar_init(smem_u32(&x.fin[i]), 1); for (int p = 0; p < G::HAND; ++p) mbar_init(smem_u32(&x.p_full[i][p]), 4); }
        x.failed = 0;
        x.odd.any = 0;
        fence_barrier_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    const int head = blockIdx.x % a.n_head;
    const QBlock b = find_rows(a, blockIdx.x / a.n_head, lane);
    if (b.s < 0) return;
    const int kh = head / a.G, q0 = b.i * TQ, tiles = (min(q0 + TQ, b.T) + G::TK - 1) / G::TK;   // q0: first row of the block in its sequence
    auto fetch_q = [&] {
        mbar_expect_tx(smem_u32(&x.q_full), TQ * D * 2);
#pragma unroll
        for (int i = 0; i < G::PARTS; ++i) tma3(base + G::OFF_Q + i * (TQ * 128), &mq, i * 64, head, b.row0 + q0, smem_u32(&x.q_full));
    };
    auto fetch_k = [&](int n, int p) {
        const int bar = n % G::ST * G::KP + p;
        const uint32_t full = smem_u32(&x.k_full[bar]), dst = base + G::OFF_K + n % G::ST * G::TILE + p * G::K_PART;
        mbar_expect_tx(full, G::K_PART);
#pragma unroll
        for (int i = 0; i < G::PARTS / G::KP; ++i) tma3(dst + i * G::K_GROUP, &mk, (p * (G::PARTS / G::KP) + i) * 64, kh, b.row0 + n * G::TK, full);
    };
    auto fetch_v = [&](int n, int p) {
        const int bar = n % G::ST * G::VP + p;
        const uint32_t full = smem_u32(&x.v_full[bar]), dst = base + G::OFF_V + n % G::ST * G::TILE + p * G::V_PART;
        mbar_expect_tx(full, G::V_PART);
#pragma unroll
        for (int i = 0; i < G::PARTS; ++i) tma3(dst + i * (G::VROWS * 128), &mv, i * 64, kh, b.row0 + n * G::TK + p * G::VROWS, full);
    };
    // the first copies are under way while accumulator memory is taken (behind the dependency wait: a CTA that waits holds none)
    constexpr int W_FETCH = G::COPIER ? 6 : 4;
    if (warp == W_FETCH && tc_elect()) {
        fetch_q();
        for (int p = 0; p < G::KP; ++p) fetch_k(0, p);
    }
    __syncwarp();
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&x.tmem)), "n"(G::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = x.tmem;
    bool ok = true;
    constexpr bool SHARED = G::OUT_WARPS == 8;
    const int there = min(32, b.T - q0 - 32 * (warp & 3));   // rows of this warp's outputs
    const uint32_t at = tmem + ((uint32_t)(warp & 3) << 21);
    // Outputs, 64 dims at a time through shared memory, which nothing else uses any more: a thread has a row, and 16 lanes write one
    auto write_outputs = [&](float inv) {
        if (there <= 0) return;
        const int from = (warp >> 2) * (D / 2), end = from + D * 4 / G::OUT_WARPS, r = b.row0 + q0 + 32 * (warp & 3), own = 32 * (warp & 3) + lane;
        const bool odd = x.odd.any;
        float* const pass = reinterpret_cast<float*>(sm + (GATE ? G::OFF_V : 0)) + warp * (32 * PASS);
        // Short loops: this runs once per block, from a cold instruction cache
        if (!GATE && !a.oq) {   // 16 bits through shared memory, rows of 144 bytes; 8 lanes write a row
            T* to = (T*)a.out + ((size_t)(r + lane / 8) * a.n_head + head) * D + from + lane % 8 * 8;
#pragma unroll 1
            for (int i = from; i < end; i += 64, to += 64) {
                float o[64];
                ld32(o, at + G::T_O + i); ld32(o + 32, at + G::T_O + i + 32); ld_wait<64>(o);
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 64; e += 8)
                    *reinterpret_cast<uint4*>(pass + lane * 36 + e / 2) = make_uint4(pack2<T>(o[e] * inv, o[e + 1] * inv), pack2<T>(o[e + 2] * inv, o[e + 3] * inv), pack2<T>(o[e + 4] * inv, o[e + 5] * inv), pack2<T>(o[e + 6] * inv, o[e + 7] * inv));
                if (odd) {   // a row each
                    uint16_t* const y = reinterpret_cast<uint16_t*>(pass + lane * 36);
#pragma unroll 1
                    for (int e = 0; e < 64; ++e) { const float add = put_in(x.odd, own, i + e); if (add != 0.f) y[e] = (uint16_t)pack2<T>(to_f32<T>(y[e]) + add, 0.f); }
                }
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (4 * j + lane / 8 < there) *reinterpret_cast<uint4*>(to + (size_t)(4 * j) * a.n_head * D) = *reinterpret_cast<const uint4*>(pass + (4 * j + lane / 8) * 36 + lane % 8 * 4);
            }
        } else {
            // 16 lanes have a row, every second one theirs
            const int d0 = lane % 16 * 4, j0 = lane / 16;
            float* const mine = pass + d0;
#pragma unroll 1
            for (int i = from; i < end; i += 64) {
                const int d = i + d0;
                float o[64];
                ld32(o, at + G::T_O + i); ld32(o + 32, at + G::T_O + i + 32); ld_wait<64>(o);
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 64; e += 4) *reinterpret_cast<float4*>(pass + lane * PASS + e) = make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
                if (odd) {
#pragma unroll 1
                    for (int e = 0; e < 64; ++e) { const float add = put_in(x.odd, own, i + e); if (add != 0.f) pass[lane * PASS + e] += add; }
                }
                __syncwarp();
                if (GATE) {   // all rows at once, those that are not there too: a row after the other would wait for each
                    const float* const g = reinterpret_cast<const float*>(sm) + (32 * (warp & 3) + j0) * D + d;
                    float4 y[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float4 o4 = *reinterpret_cast<const float4*>(mine + (2 * j + j0) * PASS), g4 = *reinterpret_cast<const float4*>(g + 2 * j * D);
                        y[j] = make_float4(o4.x * sigmoid16(g4.x), o4.y * sigmoid16(g4.y), o4.z * sigmoid16(g4.z), o4.w * sigmoid16(g4.w));
                    }
                    if (a.out) {
                        T* const to = (T*)a.out + ((size_t)(r + j0) * a.n_head + head) * D + d;
#pragma unroll
                        for (int j = 0; j < 16; ++j) if (2 * j + j0 < there) *reinterpret_cast<uint2*>(to + (size_t)(2 * j) * a.n_head * D) = make_uint2(pack2<T>(y[j].x, y[j].y), pack2<T>(y[j].z, y[j].w));
                    }
                    if (a.oq) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) *reinterpret_cast<float4*>(mine + (2 * j + j0) * PASS) = y[j];
                    }
                } else if (a.out) {
                    T* to = (T*)a.out + ((size_t)(r + j0) * a.n_head + head) * D + d;
#pragma unroll 4
                    for (int j = j0; j < there; j += 2, to += 2 * (size_t)a.n_head * D) {
                        const float4 y = *reinterpret_cast<const float4*>(mine + j * PASS);
                        *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
                    }
                }
                if (a.oq)
#pragma unroll 1
                    for (int j = j0; j < there; j += 2) quant_four(*reinterpret_cast<const float4*>(mine + j * PASS), r + j, head * D + d, a.n_head * D, a.oq, a.osc);
            }
        }
    };

    if (warp < 4) {   // ---- weights
        constexpr int TK = G::TK;
        const int row = tid;                              // of the block
        const float c = a.scale2;
        float mu = MU_NONE, l = 0.f;
        auto take = [&](int n) { return take_out<D, T>(sm + G::OFF_V + n % G::ST * G::TILE, x.v_full + n % G::ST * G::VP, x.odd, n * TK - q0, n / G::ST & 1, tid, a.err); };
        bool ready = false, far = false;   // scores of the next tile; a row of the warp has a reference from 2^24 on
#pragma unroll 1
        for (int n = 0; n < tiles; ++n) {
            const uint32_t sc = at + G::T_S + (n & 1) * TK;
            if (!n && TK - 1 > q0) ok = take(0) && ok;   // of the first tile while its scores are formed
            if (!__all_sync(0xffffffffu, ready)) ok = ok && warp_wait(smem_u32(&x.s_full[n & 1]), n >> 1 & 1, a.err);
            if (!ok) break;
            tc_fence_after();
            float s[TK];
#pragma unroll
            for (int i = 0; i < TK; i += 32) ld32(s + i, sc + i);
            ld_wait<TK>(s);
            if (GATE && n == tiles - 1) {   // the last scores are there, so nothing reads q and k any more: the gates of this warp's rows in their place, each thread its own copies
                constexpr int LPR = D / 4 < 32 ? D / 4 : 32, RPI = 32 / LPR;   // lanes of a row, rows of an instruction
                const int j0 = lane / LPR, c0 = lane % LPR * 4;
                const float* from = a.gate + (size_t)(b.row0 + q0 + 32 * warp + j0) * a.g_ld + (size_t)head * a.g_hs + c0;
                uint32_t to = base + (32 * warp + j0) * (D * 4) + c0 * 4;
#pragma unroll 4
                for (int j = j0; j < there; j += RPI, from += RPI * a.g_ld, to += RPI * D * 4)
#pragma unroll
                    for (int c = 0; c < D; c += 128) cp_async16(to + c * 4, from + c);
                __syncwarp();
            }
            const int lim = q0 + row - n * TK;   // last key of the tile that the row sees
            const bool hides = n * TK + TK - 1 > q0;
            if (hides) {
#pragma unroll
                for (int i = 0; i < TK; ++i) if (i > lim) s[i] = -INFINITY;
            }
            float t[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i + 7 < TK; i += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = max3(t[e], s[i + e], s[i + 4 + e]);
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = fmaxf(t[e], s[TK - 4 + e]);
            const float top = fmaxf(max3(t[0], t[1], t[2]), t[3]) * c;
            const bool moves = top - mu > Ref<T>::LIMIT;   // the difference of neighbours is exact, a sum of large numbers is not: mu + 8 may be mu + 16, and weights of 2^16 are more than f16 holds
            if (__any_sync(0xffffffffu, moves)) {   // a row moves by its own scores alone
                float al = 1.f;
                if (moves) { const float next = top - Ref<T>::TOP; al = ex2(mu - next); mu = next; l = l * al; }   // the first reference: 0
                far = __any_sync(0xffffffffu, fabsf(mu) >= FAR && mu != MU_NONE);
                if (n) {
                    ok = warp_wait(smem_u32(&x.pv_done[(n - 1) & 1]), (n - 1) >> 1 & 1, a.err);
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
            // distances from the reference. Logarithms from 2^24 on lie in steps of 2 and more: there the product is rounded as it was for the reference, in the rows that have such a one, so that a distance is LIMIT at most (LIMIT and a
            // half step of the logarithm, 1 next to 2^24, else)
            if (far) {
                const bool own = fabsf(mu) >= FAR;
#pragma unroll
                for (int i = 0; i < TK; ++i) s[i] = own ? s[i] * c - mu : fmaf(s[i], c, -mu);
            } else {
#pragma unroll
                for (int i = 0; i < TK; i += 2) { float2 d = make_float2(-mu, -mu); fma2(d, make_float2(s[i], s[i + 1]), make_float2(c, c)); s[i] = d.x; s[i + 1] = d.y; }
            }
            if (hides && n) {
                // One stage: V(n) comes behind the products of n - 1, and until V(n - 1) is there its barrier has the bit of n. With two stages the scores of n come behind the products of n - 2
                if (G::ST == 1) ok = warp_wait(smem_u32(&x.pv_done[(n - 1) & 1]), (n - 1) >> 1 & 1, a.err);
                ok = ok && take(n);
            }
            // weights of 32 keys are handed over as soon as they are there: their products run under the next ones' exponentials
            float2 l2 = make_float2(0.f, 0.f);
#pragma unroll
            for (int p = 0; p < G::HAND; ++p) {
                constexpr int KEYS = TK / G::HAND;
                if (p == G::HAND - 1) ready = n + 1 < tiles && mbar_test(smem_u32(&x.s_full[(n + 1) & 1]), (n + 1) >> 1 & 1);   // an answer takes some 200 clocks
#pragma unroll
                for (int i = p * KEYS; i < p * KEYS + KEYS; i += 16) {
                    uint32_t w[8];
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float2 y = make_float2(ex2(s[i + e]), ex2(s[i + e + 1]));
                        l2 = add2(l2, y);
                        w[e / 2] = pack2<T>(y.x, y.y);
                    }
                    st8(sc + i, w);   // 16 keys in the first half of their scores' columns
                }
                st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0 && ok) mbar_arrive(smem_u32(&x.p_full[n & 1][p]));
            }
            l = l + (l2.x + l2.y);
            if (!ok) break;
        }
        ok = ok && warp_wait(smem_u32(&x.pv_done[(tiles - 1) & 1]), (tiles - 1) >> 1 & 1, a.err);
        tc_fence_after();
        if (GATE) cp_async_wait_all();   // no copy outlives its thread
        __syncwarp();
        asm volatile("bar.sync 1, 128;" ::: "memory");   // what all four warps took out; they all come here
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if constexpr (SHARED) x.inv[row] = inv;
        else if (ok) write_outputs(inv);
    } else {   // ---- products and copies: K and scores in one warp, V and outputs in another, so that neither waits for what the other one waits for
        if (warp < 6 && tc_elect()) {
            constexpr uint32_t TYPE = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
            constexpr uint32_t ID = (1u << 4) | TYPE | ((uint32_t)(TQ >> 4) << 24), ID_S = ID | ((uint32_t)(G::TK >> 3) << 17), ID_O = ID | ((uint32_t)(D >> 3) << 17) | (1u << 16);   // O: V is N-major
            const uint32_t q_desc = desc_low(base + G::OFF_Q, 16), k_desc = desc_low(base + G::OFF_K, 16), v_desc = desc_low(base + G::OFF_V, G::VROWS * 128);
            auto scores = [&](int n) {
                if (n >= 2 && !mma_wait<D>(smem_u32(&x.pv_done[n & 1]), (n >> 1 & 1) ^ 1, a.err)) return false;   // the weights of n - 2, in its place, are read
                const uint32_t st = tmem + G::T_S + (n & 1) * G::TK;
                uint32_t qd = q_desc, kd = k_desc + n % G::ST * (G::TILE / 16);
#pragma unroll
                for (int p = 0; p < G::PARTS; ++p, qd += TQ * 8, kd += G::K_GROUP / 16) {
                    const int bar = n % G::ST * G::KP + p * G::KP / G::PARTS;
                    if (p % (G::PARTS / G::KP) == 0) {
                        if (!mma_wait<D>(smem_u32(&x.k_full[bar]), n / G::ST & 1, a.err)) return false;
                        tc_fence_after();
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) mma_ss(st, qd + 2 * i, kd + 2 * i, ID_S, i ? 1 : p);
                    if ((p + 1) % (G::PARTS / G::KP) == 0) tc_commit(smem_u32(&x.k_empty[bar]));
                }
                tc_commit(smem_u32(&x.s_full[n & 1]));
                return true;
            };
            auto outputs = [&](int n) {
                constexpr int SLICES = G::TK / 32, PER = G::VROWS / 32, GIVEN = SLICES / G::HAND;   // slices of 32 keys: all, of a part of V, of a hand-over
                uint32_t wt = tmem + G::T_S + (n & 1) * G::TK, vd = v_desc + n % G::ST * (G::TILE / 16);
#pragma unroll
                for (int p = 0; p < SLICES; ++p, wt += 32, vd += (G::VP > 1 ? G::V_PART : 4096) / 16) {
                    const int bar = n % G::ST * G::VP + p / PER;
                    if (p % PER == 0 && !mma_wait<D>(smem_u32(&x.v_full[bar]), n / G::ST & 1, a.err)) return false;
                    if (p % GIVEN == 0) {
                        if (!mma_wait<D>(smem_u32(&x.p_full[n & 1][p / GIVEN]), n >> 1 & 1, a.err)) return false;
                    }
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < 2; ++i) mma_ts(tmem + G::T_O, wt + 16 * i, vd + 128 * i, ID_O, i ? 1 : n | p);
                    if ((p + 1) % PER == 0) tc_commit(smem_u32(&x.v_empty[bar]));
                }
                tc_commit(smem_u32(&x.pv_done[n & 1]));
                return true;
            };
            const bool first = warp == 4;
            if (G::COPIER) {
                if (first) ok = mma_wait<D>(smem_u32(&x.q_full), 0, a.err);
                for (int n = 0; n < tiles && ok; ++n) ok = first ? scores(n) : outputs(n);
            } else {   // a stage is fetched again when the products of the tile that it held are through
                uint64_t *const full = first ? x.k_full : x.v_full, *const empty = first ? x.k_empty : x.v_empty;
                const int parts = first ? G::KP : G::VP;
                int fetched = first;   // tiles whose copies have been issued
                for (; fetched < min(G::ST, tiles); ++fetched)
                    for (int p = 0; p < parts; ++p) { if (first) fetch_k(fetched, p); else fetch_v(fetched, p); }
                if (first) ok = mma_wait<D>(smem_u32(&x.q_full), 0, a.err);
                for (int n = 0; n < tiles && ok; ++n) {
                    if (n && fetched < tiles) {
                        for (int p = 0; p < parts && ok; ++p) {
                            ok = tc_wait(smem_u32(&empty[(n - 1) % G::ST * parts + p]), (n - 1) / G::ST & 1, a.err);
                            if (ok) { if (first) fetch_k(fetched, p); else fetch_v(fetched, p); }
                        }
                        if (!ok) break;
                        ++fetched;
                    }
                    ok = first ? scores(n) : outputs(n);
                }
                if (!ok) {   // gave up: no copy outlives the CTA
                    for (int n = max(0, fetched - G::ST); n < fetched; ++n)
                        for (int p = 0; p < parts; ++p) tc_wait(smem_u32(&full[n % G::ST * parts + p]), n / G::ST & 1, a.err);
                    if (first) tc_wait(smem_u32(&x.q_full), 0, a.err);
                }
            }
            tc_commit(smem_u32(&x.fin[warp - 4]));
            ok = tc_wait(smem_u32(&x.fin[warp - 4]), 0, a.err) && ok;   // nothing in flight when the accumulator memory is given back
        }
        __syncwarp();   // the other lanes wait here: what follows takes whole warps
        if (G::COPIER && warp == 6 && tc_elect()) {
            int nk = 1, nv = 0, pk = 0, pv = 0;   // tile and part next to be fetched
            uint32_t idle = 0;
            while ((nk < tiles || nv < tiles) && idle < (1u << 23)) {
                ++idle;
                if (nk < tiles && mbar_test(smem_u32(&x.k_empty[nk % G::ST * G::KP + pk]), (nk / G::ST & 1) ^ 1)) {
                    fetch_k(nk, pk);
                    if (++pk == G::KP) { pk = 0; ++nk; }
                    idle = 0;
                }
                if (nv < tiles && mbar_test(smem_u32(&x.v_empty[nv % G::ST * G::VP + pv]), (nv / G::ST & 1) ^ 1)) {
                    fetch_v(nv, pv);
                    if (++pv == G::VP) { pv = 0; ++nv; }
                    idle = 0;
                }
                if (idle) __nanosleep(40);   // its questions take the weights' warps' time
            }
            if (nk < tiles || nv < tiles) {   // gave up: no copy outlives the CTA
                if (a.err) atomicExch(a.err, HP_ETIMEOUT);
                for (int back = 0; back < G::ST; ++back) {
                    for (int i = 0; i < G::KP; ++i) { const int n = (i < pk ? nk : nk - 1) - back; if (n >= 0) tc_wait(smem_u32(&x.k_full[n % G::ST * G::KP + i]), n / G::ST & 1, a.err); }
                    for (int i = 0; i < G::VP; ++i) { const int n = (i < pv ? nv : nv - 1) - back; if (n >= 0) tc_wait(smem_u32(&x.v_full[n % G::ST * G::VP + i]), n / G::ST & 1, a.err); }
                }
                tc_wait(smem_u32(&x.q_full), 0, a.err);
            }
        }
    }
    __syncwarp();
    if constexpr (SHARED) {   // all warps write
        if (!ok) x.failed = 1;
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (!x.failed) write_outputs(x.inv[32 * (warp & 3) + lane]);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 5) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(G::TMEM) : "memory");
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// [R][heads][D] in boxes of `rows` x 64 dims of one head. Rows behind the tensor read as zeros
int encode(EncodeFn f, CUtensorMap* m, const void* p, size_t ld, size_t hs, int R, int heads, int D, int rows, int type) {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)R}, strides[2] = {(heads == 1 ? D : hs) * 2, (R == 1 ? D : ld) * 2};
    const cuuint32_t box[3] = {64, 1, (cuuint32_t)rows}, step[3] = {1, 1, 1};
    const CUresult r = f(m, type == OUT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, step,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    HP_REQUIRE(r == CUDA_SUCCESS, "attn_prompt: rows that a tensor map cannot describe (%d): ld=%zu hs=%zu", (int)r, ld, hs);
    return HP_OK;
}
template <int D, typename T, bool GATE> int launch(const CUtensorMap (&m)[3], const PromptArgs& a, long long blocks, cudaStream_t s) {
    static bool attr[MAX_DEVICES] = {};   // per device: the opt-in belongs to the device's copy of the kernel
    const int dev = current_device(); if (dev < 0) return HP_ECUDA;
    if (!attr[dev]) { HP_CUDA(cudaFuncSetAttribute(k_attn_prompt<D, T, GATE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<D, GATE>::SMEM)); attr[dev] = true; }
    HP_CUDA(launch_pdl<4>(k_attn_prompt<D, T, GATE>, dim3((unsigned)(blocks * a.n_head)), dim3(Geo<D, GATE>::THREADS), Geo<D, GATE>::SMEM, s, m[0], m[1], m[2], a));
    return HP_OK;
}
template <typename T, bool GATE> int launch(const CUtensorMap (&m)[3], const PromptArgs& a, long long blocks, int D, cudaStream_t s) {
    return D == 256 ? launch<256, T, GATE>(m, a, blocks, s) : D == 128 ? launch<128, T, GATE>(m, a, blocks, s) : launch<64, T, GATE>(m, a, blocks, s);
}

}  // namespace

int attn_prompt(const AttnPromptParams& p, cudaStream_t s) {
    static const EncodeFn f = [] {
        void* at = nullptr; cudaDriverEntryPointQueryResult found;
        return cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &at, 12000, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess ? (EncodeFn)at : nullptr;
    }();
    if (!f) { set_error("attn_prompt: the driver has no tensor maps"); return HP_ECUDA; }
    // Numbers for blocks: a CTA without one costs some 2 us of its SM, a search among 32 lengths 1000 clocks. GRID and SORTED or ALONG, us, heads of 128, 16 over 4: 24 prompts of 500 rows 66 and 71, 40 of 100 23.6 and 26.9, one
    // of 8000 beside 39 of 100 788 and 265 (SORTED by pieces of 32 sequences 275, but 46000 for one of 4000 beside 4095 of 5, where ALONG takes 1530)
    const long long per = (p.max_rows + TQ - 1) / TQ, most = p.S * per, least = (long long)p.R / TQ + p.S, blocks = std::min(most, least);
    const int order = most <= least ? GRID : p.S <= 32 ? SORTED : ALONG;
    HP_REQUIRE(blocks * p.n_head < (1ll << 31), "attn_prompt: too many rows (%d) or heads for one call", p.R);
    CUtensorMap m[3] = {};
    int rc = encode(f, &m[0], p.q, p.q_ld, p.q_hs, p.R, p.n_head, p.head_dim, TQ, p.type);
    if (!rc) rc = encode(f, &m[1], p.k, p.k_ld, p.k_hs, p.R, p.n_kv, p.head_dim, p.head_dim == 256 ? Geo<256>::TK : Geo<128>::TK, p.type);
    if (!rc) rc = encode(f, &m[2], p.v, p.v_ld, p.v_hs, p.R, p.n_kv, p.head_dim, p.head_dim == 256 ? Geo<256>::VROWS : Geo<128>::VROWS, p.type);
    if (rc) return rc;
    PromptArgs a; a.row_start = p.row_start; a.S = p.S; a.R = p.R; a.max_rows = p.max_rows; a.order = order; a.n_head = p.n_head; a.G = p.n_head / p.n_kv; a.scale2 = (float)((double)p.scale * 1.4426950408889634074);
    a.gate = p.gate; a.g_ld = p.g_ld; a.g_hs = p.g_hs; a.out = p.out; a.oq = (int8_t*)p.xq.q; a.osc = (float*)p.xq.sc; a.err = device_err_flag(); a.arg_err = device_arg_flag();
    auto type = [&](auto gate) { constexpr bool GATE = decltype(gate)::value; return p.type == OUT_F16 ? launch<__half, GATE>(m, a, blocks, p.head_dim, s) : launch<__nv_bfloat16, GATE>(m, a, blocks, p.head_dim, s); };
    return p.gate ? type(std::true_type()) : type(std::false_type());
}

}  // namespace hp
