// af_tree.cu — attention of drafted tokens over a paged cache
// (af_attention_tree_f32): the nodes of every sequence see its cached
// positions and, by a bit mask, one another,
//     out = Σ_j 2^(s_j - m)·v_j / Σ_j 2^(s_j - m),  s_j = q·k_j·scale·log2(e),  m = max s_j
// over the positions j that the row sees, in one pass with a running m.
// Three kernels: tree_mma_kernel for head_dim 64 and 128, tree_small_kernel for
// the same where the call is small (small_call), tree_row_kernel for every other
// head_dim.
#define AF_WHOLE_PROGRAM  // the register split below (setmaxnreg) holds only without separate compilation
#include <cuda.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "af_kvpages.cuh"
#include "af_ops.cuh"

namespace af {
namespace {

struct TreeParams {
    KvView kv;
    KvBatch b;
    int layer, n_rows, H, G;
    uint32_t G_inv;  // 2^32 / G, rounded up
    const float* q;
    float* out;
    long long qs, os;
    const unsigned long long* mask;
    int mask_words;
    float scale;  // of the scores, times log2(e): the softmax runs in powers of two
};

// Whether the mask row lets node j be seen (no mask: a chain).
__device__ __forceinline__ bool tree_sees(const TreeParams& p, int row, int node, int j) {
    if (!p.mask) return j <= node;
    return j < 64 * p.mask_words && ((p.mask[(long long)row * p.mask_words + (j >> 6)] >> (j & 63)) & 1);
}

constexpr int kTreeThreads = 128;

// The least factor of something that a row sees: an infinite value of V counts however small its weight is, and is not
// turned into NaN by a factor of 0.
__device__ __forceinline__ float least() { return __int_as_float(1); }

// One block per row and head: its warps take the positions in turn, a lane
// the dimensions lane, lane + 32, ...; each warp keeps a running maximum, sum
// and output, merged at the end.  Every row reads K and V again and a warp has
// one position at a time: bound by the latency of its loads.
template <int TYPE>
__global__ void __launch_bounds__(kTreeThreads) tree_row_kernel(TreeParams p) {
    using E = KvElem<TYPE>;
    constexpr int W = kTreeThreads / 32;
    __shared__ int s_seq, s_r0, s_n;
    __shared__ float s_m[W], s_l[W], s_o[W][256];
    const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) s_seq = -1;
    __syncthreads();
    for (int s = tid; s < p.b.n_seq; s += kTreeThreads) {
        int r0, n;
        kv_nodes(p.b, p.n_rows, s, r0, n);
        if (row >= r0 && row < r0 + n) {
            s_seq = s;
            s_r0 = r0;
            s_n = n;
        }
    }
    __syncthreads();
    const int seq = s_seq;
    if (seq < 0) return;
    const int len = kv_len(p.kv, p.b, seq, s_n);
    if (len < 0) return;
    const int node = row - s_r0, hd = p.kv.hd;
    const float* q = p.q + (long long)row * p.qs + (long long)h * hd;
    const long long head = p.layer * p.kv.layer_bytes + (long long)(h / p.G) * hd * sizeof(typename E::T);
    float qv[8], o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        qv[i] = lane + 32 * i < hd ? q[lane + 32 * i] * p.scale : 0.f;
        o[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int pos = warp; pos < len + s_n; pos += W) {
        if (pos >= len && !tree_sees(p, row, node, pos - len)) continue;
        const long long at = kv_row(p.kv, p.b, seq, pos);  // below 0: no page, a key and value of zeros
        if (at < 0) set_err_at(p.b.err, kErrBadArgs);
        const auto* kr = reinterpret_cast<const typename E::T*>(p.kv.k + head + at);
        const auto* vr = reinterpret_cast<const typename E::T*>(p.kv.v + head + at);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at >= 0 && lane + 32 * i < hd) s = fmaf(qv[i], E::load(kr[lane + 32 * i]), s);
        s = warp_sum(s);
        const float mn = fmaxf(m, s), c = mn == -INFINITY ? 1.f : fmaxf(exp2f(m - mn), least());
        const float w = s == -INFINITY ? 0.f : fmaxf(exp2f(s - mn), least());
        m = mn;
        l = l * c + w;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < hd) o[i] = fmaf(w, at >= 0 ? E::load(vr[lane + 32 * i]) : 0.f, o[i] * c);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s_o[warp][lane + 32 * i] = o[i];
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w]);
    float c[W];
    for (int w = 0; w < W; ++w) {
        c[w] = s_m[w] == -INFINITY && s_l[w] == 0.f ? 0.f : fmaxf(exp2f(s_m[w] - top), least());
        sum += c[w] * s_l[w];
    }
    for (int d = tid; d < hd; d += kTreeThreads) {
        float x = 0.f;
        for (int w = 0; w < W; ++w)
            if (c[w] != 0.f) x = fmaf(c[w], s_o[w][d], x);
        p.out[(long long)row * p.os + (long long)h * hd + d] = sum == 0.f ? 0.f : x / sum;
    }
}

// ------------------------------------------------------- tensor-core kernel
//
// One block per (128 query rows, kv head, sequence, split of the positions);
// a row is a node and one of the G query heads that share the kv head.  The
// scores Q·Kᵀ and the products P·V are tcgen05.mma (kind::f16, f32
// accumulation): A — the queries, then the weights — lies in tensor memory, B —
// a tile of K or V rows — in shared memory.
//
// fp32 accuracy out of f16 operands: x·2^a (a power of two that puts the
// largest of a query, or of 8 rows of f32, 32 of bf16, in [2^14, 2^15)) is
// split as hi + lo, both f16: 22 bits, and what is lost below is 2^-39 of that
// largest value.  x·y = hi·hi + hi·lo + lo·hi to 2^-22.  A cache in f16 needs
// no scale and no lo, one in bf16 a scale and no lo (8 bits in 11).  The
// powers of two are undone exactly: K's in the score, V's in the exponent of
// the weight, 2^(s_j - a_j), whose sum Σ 2^(s_j - a_j)·2^a_j is the softmax's.
// The running maximum is of s_j - a_j, a_j at most 60 (V of zeros), so that it rises by up to 46 + e + (s - s') when V
// of magnitude 2^e follows zeros: below 126, where the factor 2^-126 of the sum so far would be 0, for e up to 55 and
// scores 2^24 apart in weight.
// Weights carry a factor 2^14, so that those as small as 2^-38 of the largest
// keep f16's spacing.
//
// The tensor cores truncate when they add to an accumulator (measured: sums
// of 400 and 4000 positive products came out 3.9e-5 and 4.0e-4 low, 1e-7 an
// instruction), so no accumulator lives longer than a tile: small products
// first, then the hi·hi ones, and the output warps add each tile's P·V to sums
// in registers, which round to nearest.
//
// Warps (32): first the softmax warps, 32 of a tile's columns of 32 rows each
// (f32: 8 warps for 64 positions; others: 16 for 128); four add up the tiles'
// P·V and write the rows out; 8 for K and 8 for V (f32) or 4 and 4 put the
// tiles into the form that the products take (split, scaled; a cache in f16
// only has its V looked through); 28 issues P·V and 31 the scores, each behind
// its own barriers (one warp for both: 52 us where two take 47); 29 and 30 copy
// K and V, a box of rows per page by the TMA engine (single rows by bulk copies
// run at 2.3 TB/s).  Registers (setmaxnreg): MmaShape's REG_*, out of the
// launch's 1,024·64.
//
// Measured with inputs out of L2, device time: 26 nodes over 4,000 positions, 32
// heads of 128, f32, 45.7 us (2.9 TB/s of the 132 MB; bound by the splitting
// warps: each reads, splits and stores its rows in turn, ~2,900 cycles a tile, of
// which the stores' part 1,850; and ~15,000 cycles before the first tile's
// products); 16 sequences of 0 to 8,190 positions with 31 nodes, 16/2 heads of 128,
// f16, 48.1 us (1.6 TB/s; ~2,900 cycles a tile of 128, the softmax's chain, of
// which the exponentials fill 1,024 on the special function units, and ~16,000
// cycles of plan, queries, and sums at both ends); chunks of 509 over up to 16,001
// positions, 32/4 heads of 64, bf16, 212.7 us (321 TFLOP/s; the same chain, ~3,100
// cycles a tile).  Steps that got there: K and V by single bulk copies -> boxes;
// 4 -> 8 -> 16 softmax warps (chunk 402 -> 333 -> 266 us); tiles of 64 -> 128
// positions with a power of two per 32 bf16 rows (241 -> 218 us); V's powers of
// two said before its tile (46.4 -> 45.2 us).  Not taken: two sets of softmax warps
// that take the tiles in turn (220 us where one set took 218: 66 % of the issue slots
// are busy already).
//
// Tiles in shared memory: rows of 64 values (128 bytes) in the 128-byte
// swizzle, K-major for K, the same tile MN-major for V; for f32 the TMA engine
// leaves rows as they are in a place of their own (64 KB, a tile's K and V in
// halves) and the splitting warps write the tiles.

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// d (+)= A · B: A in tensor memory, B by descriptor.  The whole warp comes
// here, its leader's instruction runs: the operands then stay in uniform
// registers (issued by one diverged thread, each product cost 130 cycles).
__device__ __forceinline__ void tc_mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(leader)
        : "memory");
}

__device__ __forceinline__ void tc_commit(uint32_t leader, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
        "r"(leader)
        : "memory");
}

__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The largest |x|, NaN if one is NaN.
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
    return r;
}

// Descriptor of a tile in the 128-byte swizzle: strides in bytes, version 1.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}

// 32 consecutive columns of this thread's lane.
__device__ __forceinline__ void tc_ld32(uint32_t t, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
          "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
          "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(t));
}
__device__ __forceinline__ void tc_ld16(uint32_t t, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(t));
}
__device__ __forceinline__ void tc_st8(uint32_t t, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(t)
                 : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// a, b -> packed f16 hi and, of what is left, lo.
__device__ __forceinline__ void split2(f32x2 x, uint32_t& hi, uint32_t& lo) {
    float a, b;
    unpair(x, a, b);
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    unpair(fma2(pair(f.x, f.y), pair(-1.f, -1.f), x), a, b);
    const __half2 l = __floats2half2_rn(a, b);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The power of two for values whose largest has these bits: max·2^a in
// [2^14, 2^15), a within [-113, top]; -113 beside an infinity or NaN, which no other value then joins.
__device__ __forceinline__ int scale_of(uint32_t max_bits, int top) {
    if (max_bits >= 0x7f800000u) return -113;
    return min(top, 14 - ((int)(max_bits >> 23) - 127));
}
__device__ __forceinline__ float pow2(int a) { return __int_as_float((a + 127) << 23); }

constexpr int kMmaThreads = 1024;
constexpr int kMmaWarp = 28, kCopyWarp = 29, kScoreWarp = 31;  // copies of K, of V: 29, 30
constexpr int kMmaRows = 128;
constexpr int tree_tile(int type) { return type == AF_KV_F32 ? 64 : 128; }  // positions of a tile
constexpr int kMmaBadWords = 512;  // tiles of a split whose V holds something non-finite, a bit each
constexpr int kMmaMaxNodes = (1 << 20) - 128;  // of a sequence, so that every group of them has a bit (APART)

template <int TYPE, int HD>
struct MmaShape {
    static constexpr bool F32 = TYPE == AF_KV_F32;
    static constexpr int SIZE = F32 ? 4 : 2;
    static constexpr int T = tree_tile(TYPE);
    static constexpr int TERMS = F32 ? 2 : 1;           // hi, lo of K and V
    static constexpr int PARTS = T / 32;                // of a row's scores: 32 a softmax thread
    static constexpr int SW = F32 ? 8 : 4;              // splitting warps of K, of V
    static constexpr int OUT = 4 * PARTS, SPLIT_K = OUT + 4, SPLIT_V = SPLIT_K + SW;  // first warps
    static_assert(SPLIT_V + SW == kMmaWarp, "warps");
    static constexpr int QW = TYPE == AF_KV_F16 ? kMmaWarp : OUT + 4;  // warps that bring the queries in: f16 has nothing to split yet
    static constexpr int COLS = T * 128;                // 64 values of every row
    static constexpr int TILE = HD / 64 * COLS;
    static constexpr int HALF = TERMS * TILE;           // K or V of a tile: hi, lo
    static constexpr int NB = F32 ? 256 / HD : 3;       // tiles in shared memory: K V K V ...
    static constexpr int NS = F32 ? 4 : HD == 128 ? 2 : 3;  // score tiles in tensor memory (each becomes its weights)
    static constexpr int NC = NS + 1;                   // corrections (see c_full)
    static constexpr int RING = NB + NS + 1;            // barriers and powers of two (see k_full)
    static constexpr int RAWB = T / 2 * HD * 4;         // f32: half the rows of K or V as they are
    static constexpr int RPW = T / SW;                  // rows that share a power of two: a splitting warp's
    static constexpr int LPR = HD * SIZE / 16;          // lanes of a row (f32)
    static constexpr int RPC = 32 / LPR;                // rows of a warp's 512 bytes (f32)
    // queries in, rows out: 128 rows over the last tiles' place, 16-byte columns swizzled by the row
    static constexpr int QROW = HD * 4;
    static constexpr int QTILE = NB - (kMmaRows * QROW + 2 * HALF - 1) / (2 * HALF);
    static_assert(QTILE >= 1, "the first tile does not wait for the queries");
    // registers: what does not fit is spilled, where it costs least (16 bits, head_dim 64: 64 for the softmax 220 us of
    // chunks, 72 taken from the others 209; head_dim 128: 32 for the splitting warps 52 us of the batch, 40 47)
    static constexpr int REG_S = F32 ? 64 : HD == 64 ? 72 : 56, REG_O = HD == 64 ? F32 ? 104 : 96 : F32 ? 160 : 168,
                         REG_K = F32 ? 48 : 40, REG_M = F32 && HD == 128 ? 32 : 40;
    static_assert(PARTS * REG_S + REG_O + SW / 2 * REG_K + REG_M <= 8 * 64, "what the launch gives: 1,024 threads of 64");
    // tensor memory columns
    static constexpr int QH = 0, QL = HD / 2, S0 = HD, O0 = HD + NS * T;
    static_assert(O0 + HD <= 512, "tensor memory");
    // shared memory, behind 768 bytes of mbarriers
    static constexpr int BAD = 768;                       // kMmaBadWords words
    static constexpr int GROUPS = T / RPW;
    static constexpr int APART_WORDS = TYPE == AF_KV_F16 ? 0 : (1 << 20) / RPW / 32;
    static constexpr int APART = BAD + kMmaBadWords * 4;  // groups with nodes that are left to the output warps, a bit each
    static constexpr int ROWS = APART + APART_WORDS * 4;  // [128] query scales, [NC][128] corrections, [2][PARTS][128] exchange, [128] tops, [PARTS][128] sums
    static_assert(APART % 16 == 0 && ROWS % 16 == 0, "read 16 bytes at a time");
    static constexpr int SCALE = ROWS + (2 + NC + 3 * PARTS) * kMmaRows * 4;  // [RING][4][GROUPS] floats: 2^-a of K; -a, 2^a of V; 0 of K
    static constexpr int TILES = (SCALE + RING * 4 * GROUPS * 4 + 1023) / 1024 * 1024;
    static constexpr int RAW = TILES + NB * 2 * HALF;
    static constexpr int BYTES = RAW + (F32 ? 4 * RAWB : 0);  // K, K, V, V
    static_assert(BYTES <= 227 * 1024 - 128, "shared memory");
};

// A box of rows of one kv head (TMA engine): x value, y head, z row.
// The whole warp comes here, its leader's instruction runs (see tc_mma_ts).
__device__ __forceinline__ void tma_rows(uint32_t leader, uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %6, 0;\n\t"
        "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}\n" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(leader)
        : "memory");
}

// Zeros for what is not finite; the largest of the rest, over the warp.
template <int N>
__device__ __noinline__ uint32_t clean(float4 (&x)[N]) {
    uint32_t b = 0;
    for (int i = 0; i < N; ++i) {
        float* e = &x[i].x;
        for (int j = 0; j < 4; ++j) {
            if (!(fabsf(e[j]) < INFINITY)) e[j] = 0.f;
            b = max(b, __float_as_uint(e[j]) & 0x7fffffffu);
        }
    }
    return __reduce_max_sync(0xffffffffu, b);
}

// Nodes are not seen by every row, so what one holds must not cost its neighbours their bits: 2^-39 of a group's largest
// value is lost.  A group with nodes that has a row whose largest is far below, or a key that is not finite, is left out
// of the products (its -a of V, or what stands beside K's power of two, is -inf, so that no row gives it a weight) and
// added position by position in the end, 4 to 9 us each.  Looked at is the smallest largest value of any 16 bytes (bf16:
// of every other value there) that hold something; 2^14 below is far for f32, which leaves 2^-25 of such values; bf16
// groups, of four times the rows, that have one 2^12 below are looked at row by row, so that channels that are large in
// every row are none of it.  (f32 by rows too: 26 nodes over 3,989 positions 45.5 -> 46.8 us.)  Looking costs 3 to 10 %
// where all tiles have nodes (500 tokens: bf16 32/4 heads of 64 19.9 -> 20.6 us, 16/2 of 128 25.7 -> 27.4, f32 28.4 ->
// 29.9; 4 trees of 196, 32/32 heads of 128, bf16 34.7 -> 37.9) and 0 to 2 % over long caches.  Not taken: a power of two
// per row, which the softmax then has to take apart (chunk 209 -> 222 us).
// `mx`: the group's largest value, `low`: the smallest as above (bits, less 1: zeros are all ones).
template <int TYPE>
__device__ __forceinline__ bool far_apart(uint32_t mx, uint32_t low) {
    low = __reduce_min_sync(0xffffffffu, low);
    return mx >= 0x7f800000u || (low != 0xffffffffu && (mx >> 23) > ((low + 1u) >> 23) + (TYPE == AF_KV_F32 ? 14 : 12));
}

// The lane's part of `low` by whole rows, of a group of bf16 rows in shared memory: 4 rows of 64 values an access, HALVES
// accesses of a row COLS bytes apart, `left` rows in front of the end; what is not finite is none.
template <int RUNS, int HALVES, int COLS>
__device__ __noinline__ uint32_t lowest_row(const uint8_t* at, int left) {
    uint32_t low = 0xffffffffu;
    for (int i = 0; i < RUNS; ++i) {
        uint32_t r = 0;
        for (int h = 0; h < HALVES; ++h) {
            const uint4 x = *reinterpret_cast<const uint4*>(at + h * COLS + i * 512);
            const uint32_t e[4] = {x.x, x.y, x.z, x.w};
            for (int j = 0; j < 4; ++j) {
                const uint32_t a = e[j] << 16 & 0x7fff0000u, b = e[j] & 0x7fff0000u;
                r = max(r, max(a < 0x7f800000u ? a : 0u, b < 0x7f800000u ? b : 0u));
            }
        }
        if (i * 4 >= left) r = 0;
        for (int o = 1; o < 8; o <<= 1) r = max(r, __shfl_xor_sync(0xffffffffu, r, o));
        low = min(low, r - 1u);
    }
    return low;
}

// Work: an item is 128 rows of a sequence with one kv head, its tiles split
// over blocks of at most t tiles.  How many tiles there are is known on the
// device alone (lengths, counts), so every block finds its place itself: the
// smallest t for which the blocks fit the waves that the items need anyway.  A
// ragged batch then costs its average and not its longest: 16 sequences of
// 8190 to 0 positions, 120 -> 82 us when it came in.
constexpr int kTreeSms = 148;
constexpr int kTreeWaves = 4;                                // beyond so many the items balance one another
constexpr int kTreeItems = kTreeSms * kTreeWaves;
constexpr int kTreeMinTiles = 3;                             // a shorter split costs more than it saves: a block's set-up is 10,000 cycles, a tile ~3,000

struct MmaParams {
    CUtensorMap k_map, v_map;  // [rows of the layer's pool][kv heads][HD], boxes of box_rows rows
    TreeParams t;
    int box_rows;
    int blocks, slots;  // blocks launched; rooms for the sums of a split item
    float* part;        // [slots][128][HD], then [slots][128][2]: top, sum
    int2* plan;         // [n_seq] first slot, splits of an item; null where no item can be split
};

struct TreeSpot {
    int seq, rt, kvh, split, splits, slot, first_slot;
    int r0, n, len;  // the sequence's rows and cached positions
};

// Rows, items and tiles of sequence s.
struct TreeSeq {
    int r0, n, len, items, tiles;
};
__device__ __forceinline__ TreeSeq tree_seq(const MmaParams& mp, int T, int s) {
    TreeSeq q = {};
    const KvBatch& b = mp.t.b;
    if (s >= b.n_seq) return q;
    q.len = b.len[s];  // beside the counts, not behind them
    kv_nodes(b, mp.t.n_rows, s, q.r0, q.n);
    if (q.len < 0 || (long long)q.len + q.n > ((long long)b.max_blocks << mp.t.kv.ps_shift)) {
        set_err_at(b.err, kErrBadArgs);
        q.n = 0;
    }
    if (q.n) {
        q.items = (q.n * mp.t.G + kMmaRows - 1) / kMmaRows * mp.t.kv.kv_heads;
        q.tiles = (q.len + q.n + T - 1) / T;
    }
    return q;
}

__device__ __forceinline__ int warp_scan(int v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}

// Where block b works (by a whole warp); seq -1: nowhere.
__device__ __forceinline__ TreeSpot tree_spot(const MmaParams& mp, int T, int b) {
    const int lane = threadIdx.x & 31, n_seq = mp.t.b.n_seq;
    const TreeSeq first = tree_seq(mp, T, lane);  // of sequence `lane`; later ones are looked up each time
    auto of = [&](int s0) { return s0 ? tree_seq(mp, T, s0 + lane) : first; };
    int all = 0, longest = 0;
    float work = 0.f;
    for (int s0 = 0; s0 < n_seq; s0 += 32) {
        const TreeSeq q = of(s0);
        all += __reduce_add_sync(0xffffffffu, q.items);
        longest = max(longest, __reduce_max_sync(0xffffffffu, q.tiles));
        work += warp_sum((float)q.items * (float)q.tiles);
    }
    const int need = (all + kTreeSms - 1) / kTreeSms, waves = min(max(need, 1), kTreeWaves);
    const int cap = all <= kTreeItems ? min(need * kTreeSms, mp.blocks) : mp.blocks;
    // the splits of an item at 1/t tiles each: one rule for everybody, whatever it rounds to
    auto splits_of = [](int tiles, float inv_t) { return max(1, (int)ceilf((float)tiles * inv_t - 1e-4f)); };
    const float t_min = fmaxf((float)kTreeMinTiles, work / (float)(waves * kTreeSms));
    float inv_t = 0.f;  // nothing is split
    // 32 candidates, a lane each, 1/32 further apart every time: the first that fits
    for (float base = t_min; base < (float)longest; base *= 2.f) {
        const float mine = 1.f / (base * (1.f + (float)lane * (1.f / 32.f)));
        int blocks = 0, slots = 0;
        for (int s0 = 0; s0 < n_seq; s0 += 32) {
            const TreeSeq q = of(s0);
            const int m = min(32, n_seq - s0);
            for (int j = 0; j < m; ++j) {
                const int items = __shfl_sync(0xffffffffu, q.items, j), tiles = __shfl_sync(0xffffffffu, q.tiles, j);
                const int k = splits_of(tiles, mine);
                blocks += items * k;
                slots += k > 1 ? items * k : 0;
            }
        }
        const unsigned fits = __ballot_sync(0xffffffffu, blocks <= cap && slots <= mp.slots);
        if (fits) {
            inv_t = __shfl_sync(0xffffffffu, mine, __ffs(fits) - 1);
            break;
        }
    }
    TreeSpot w = {};
    w.seq = -1;
    int front = 0, slots = 0;
    for (int s0 = 0; s0 < n_seq; s0 += 32) {
        const TreeSeq q = of(s0);
        const int k = splits_of(q.tiles, inv_t), mine = q.items * k, split = k > 1 ? mine : 0;
        const int end = warp_scan(mine, lane), send = warp_scan(split, lane);
        const unsigned hit = __ballot_sync(0xffffffffu, b < front + end);
        if (hit) {
            const int src = __ffs(hit) - 1;
            if (lane == src) {  // items in order, an item's splits side by side
                const int r = b - front - (end - mine), item = r / k;
                w.seq = s0 + src;
                w.splits = k;
                w.split = r - item * k;
                w.rt = item / mp.t.kv.kv_heads;
                w.kvh = item - w.rt * mp.t.kv.kv_heads;
                w.first_slot = slots + send - split;
                w.slot = w.first_slot + r;
                w.r0 = q.r0, w.n = q.n, w.len = q.len;
            }
            w.seq = __shfl_sync(0xffffffffu, w.seq, src);
            break;
        }
        front += __shfl_sync(0xffffffffu, end, 31);
        slots += __shfl_sync(0xffffffffu, send, 31);
    }
    return w;  // whole in the lane whose first_slot, n, ... are set: the one that `src` was
}

// x / G for row x of a sequence's n·G: exact while x·G < 2^32, which the call is checked for.
__device__ __forceinline__ int node_of(const TreeParams& p, int x) { return p.G == 1 ? x : (int)__umulhi((uint32_t)x, p.G_inv); }

// Which of positions p0 .. p0+63 the row sees, bit by bit.
__device__ __forceinline__ unsigned long long tree_window(const TreeParams& p, int row, int node, int n, int len, int p0) {
    auto ones = [](int c) -> unsigned long long { return c >= 64 ? ~0ull : c <= 0 ? 0ull : (1ull << c) - 1; };
    if (!p.mask) return ones(len + node + 1 - p0);
    const unsigned long long* m = p.mask + (long long)row * p.mask_words;
    const int j0 = p0 - len;
    unsigned long long w = 0;
    if (j0 >= 0) {
        const int i = j0 >> 6, o = j0 & 63;
        if (i < p.mask_words) w = m[i] >> o;
        if (o && i + 1 < p.mask_words) w |= m[i + 1] << (64 - o);
    } else if (j0 > -64) {
        w = m[0] << -j0;
    }
    return (w & ones(len + n - p0)) | ones(len - p0);
}

// Groups whose nodes differ too much (far_apart), position by position on the f32 units, as the softmax would have had
// them: `mine` holds the row's sums (columns as staged_at has them, by turn), m and *l their maximum and sum of weights.
// Ends with what the row's place is to hold.
template <int TYPE, int HD>
__device__ __noinline__ float add_apart(const MmaParams& mp, const TreeSpot& spot, const uint32_t* apart, int end, int row, int head,
                                        float4* mine, int turn, float m, float* l) {
    using SH = MmaShape<TYPE, HD>;
    using E = KvElem<TYPE>;
    const TreeParams& p = mp.t;
    const int tiles = (end + SH::T - 1) / SH::T, n = spot.n, len = spot.len, node = row - spot.r0;
    const int t0 = (int)((long long)tiles * spot.split / spot.splits), t1 = (int)((long long)tiles * (spot.split + 1) / spot.splits);
    const int first = max(t0, len / SH::T);  // tile with nodes
    const float* q = p.q + (long long)row * p.qs + (long long)head * HD;
    float sum = *l;
    for (int g = 0; g < (t1 - first) * SH::GROUPS; ++g) {
        if (!((apart[g >> 5] >> (g & 31)) & 1)) continue;
        const int p0 = first * SH::T + g * SH::RPW;
        for (int pos = p0; pos < min(p0 + SH::RPW, end); ++pos) {
            if (!(tree_window(p, row, node, n, len, pos) & 1)) continue;
            const long long at = kv_row(p.kv, p.b, spot.seq, pos);  // below 0: no page, a key and value of zeros
            const long long from = p.layer * p.kv.layer_bytes + at + (long long)spot.kvh * HD * SH::SIZE;
            const auto* kr = reinterpret_cast<const typename E::T*>(p.kv.k + from);
            const auto* vr = reinterpret_cast<const typename E::T*>(p.kv.v + from);
            float s = 0.f;
            if (at >= 0) {
#pragma unroll 32
                for (int d = 0; d < HD; ++d) s = fmaf(q[d], E::load(kr[d]), s);
            }
            s *= p.scale;
            const float mn = fmaxf(m, s), c = fmaxf(ex2(m - mn), least()), w = ex2(s - mn + 14.f);
            m = mn;
            sum = fmaf(sum, c, w);
            auto v = [&](int d) {
                const float x = at >= 0 ? E::load(vr[d]) : 0.f;
                return fabsf(x) < INFINITY ? x : 0.f;
            };
#pragma unroll 4
            for (int d = 0; d < HD; d += 4) {
                float4 f = mine[(d >> 2) ^ turn];
                f.x = fmaf(w, v(d), f.x * c), f.y = fmaf(w, v(d + 1), f.y * c);
                f.z = fmaf(w, v(d + 2), f.z * c), f.w = fmaf(w, v(d + 3), f.w * c);
                mine[(d >> 2) ^ turn] = f;
            }
        }
    }
    *l = sum;
    const float inv = spot.splits > 1 ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
    for (int d = 0; d < HD / 4; ++d) {
        const float4 f = mine[d];
        mine[d] = make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
    }
    return m;
}

template <int TYPE, int HD>
__global__ void __launch_bounds__(kMmaThreads, 1) tree_mma_kernel(const __grid_constant__ MmaParams mp) {
    using SH = MmaShape<TYPE, HD>;
    using E = KvElem<TYPE>;
    constexpr int T = SH::T, NB = SH::NB, NS = SH::NS, NC = SH::NC, RING = SH::RING, SW = SH::SW, PARTS = SH::PARTS;
    constexpr int kOutWarp = SH::OUT, kSplitWarp = SH::SPLIT_K;
    extern __shared__ __align__(1024) uint8_t sm[];
    const TreeParams& p = mp.t;
    // A waiter never falls a whole ring behind.  Scores of tile u are issued when the products of u - NS are done, and
    // those are issued when the weights of u - NS are there and the products before them were taken.  K's powers of
    // two of t + RING are written behind the tile before, whose place is free when the scores of t + RING - 1 - NB =
    // t + NS are done, so the softmax is through with tile t, and the correction of t + NC finds that of t taken;
    // V's are written when the products of t + RING - 1 - NB are done.  Every other barrier's next phase needs what
    // the waiter of this one does.
    uint64_t* k_full = reinterpret_cast<uint64_t*>(sm);  // [RING] K of a tile is ready: its splitting warps (f16: the copy)
    uint64_t* v_full = k_full + RING;                    // [NB] V, its splitting warps
    uint64_t* k_empty = v_full + NB;                     // [NB] scores done
    uint64_t* v_empty = k_empty + NB;                    // [NB] P·V done
    uint64_t* k_land = v_empty + NB;                     // [NB] copies of K landed (f32: [2] halves of its rows)
    uint64_t* v_land = k_land + NB;                      // [NB] copies of V
    uint64_t* raw_free = v_land + NB;                    // [2][2] f32: the splitting warps have half of K's, V's rows in registers
    uint64_t* s_full = raw_free + 4;              // [NS] scores done
    uint64_t* p_full = s_full + NS;                      // [NS] softmax warps: weights written
    uint64_t* c_full = p_full + NS;                      // [NC] softmax warps: correction written
    uint64_t* o_full = c_full + NC;                      // P·V done
    uint64_t* o_free = o_full + 1;                       // output warps: P·V and correction taken
    uint64_t* q_full = o_free + 1;                       // QW warps: queries written
    uint64_t* fin = q_full + 1;                          // softmax warps: tops and sums written
    uint64_t* done = fin + 1;                            // everything issued is done: scores, products
    uint64_t* w_empty = done + 1;                        // [NS] P·V done: the weights' place is free
    uint64_t* v_scale = w_empty + NS;                    // [RING] V's powers of two are written: its splitting warps
    static_assert((2 * RING + 5 * NB + 3 * NS + NC + 9) * 8 + 16 <= SH::BAD, "barriers");
    uint32_t* tslot = reinterpret_cast<uint32_t*>(v_scale + RING);
    volatile int* flag = reinterpret_cast<volatile int*>(tslot + 1);
    int* any_apart = reinterpret_cast<int*>(tslot + 2);  // whether apart[] has a bit set
    uint32_t* bad = reinterpret_cast<uint32_t*>(sm + SH::BAD);
    uint32_t* apart = reinterpret_cast<uint32_t*>(sm + SH::APART);
    float* s_rs = reinterpret_cast<float*>(sm + SH::ROWS);
    float* s_corr = s_rs + kMmaRows;
    float* s_other = s_corr + NC * kMmaRows;
    float* s_top = s_other + 2 * PARTS * kMmaRows;
    float* s_sum = s_top + kMmaRows;
    float* scales = reinterpret_cast<float*>(sm + SH::SCALE);
    uint8_t* tiles = sm + SH::TILES;
    uint8_t* staged = tiles + SH::QTILE * 2 * SH::HALF;
    auto staged_at = [&](int row, int byte) { return staged + row * SH::QROW + (((byte >> 4) ^ (row & 7)) << 4) + (byte & 15); };
    // A whole warp waits and stays together: the first look is cheap, the rest bounded (kSpinLimit, or another's flag).
    auto wait_warp = [&](uint64_t* bar, int phase) -> bool {
        bool ok = mbar_try_wait(bar, (uint32_t)phase & 1u);
        if (__all_sync(0xffffffffu, ok)) return true;
        for (uint32_t i = 0; i < kSpinLimit; ++i) {
            ok = ok || mbar_try_wait(bar, (uint32_t)phase & 1u);
            if (__all_sync(0xffffffffu, ok)) return true;
            if ((i & 15) == 15 && __any_sync(0xffffffffu, *flag != 0)) return false;
        }
        set_err_at(p.b.err, kErrMbarTimeout);
        return false;
    };
    // Several at once: the looks overlap where all have come already.
    auto wait_both = [&](uint64_t* a, int pa, uint64_t* b, int pb) -> bool {
        const bool x = mbar_try_wait(a, (uint32_t)pa & 1u), y = mbar_try_wait(b, (uint32_t)pb & 1u);
        return __all_sync(0xffffffffu, x && y) || (wait_warp(a, pa) && wait_warp(b, pb));
    };
    auto wait_three = [&](uint64_t* a, int pa, uint64_t* b, int pb, uint64_t* c, int pc) -> bool {
        const bool x = mbar_try_wait(a, (uint32_t)pa & 1u), y = mbar_try_wait(b, (uint32_t)pb & 1u), z = mbar_try_wait(c, (uint32_t)pc & 1u);
        return __all_sync(0xffffffffu, x && y && z) || (wait_warp(a, pa) && wait_warp(b, pb) && wait_warp(c, pc));
    };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    __shared__ TreeSpot spot;
    pdl_launch_dependents();
    if (warp == 0) {
        const TreeSpot w = tree_spot(mp, T, blockIdx.x);
        if (w.seq < 0 ? lane == 0 : w.splits > 0) {
            spot = w;
            if (w.seq >= 0 && mp.plan && w.split == 0 && w.rt == 0 && w.kvh == 0) mp.plan[w.seq] = make_int2(w.first_slot, w.splits);
        }
    } else if (warp == 1 && lane == 0) {
        for (int i = 0; i < NB; ++i) {
            mbar_init(&v_full[i], SW);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&k_land[i], 1);
            mbar_init(&v_land[i], 1);
        }
        for (int i = 0; i < RING; ++i) {
            mbar_init(&k_full[i], TYPE == AF_KV_F16 ? 1 : SW);
            mbar_init(&v_scale[i], SW);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&raw_free[i], SW / 2);
        for (int i = 0; i < NS; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&w_empty[i], 1);
        }
        mbar_init(o_full, 1);
        mbar_init(q_full, SH::QW);
        mbar_init(done, 2);
        *flag = 0;
        *any_apart = 0;
    } else if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (warp == kCopyWarp && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mp.k_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&mp.v_map) : "memory");
    }
    for (int i = tid; i < kMmaBadWords + SH::APART_WORDS; i += kMmaThreads) bad[i] = 0;  // and apart[], behind it
    __syncthreads();
    const int seq = spot.seq, kvh = spot.kvh, r0 = spot.r0, n = spot.n, len = spot.len;
    // the block's rows and tiles (the same in every thread)
    const int row_lo = spot.rt * kMmaRows, row_hi = min(row_lo + kMmaRows, n * p.G);
    const int live_warps = (row_hi - row_lo + 31) / 32;  // of every 4 that work on rows; the others have none
    if (tid == 0 && seq >= 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&p_full[i], PARTS * live_warps);
        }
        for (int i = 0; i < NC; ++i) mbar_init(&c_full[i], live_warps);
        mbar_init(o_free, live_warps);
        mbar_init(fin, PARTS * live_warps);
    }
    if (tid < 64) fence_mbar_init();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tslot;
    if (seq < 0) {
        if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        return;
    }
    const int end = p.mask ? len + n : len + node_of(p, row_hi - 1) + 1;  // positions that some row may see
    const int nt_all = (end + T - 1) / T;
    const int t0 = (int)((long long)nt_all * spot.split / spot.splits),
              t1 = (int)((long long)nt_all * (spot.split + 1) / spot.splits);
    const int nt = t1 - t0;
    int bs = 0;  // tiles of a bit of bad[]: 1 << bs
    while (nt > (kMmaBadWords * 32) << bs) ++bs;

    // Queries, by QW warps: a row a warp in turn — its largest value, hi and lo — into the staging
    // place, from there a row a thread (hi by softmax warps 0-3, lo by 4-7) into tensor memory.  Rows that are
    // none keep what is there: what comes of them stays in their own row.
    auto queries = [&]() {
        constexpr int QW = SH::QW, Q4 = HD / 4, QR = 32 / Q4, QN = (128 / QR + QW - 1) / QW;  // lanes of a row at 16 bytes, rows and number of a warp's loads
        const int sub = lane / Q4, col = lane % Q4, rows = row_hi - row_lo;
        const bool wide = ((reinterpret_cast<uintptr_t>(p.q) & 15) | (p.qs & 3)) == 0;
        float4 f[QN];  // all in flight
#pragma unroll
        for (int j = 0; j < QN; ++j) {
            if ((warp + QW * j) * QR >= rows) break;
            const int x = row_lo + min((warp + QW * j) * QR + sub, rows - 1), node = node_of(p, x);
            const float* q = p.q + (long long)(r0 + node) * p.qs + (kvh * p.G + x - node * p.G) * HD + 4 * col;
            if (wide) f[j] = __ldg(reinterpret_cast<const float4*>(q));
            else f[j] = make_float4(q[0], q[1], q[2], q[3]);
        }
#pragma unroll
        for (int j = 0; j < QN; ++j) {
            if ((warp + QW * j) * QR >= rows) break;
            const int i = (warp + QW * j) * QR + sub;
            uint32_t mx = __float_as_uint(max3_abs_nan(max3_abs_nan(0.f, f[j].x, f[j].y), f[j].z, f[j].w));
            if (QR == 1) {
                mx = __reduce_max_sync(0xffffffffu, mx);
            } else {
#pragma unroll
                for (int o = 1; o < Q4; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            }
            const int a = scale_of(mx, 100);
            const float sg = copysignf(pow2(a), p.scale);  // a negative scale turns the query around
            const f32x2 s = pair(sg, sg);
            uint2 hi, lo;
            split2(mul2(pair(f[j].x, f[j].y), s), hi.x, lo.x);
            split2(mul2(pair(f[j].z, f[j].w), s), hi.y, lo.y);
            if (i < rows) {
                *reinterpret_cast<uint2*>(staged_at(i, 8 * col)) = hi;
                *reinterpret_cast<uint2*>(staged_at(i, 2 * HD + 8 * col)) = lo;
                if (col == 0) s_rs[i] = fmaxf(fabsf(p.scale) * pow2(-a), FLT_MIN);
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(QW * 32) : "memory");
        const int mine = tid & 127;
        if (warp < 8 && (mine & ~31) < rows) {
            const int from = warp < 4 ? 0 : 2 * HD;
            const uint32_t to = tmem + ((uint32_t)(mine & ~31) << 16) + (warp < 4 ? SH::QH : SH::QL);
#pragma unroll 2
            for (int c = 0; c < HD / 16; ++c) {
                const uint4 x = *reinterpret_cast<const uint4*>(staged_at(mine, from + 32 * c));
                const uint4 y = *reinterpret_cast<const uint4*>(staged_at(mine, from + 32 * c + 16));
                const uint32_t v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                tc_st8(to + 8 * c, v);
            }
            tc_wait_st();
        }
        tc_fence_before();
        fence_proxy_async_smem();  // the copies may write over the staging place now
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
    };

    if (warp < kOutWarp) {
        // ------------------------------------------------------- softmax
        // Four warps have 32 of a tile's columns, the next four the next 32, of the same rows.  A row's threads tell
        // one another their largest value and keep sums of their own.
        if constexpr (SH::REG_S > 64) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SH::REG_S));
        else if constexpr (SH::REG_S < 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SH::REG_S));
        constexpr int C = 32;
        const int part = warp >> 2, ti = tid & 127, w4 = warp & 3;
        const uint32_t lanes = (uint32_t)(w4 * 32) << 16;
        const int r = row_lo + ti;
        const bool live = r < row_hi;
        const int node = live ? node_of(p, r) : 0, row = r0 + node;
        queries();
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        const float rs = s_rs[ti];  // what a raw score is times, but for K's power of two
        auto publish = [&](int sl) {
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[sl]);
        };
        const int tiles_mine = w4 < live_warps ? nt : 0;
        int sl = 0, sl_ph = 0, kt = 0, kt_ph = 0, co = 0;  // rings of NS, RING, NC and their phases
        int met = 0;  // the tiles at which the row's warps have met
        for (int t = 0; t < tiles_mine; ++t) {
            ok = TYPE == AF_KV_F16 ? wait_warp(&s_full[sl], sl_ph)
                                   : wait_three(&k_full[kt], kt_ph, &s_full[sl], sl_ph, &v_scale[kt], kt_ph);
            if (!ok) break;
            tc_fence_after();
            const uint32_t sb = tmem + lanes + SH::S0 + sl * T + part * C;
            float v[C];
#pragma unroll
            for (int c = 0; c < C / 32; ++c) tc_ld32(sb + 32 * c, v + 32 * c);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < C; ++i) asm volatile("" : "+f"(v[i]));  // no use may move above the wait
            // f32: a power of two per 8 columns; bf16: one for the thread's 32, taken care of in the exponent
            const float* sc = scales + kt * 4 * SH::GROUPS + part * (C / SH::RPW);  // 2^-a of K, -a of V, 2^a of V, 0 of K
            float scale = rs, shift = 0.f, share = 1.f;
            if (TYPE == AF_KV_BF16) scale = fmaxf(rs * sc[0], FLT_MIN), shift = sc[SH::GROUPS] + sc[3 * SH::GROUPS], share = sc[2 * SH::GROUPS];
            if (SH::F32) {
                const float4 x = *reinterpret_cast<const float4*>(sc), z = *reinterpret_cast<const float4*>(sc + SH::GROUPS),
                             y = *reinterpret_cast<const float4*>(sc + 3 * SH::GROUPS);
                const float c[4] = {rs * x.x, rs * x.y, rs * x.z, rs * x.w}, f[4] = {z.x + y.x, z.y + y.y, z.z + y.z, z.w + y.w};
#pragma unroll
                for (int e = 0; e < C; e += 2)
                    unpair(fma2(pair(v[e], v[e + 1]), pair(c[e / 8], c[e / 8]), pair(f[e / 8], f[e / 8])), v[e], v[e + 1]);
            }
            const int p0 = (t0 + t) * T + part * C;
            if (p0 + C > len) {
                unsigned long long see = live ? tree_window(p, row, node, n, len, p0) : 0ull;
#pragma unroll
                for (int i = 0; i < C; ++i)
                    if (!((see >> i) & 1)) v[i] = -INFINITY;
            }
            float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
            for (int i = 4; i + 1 < C; i += 2) top[(i >> 1) & 3] = max3(top[(i >> 1) & 3], v[i], v[i + 1]);
            float mn = max3(top[0], top[1], fmaxf(top[2], top[3]));
            if (!SH::F32 && mn != -INFINITY) mn = fmaf(mn, scale, shift);  // scale > 0: raw scores have the same largest one
            mn = fmaxf(m, mn);
            // the row's other parts, in two places in turn: this one is written again when all have read it
            float* others = s_other + (t & 1) * PARTS * kMmaRows + ti;
            others[part * kMmaRows] = mn;
            asm volatile("bar.sync %0, %1;" ::"r"(2 + w4), "n"(PARTS * 32) : "memory");
            ++met;
#pragma unroll
            for (int i = 0; i < PARTS; ++i) mn = fmaxf(mn, others[i * kMmaRows]);
            const float ms = mn == -INFINITY ? 0.f : mn - 14.f;  // weights times 2^14
            const float corr = ex2(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            if (part == 0) {
                s_corr[co * kMmaRows + ti] = corr;
                __syncwarp();
                if (lane == 0) mbar_arrive(&c_full[co]);
            }
            if (++co == NC) co = 0;
            f32x2 sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
            const f32x2 ms2 = pair(shift - ms, shift - ms), rs2 = pair(scale, scale);
            float g4[4];
            if (SH::F32) {
                const float4 x = *reinterpret_cast<const float4*>(sc + 2 * SH::GROUPS);
                g4[0] = x.x, g4[1] = x.y, g4[2] = x.z, g4[3] = x.w;
            }
#pragma unroll
            for (int c = 0; c < C / 16; ++c) {
                uint32_t hi[8], lo[8];
                float w[16];
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const f32x2 x = pair(v[16 * c + i], v[16 * c + i + 1]);
                    unpair(SH::F32 ? add2(x, ms2) : fma2(x, rs2, ms2), w[i], w[i + 1]);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = ex2(w[i]);
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const f32x2 x = pair(w[i], w[i + 1]);
                    if (SH::F32) {
                        const float g = g4[(16 * c + i) / 8];
                        sum[(i >> 1) & 1] = fma2(x, pair(g, g), sum[(i >> 1) & 1]);
                    } else {
                        sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], x);
                    }
                    split2(x, hi[i / 2], lo[i / 2]);
                }
                tc_st8(sb + 16 * c, hi);  // over the 16 scores that they came from
                tc_st8(sb + 16 * c + 8, lo);
            }
            {
                float a, b;
                unpair(add2(sum[0], sum[1]), a, b);
                l = fmaf(l, corr, share * (a + b));
            }
            publish(sl);
            if (++sl == NS) sl = 0, sl_ph ^= 1;
            if (++kt == RING) kt = 0, kt_ph ^= 1;
        }
        // one that leaves early is counted at the others' remaining meetings: nobody is left waiting
        for (; met < tiles_mine; ++met) asm volatile("bar.arrive %0, %1;" ::"r"(2 + w4), "n"(PARTS * 32) : "memory");
        if (!ok) *flag = 1;
        if (part == 0) s_top[ti] = m;
        s_sum[part * kMmaRows + ti] = l;
        __syncwarp();
        if (lane == 0 && w4 < live_warps) mbar_arrive(fin);
    } else if (warp < kSplitWarp) {
        // ------------------------------------------------ sums, rows out
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SH::REG_O));
        queries();
        constexpr int Q4 = HD / 4, QR = 32 / Q4;  // lanes of a row at 16 bytes each, rows of a warp's store
        const int w = warp - kOutWarp, ti = tid - kOutWarp * 32;
        const uint32_t lanes = (uint32_t)(w * 32) << 16;
        const int sub = lane / Q4, col = lane % Q4;
        float acc[HD];
#pragma unroll
        for (int i = 0; i < HD; ++i) acc[i] = 0.f;
        bool ok = w < live_warps;
        int co = 0, co_ph = 0;
        for (int t = 0; ok && t < nt; ++t) {  // acc = acc·corr + (P·V)(t)
            ok = wait_both(&c_full[co], co_ph, o_full, t);
            if (!ok) break;
            tc_fence_after();
            const float corr = s_corr[co * kMmaRows + ti];
            if (++co == NC) co = 0, co_ph ^= 1;
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {
                float o[16];
                tc_ld16(tmem + lanes + SH::O0 + 16 * c, o);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) asm volatile("" : "+f"(o[i]));  // no use may move above the wait
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    float& x = acc[16 * c + i];
                    float& y = acc[16 * c + i + 1];
                    unpair(fma2(pair(x, y), pair(corr, corr), pair(o[i], o[i + 1])), x, y);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_free);
        }
        ok = ok && wait_warp(fin, 0);
        if (!ok && w < live_warps) *flag = 1;
        const int r = row_lo + ti;
        const bool live = r < row_hi;
        const int node = live ? node_of(p, r) : 0, row = r0 + node, head = kvh * p.G + (live ? r - node * p.G : 0);
        // non-finite values of V were taken out of the products: the rows that see them get them back
        for (int wd = 0; ok && wd < kMmaBadWords && (32 * wd) << bs < nt; ++wd) {
            uint32_t b = bad[wd];
            while (b) {
                const int t = (32 * wd + __ffs(b) - 1) << bs;
                b &= b - 1;
                for (int pos = (t0 + t) * T; pos < min((t0 + min(t + (1 << bs), nt)) * T, end); ++pos) {
                    if (!live || !(tree_window(p, row, node, n, len, pos) & 1)) continue;
                    const long long at = kv_row(p.kv, p.b, seq, pos);
                    if (at < 0) continue;
                    const auto* vr = reinterpret_cast<const typename E::T*>(p.kv.v + p.layer * p.kv.layer_bytes + at) + kvh * HD;
#pragma unroll
                    for (int d = 0; d < HD; ++d) {
                        const float x = E::load(vr[d]);
                        if (!(fabsf(x) < INFINITY)) acc[d] += x;
                    }
                }
            }
        }
        if (ok) {
            const int splits = spot.splits, mine_rows = min(32, row_hi - row_lo - w * 32);
            float l = 0.f;
#pragma unroll
            for (int i = 0; i < PARTS; ++i) l += s_sum[i * kMmaRows + ti];
            const bool more = TYPE != AF_KV_F16 && *any_apart != 0;
            const float inv = splits > 1 || more ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int i = 0; i < HD; i += 4)
                *reinterpret_cast<float4*>(staged_at(ti, 4 * i)) =
                    make_float4(acc[i] * inv, acc[i + 1] * inv, acc[i + 2] * inv, acc[i + 3] * inv);
            if constexpr (TYPE != AF_KV_F16) {
                if (more && live) s_top[ti] = add_apart<TYPE, HD>(mp, spot, apart, end, row, head, reinterpret_cast<float4*>(staged + ti * SH::QROW), ti & 7, s_top[ti], &l);
            }
            __syncwarp();
            auto from = [&](int i) { return *reinterpret_cast<const float4*>(staged_at(w * 32 + i + sub, 16 * col)); };
            if (splits > 1) {  // the split's place in the workspace, rows of HD values side by side
                const long long at = (long long)spot.slot * kMmaRows + w * 32;
                float* o = mp.part + (at + sub) * HD + 4 * col;
#pragma unroll 8
                for (int i = 0; i < mine_rows; i += QR)
                    if (i + sub < mine_rows)
                        *reinterpret_cast<float4*>(o + i * HD) = from(i);
                if (lane < mine_rows)
                    *reinterpret_cast<float2*>(mp.part + (long long)mp.slots * kMmaRows * HD + (at + lane) * 2) =
                        make_float2(s_top[ti], l);
            } else {
                float* orow = live ? p.out + (long long)row * p.os + (long long)head * HD : nullptr;
                const bool wide_out = ((reinterpret_cast<uintptr_t>(p.out) & 15) | (p.os & 3)) == 0;
#pragma unroll 4
                for (int i = 0; i < mine_rows; i += QR) {
                    float* o = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(orow), i + sub));
                    const float4 f = from(i);
                    if (o) {
                        o += 4 * col;
                        if (wide_out) *reinterpret_cast<float4*>(o) = f;
                        else o[0] = f.x, o[1] = f.y, o[2] = f.z, o[3] = f.w;
                    }
                }
            }
        }
    } else if (warp < kMmaWarp) {
        // ------------------------------------------------- splitting K and V
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SH::REG_K));
        if (TYPE == AF_KV_F16) queries();
        const bool isv = warp >= kSplitWarp + SW;
        const int w = (warp - kSplitWarp) % SW;
        uint64_t *full = isv ? v_full : k_full, *empty = isv ? v_empty : k_empty, *land = isv ? v_land : k_land;
        const int ring = isv ? NB : RING;
        auto hand_over = [&](uint64_t* bar) {
            fence_proxy_async_smem();  // these stores, before the products read them
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        auto note_bad = [&](int t) {
            if (lane == 0) atomicOr(&bad[(t >> bs) >> 5], 1u << ((t >> bs) & 31));
        };
        bool ok = true;
        int st = 0, ph = 0, fu = 0, sc_at = 0;  // ring of NB tiles and its phase, of `full`, of the scales
        auto note_apart = [&](int t) {  // the group is left out of the products
            const int i = (t - max(len / T - t0, 0)) * SH::GROUPS + w;  // of those of the tiles with nodes
            if (lane == 0) {
                atomicOr(&apart[i >> 5], 1u << (i & 31));
                *any_apart = 1;
            }
        };
        auto put_scale = [&](int a, float f, bool out) {  // the group's power of two
            if (lane != 0) return;
            float* sc = scales + sc_at * 4 * SH::GROUPS + w;
            if (isv) {
                sc[SH::GROUPS] = out ? -INFINITY : (float)-a;
                sc[2 * SH::GROUPS] = f;
                mbar_arrive(&v_scale[sc_at]);  // the softmax need not wait for the tile itself
            } else {
                sc[0] = out ? 0.f : pow2(-a);
                sc[3 * SH::GROUPS] = out ? -INFINITY : 0.f;
            }
        };
        auto next = [&]() {
            if (++st == NB) st = 0, ph ^= 1;
            if (++fu == ring) fu = 0;
            if (++sc_at == RING) sc_at = 0;
        };
        if (SH::F32) {
            // RPW rows of the tile, half a tile being in flight: out of the raw place into registers, which frees it, then
            // split and stored.
            constexpr int NX = SH::RPW * HD * 4 / 512;  // a warp's loads of its rows
            const int sub = lane / SH::LPR, col = lane % SH::LPR;
            const uint8_t* raw = sm + SH::RAW + (isv ? 2 * SH::RAWB : 0) + w * SH::RPW * HD * 4 + lane * 16;
            uint64_t* freed = raw_free + (isv ? 2 : 0);
            const int in_half = (4 * col) % 64 * 2;  // byte of the lane's 4 values in a 128-byte row
            uint8_t* home = tiles + (isv ? SH::HALF : 0) + (4 * col) / 64 * SH::COLS + w * SH::RPW * 128 + (in_half & 8);
            uint64_t* due = nullptr;                 // a tile that is stored and not yet handed over
#pragma unroll 1
            for (int t = 0; ok && t < nt; ++t) {
                ok = wait_warp(&land[w / (SW / 2)], t);
                if (!ok) break;
                float4 x[NX];
                float big[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NX; ++i) x[i] = *reinterpret_cast<const float4*>(raw + i * 512);
                const int left = end - (t0 + t) * T - w * SH::RPW - sub;  // rows in front of the end
                if (left < SH::RPW) {                                               // the last tile: what lies behind is nothing
#pragma unroll
                    for (int i = 0; i < NX; ++i)
                        if (i * SH::RPC >= left) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int i = 0; i < NX; ++i) {
                    big[(2 * i) & 3] = max3_abs_nan(big[(2 * i) & 3], x[i].x, x[i].y);
                    big[(2 * i + 1) & 3] = max3_abs_nan(big[(2 * i + 1) & 3], x[i].z, x[i].w);
                }
                uint32_t mx = __reduce_max_sync(
                    0xffffffffu, __float_as_uint(max3_abs_nan(max3_abs_nan(big[0], big[1], big[2]), big[3], 0.f)));
                if (lane == 0) mbar_arrive(&freed[w / (SW / 2)]);  // all lanes hold theirs
                if (isv && mx >= 0x7f800000u) {  // rare: take what is not finite out, and remember the tile
                    float4 y[NX];
#pragma unroll
                    for (int i = 0; i < NX; ++i) y[i] = x[i];
                    mx = clean(y);
#pragma unroll
                    for (int i = 0; i < NX; ++i) x[i] = y[i];
                    note_bad(t);
                }
                bool differ = false;
                if ((t0 + t) * T + (w + 1) * SH::RPW > len) {  // the group has nodes
                    uint32_t low = 0xffffffffu;
#pragma unroll
                    for (int i = 0; i < NX; ++i)
                        low = min(low, __float_as_uint(max3_abs_nan(max3_abs_nan(0.f, x[i].x, x[i].y), x[i].z, x[i].w)) - 1u);
                    differ = far_apart<TYPE>(mx, low);
                    if (differ) note_apart(t);
                }
                const int a = scale_of(mx, isv ? 60 : 100);
                const float f = pow2(a);
                const f32x2 f2 = pair(f, f);
                put_scale(a, f, differ);
                if (due) hand_over(due);                        // the tile before: its stores are through by now
                if (t == SH::QTILE) ok = wait_warp(q_full, 0);  // the staged queries' place is written over
                if (ok && t >= NB) ok = wait_warp(&empty[st], ph ^ 1);
                if (!ok) break;
                uint8_t* dst = home + st * 2 * SH::HALF;
#pragma unroll
                for (int i = 0; i < NX; ++i) {
                    uint2 hi, lo;
                    split2(mul2(pair(x[i].x, x[i].y), f2), hi.x, lo.x);
                    split2(mul2(pair(x[i].z, x[i].w), f2), hi.y, lo.y);
                    const int rr = i * SH::RPC + sub;
                    uint8_t* d = dst + rr * 128 + (((in_half >> 4) ^ ((w * SH::RPW + rr) & 7)) << 4);
                    *reinterpret_cast<uint2*>(d) = hi;
                    *reinterpret_cast<uint2*>(d + SH::TILE) = lo;
                }
                due = &full[fu];
                next();
            }
            if (ok && due) hand_over(due);
        } else if (TYPE == AF_KV_BF16 || isv) {
            // in place; an access takes 512 bytes: 4 rows of 64 values
            constexpr int ALL = SH::RPW * HD * 2 / 512, NC = 4, PER = SH::RPW / 4;  // accesses; at a time; of the rows' 64 values
            auto fix = [&](int t, auto with_nodes) {
                constexpr bool NODES = decltype(with_nodes)::value;
                uint8_t* at = tiles + (st * 2 + (isv ? 1 : 0)) * SH::HALF + w * SH::RPW * 128 + lane * 16;
                auto place = [&](int i) { return reinterpret_cast<uint4*>(at + (i / PER) * SH::COLS + (i % PER) * 512); };
                uint4 x[NC];
                uint32_t* e = &x[0].x;
                const int left = end - (t0 + t) * T - w * SH::RPW - lane / 8;  // rows in front of the end
                const bool last = NODES && left + lane / 8 < SH::RPW;          // the same in the whole warp
                auto load = [&](int i0) {
#pragma unroll
                    for (int i = 0; i < NC; ++i) x[i] = *place(i0 + i);
                    if (last) {  // what lies behind the end is nothing: whatever was in that place before
#pragma unroll
                        for (int i = 0; i < NC; ++i)
                            if ((i0 + i) % PER * 4 >= left) x[i] = make_uint4(0u, 0u, 0u, 0u);
                    }
                };
                auto without = [&]() {  // zeros for what is not finite
                    constexpr uint32_t top = TYPE == AF_KV_F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
                    for (int i = 0; i < 4 * NC; ++i) {
                        if ((e[i] & top) == top) e[i] &= 0xffff0000u;
                        if ((e[i] & top << 16) == top << 16) e[i] &= 0x0000ffffu;
                    }
                };
                if (TYPE == AF_KV_F16) {
#pragma unroll 1
                    for (int i0 = 0; i0 < ALL; i0 += NC) {
                        load(i0);
                        __half2 z = __float2half2_rn(0.f);  // x·0 is 0 for what is finite, NaN otherwise
#pragma unroll
                        for (int i = 0; i < 4 * NC; ++i)
                            z = __hfma2(*reinterpret_cast<const __half2*>(&e[i]), __float2half2_rn(0.f), z);
                        const uint32_t zz = *reinterpret_cast<const uint32_t*>(&z) & 0x7fff7fffu;
                        const bool odd = __any_sync(0xffffffffu, zz != 0);
                        if (odd) {
                            without();
                            note_bad(t);
                        }
                        if (odd || last) {
#pragma unroll
                            for (int i = 0; i < NC; ++i) *place(i0 + i) = x[i];
                        }
                    }
                    return;
                }
                const bool nodes = NODES && (t0 + t) * T + (w + 1) * SH::RPW > len;
                uint32_t low = 0xffffffffu;  // see far_apart
                auto largest = [&](bool finite, auto with_low) {
                    uint32_t b = 0, least = 0xffffffffu;  // two at once: bf16's magnitudes are ordered as 16-bit numbers
#pragma unroll 1
                    for (int i0 = 0; i0 < ALL; i0 += NC) {
                        load(i0);
                        if (finite) without();
#pragma unroll
                        for (int i = 0; i < NC; ++i) {
                            uint32_t z = e[4 * i] & 0x7fff7fffu;
#pragma unroll
                            for (int j = 1; j < 4; ++j) z = __vmaxu2(z, e[4 * i + j] & 0x7fff7fffu);
                            b = __vmaxu2(b, z);
                            if (decltype(with_low)::value) least = __vminu2(least, ((z | 0x80008000u) - 0x00010001u) ^ 0x80008000u);  // less 1, 0 the largest
                        }
                    }
                    if (decltype(with_low)::value) {
                        least = min(least & 0xffffu, least >> 16);
                        low = least == 0xffffu ? 0xffffffffu : (least << 16) + 0xffffu;
                    }
                    return __reduce_max_sync(0xffffffffu, max(b << 16, b & 0xffff0000u));
                };
                uint32_t mx = largest(false, std::integral_constant<bool, NODES>());
                const bool odd = isv && mx >= 0x7f800000u;
                if (odd) {
                    low = 0xffffffffu;
                    mx = largest(true, std::integral_constant<bool, NODES>());
                    note_bad(t);
                }
                const bool differ = nodes && far_apart<TYPE>(mx, low) && far_apart<TYPE>(mx, lowest_row<PER, HD / 64, SH::COLS>(at, left));
                if (differ) note_apart(t);
                const int a = scale_of(mx, isv ? 60 : 100);
                const float f = pow2(a);
                const f32x2 f2 = pair(f, f);
                put_scale(a, f, differ);
#pragma unroll 1
                for (int i0 = 0; i0 < ALL; i0 += NC) {
                    load(i0);
                    if (odd) without();
#pragma unroll
                    for (int i = 0; i < 4 * NC; ++i) {
                        float lo, hi;
                        unpair(mul2(pair(__uint_as_float(e[i] << 16), __uint_as_float(e[i] & 0xffff0000u)), f2), lo, hi);
                        e[i] = pack2(lo, hi);
                    }
#pragma unroll
                    for (int i = 0; i < NC; ++i) *place(i0 + i) = x[i];
                }
            };
            auto take = [&](int t, auto with_nodes) {
                ok = wait_warp(&land[st], ph);
                if (!ok) return;
                fix(t, with_nodes);
                hand_over(&full[fu]);
                next();
            };
            int t = 0;
#pragma unroll 1
            for (; TYPE != AF_KV_F16 && ok && t < nt && (t0 + t + 1) * T <= len; ++t) take(t, std::false_type());
#pragma unroll 1
            for (; ok && t < nt; ++t) take(t, std::true_type());
        }
        if (!ok) *flag = 1;
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SH::REG_M));
        if ((warp == kCopyWarp || warp == kCopyWarp + 1) && nt > 0) {
            // --------------------------------------------------- copies
            const bool isv = warp != kCopyWarp;
            const CUtensorMap* map = isv ? &mp.v_map : &mp.k_map;
            const uint32_t leader = elect_one();
            const int R = mp.box_rows;  // a box never crosses a page
            const int* table = p.b.table ? p.b.table + (long long)seq * p.b.max_blocks : nullptr;
            const int page0 = (int)min((long long)seq * p.b.max_blocks, (long long)p.kv.n_pages);  // no table: pages in order
            const int in_page = (1 << p.kv.ps_shift) - 1;
            auto fetch = [&](int t, int box) -> int {  // the page of a box, asked for early
                const int pos = min((t0 + min(t, nt - 1)) * T + box * R, end - 1);
                const int blk = pos >> p.kv.ps_shift;
                return table ? __ldg(table + blk) : page0 + blk;
            };
            // pool row of this lane's box of tile t; a page that is none: the error word, and rows in front of the pool,
            // which the copy fills with zeros
            auto row_of = [&](int t, int box, int page) -> int {
                if ((unsigned)page >= (unsigned)p.kv.n_pages) {
                    set_err_at(p.b.err, kErrBadArgs);
                    return -R;
                }
                return (page << p.kv.ps_shift) + (((t0 + t) * T + box * R) & in_page);
            };
            // boxes [first, first + n) of tile t, as far as they are in front of the end, to dst
            auto send = [&](int t, int first, int n_boxes, uint8_t* dst, uint64_t* bar, int row) {
                constexpr int HALVES = SH::F32 ? 1 : HD / 64, ROWB = SH::F32 ? HD * 4 : 128;
                const int live = max(0, min(n_boxes, (end - (t0 + t) * T + R - 1) / R - first));
                const uint32_t b = smem_u32(bar), d = smem_u32(dst);
                if (leader) mbar_arrive_expect_tx(bar, (uint32_t)(live * R * HD * SH::SIZE));
                __syncwarp();
                for (int i = 0; i < live; ++i) {
                    const int box = first + i;
                    if (box && !(box & 31)) row = row_of(t, box + lane, fetch(t, box + lane));  // pages of one or two rows
                    const int z = __shfl_sync(0xffffffffu, row, box & 31);
#pragma unroll
                    for (int c = 0; c < HALVES; ++c)
                        tma_rows(leader, d + c * SH::COLS + i * R * ROWB, map, 64 * c, kvh, z, b);
                }
                return row;
            };
            bool ok = true;
            int page = fetch(0, lane);
            int st = 0, ph = 0, kt = 0;
            for (int t = 0; t < nt; ++t) {
                int row = row_of(t, lane, page);
                page = fetch(t + 1, lane);
                if (SH::F32) {
                    const int half = T / 2 / R;
#pragma unroll 1
                    for (int s = 0; ok && s < 2; ++s) {
                        if (t) ok = wait_warp(&raw_free[(isv ? 2 : 0) + s], t - 1);
                        if (ok)
                            row = send(t, s * half, half, sm + SH::RAW + ((isv ? 2 : 0) + s) * SH::RAWB, (isv ? v_land : k_land) + s, row);
                    }
                } else {
                    if (t == SH::QTILE) ok = wait_warp(q_full, 0);  // the staged queries' place is written over
                    if (ok && t >= NB) ok = wait_warp(isv ? &v_empty[st] : &k_empty[st], ph ^ 1);
                    if (ok)
                        send(t, 0, T / R, tiles + (st * 2 + (isv ? 1 : 0)) * SH::HALF,
                             isv ? &v_land[st] : TYPE == AF_KV_F16 ? &k_full[kt] : &k_land[st], row);
                }
                if (!ok) break;
                if (++st == NB) st = 0, ph ^= 1;
                if (++kt == RING) kt = 0;
            }
            if (!ok) *flag = 1;
        } else if ((warp == kMmaWarp || warp == kScoreWarp) && nt > 0) {
            // --------------------------------------------------- products
            constexpr uint32_t base = (1u << 4) | ((uint32_t)(kMmaRows >> 4) << 24);  // f32 accumulators, f16 operands
            constexpr uint32_t ids = base | ((uint32_t)(T >> 3) << 17);
            constexpr uint32_t ido = base | ((uint32_t)(HD >> 3) << 17) | (1u << 16);  // B MN-major
            const uint32_t leader = elect_one();
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const int n_tiles = __shfl_sync(0xffffffffu, nt, 0);
            bool ok = true;
            int st = 0, ph = 0, sl = 0, sl_ph = 0;
            if (warp == kScoreWarp) {
                // K: 8-row groups 1,024 bytes apart, 16 values 32 bytes on
                const uint64_t kd = tile_desc(smem_u32(tiles), 16, 1024);
                auto k_step = [](int ks) { return (uint32_t)((ks >> 2) * SH::COLS + (ks & 3) * 32) >> 4; };
                int kt = 0, kt_ph = 0;
                ok = wait_warp(q_full, 0);
                for (int t = 0; ok && t < n_tiles; ++t) {
                    ok = t < NS ? wait_warp(&k_full[kt], kt_ph) : wait_both(&k_full[kt], kt_ph, &w_empty[sl], sl_ph ^ 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t k = kd + (uint32_t)(st * (2 * SH::HALF >> 4));
                    const uint32_t d = tm + SH::S0 + sl * T;
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks) tc_mma_ts(leader, d, tm + SH::QL + 8 * ks, k + k_step(ks), ids, ks > 0);
                    if (SH::TERMS == 2) {
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ++ks)
                            tc_mma_ts(leader, d, tm + SH::QH + 8 * ks, k + (SH::TILE >> 4) + k_step(ks), ids, true);
                    }
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks) tc_mma_ts(leader, d, tm + SH::QH + 8 * ks, k + k_step(ks), ids, true);
                    tc_commit(leader, &s_full[sl]);
                    tc_commit(leader, &k_empty[st]);
                    if (++st == NB) st = 0;
                    if (++sl == NS) sl = 0, sl_ph ^= 1;
                    if (++kt == RING) kt = 0, kt_ph ^= 1;
                }
            } else {
                // V: 64 values COLS bytes apart, 16 positions 2,048 on
                const uint64_t vd = tile_desc(smem_u32(tiles) + SH::HALF, SH::COLS, 1024);
                for (int t = 0; ok && t < n_tiles; ++t) {
                    ok = t ? wait_three(&p_full[sl], sl_ph, &v_full[st], ph, o_free, t - 1) : wait_both(&p_full[sl], sl_ph, &v_full[st], ph);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t v = vd + (uint32_t)(st * (2 * SH::HALF >> 4));
                    const uint32_t w = tm + SH::S0 + sl * T, d = tm + SH::O0;
#pragma unroll
                    for (int ks = 0; ks < T / 16; ++ks) tc_mma_ts(leader, d, w + 8 + 16 * ks, v + (2048 * ks >> 4), ido, ks > 0);
                    if (SH::TERMS == 2) {
#pragma unroll
                        for (int ks = 0; ks < T / 16; ++ks)
                            tc_mma_ts(leader, d, w + 16 * ks, v + ((SH::TILE + 2048 * ks) >> 4), ido, true);
                    }
#pragma unroll
                    for (int ks = 0; ks < T / 16; ++ks) tc_mma_ts(leader, d, w + 16 * ks, v + (2048 * ks >> 4), ido, true);
                    tc_commit(leader, o_full);
                    tc_commit(leader, &v_empty[st]);
                    tc_commit(leader, &w_empty[sl]);
                    if (++st == NB) st = 0, ph ^= 1;
                    if (++sl == NS) sl = 0, sl_ph ^= 1;
                }
            }
            if (!ok) *flag = 1;
            // whatever was issued ends before tensor memory is given back
            tc_commit(leader, done);
            __syncwarp();
            if (warp == kMmaWarp) mbar_wait_at(done, 0u, p.b.err, nullptr);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// The splits of a row, a warp each: out = Σ 2^(m_s - m)·O_s / Σ 2^(m_s - m)·l_s, in split order.
template <int HD>
__global__ void __launch_bounds__(256) tree_merge_kernel(const __grid_constant__ MmaParams mp) {
    const TreeParams& p = mp.t;
    constexpr int PER = HD / 32;
    const int lane = threadIdx.x & 31, seq = blockIdx.y;
    int r0, n;
    kv_nodes(p.b, p.n_rows, seq, r0, n);
    const int len = kv_len(p.kv, p.b, seq, n);
    const int i = blockIdx.x * 8 + (threadIdx.x >> 5), r = i / p.H * p.G + i % p.H % p.G, kvh = i % p.H / p.G;
    pdl_wait();
    if (len < 0 || i >= n * p.H) return;
    const int2 plan = mp.plan[seq];
    const int item = (r / kMmaRows) * p.kv.kv_heads + kvh;
    if (plan.y <= 1 || plan.x < 0 || plan.x + (long long)(item + 1) * plan.y > mp.slots) return;
    const int row = r0 + i / p.H, head = i % p.H;
    const long long at = (plan.x + (long long)item * plan.y) * kMmaRows + r % kMmaRows;
    const float* o = mp.part + at * HD + lane * PER;
    const float* ml = mp.part + (long long)mp.slots * kMmaRows * HD + at * 2;
    float top = -INFINITY;
    for (int s = lane; s < plan.y; s += 32) top = fmaxf(top, ml[s * (2 * kMmaRows)]);
    top = warp_max(top);
    float acc[PER], sum = 0.f;
#pragma unroll
    for (int d = 0; d < PER; ++d) acc[d] = 0.f;
#pragma unroll 4
    for (int s = 0; s < plan.y; ++s) {
        const float2 x = *reinterpret_cast<const float2*>(ml + s * (2 * kMmaRows));
        if (x.y == 0.f && x.x == -INFINITY) continue;  // a split that the row sees nothing of
        const float c = fmaxf(ex2(x.x - top), least());
        sum = fmaf(c, x.y, sum);
        float v[PER];
        if (PER == 4) {
            const float4 f = *reinterpret_cast<const float4*>(o + (long long)s * kMmaRows * HD);
            v[0] = f.x, v[1] = f.y, v[2 % PER] = f.z, v[3 % PER] = f.w;
        } else {
            const float2 f = *reinterpret_cast<const float2*>(o + (long long)s * kMmaRows * HD);
            v[0] = f.x, v[1] = f.y;
        }
#pragma unroll
        for (int d = 0; d < PER; ++d) acc[d] = fmaf(c, v[d], acc[d]);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    float* out = p.out + (long long)row * p.os + (long long)head * HD + lane * PER;
#pragma unroll
    for (int d = 0; d < PER; ++d) out[d] = acc[d] * inv;
}

// ------------------------------------------------------------ small calls
//
// Few rows over few positions, where the kernel above spends its time on
// setting up: a cluster of blocks per (16 query rows, kv head, sequence) takes
// tiles of 32 positions in turn, K and V in shared memory as f32 with the next
// tile's on their way, products on the f32 units.  A warp has two rows: their
// scores, a position a lane, and their softmax; in P·V a thread has a dimension
// and some rows.  In the end the blocks read one another's sums.  What bounds
// it is the latency of its steps: lengths, pages, K and V, three passes over
// shared memory.

constexpr int kSmallThreads = 256;
constexpr int kSmallRows = 16;
constexpr int kSmallTile = 32;

template <int HD>
struct SmallShape {
    static constexpr int T = kSmallTile;
    static constexpr int KS = HD + 4, PS = kSmallRows + 4;  // floats from row to row: K's, the weights' of a position
    static constexpr int DR = kSmallRows * HD / kSmallThreads;  // rows of a thread in P·V
    static constexpr int BYTES = (T * (KS + HD + PS) + 2 * kSmallRows * HD + 3 * kSmallRows) * 4;
};

// 16 bytes of the cache as f32.
template <int TYPE>
__device__ __forceinline__ void widen(const uint4& x, float* f) {
    const uint32_t e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (TYPE == AF_KV_F32) {
            f[i] = __uint_as_float(e[i]);
        } else if (TYPE == AF_KV_F16) {
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&e[i]));
            f[2 * i] = y.x, f[2 * i + 1] = y.y;
        } else {
            f[2 * i] = __uint_as_float(e[i] << 16), f[2 * i + 1] = __uint_as_float(e[i] & 0xffff0000u);
        }
    }
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float cluster_ld(const float* mine, int rank) {
    uint32_t a;
    float f;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(a) : "memory");
    return f;
}

template <int TYPE, int HD>
__global__ void __launch_bounds__(kSmallThreads, 2) tree_small_kernel(TreeParams p, int blocks) {  // of a cluster
    using SH = SmallShape<HD>;
    using E = KvElem<TYPE>;
    constexpr int T = SH::T, KS = SH::KS, PS = SH::PS, DR = SH::DR;
    extern __shared__ __align__(1024) uint8_t sm[];  // declared alike everywhere: the strictest alignment is tree_mma_kernel's
    float* sk = reinterpret_cast<float*>(sm);        // [T][KS]
    float* sv = sk + T * KS;                         // [T][HD]
    float* sw = sv + T * HD;                         // [T][PS] weights
    float* sq = sw + T * PS;                         // [16][HD] queries, times the scale
    float* so = sq + kSmallRows * HD;                // [16][HD] this block's sums of weighted V
    float* s_m = so + kSmallRows * HD;               // [16] its largest score
    float* s_l = s_m + kSmallRows;                   // [16] its sum of weights
    float* s_c = s_l + kSmallRows;                   // [16] the tile's correction
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, seq = blockIdx.y;
    const int rank = blocks > 1 ? blockIdx.x % blocks : 0, kvh = blocks > 1 ? blockIdx.x / blocks : blockIdx.x;
    int r0, n;
    kv_nodes(p.b, p.n_rows, seq, r0, n);
    const int len = kv_len(p.kv, p.b, seq, n);
    const int x0 = blockIdx.z * kSmallRows, rows = min(kSmallRows, n * p.G - x0);
    if (len < 0 || rows <= 0) return;  // the whole cluster
    const int end = p.mask ? len + n : len + node_of(p, x0 + rows - 1) + 1;
    // K and V of a tile, 16 bytes a load
    constexpr int VPL = 16 / (int)sizeof(typename E::T), LPR = HD / VPL, N = T * LPR / kSmallThreads;
    uint4 k[N], v[N];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = tid + j * kSmallThreads, pos = t0 + i / LPR;
            k[j] = v[j] = make_uint4(0u, 0u, 0u, 0u);
            if (pos >= end) continue;
            const long long at = kv_row(p.kv, p.b, seq, pos);
            if (at < 0) {
                set_err_at(p.b.err, kErrBadArgs);
                continue;
            }
            const long long from = p.layer * p.kv.layer_bytes + at + (kvh * HD + i % LPR * VPL) * (int)sizeof(typename E::T);
            k[j] = __ldg(reinterpret_cast<const uint4*>(p.kv.k + from));
            v[j] = __ldg(reinterpret_cast<const uint4*>(p.kv.v + from));
        }
    };
    fetch(rank * T);
    for (int i = tid; i < kSmallRows * HD; i += kSmallThreads) {
        float q = 0.f;
        if (i / HD < rows) {
            const int x = x0 + i / HD, node = node_of(p, x);
            q = p.q[(long long)(r0 + node) * p.qs + (kvh * p.G + x - node * p.G) * HD + i % HD] * p.scale;
        }
        sq[i] = q;
    }
    const int r2 = 2 * warp;  // the warp's rows
    int row[2], node[2];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        node[i] = r2 + i < rows ? node_of(p, x0 + r2 + i) : -1;
        row[i] = r0 + node[i];
    }
    const int d = tid % HD, dr = tid / HD * DR;  // of P·V: a dimension, the first row
    float acc[DR];
#pragma unroll
    for (int i = 0; i < DR; ++i) acc[i] = 0.f;
    for (int t0 = rank * T; t0 < end; t0 += blocks * T) {
        bool odd = false;  // V with something that is not finite
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = tid + j * kSmallThreads, at = i / LPR, col = i % LPR * VPL;
            float f[VPL], g[VPL];
            widen<TYPE>(k[j], f);
            widen<TYPE>(v[j], g);
#pragma unroll
            for (int c = 0; c < VPL; c += 4) {
                *reinterpret_cast<float4*>(sk + at * KS + col + c) = make_float4(f[c], f[c + 1], f[c + 2], f[c + 3]);
                *reinterpret_cast<float4*>(sv + at * HD + col + c) = make_float4(g[c], g[c + 1], g[c + 2], g[c + 3]);
                const float z = fmaf(g[c], 0.f, fmaf(g[c + 1], 0.f, fmaf(g[c + 2], 0.f, g[c + 3] * 0.f)));
                odd = odd || z != 0.f;  // NaN
            }
        }
        odd = __syncthreads_or(odd);
        if (t0 + blocks * T < end) fetch(t0 + blocks * T);
        if (r2 < rows) {
            float s[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll 8
            for (int c = 0; c < HD; c += 4) {
                const float4 x = *reinterpret_cast<const float4*>(sk + lane * KS + c);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 q = *reinterpret_cast<const float4*>(sq + (r2 + i) * HD + c);
                    s[i][0] = fmaf(q.y, x.y, fmaf(q.x, x.x, s[i][0]));
                    s[i][1] = fmaf(q.w, x.w, fmaf(q.z, x.z, s[i][1]));
                }
            }
            float w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = t0 + lane - len;
                const bool sees = node[i] >= 0 && t0 + lane < end && (j < 0 || tree_sees(p, row[i], node[i], j));
                const float x = sees ? s[i][0] + s[i][1] : -INFINITY;
                const float mn = fmaxf(m[i], warp_max(x)), ms = mn == -INFINITY ? 0.f : mn;
                w[i] = !sees ? 0.f : isnan(x) ? x : fmaxf(ex2(x - ms), least());  // NaN stays
                const float corr = fmaxf(ex2(m[i] - ms), least());
                l[i] = fmaf(l[i], corr, warp_sum(w[i]));
                m[i] = mn;
                if (lane == 0) s_c[r2 + i] = corr;
            }
            *reinterpret_cast<float2*>(sw + lane * PS + r2) = make_float2(w[0], w[1]);
        }
        __syncthreads();
        if (dr < rows) {
#pragma unroll
            for (int i = 0; i < DR; ++i) acc[i] *= dr + i < rows ? s_c[dr + i] : 0.f;
            const int last = min(T, end - t0);
            auto add = [&](bool guard) {
#pragma unroll 8
                for (int j = 0; j < last; ++j) {
                    const float y = sv[j * HD + d];
#pragma unroll
                    for (int i = 0; i < DR; i += 4) {
                        const float4 w = *reinterpret_cast<const float4*>(sw + j * PS + dr + i);
                        if (!guard || w.x != 0.f) acc[i] = fmaf(w.x, y, acc[i]);
                        if (!guard || w.y != 0.f) acc[i + 1] = fmaf(w.y, y, acc[i + 1]);
                        if (!guard || w.z != 0.f) acc[i + 2] = fmaf(w.z, y, acc[i + 2]);
                        if (!guard || w.w != 0.f) acc[i + 3] = fmaf(w.w, y, acc[i + 3]);
                    }
                }
            };
            if (odd) add(true);
            else add(false);
        }
        __syncthreads();
    }
    if (lane < 2 && r2 + lane < rows) {
        s_m[r2 + lane] = lane ? m[1] : m[0];
        s_l[r2 + lane] = lane ? l[1] : l[0];
    }
#pragma unroll
    for (int i = 0; i < DR; ++i) so[(dr + i) * HD + d] = acc[i];
    if (blocks > 1) cluster_sync();
    else __syncthreads();
    for (int i = rank * kSmallThreads + tid; i < rows * HD; i += blocks * kSmallThreads) {
        const int r = i / HD, c = i % HD, x = x0 + r, nd = node_of(p, x);
        float top = s_m[r], sum = s_l[r], o = so[i];
        if (blocks > 1) {  // Σ 2^(m_b - m)·O_b / Σ 2^(m_b - m)·l_b, in the blocks' order
            top = -INFINITY;
            for (int b = 0; b < blocks; ++b) top = fmaxf(top, cluster_ld(s_m + r, b));
            sum = o = 0.f;
            for (int b = 0; b < blocks; ++b) {
                const float lb = cluster_ld(s_l + r, b), mb = cluster_ld(s_m + r, b);
                if (mb == -INFINITY && lb == 0.f) continue;  // a block that the row sees nothing of
                const float f = fmaxf(ex2(mb - top), least());
                sum = fmaf(f, lb, sum);
                o = fmaf(f, cluster_ld(so + i, b), o);
            }
        }
        p.out[(long long)(r0 + nd) * p.os + (kvh * p.G + x - nd * p.G) * HD + c] = sum == 0.f ? 0.f : o / sum;
    }
    if (blocks > 1) cluster_sync();  // a block's sums stay until all have read them
}

// ------------------------------------------------------------------ launch

struct TreePlan {
    bool mma, small;
    long long max_len;
    int nodes;          // of a sequence, at most: max_nodes may be far above the call's rows
    int blocks, slots;  // slots 0: nothing is split, no second launch
    size_t ws;
};

constexpr int kSmallFill = 2 * kTreeSms;  // blocks up to which a small call's items are split over clusters

// Which kernel: the smaller of two estimates in µs, from the sizes alone.  A
// small call's tile costs its block about 1.2 µs (head_dim 64) or 2.2 µs (128;
// 1.2 where three blocks share an SM), and up to 8 blocks share an item; the
// tensor-core kernel costs 10 to 12 µs a wave of 148 items and its tiles.
// Measured, small / tensor-core kernel, f32, 32/4 heads of 64: one row of 137
// and 1,000 positions 5.9 / 11.9 and 11.6 / 14.7 µs; 16 sequences of 250 8.1 /
// 15.3, of 1,000 20.4 / 19.8; 16 rows each of 250 40 / 18.  16 sequences with 32
// kv heads of 128, a row each of 137: 19.7 / 45.5, of 1,000 95 / 98.
bool small_call(const af_attention_tree_args& a, int nodes, long long max_len) {
    const bool f32 = a.kv.type == AF_KV_F32, narrow = a.kv.head_dim == 64;
    const long long rows = (long long)nodes * (a.n_heads / a.kv.n_kv_heads), heads = (long long)a.batch.n_seq * a.kv.n_kv_heads;
    const long long items = (rows + kSmallRows - 1) / kSmallRows * heads, tiles = (max_len + kSmallTile - 1) / kSmallTile;
    const double each = narrow || items >= kSmallFill ? 1.2 : 2.2;
    const double small = 5. + std::max(each * (double)items * (double)tiles / kTreeSms, (narrow ? 1.6 : 2.4) * (double)((tiles + 7) / 8));
    const double work = (double)((rows + kMmaRows - 1) / kMmaRows * heads) / kTreeSms;
    const double mma = (f32 ? 12. : 10.) * std::max(1., work) + work * (double)((max_len + 63) / 64) * (narrow ? .5 : 1.) * (f32 ? 1. : .5);
    return rows <= 65535ll * kSmallRows && a.batch.n_seq <= 65535 && small < mma;
}

TreePlan tree_plan(const af_attention_tree_args& a) {
    TreePlan pl = {};
    const int hd = a.kv.head_dim, G = a.n_heads / a.kv.n_kv_heads;
    pl.mma = hd == 64 || hd == 128;
    if (!pl.mma) return pl;
    const long long cap = (long long)a.batch.max_blocks * a.kv.page_size;
    const long long max_len = a.max_len > 0 ? std::min((long long)a.max_len, cap) : cap;
    pl.max_len = max_len;
    pl.nodes = std::max(1, std::min(a.batch.max_nodes, a.n_rows));
    pl.small = small_call(a, pl.nodes, max_len);
    // the workspace does not ask which kernel: it grows with every size, so one for the largest call serves smaller
    // ones, which may go to the other kernel
    const int T = tree_tile(a.kv.type);
    const long long tiles = (max_len + T - 1) / T, most = (tiles + kTreeMinTiles - 1) / kTreeMinTiles;
    auto blocks = [&](long long items) {
        const long long split = items <= kTreeItems ? (items + kTreeSms - 1) / kTreeSms * kTreeSms : items + 2 * kTreeItems;
        return std::min({split, items * std::max(1ll, most), (long long)INT_MAX});
    };
    const long long n_seq = a.batch.n_seq, kv = a.kv.n_kv_heads;
    auto items = [&](long long nodes) { return (nodes * G + kMmaRows - 1) / kMmaRows * n_seq; };  // of a kv head
    // the launch also knows the call's rows, of which a sequence leaves one item partly filled
    pl.blocks = (int)blocks(std::min(items(pl.nodes), (long long)a.n_rows * G / kMmaRows + n_seq) * kv);
    if (most > 1) pl.slots = (int)std::min(blocks(items(a.batch.max_nodes) * kv), 2ll * kTreeItems);
    if (pl.slots) pl.ws = (size_t)pl.slots * kMmaRows * (hd + 2) * sizeof(float) + (size_t)a.batch.n_seq * sizeof(int2);
    return pl;
}

// The driver's cuTensorMapEncodeTiled, through the runtime (the library does not link libcuda).
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess) f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}

// Rows of a layer's pool as boxes of up to a tile's or a page's rows: f32 rows whole, others 64 values swizzled.
bool tree_map(CUtensorMap* map, const TreeParams& p, int type, uint8_t* pool, int box_rows) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    const bool f32 = type == AF_KV_F32;
    const int size = kv_type_bytes(type);
    const cuuint64_t dims[3] = {(cuuint64_t)p.kv.hd, (cuuint64_t)p.kv.kv_heads, (cuuint64_t)p.kv.n_pages << p.kv.ps_shift};
    const cuuint64_t strides[2] = {(cuuint64_t)p.kv.hd * size, (cuuint64_t)p.kv.row_bytes};
    const cuuint32_t box[3] = {(cuuint32_t)(f32 ? p.kv.hd : 64), 1u, (cuuint32_t)box_rows}, step[3] = {1, 1, 1};
    return encode(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3,
                  pool + (size_t)p.layer * p.kv.layer_bytes, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  f32 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TYPE, int HD>
cudaError_t mma_launch(const MmaParams& mp, int n_seq, int nodes, cudaStream_t st) {
    constexpr int smem = MmaShape<TYPE, HD>::BYTES;
    AF_CUDA_TRY(cudaFuncSetAttribute(tree_mma_kernel<TYPE, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    tree_mma_kernel<TYPE, HD><<<mp.blocks, kMmaThreads, smem, st>>>(mp);
    AF_CUDA_TRY(cudaGetLastError());
    if (!mp.slots) return cudaSuccess;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((long long)nodes * mp.t.H + 7) / 8), n_seq);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, tree_merge_kernel<HD>, mp);
}

template <int TYPE, int HD>
cudaError_t small_launch(const TreeParams& p, int nodes, long long max_len, cudaStream_t st) {
    constexpr int smem = SmallShape<HD>::BYTES;
    AF_CUDA_TRY(cudaFuncSetAttribute(tree_small_kernel<TYPE, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    // as many blocks a cluster (a power of two up to 8) as keep the SMs at most twice filled
    const long long tiles = (nodes * p.G + kSmallRows - 1) / kSmallRows, items = tiles * p.b.n_seq * p.kv.kv_heads;
    int blocks = 1;
    while (blocks < 8 && 2 * blocks * items <= kSmallFill && blocks * kSmallTile < max_len) blocks *= 2;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)blocks, 1, 1};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.kv.kv_heads * blocks, p.b.n_seq, (unsigned)tiles);
    cfg.blockDim = dim3(kSmallThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, tree_small_kernel<TYPE, HD>, p, blocks);
}

template <int TYPE>
cudaError_t tree_launch(const TreeParams& p, const TreePlan& pl, void* ws, cudaStream_t st) {
    if (pl.small) return p.kv.hd == 64 ? small_launch<TYPE, 64>(p, pl.nodes, pl.max_len, st)
                                       : small_launch<TYPE, 128>(p, pl.nodes, pl.max_len, st);
    if (pl.mma) {
        MmaParams mp = {};
        mp.t = p;
        mp.blocks = pl.blocks;
        mp.slots = pl.slots;
        mp.part = static_cast<float*>(ws);
        mp.box_rows = std::min(1 << p.kv.ps_shift, tree_tile(TYPE) / (TYPE == AF_KV_F32 ? 2 : 1));
        if (!tree_map(&mp.k_map, p, TYPE, p.kv.k, mp.box_rows) || !tree_map(&mp.v_map, p, TYPE, p.kv.v, mp.box_rows)) {
            set_last_error("af_attention_tree_f32: the cache cannot be described to the copy engine");
            return cudaErrorInvalidValue;
        }
        if (pl.slots) mp.plan = reinterpret_cast<int2*>(mp.part + (size_t)pl.slots * kMmaRows * (p.kv.hd + 2));
        return p.kv.hd == 64 ? mma_launch<TYPE, 64>(mp, p.b.n_seq, pl.nodes, st) : mma_launch<TYPE, 128>(mp, p.b.n_seq, pl.nodes, st);
    }
    tree_row_kernel<TYPE><<<dim3(p.n_rows, p.H), kTreeThreads, 0, st>>>(p);
    return cudaGetLastError();
}

std::string tree_wrong(const af_attention_tree_args& a) {
    std::string why = kv_cache_wrong(a.kv);
    if (why.empty()) why = kv_batch_wrong(a.batch, a.kv, true);
    if (!why.empty()) return why;
    if (a.layer < 0 || a.layer >= a.kv.n_layers) return "layer outside the cache";
    if (a.n_rows < 0 || a.n_heads <= 0 || a.n_heads > 65535 || a.n_heads % a.kv.n_kv_heads)
        return "need n_rows >= 0 and n_heads a multiple of n_kv_heads";
    if (a.max_len < 0) return "max_len must not be negative";
    const long long G = a.n_heads / a.kv.n_kv_heads;
    if (a.batch.max_nodes * G > (1ll << 31) / G) return "max_nodes times the square of n_heads / n_kv_heads must be at most 2^31";
    const bool mma = a.kv.head_dim == 64 || a.kv.head_dim == 128;  // its merge numbers rows and heads with 32 bits
    if (mma && (long long)std::min(a.batch.max_nodes, a.n_rows) * a.n_heads > INT_MAX - 8)
        return "n_rows times n_heads must be below 2^31";
    if (a.mask && (a.mask_words <= 0 || (long long)a.mask_words * 64 < a.batch.max_nodes))
        return "mask_words must cover max_nodes";
    if (mma && std::min(a.batch.max_nodes, a.n_rows) > kMmaMaxNodes) return "a sequence has at most 1,048,448 nodes";
    const long long qd = (long long)a.n_heads * a.kv.head_dim;
    if ((a.q_stride && a.q_stride < qd) || (a.out_stride && a.out_stride < qd)) return "a row stride is shorter than a row";
    return "";
}

cudaError_t refuse(const std::string& why) {
    set_last_error("af_attention_tree_f32: " + why);
    return cudaErrorInvalidValue;
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" size_t af_attention_tree_f32_workspace(const af_attention_tree_args* a) {
    return a && tree_wrong(*a).empty() ? tree_plan(*a).ws : 0;
}

extern "C" cudaError_t af_attention_tree_f32(const af_attention_tree_args* a, cudaStream_t stream) {
    if (!a) return refuse("null arguments");
    const std::string why = tree_wrong(*a);
    if (!why.empty()) return refuse(why);
    if (a->n_rows == 0 || a->batch.n_seq == 0) return cudaSuccess;
    if (!a->q || !a->out) return refuse("null q or out");
    const TreePlan pl = tree_plan(*a);
    if (!pl.small && pl.ws && (!a->ws || a->ws_bytes < pl.ws || (reinterpret_cast<uintptr_t>(a->ws) & 15)))
        return refuse("ws must hold af_attention_tree_f32_workspace bytes, 16-byte aligned");
    const long long qd = (long long)a->n_heads * a->kv.head_dim;
    TreeParams p = {};
    p.kv = kv_view(a->kv);
    int* err = nullptr;
    AF_CUDA_TRY(device_error_word(&err));
    p.b = kv_batch(a->batch, err);
    p.layer = a->layer;
    p.n_rows = a->n_rows;
    p.H = a->n_heads;
    p.G = a->n_heads / a->kv.n_kv_heads;
    p.G_inv = (uint32_t)(((1ull << 32) + p.G - 1) / p.G);
    p.q = a->q;
    p.out = a->out;
    p.qs = a->q_stride ? a->q_stride : qd;
    p.os = a->out_stride ? a->out_stride : qd;
    p.mask = reinterpret_cast<const unsigned long long*>(a->mask);
    p.mask_words = a->mask_words;
    p.scale = (a->scale != 0.f ? a->scale : 1.f / std::sqrt((float)a->kv.head_dim)) * 1.4426950408889634f;
    switch (a->kv.type) {
        case AF_KV_F32: return tree_launch<AF_KV_F32>(p, pl, a->ws, stream);
        case AF_KV_F16: return tree_launch<AF_KV_F16>(p, pl, a->ws, stream);
        default: return tree_launch<AF_KV_BF16>(p, pl, a->ws, stream);
    }
}
