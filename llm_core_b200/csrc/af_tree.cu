// af_tree.cu — attention of drafted tokens over a paged cache
// (af_attention_tree_f32): the nodes of every sequence see its cached
// positions and, by a bit mask, one another.
#define AF_WHOLE_PROGRAM  // the register split below (setmaxnreg) holds only without separate compilation
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "af_kvpages.cuh"
#include "af_ops.cuh"

namespace af {
namespace {

struct TreeParams {
    KvView kv;
    KvBatch b;
    int layer, n_rows, H, G;
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

// One block per row and head: its warps take the positions in turn, a lane
// the dimensions lane, lane + 32, ...; each warp keeps a running maximum, sum
// and output, merged at the end.
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
        const long long at = kv_row(p.kv, p.b, seq, pos);
        if (at < 0) {
            set_err_at(p.b.err, kErrBadArgs);
            continue;
        }
        const auto* kr = reinterpret_cast<const typename E::T*>(p.kv.k + head + at);
        const auto* vr = reinterpret_cast<const typename E::T*>(p.kv.v + head + at);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < hd) s = fmaf(qv[i], E::load(kr[lane + 32 * i]), s);
        s = warp_sum(s);
        const float mn = fmaxf(m, s), c = mn == -INFINITY ? 1.f : exp2f(m - mn);
        const float w = s == -INFINITY ? 0.f : exp2f(s - mn);
        m = mn;
        l = l * c + w;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < hd) o[i] = fmaf(w, E::load(vr[lane + 32 * i]), o[i] * c);
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
        c[w] = s_m[w] == -INFINITY && s_l[w] == 0.f ? 0.f : exp2f(s_m[w] - top);
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
// largest of a row, or of the rows of one 512-byte load, in [2^14, 2^15)) is
// split as hi + lo, both f16: 22 bits, and what is lost below is 2^-39 of that
// largest value.  x·y = hi·hi + hi·lo + lo·hi to 2^-22.  A cache in f16 needs
// no scale and no lo, one in bf16 a scale and no lo (8 bits in 11).  The
// powers of two are undone exactly: K's in the score, V's in the exponent of
// the weight, 2^(s_j - a_j), whose sum Σ 2^(s_j - a_j)·2^a_j is the softmax's.
// Weights carry a factor 2^14, so that those as small as 2^-38 of the largest
// keep f16's spacing.
//
// The tensor cores truncate when they add to an accumulator (measured: sums
// of 400 and 4000 positive products came out 3.9e-5 and 4.0e-4 low, 1e-7 an
// instruction), so no accumulator lives longer than a tile: small products
// first, then the hi·hi ones, and the softmax warps add each tile's P·V to
// sums in registers, which round to nearest.
//
// Warps 0-3 (one query row a thread) run the softmax; warps 4-11 load K and V
// rows, page by page, straight into registers (16 loads of 16 bytes a lane
// in flight, 64 KB an SM), split them and store them in the layout that
// tcgen05 reads; warp 12 issues the products.  registers: 232 / 120 / 40 a
// thread (setmaxnreg; 232·128 + 120·256 + 40·128 = 65,536, the launch's 128·512).
//
// Shared-memory tiles: 8-row × 16-byte core matrices without swizzle, 144
// bytes apart along the row (16 bytes of padding: the stores of a warp then
// fall into all banks) — K-major for K, and the same tile MN-major for V.

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// d (+)= A · B: A in tensor memory, B by descriptor.
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}

__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// No-swizzle descriptor: strides in bytes, version 1.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46);
}

// 32 consecutive columns of this thread's lane.
__device__ __forceinline__ void tc_ld32(uint32_t t, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(t));
}
__device__ __forceinline__ void tc_st16(uint32_t t, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(t)
        : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// a, b -> packed f16 hi and, of what is left, lo.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The power of two for values whose largest has these bits: max·2^a in
// [2^14, 2^15), a within [-113, top]; 0 for an infinity or NaN.
__device__ __forceinline__ int scale_of(uint32_t max_bits, int top) {
    if (max_bits >= 0x7f800000u) return 0;
    return min(top, 14 - ((int)(max_bits >> 23) - 127));
}
__device__ __forceinline__ float pow2(int a) { return __int_as_float((a + 127) << 23); }

constexpr int kMmaThreads = 512;
constexpr int kMmaRows = 128;
constexpr int kMmaBadWords = 512;  // tiles of a split whose V holds something non-finite, a bit each

template <int TYPE, int HD>
struct MmaShape {
    static constexpr int SIZE = TYPE == AF_KV_F32 ? 4 : 2;
    static constexpr int T = HD == 128 ? 64 : 128;      // positions of a tile
    static constexpr int TERMS = TYPE == AF_KV_F32 ? 2 : 1;  // hi, lo of K and V
    static constexpr int CS = 144;                      // between 16-byte columns of a tile
    static constexpr int RS = HD / 8 * CS;              // between groups of 8 rows
    static constexpr int TILE = T / 8 * RS;             // 18,432
    static constexpr int STAGE = 2 * TERMS * TILE;      // K hi, K lo, V hi, V lo
    static constexpr int NB = TYPE == AF_KV_F32 ? 3 : HD == 128 ? 6 : 5;
    static constexpr int RPW = T / 8;                   // rows of a loading warp in a tile
    static constexpr int LPR = HD * SIZE / 16;          // lanes of a row
    static constexpr int RPC = 32 / LPR;                // rows of one load
    static constexpr int NCK = RPW / RPC;               // loads of a lane for K (and for V)
    static constexpr int RING = 16 / (2 * NCK);         // tiles in flight in registers
    // tensor memory columns
    static constexpr int QH = 0, QL = HD / 2, S0 = HD, O0 = HD + 2 * T;
    static_assert(O0 + 2 * HD <= 512, "tensor memory");
    // shared memory
    static constexpr int BAD = 256;                     // behind the mbarriers: kMmaBadWords words
    static constexpr int SCALE = BAD + kMmaBadWords * 4;  // [NB][3][T] floats
    static constexpr int TILES = (SCALE + NB * 3 * T * 4 + 127) / 128 * 128;
    static constexpr int BYTES = TILES + NB * STAGE;
    static_assert(BYTES <= 227 * 1024, "shared memory");
};

struct MmaParams {
    TreeParams t;
    int nsplit, row_tiles;
    float* part;  // [nsplit][n_rows][H][HD], then [nsplit][n_rows][H][2]: top, sum (nsplit > 1)
};

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

template <int TYPE, int HD>
__global__ void __launch_bounds__(kMmaThreads, 1) tree_mma_kernel(MmaParams mp) {
    using SH = MmaShape<TYPE, HD>;
    using E = KvElem<TYPE>;
    constexpr int T = SH::T, NB = SH::NB, RING = SH::RING, NCK = SH::NCK;
    extern __shared__ __align__(1024) uint8_t sm[];
    const TreeParams& p = mp.t;
    uint64_t* full = reinterpret_cast<uint64_t*>(sm);  // [NB] 8 loading warps
    uint64_t* empty = full + NB;                       // [NB] P·V done
    uint64_t* s_full = empty + NB;                     // [2] scores done
    uint64_t* p_full = s_full + 2;                     // [2] 4 softmax warps: weights written
    uint64_t* o_full = p_full + 2;                     // [2] P·V done
    uint64_t* o_free = o_full + 2;                     // [2] 4 softmax warps: P·V taken
    uint64_t* q_full = o_free + 2;                     // 4 softmax warps: queries written
    uint64_t* done = q_full + 1;                       // every product done
    uint32_t* tslot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* flag = reinterpret_cast<volatile int*>(tslot + 1);
    uint32_t* bad = reinterpret_cast<uint32_t*>(sm + SH::BAD);
    float* scales = reinterpret_cast<float*>(sm + SH::SCALE);
    uint8_t* tiles = sm + SH::TILES;
    auto wait = [&](uint64_t* bar, uint32_t parity, const volatile int* abort) -> bool {
        return mbar_wait_at(bar, parity, p.b.err, abort);
    };
    // the same for a whole warp, which stays together
    auto wait_warp = [&](uint64_t* bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, mbar_wait_at(bar, parity, p.b.err, flag));
    };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x % mp.nsplit, rt = blockIdx.x / mp.nsplit, kvh = blockIdx.y, seq = blockIdx.z;

    // the block's rows and tiles (the same in every thread)
    int r0, n;
    kv_nodes(p.b, p.n_rows, seq, r0, n);
    const int len = kv_len(p.kv, p.b, seq, n);
    const int row_lo = rt * kMmaRows, row_hi = min(row_lo + kMmaRows, n * p.G);
    if (len < 0 || row_lo >= row_hi) return;
    const int end = p.mask ? len + n : len + (row_hi - 1) / p.G + 1;  // positions that some row may see
    const int nt_all = (end + T - 1) / T;
    const int t0 = (int)((long long)nt_all * split / mp.nsplit), t1 = (int)((long long)nt_all * (split + 1) / mp.nsplit);
    const int nt = t1 - t0;
    int bs = 0;  // tiles of a bit of bad[]: 1 << bs
    while (nt > (kMmaBadWords * 32) << bs) ++bs;
    pdl_launch_dependents();

    if (tid == 0) {
        for (int i = 0; i < NB; ++i) {
            mbar_init(&full[i], 8);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
            mbar_init(&o_free[i], 4);
        }
        mbar_init(q_full, 4);
        mbar_init(done, 1);
        *flag = 0;
        fence_mbar_init();
    }
    for (int i = tid; i < kMmaBadWords; i += kMmaThreads) bad[i] = 0;
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tslot;

    if (warp < 4) {
        // ------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const int r = row_lo + tid;
        const bool live = r < row_hi;
        const int node = live ? r / p.G : 0, row = r0 + node, head = kvh * p.G + (live ? r % p.G : 0);
        float rs;  // what a raw score is times, but for K's power of two
        {
            const float* q = p.q + (long long)row * p.qs + (long long)head * HD;
            float x[HD];
            uint32_t mx = 0;
            if ((reinterpret_cast<uintptr_t>(q) & 15) == 0) {
#pragma unroll
                for (int i = 0; i < HD; i += 4) {
                    const float4 f = live ? __ldg(reinterpret_cast<const float4*>(q + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[i] = f.x, x[i + 1] = f.y, x[i + 2] = f.z, x[i + 3] = f.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < HD; ++i) x[i] = live ? q[i] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < HD; ++i) mx = max(mx, __float_as_uint(x[i]) & 0x7fffffffu);
            const int a = scale_of(mx, 100);
            const float s = pow2(a);
            rs = p.scale * pow2(-a);
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) split2(x[32 * c + 2 * i] * s, x[32 * c + 2 * i + 1] * s, hi[i], lo[i]);
                tc_st16(tmem + lanes + SH::QH + 16 * c, hi);
                tc_st16(tmem + lanes + SH::QL + 16 * c, lo);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        float acc[HD];
#pragma unroll
        for (int i = 0; i < HD; ++i) acc[i] = 0.f;
        float m = -INFINITY, l = 0.f, corr = 0.f;  // corr: of the sums, for the tile whose P·V is due
        bool ok = true;
        auto take = [&](int t) -> bool {           // acc = acc·corr + (P·V)(t)
            if (!wait_warp(&o_full[t & 1], (uint32_t)(t >> 1) & 1u)) return false;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                tc_ld32(tmem + lanes + SH::O0 + (t & 1) * HD + 32 * c, o);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[32 * c + i] = fmaf(acc[32 * c + i], corr, __uint_as_float(o[i]));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free[t & 1]);
            return true;
        };
        for (int t = 0; t < nt; ++t) {
            const int st = t % NB;
            if (!wait_warp(&full[st], (uint32_t)(t / NB) & 1u) || !wait_warp(&s_full[t & 1], (uint32_t)(t >> 1) & 1u)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t sb = tmem + lanes + SH::S0 + (t & 1) * T;
            float v[T];
#pragma unroll
            for (int c = 0; c < T / 32; ++c) {
                uint32_t x[32];
                tc_ld32(sb + 32 * c, x);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) v[32 * c + i] = __uint_as_float(x[i]);
            }
            const float4* kc = reinterpret_cast<const float4*>(scales + (st * 3 + 0) * T);  // 2^-a of K
            const float4* vf = reinterpret_cast<const float4*>(scales + (st * 3 + 1) * T);  // -a of V
            const float4* vg = reinterpret_cast<const float4*>(scales + (st * 3 + 2) * T);  // 2^a of V
            if (TYPE == AF_KV_F16) {
#pragma unroll
                for (int i = 0; i < T; ++i) v[i] *= rs;
            } else {
#pragma unroll
                for (int i = 0; i < T; i += 4) {
                    const float4 c = kc[i / 4], f = vf[i / 4];
                    v[i] = fmaf(v[i] * rs, c.x, f.x);
                    v[i + 1] = fmaf(v[i + 1] * rs, c.y, f.y);
                    v[i + 2] = fmaf(v[i + 2] * rs, c.z, f.z);
                    v[i + 3] = fmaf(v[i + 3] * rs, c.w, f.w);
                }
            }
            const int p0 = (t0 + t) * T;
            if (p0 + T > len) {
#pragma unroll
                for (int w = 0; w < T / 64; ++w) {
                    const unsigned long long see = live ? tree_window(p, row, node, n, len, p0 + 64 * w) : 0ull;
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (!((see >> i) & 1)) v[64 * w + i] = -INFINITY;
                }
            }
            float top = v[0];
#pragma unroll
            for (int i = 1; i < T; ++i) top = fmaxf(top, v[i]);
            const float mn = fmaxf(m, top);
            const float ms = mn == -INFINITY ? 0.f : mn - 14.f;  // weights times 2^14
            const float c_new = ex2(m - (mn == -INFINITY ? 0.f : mn));
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < T / 32; ++c) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const int e = 32 * c + i;
                    float w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = ex2(v[e + j] - ms);
                    if (TYPE == AF_KV_F16) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum[j] += w[j];
                    } else {
                        const float4 g = vg[e / 4];
                        sum[0] = fmaf(w[0], g.x, sum[0]);
                        sum[1] = fmaf(w[1], g.y, sum[1]);
                        sum[2] = fmaf(w[2], g.z, sum[2]);
                        sum[3] = fmaf(w[3], g.w, sum[3]);
                    }
                    split2(w[0], w[1], hi[i / 2], lo[i / 2]);
                    split2(w[2], w[3], hi[i / 2 + 1], lo[i / 2 + 1]);
                }
                tc_st16(sb + 16 * c, hi);
                tc_st16(sb + T / 2 + 16 * c, lo);
            }
            l = fmaf(l, c_new, (sum[0] + sum[1]) + (sum[2] + sum[3]));
            m = mn;
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t & 1]);
            if (t > 0 && !take(t - 1)) {
                ok = false;
                break;
            }
            corr = c_new;
        }
        if (ok && nt > 0) ok = take(nt - 1);
        if (!ok) *flag = 1;
        // non-finite values of V were taken out of the products: the rows that see them get them back
        for (int w = 0; ok && w < kMmaBadWords && (32 * w) << bs < nt; ++w) {
            uint32_t b = bad[w];
            while (b) {
                const int t = (32 * w + __ffs(b) - 1) << bs;
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
        if (live && ok) {
            if (mp.nsplit == 1) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                float* o = p.out + (long long)row * p.os + (long long)head * HD;
                if ((reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
                    for (int i = 0; i < HD; i += 4)
                        *reinterpret_cast<float4*>(o + i) =
                            make_float4(acc[i] * inv, acc[i + 1] * inv, acc[i + 2] * inv, acc[i + 3] * inv);
                } else {
#pragma unroll
                    for (int i = 0; i < HD; ++i) o[i] = acc[i] * inv;
                }
            } else {
                const long long at = ((long long)split * p.n_rows + row) * p.H + head;
                float* o = mp.part + at * HD;
#pragma unroll
                for (int i = 0; i < HD; i += 4)
                    *reinterpret_cast<float4*>(o + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
                float* ml = mp.part + (long long)mp.nsplit * p.n_rows * p.H * HD + at * 2;
                *reinterpret_cast<float2*>(ml) = make_float2(m, l);
            }
        }
    } else if (warp < 12) {
        // ------------------------------------------------------- K and V
        asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
        const int w = warp - 4, sub = lane / SH::LPR, col = lane % SH::LPR;
        const long long hoff = p.layer * p.kv.layer_bytes + (long long)kvh * HD * SH::SIZE + col * 16;
        const uint8_t* kb = p.kv.k + hoff;
        const uint8_t* vb = p.kv.v + hoff;
        const int mine = w * SH::RPW + lane;  // lane < RPW: the row that this lane looks up
        auto lookup = [&](int t) -> int {     // pool row of the lane's position, -1: none
            const int pos = (t0 + t) * T + mine;
            if (t >= nt || lane >= SH::RPW || pos >= end) return -1;
            const int page = kv_page(p.b, p.kv.n_pages, seq, pos >> p.kv.ps_shift);
            if (page < 0) {
                set_err_at(p.b.err, kErrBadArgs);
                return -1;
            }
            return (page << p.kv.ps_shift) + (pos & ((1 << p.kv.ps_shift) - 1));
        };
        uint4 ring[RING][2 * NCK];
        auto load = [&](int idx, int c) -> uint4 {  // chunk c: K rows first, then V
            const int at = __shfl_sync(0xffffffffu, idx, (c % NCK) * SH::RPC + sub);
            if (at < 0) return make_uint4(0u, 0u, 0u, 0u);
            return __ldg(reinterpret_cast<const uint4*>((c < NCK ? kb : vb) + (long long)at * p.kv.row_bytes));
        };
        int idx = lookup(0);
#pragma unroll
        for (int s = 0; s < RING; ++s) {
#pragma unroll
            for (int c = 0; c < 2 * NCK; ++c) ring[s][c] = load(idx, c);
            idx = lookup(s + 1);
        }
        bool ok = true;
        for (int tb = 0; tb < nt && ok; tb += RING) {
#pragma unroll
            for (int s = 0; s < RING; ++s) {
                const int t = tb + s, st = t % NB;
                if (t >= nt) break;
                if (t >= NB && !wait_warp(&empty[st], (uint32_t)(t / NB - 1) & 1u)) {
                    ok = false;
                    break;
                }
                uint8_t* stage = tiles + st * SH::STAGE;
                float* sc = scales + st * 3 * T;
#pragma unroll
                for (int c = 0; c < 2 * NCK; ++c) {
                    const bool isv = c >= NCK;
                    const int trow = w * SH::RPW + (c % NCK) * SH::RPC + sub;  // row of the tile
                    uint8_t* dst = stage + (isv ? SH::TERMS * SH::TILE : 0) + (trow >> 3) * SH::RS + (trow & 7) * 16;
                    uint4 x = ring[s][c];
                    ring[s][c] = load(idx, c);
                    if (TYPE == AF_KV_F32) {
                        uint32_t b = max(max(x.x & 0x7fffffffu, x.y & 0x7fffffffu), max(x.z & 0x7fffffffu, x.w & 0x7fffffffu));
                        uint32_t mx = __reduce_max_sync(0xffffffffu, b);
                        if (isv && mx >= 0x7f800000u) {  // rare: take what is not finite out, and remember the tile
                            uint32_t* e = &x.x;
                            b = 0;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if ((e[i] & 0x7fffffffu) >= 0x7f800000u) e[i] = 0u;
                                b = max(b, e[i] & 0x7fffffffu);
                            }
                            mx = __reduce_max_sync(0xffffffffu, b);
                            if (lane == 0) atomicOr(&bad[(t >> bs) >> 5], 1u << ((t >> bs) & 31));
                        }
                        const int a = scale_of(mx, isv ? 60 : 100);
                        const float f = pow2(a);
                        uint2 hi, lo;
                        split2(__uint_as_float(x.x) * f, __uint_as_float(x.y) * f, hi.x, lo.x);
                        split2(__uint_as_float(x.z) * f, __uint_as_float(x.w) * f, hi.y, lo.y);
                        dst += (col >> 1) * SH::CS + (col & 1) * 8;
                        *reinterpret_cast<uint2*>(dst) = hi;
                        *reinterpret_cast<uint2*>(dst + SH::TILE) = lo;
                        if (col == 0) {
                            if (isv) {
                                sc[T + trow] = (float)-a;
                                sc[2 * T + trow] = f;
                            } else {
                                sc[trow] = pow2(-a);
                            }
                        }
                    } else if (TYPE == AF_KV_BF16) {
                        uint32_t* e = &x.x;
                        uint32_t b = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) b = max(b, max((e[i] << 16) & 0x7fff0000u, e[i] & 0x7fff0000u));
                        uint32_t mx = __reduce_max_sync(0xffffffffu, b);
                        if (isv && mx >= 0x7f800000u) {
                            b = 0;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (((e[i] << 16) & 0x7fff0000u) >= 0x7f800000u) e[i] &= 0xffff0000u;
                                if ((e[i] & 0x7fff0000u) >= 0x7f800000u) e[i] &= 0x0000ffffu;
                                b = max(b, max((e[i] << 16) & 0x7fff0000u, e[i] & 0x7fff0000u));
                            }
                            mx = __reduce_max_sync(0xffffffffu, b);
                            if (lane == 0) atomicOr(&bad[(t >> bs) >> 5], 1u << ((t >> bs) & 31));
                        }
                        const int a = scale_of(mx, isv ? 60 : 100);
                        const float f = pow2(a);
                        uint4 h;
                        uint32_t* o = &h.x;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            o[i] = pack2(__uint_as_float(e[i] << 16) * f, __uint_as_float(e[i] & 0xffff0000u) * f);
                        *reinterpret_cast<uint4*>(dst + col * SH::CS) = h;
                        if (col == 0) {
                            if (isv) {
                                sc[T + trow] = (float)-a;
                                sc[2 * T + trow] = f;
                            } else {
                                sc[trow] = pow2(-a);
                            }
                        }
                    } else {
                        if (isv) {
                            uint32_t* e = &x.x;
                            __half2 z = __float2half2_rn(0.f);  // x·0 is 0 for what is finite, NaN otherwise
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                z = __hfma2(*reinterpret_cast<const __half2*>(&e[i]), __float2half2_rn(0.f), z);
                            const uint32_t zz = *reinterpret_cast<const uint32_t*>(&z) & 0x7fff7fffu;
                            if (__any_sync(0xffffffffu, zz != 0)) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    if ((e[i] & 0x7c00u) == 0x7c00u) e[i] &= 0xffff0000u;
                                    if ((e[i] & 0x7c000000u) == 0x7c000000u) e[i] &= 0x0000ffffu;
                                }
                                if (lane == 0) atomicOr(&bad[(t >> bs) >> 5], 1u << ((t >> bs) & 31));
                            }
                        }
                        *reinterpret_cast<uint4*>(dst + col * SH::CS) = x;
                    }
                }
                idx = lookup(t + RING + 1);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[st]);
            }
        }
        if (!ok) *flag = 1;
    } else {
        // ------------------------------------------------------- products
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 12 && lane == 0 && nt > 0) {
            constexpr uint32_t base = (1u << 4) | ((uint32_t)(kMmaRows >> 4) << 24);  // f32 accumulators, f16 operands
            constexpr uint32_t ids = base | ((uint32_t)(T >> 3) << 17);
            constexpr uint32_t ido = base | ((uint32_t)(HD >> 3) << 17) | (1u << 16);  // B MN-major
            auto scores = [&](int t) {
                const uint32_t k0 = smem_u32(tiles + (t % NB) * SH::STAGE), d = tmem + SH::S0 + (t & 1) * T;
                bool acc = false;
                auto pass = [&](uint32_t q, uint32_t k) {
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks) {
                        tc_mma_ts(d, tmem + q + 8 * ks, tile_desc(k + 2 * ks * SH::CS, SH::CS, SH::RS), ids, acc);
                        acc = true;
                    }
                };
                pass(SH::QL, k0);
                if (SH::TERMS == 2) pass(SH::QH, k0 + SH::TILE);
                pass(SH::QH, k0);
                tc_commit(&s_full[t & 1]);
            };
            auto values = [&](int t) {
                const uint32_t v0 = smem_u32(tiles + (t % NB) * SH::STAGE + SH::TERMS * SH::TILE);
                const uint32_t w = tmem + SH::S0 + (t & 1) * T, d = tmem + SH::O0 + (t & 1) * HD;
                bool acc = false;
                auto pass = [&](uint32_t a, uint32_t v) {
#pragma unroll
                    for (int ks = 0; ks < T / 16; ++ks) {
                        tc_mma_ts(d, a + 8 * ks, tile_desc(v + 2 * ks * SH::RS, SH::RS, SH::CS), ido, acc);
                        acc = true;
                    }
                };
                pass(w + T / 2, v0);
                if (SH::TERMS == 2) pass(w, v0 + SH::TILE);
                pass(w, v0);
                tc_commit(&empty[t % NB]);
                tc_commit(&o_full[t & 1]);
            };
            bool ok = wait(q_full, 0u, flag) && wait(&full[0], 0u, flag);
            if (ok) {
                tc_fence_after();
                scores(0);
            }
            for (int t = 0; ok && t < nt; ++t) {
                if (t + 1 < nt) {  // the next tile's scores, over the weights of the tile before this one
                    ok = wait(&full[(t + 1) % NB], (uint32_t)((t + 1) / NB) & 1u, flag) &&
                         (t < 1 || wait(&o_full[(t + 1) & 1], (uint32_t)((t - 1) >> 1) & 1u, flag));
                    if (!ok) break;
                    tc_fence_after();
                    scores(t + 1);
                }
                ok = wait(&p_full[t & 1], (uint32_t)(t >> 1) & 1u, flag) &&
                     (t < 2 || wait(&o_free[t & 1], (uint32_t)((t >> 1) - 1) & 1u, flag));
                if (!ok) break;
                tc_fence_after();
                values(t);
            }
            if (!ok) *flag = 1;
            // whatever was issued ends before tensor memory is given back
            tc_commit(done);
            wait(done, 0u, nullptr);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// The splits of a row, a warp each: out = Σ 2^(m_s - m)·O_s / Σ 2^(m_s - m)·l_s, in split order.
template <int HD>
__global__ void __launch_bounds__(256) tree_merge_kernel(MmaParams mp) {
    const TreeParams& p = mp.t;
    constexpr int PER = HD / 32;
    const int lane = threadIdx.x & 31, seq = blockIdx.y;
    int r0, n;
    kv_nodes(p.b, p.n_rows, seq, r0, n);
    if (kv_len(p.kv, p.b, seq, n) < 0) return;
    const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_wait();
    if (i >= n * p.H) return;
    const int row = r0 + i / p.H, head = i % p.H;
    const long long step = (long long)p.n_rows * p.H, at = (long long)row * p.H + head;
    const float* o = mp.part + at * HD + lane * PER;
    const float* ml = mp.part + mp.nsplit * step * HD + at * 2;
    float top = -INFINITY;
    for (int s = lane; s < mp.nsplit; s += 32) top = fmaxf(top, ml[s * step * 2]);
    top = warp_max(top);
    float acc[PER], sum = 0.f;
#pragma unroll
    for (int d = 0; d < PER; ++d) acc[d] = 0.f;
#pragma unroll 4
    for (int s = 0; s < mp.nsplit; ++s) {
        const float2 x = *reinterpret_cast<const float2*>(ml + s * step * 2);
        if (x.y == 0.f && x.x == -INFINITY) continue;  // a split that the row sees nothing of
        const float c = ex2(x.x - top);
        sum = fmaf(c, x.y, sum);
        float v[PER];
        if (PER == 4) {
            const float4 f = *reinterpret_cast<const float4*>(o + s * step * HD);
            v[0] = f.x, v[1] = f.y, v[2 % PER] = f.z, v[3 % PER] = f.w;
        } else {
            const float2 f = *reinterpret_cast<const float2*>(o + s * step * HD);
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

// ------------------------------------------------------------------ launch

// Splits of the positions: enough blocks for every SM, none below 4 tiles.
struct TreePlan {
    bool mma;
    int row_tiles, nsplit;
    size_t ws;
};

TreePlan tree_plan(const af_attention_tree_args& a) {
    TreePlan pl = {};
    const int hd = a.kv.head_dim, G = a.n_heads / a.kv.n_kv_heads;
    pl.nsplit = 1;
    pl.mma = hd == 64 || hd == 128;
    if (!pl.mma) return pl;
    const long long cap = (long long)a.batch.max_blocks * a.kv.page_size;
    const long long max_len = a.max_len > 0 ? std::min((long long)a.max_len, cap) : cap;
    pl.row_tiles = (int)(((long long)a.batch.max_nodes * G + kMmaRows - 1) / kMmaRows);
    const long long base = (long long)pl.row_tiles * a.kv.n_kv_heads * std::max(1, a.batch.n_seq);
    const int T = hd == 128 ? 64 : 128;
    const long long tiles = (max_len + T - 1) / T;
    long long want = 148 / base;
    pl.nsplit = (int)std::max(1ll, std::min({want, tiles / 2, 148ll}));
    if (pl.nsplit > 1) pl.ws = (size_t)pl.nsplit * a.n_rows * a.n_heads * (hd + 2) * sizeof(float);
    return pl;
}

template <int TYPE, int HD>
cudaError_t mma_launch(const MmaParams& mp, int n_seq, int max_nodes, cudaStream_t st) {
    constexpr int smem = MmaShape<TYPE, HD>::BYTES;
    AF_CUDA_TRY(cudaFuncSetAttribute(tree_mma_kernel<TYPE, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    tree_mma_kernel<TYPE, HD><<<dim3(mp.nsplit * mp.row_tiles, mp.t.kv.kv_heads, n_seq), kMmaThreads, smem, st>>>(mp);
    AF_CUDA_TRY(cudaGetLastError());
    if (mp.nsplit == 1) return cudaSuccess;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((long long)max_nodes * mp.t.H + 7) / 8), n_seq);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, tree_merge_kernel<HD>, mp);
}

template <int TYPE>
cudaError_t tree_launch(const TreeParams& p, const TreePlan& pl, int max_nodes, void* ws, cudaStream_t st) {
    if (pl.mma) {
        MmaParams mp = {p, pl.nsplit, pl.row_tiles, static_cast<float*>(ws)};
        return p.kv.hd == 64 ? mma_launch<TYPE, 64>(mp, p.b.n_seq, max_nodes, st) : mma_launch<TYPE, 128>(mp, p.b.n_seq, max_nodes, st);
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
    if (a.mask && (a.mask_words <= 0 || (long long)a.mask_words * 64 < a.batch.max_nodes))
        return "mask_words must cover max_nodes";
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
    if (pl.ws && (!a->ws || a->ws_bytes < pl.ws || (reinterpret_cast<uintptr_t>(a->ws) & 15)))
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
    p.q = a->q;
    p.out = a->out;
    p.qs = a->q_stride ? a->q_stride : qd;
    p.os = a->out_stride ? a->out_stride : qd;
    p.mask = reinterpret_cast<const unsigned long long*>(a->mask);
    p.mask_words = a->mask_words;
    p.scale = (a->scale != 0.f ? a->scale : 1.f / std::sqrt((float)a->kv.head_dim)) * 1.4426950408889634f;
    switch (a->kv.type) {
        case AF_KV_F32: return tree_launch<AF_KV_F32>(p, pl, a->batch.max_nodes, a->ws, stream);
        case AF_KV_F16: return tree_launch<AF_KV_F16>(p, pl, a->batch.max_nodes, a->ws, stream);
        default: return tree_launch<AF_KV_BF16>(p, pl, a->batch.max_nodes, a->ws, stream);
    }
}
