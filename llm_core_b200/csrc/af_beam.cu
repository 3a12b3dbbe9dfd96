// af_beam.cu — one step of a beam search (af_beam_select_f32): of every
// sequence's beams the n_out best continuations by cumulative log-probability,
//     score(b, t) = scores[b] + x[b][t] - log Σ_t' exp x[b][t'],
// in one pass over the logits.
//
//  * Segment kernel: a block streams a segment of a row, 4096 logits a step
//    (four 16-byte loads a thread, the next step's in flight): the running
//    maximum, Σ exp(x - max), and a buffer of what may be among the segment's
//    K = n_out largest.  Within a beam scores are ordered as logits, so the K
//    best of a segment are its K largest, ties to the lower token: 64-bit
//    keys (ordered value, ~token) are distinct.  The first step's threshold:
//    of each warp's threads' largest values the ceil(K/8)-th; the smallest of
//    these has at least K values at or above it.  Later logits have higher
//    tokens, so one that only equals the threshold has K better ones in front
//    of it and is passed over: what enters the buffer is rare, and where it is
//    not (rising or equal logits) the buffer is cut back to its K best, which
//    raises the threshold.  16 sequences of 8 beams over 151,936 logits (78 MB)
//    take 33 us with the merge, 2.4 TB/s: with all of a step's data there it
//    still takes ~2,200 cycles, the exponentials 600, the keys that pass up to
//    1,500 in some warp, which the block's barrier then waits for; the first
//    step and the last cut add 8,000.
//  * Merge kernel, a block per sequence: the segments' sums to one base
//    scores[b] - log Σ per beam in 64 bits, so that scores of different beams
//    compare as their definition does, and the K best of the segment lists: the
//    K-th best list head is again a threshold, which at most K lists of K pass.
//    Latency alone: 4 beams of 32,000 logits take 10 us, both kernels.
//  * A beam that is dead before the call (score not finite) is not read.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "af_common.cuh"
#include "af_ops.cuh"

namespace af {
namespace {

typedef unsigned long long u64;

constexpr int kBeamThreads = 256;
constexpr int kBeamBlocks = 3;                          // on an SM
constexpr int kBeamPer = 16;                            // logits of a thread in a step
constexpr int kBeamStep = kBeamThreads * kBeamPer;      // 4096
constexpr int kBeamFull = 2048;                         // keys kept: cut back when more are there
constexpr int kBeamBuffer = kBeamFull + kBeamStep;
constexpr int kBeamSelect = 512;                        // of those, near the best
constexpr int kBeamChunk = 8192;                        // shortest segment
constexpr int kBeamMaxK = 64;
constexpr int kBeamLists = 1024;                        // chunk lists of a sequence
constexpr int kMergeThreads = 256;

struct BeamParams {
    const float *logits, *scores;
    long long stride;
    int n_seq, beams, vocab, K, chunks, seg, vec;  // chunks: segments of a row, of seg logits
    float* out_score;
    int *out_beam, *out_token;
    u64* keys;      // [rows][chunks][K] the segments' largest, in order; 0: none
    double* sums;   // [rows][chunks]
    float* tops;    // [rows][chunks]
};

// -0 and 0 are one value: v + 0 is never -0.
__device__ __forceinline__ u64 logit_key(float v, int token) { return argmax_key(v + 0.f, (uint32_t)token); }

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ bool dead_score(float s) { return !(fabsf(s) < INFINITY); }  // infinities and NaN

// This lane's value of the warp's 32 in descending order.
template <typename T>
__device__ __forceinline__ T warp_sort_desc(T v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1) {
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const T o = __shfl_xor_sync(0xffffffffu, v, j);
            const bool up = (lane & k) != 0, low = (lane & j) == 0;  // ascending run; lower partner
            v = (low != up) == (v > o) ? v : o;
        }
    }
    return v;
}

// The warp's n-th largest value, equal ones counted one by one, n <= 32 (values > 0).
__device__ __forceinline__ uint32_t warp_nth(uint32_t v, int n) {
    for (;;) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, v);
        n -= __popc(__ballot_sync(0xffffffffu, v == m));
        if (n <= 0 || m == 0) return m;
        if (v == m) v = 0;
    }
}

__device__ __forceinline__ float beam_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct BeamShared {
    u64 key[kBeamBuffer];
    u64 sel[kBeamSelect];
    u64 out[kBeamMaxK];
    u64 wkey[kBeamThreads / 32];
    float wval[kBeamThreads / 32];
    double wsum[kBeamThreads / 32];
    int count, kept;
};

// The buffer's K best keys, in order, to its front (fewer where it has fewer).
__device__ void beam_cut(BeamShared& sh, int K) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = sh.count;
    u64 best = 0;
    // every warp has its share of them: key i is warp i % W's; a warp's n-th is of its threads' best values
    constexpr int W = kBeamThreads / 32;
    for (int i = lane * W + warp; i < n; i += kBeamThreads) best = max(best, sh.key[i]);
    const uint32_t nth = warp_nth((uint32_t)(best >> 32), (K + W - 1) / W);  // 0 where the warp has fewer: everything passes
    if (lane == 0) sh.wkey[warp] = (u64)nth << 32;
    if (tid == 0) sh.kept = 0;
    __syncthreads();
    u64 thr = sh.wkey[0];
#pragma unroll
    for (int w = 1; w < W; ++w) thr = min(thr, sh.wkey[w]);
    // their order among what passes, or, where that is more than sel holds (rising logits), among all
    for (int i = tid; i < n; i += kBeamThreads) {
        const u64 k = sh.key[i];
        if (k >= thr) {
            const int at = atomicAdd(&sh.kept, 1);
            if (at < kBeamSelect) sh.sel[at] = k;
        }
    }
    __syncthreads();
    const int kept = sh.kept;
    const bool few = kept <= kBeamSelect;
    const u64* from = few ? sh.sel : sh.key;
    const int m = few ? kept : n;
    for (int c = tid; c < m; c += kBeamThreads) {
        const u64 k = from[c];
        if (k < thr) continue;
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < m; ++i) rank += from[i] > k;
        if (rank < K) sh.out[rank] = k;
    }
    __syncthreads();
    const int have = min(K, kept);
    if (tid < have) sh.key[tid] = sh.out[tid];
    if (tid == 0) sh.count = have;
    __syncthreads();
}

__global__ void __launch_bounds__(kBeamThreads, kBeamBlocks) beam_segment_kernel(BeamParams p) {
    constexpr int W = kBeamThreads / 32;
    extern __shared__ __align__(16) uint8_t sm[];
    BeamShared& sh = *reinterpret_cast<BeamShared*>(sm);
    pdl_launch_dependents();  // the merge kernel may start launching
    const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float score = p.scores[row];
    const int lo = blockIdx.x * p.seg, hi = min(lo + p.seg, p.vocab), K = p.K;
    const float* x = p.logits + (long long)row * p.stride;
    auto token = [&](int t0, int j) { return t0 + (j >> 2) * (4 * kBeamThreads) + 4 * tid + (j & 3); };
    auto load = [&](int t0, float (&v)[kBeamPer]) {
        if (p.vec && t0 + kBeamStep <= hi) {
#pragma unroll
            for (int h = 0; h < kBeamPer / 4; ++h) {
                const float4 f = __ldcs(reinterpret_cast<const float4*>(x + token(t0, 4 * h)));
                v[4 * h] = f.x, v[4 * h + 1] = f.y, v[4 * h + 2] = f.z, v[4 * h + 3] = f.w;
            }
            return;
        }
#pragma unroll
        for (int h = 0; h < kBeamPer / 4; ++h) {
            const int t = token(t0, 4 * h);
            if (p.vec && t + 4 <= hi) {
                const float4 f = __ldcs(reinterpret_cast<const float4*>(x + t));
                v[4 * h] = f.x, v[4 * h + 1] = f.y, v[4 * h + 2] = f.z, v[4 * h + 3] = f.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * h + j] = t + j < hi ? x[t + j] : -INFINITY;
            }
        }
    };
    float even[kBeamPer], odd[kBeamPer];  // a step's logits, and the next one's, on their way
    load(lo, even);                       // beside the beam's score, not behind it
    if (dead_score(score)) return;
    if (lo + kBeamStep < hi) load(lo + kBeamStep, odd);
    if (tid == 0) sh.count = 0;
    __syncthreads();
    float top = -INFINITY, thr = 0.f;
    double sum = 0.;
    constexpr float kLog2e = 1.4426950408889634f;
    auto lowest = [&]() {
        float m = sh.wval[0];
#pragma unroll
        for (int w = 1; w < W; ++w) m = fminf(m, sh.wval[w]);
        return m;
    };
    auto step = [&](int t0, float (&v)[kBeamPer]) {
        float m[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = fmaxf(fmaxf(v[4 * j], v[4 * j + 1]), fmaxf(v[4 * j + 2], v[4 * j + 3]));
        const float big = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
        if (big > top) {
            sum *= (double)beam_exp2((top - big) * kLog2e);
            top = big;
        }
        // a step's terms in 32 bits, the rest in 64; NaN stays NaN, and where all is -inf, nothing is added
        const float off = top > -INFINITY ? top : 0.f;
        f32x2 part[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
        const f32x2 less = pair(-off, -off), log2e = pair(kLog2e, kLog2e);
#pragma unroll
        for (int j = 0; j < kBeamPer; j += 2) {
            float a, b;
            unpair(mul2(add2(pair(v[j], v[j + 1]), less), log2e), a, b);
            part[(j >> 1) & 1] = add2(part[(j >> 1) & 1], pair(beam_exp2(a), beam_exp2(b)));
        }
        float pa, pb;
        unpair(add2(part[0], part[1]), pa, pb);
        sum += (double)(pa + pb);
        const bool begin = t0 == lo;
        // The threshold, of the first step before anything is kept; of all steps so far behind steps 1, 2, 4, 8, ...,
        // which halves how many pass each time (top is the thread's largest so far).
        const int nr = (t0 - lo) / kBeamStep + 1;
        const bool raise = (nr & (nr - 1)) == 0;
        if (raise) {
            const uint32_t s = warp_nth(float_to_ordered(top), (K + 7) / 8);
            if (lane == 0) sh.wval[warp] = ordered_to_float(s);
        }
        if (begin) {
            __syncthreads();
            thr = lowest();
        }
        bool full = false;  // this thread's last key came behind kBeamFull others
        auto keep = [&](int j) {
            const int at = atomicAdd(&sh.count, 1);
            sh.key[at] = logit_key(v[j], token(t0, j));
            full = at >= kBeamFull;
        };
        if (begin) {
            if (big >= thr) {
#pragma unroll
                for (int j = 0; j < kBeamPer; ++j)
                    if (v[j] >= thr && token(t0, j) < hi) keep(j);
            }
        } else if (big > thr) {  // what lies behind the segment is -inf
#pragma unroll
            for (int j = 0; j < kBeamPer; j += 4) {
                if (m[(j >> 2) & 3] <= thr) continue;
#pragma unroll
                for (int i = j; i < j + 4; ++i)
                    if (v[i] > thr) keep(i);
            }
        }
        if (t0 + 2 * kBeamStep < hi) load(t0 + 2 * kBeamStep, v);
        // Whoever added the last key knows that it was one too many; the count itself may still grow when another looks.
        // So at most a step's keys come on top of at most kBeamFull.
        if (__syncthreads_or(full)) {
            beam_cut(sh, K);
            thr = fmaxf(thr, ordered_to_float((uint32_t)(sh.key[K - 1] >> 32)));
            __syncthreads();
        }
        if (raise && !begin) {
            thr = fmaxf(thr, lowest());
            __syncthreads();
        }
    };
    for (int t0 = lo; t0 < hi; t0 += 2 * kBeamStep) {
        step(t0, even);
        if (t0 + kBeamStep < hi) step(t0 + kBeamStep, odd);
    }
    beam_cut(sh, K);
    const long long list = (long long)row * p.chunks + blockIdx.x;
    const int have = sh.count;
    if (tid < K) p.keys[list * K + tid] = tid < have ? sh.key[tid] : 0;
    // one maximum and one sum
    const float wtop = warp_max(top);
    if (lane == 0) sh.wval[warp] = wtop;
    __syncthreads();
    float all = sh.wval[0];
#pragma unroll
    for (int w = 1; w < W; ++w) all = fmaxf(all, sh.wval[w]);
    sum = warp_sum_d(top == all ? sum : sum * (double)expf(top - all));  // 0·exp(-inf) = 0
    if (lane == 0) sh.wsum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.;
        for (int w = 0; w < W; ++w) sum += sh.wsum[w];
        p.sums[list] = sum;
        p.tops[list] = all;
    }
}

// Order-preserving map of a double to u64.
__device__ __forceinline__ u64 double_ordered(double d) {
    const u64 u = (u64)__double_as_longlong(d);
    return (u >> 63) ? ~u : (u | (1ull << 63));
}
__device__ __forceinline__ double ordered_double(u64 k) {
    return __longlong_as_double((long long)((k >> 63) ? (k & ~(1ull << 63)) : ~k));
}

// Candidates: the higher score, then the lower (beam, token) first.
__device__ __forceinline__ bool better(u64 s, unsigned f, u64 s2, unsigned f2) { return s > s2 || (s == s2 && f < f2); }

constexpr int kMergeKeys = 4096;  // keys of a sequence that are brought to shared memory, when they are no more
constexpr int kMergeSmem = kBeamLists * 12 + kBeamMaxK * kBeamMaxK * 12 + 64 * 8 + kMergeKeys * 8 + (2 + kBeamMaxK) * 4;

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(BeamParams p) {
    extern __shared__ __align__(16) uint8_t sm[];
    u64* hs = reinterpret_cast<u64*>(sm);                        // [lists] heads
    u64* cs = hs + kBeamLists;                                   // [K*K] candidates
    double* base = reinterpret_cast<double*>(cs + kBeamMaxK * kBeamMaxK);  // [beams]
    u64* near = reinterpret_cast<u64*>(base + 64);               // [lists][K], if they fit
    unsigned* hf = reinterpret_cast<unsigned*>(near + kMergeKeys);
    unsigned* cf = hf + kBeamLists;
    int* ctl = reinterpret_cast<int*>(cf + kBeamMaxK * kBeamMaxK);  // candidates, lists, the lists with the best heads
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row0 = seq * p.beams, K = p.K;
    const int lists = p.beams * p.chunks;
    const bool here = lists * K <= kMergeKeys;
    const u64* keys = p.keys + (long long)row0 * p.chunks * K;
    pdl_wait();
    if (here)
        for (int i = tid; i < lists * K; i += kMergeThreads) near[i] = keys[i];
    if (here) keys = near;
    // a beam's base: scores[b] - log Σ exp, -inf for a dead one
    for (int b = warp; b < p.beams; b += kMergeThreads / 32) {
        const float s = p.scores[row0 + b];
        double d = -INFINITY;
        if (!dead_score(s)) {
            const long long l0 = (long long)(row0 + b) * p.chunks;
            float t = lane < p.chunks ? p.tops[l0 + lane] : -INFINITY, top = t;
            double sum = lane < p.chunks ? p.sums[l0 + lane] : 0.;
            for (int c = lane + 32; c < p.chunks; c += 32) top = fmaxf(top, p.tops[l0 + c]);
            top = warp_max(top);
            if (lane < p.chunks && t != top) sum *= (double)expf(t - top);  // NaN sums stay
            for (int c = lane + 32; c < p.chunks; c += 32) {
                t = p.tops[l0 + c];
                sum += p.sums[l0 + c] * (t == top ? 1. : (double)expf(t - top));
            }
            sum = warp_sum_d(sum);
            d = (double)s - ((double)top + log(sum));
            if (!(d > -INFINITY) || top == -INFINITY || top == INFINITY) d = -INFINITY;  // NaN or ±inf logits
        }
        if (lane == 0) base[b] = d;
    }
    if (tid == 0) ctl[0] = 0;
    __syncthreads();
    // entry c of a list: (score, beam*vocab + token); a dead beam's first list
    // holds its tokens 0..K-1 at -inf, its others nothing
    auto entry = [&](int list, int c, u64& s, unsigned& f) -> bool {
        const int b = list / p.chunks, chunk = list % p.chunks;
        if (base[b] == -INFINITY) {
            if (chunk || c >= p.vocab) return false;
            s = double_ordered(-INFINITY);
            f = (unsigned)b * p.vocab + c;
            return true;
        }
        const u64 k = keys[list * K + c];
        if (!k) return false;
        const double x = (double)ordered_to_float((uint32_t)(k >> 32));
        s = double_ordered(base[b] + x);
        f = (unsigned)b * p.vocab + (0xFFFFFFFFu - (uint32_t)k);
        return true;
    };
    for (int l = tid; l < lists; l += kMergeThreads) {
        u64 ms = 0;
        unsigned mf = UINT_MAX;  // no entry at all
        if (!entry(l, 0, ms, mf)) ms = 0, mf = UINT_MAX;
        hs[l] = ms;
        hf[l] = mf;
    }
    __syncthreads();
    // only the K lists with the best heads can hold the K best, and of the one of rank r only its first K - r entries
    for (int l = tid; l < lists; l += kMergeThreads) {
        const u64 ms = hs[l];
        const unsigned mf = hf[l];
        if (mf == UINT_MAX) continue;
        int rank = 0;
#pragma unroll 4
        for (int i = 0; i < lists; ++i) rank += better(hs[i], hf[i], ms, mf);
        if (rank < K) ctl[2 + rank] = l;
    }
    if (tid < 32) {  // how many lists have a head at all
        int any = 0;
        for (int i = tid; i < lists; i += 32) any += hf[i] != UINT_MAX;
        any = __reduce_add_sync(0xffffffffu, any);
        if (tid == 0) ctl[1] = min(any, K);
    }
    __syncthreads();
    const int good = ctl[1];
    u64 best = 0;
    for (int i = tid; i < good * K; i += kMergeThreads) {
        const int r = i / K, c = i % K;
        u64 s;
        unsigned f;
        if (r + c < K && entry(ctl[2 + r], c, s, f)) {
            const int at = atomicAdd(&ctl[0], 1);
            cs[at] = s;
            cf[at] = f;
            best = max(best, s);
        }
    }
    unsigned* sel = hf;  // the candidates to rank, up to kBeamLists
    __syncthreads();
    const int cnt = ctl[0];
    if (cnt > kMergeThreads) {
        // a score that at least K reach: the smallest of the warps' ceil(K/8)-th best
        best = warp_sort_desc(best, lane);
        if (lane == (K + 7) / 8 - 1) hs[warp] = best;
        if (tid == 0) ctl[1] = 0;
        __syncthreads();
        u64 thr = hs[0];
        for (int w = 1; w < kMergeThreads / 32; ++w) thr = min(thr, hs[w]);
        for (int c = tid; c < cnt; c += kMergeThreads)
            if (cs[c] >= thr) {
                const int at = atomicAdd(&ctl[1], 1);
                if (at < kBeamLists) sel[at] = c;
            }
        __syncthreads();
    }
    const bool few = cnt > kMergeThreads && ctl[1] <= kBeamLists;
    const int m = few ? ctl[1] : cnt;
    for (int i = tid; i < m; i += kMergeThreads) {
        const int c = few ? sel[i] : i;
        const u64 s = cs[c];
        const unsigned f = cf[c];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < m; ++j) {
            const int o = few ? sel[j] : j;
            rank += better(cs[o], cf[o], s, f);
        }
        if (rank < K) {
            const long long at = (long long)seq * K + rank;
            p.out_score[at] = (float)ordered_double(s);
            p.out_beam[at] = row0 + (int)(f / (unsigned)p.vocab);
            p.out_token[at] = (int)(f % (unsigned)p.vocab);
        }
    }
}

cudaError_t refuse(const std::string& why) {
    set_last_error("af_beam_select_f32: " + why);
    return cudaErrorInvalidValue;
}

std::string beam_wrong(const af_beam_select_args& a) {
    if (a.n_seq < 0 || a.n_beams <= 0 || a.n_beams > 64 || a.vocab <= 0) return "need n_seq >= 0, 1 <= n_beams <= 64, vocab > 0";
    if ((long long)a.n_seq * a.n_beams > 65535) return "n_seq * n_beams must be at most 65535";
    if (a.n_out <= 0 || a.n_out > kBeamMaxK || a.n_out > (long long)a.n_beams * a.vocab)
        return "n_out must be in 1..64 and at most n_beams * vocab";
    if ((long long)a.n_beams * ((a.vocab + (long long)kBeamChunk - 1) / kBeamChunk) > kBeamLists)
        return "n_beams * ceil(vocab / 8192) must be at most 1024";
    if (a.logits_stride && a.logits_stride < a.vocab) return "logits_stride is shorter than a row";
    return "";
}

constexpr int kBeamFill = kBeamBlocks * 148;  // blocks that the SMs hold at once

int beam_most(int vocab) { return (int)(((long long)vocab + kBeamChunk - 1) / kBeamChunk); }

// Segments of a row: as many blocks as the SMs hold at once, none below kBeamChunk logits.
int beam_segments(const af_beam_select_args& a) {
    const long long rows = std::max(1ll, (long long)a.n_seq * a.n_beams);
    return (int)std::min((long long)beam_most(a.vocab), std::max(1ll, kBeamFill / rows));
}

// Fewer rows have more segments each: room for the most lists that any number of rows up to this one makes.
size_t beam_ws(const af_beam_select_args& a) {
    const size_t rows = (size_t)a.n_seq * a.n_beams;
    const size_t lists = std::min(rows * beam_most(a.vocab), std::max(rows, (size_t)kBeamFill));
    return lists * ((size_t)a.n_out * 8 + 16);
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" size_t af_beam_select_f32_workspace(const af_beam_select_args* a) {
    return a && beam_wrong(*a).empty() ? beam_ws(*a) : 0;
}

extern "C" cudaError_t af_beam_select_f32(const af_beam_select_args* a, cudaStream_t stream) {
    if (!a) return refuse("null arguments");
    const std::string why = beam_wrong(*a);
    if (!why.empty()) return refuse(why);
    if (a->n_seq == 0) return cudaSuccess;
    if (!a->logits || !a->scores || !a->out_score || !a->out_beam || !a->out_token) return refuse("null arguments");
    if (!a->ws || a->ws_bytes < beam_ws(*a) || (reinterpret_cast<uintptr_t>(a->ws) & 15))
        return refuse("ws must hold af_beam_select_f32_workspace bytes, 16-byte aligned");
    BeamParams p = {};
    p.logits = a->logits;
    p.scores = a->scores;
    p.stride = a->logits_stride ? a->logits_stride : a->vocab;
    p.n_seq = a->n_seq;
    p.beams = a->n_beams;
    p.vocab = a->vocab;
    p.K = a->n_out;
    p.chunks = beam_segments(*a);
    p.seg = ((a->vocab + p.chunks - 1) / p.chunks + kBeamStep - 1) / kBeamStep * kBeamStep;
    p.chunks = (a->vocab + p.seg - 1) / p.seg;
    p.vec = !(reinterpret_cast<uintptr_t>(a->logits) & 15) && p.stride % 4 == 0;
    p.out_score = a->out_score;
    p.out_beam = a->out_beam;
    p.out_token = a->out_token;
    const size_t lists = (size_t)a->n_seq * a->n_beams * p.chunks;
    p.keys = static_cast<u64*>(a->ws);
    p.sums = reinterpret_cast<double*>(p.keys + lists * p.K);
    p.tops = reinterpret_cast<float*>(p.sums + lists);
    AF_CUDA_TRY(cudaFuncSetAttribute(beam_segment_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(BeamShared)));
    beam_segment_kernel<<<dim3(p.chunks, p.n_seq * p.beams), kBeamThreads, sizeof(BeamShared), stream>>>(p);
    AF_CUDA_TRY(cudaGetLastError());
    AF_CUDA_TRY(cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMergeSmem));
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.n_seq);
    cfg.blockDim = dim3(kMergeThreads);
    cfg.dynamicSmemBytes = kMergeSmem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, beam_merge_kernel, p);
}
