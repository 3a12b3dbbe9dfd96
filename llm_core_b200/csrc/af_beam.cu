// af_beam.cu — one step of a beam search (af_beam_select_f32): of every
// sequence's beams the n_out best continuations by cumulative log-probability,
//     score(b, t) = scores[b] + x[b][t] - log Σ_t' exp x[b][t'],
// in one pass over the logits.
//
//  * Chunk kernel: a block holds up to 8192 logits of a row in registers
//    (32 a thread): their maximum, Σ exp(x - max), and their K = n_out largest
//    in order.  Within a beam scores are ordered as logits, so the K best of a
//    chunk are its K largest logits, ties to the lower token: 64-bit keys
//    (ordered value, ~token) are distinct.  The K-th largest of the threads'
//    own largest keys is a threshold with at least K keys at or above it and
//    at most K·32 (those of K threads), so what passes it fits a fixed buffer
//    whatever the logits (all equal, say), and its order is found by counting.
//  * Merge kernel, a block per sequence: the chunks' sums to one base
//    scores[b] - log Σ per beam in 64 bits, so that scores of different beams
//    compare as their definition does, and the K best of the chunk lists: the
//    K-th best list head is again a threshold, which at most K lists of K pass.
//  * A beam that is dead before the call (score -inf or NaN) is not read.
#include <climits>
#include <cmath>
#include <cstdint>

#include "af_common.cuh"
#include "af_ops.cuh"

namespace af {
namespace {

typedef unsigned long long u64;

constexpr int kBeamThreads = 256;
constexpr int kBeamPer = 32;                            // logits of a thread
constexpr int kBeamChunk = kBeamThreads * kBeamPer;     // 8192
constexpr int kBeamMaxK = 64;
constexpr int kBeamLists = 1024;                        // chunk lists of a sequence
constexpr int kMergeThreads = 1024;

struct BeamParams {
    const float *logits, *scores;
    long long stride;
    int n_seq, beams, vocab, K, chunks, vec;
    float* out_score;
    int *out_beam, *out_token;
    u64* keys;      // [rows][chunks][K] the chunks' largest, in order; 0: none
    double* sums;   // [rows][chunks]
    float* tops;    // [rows][chunks]
};

__device__ __forceinline__ u64 logit_key(float v, int token) { return argmax_key(v, (uint32_t)token); }

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ bool dead_score(float s) { return !(s > -INFINITY); }  // -inf and NaN

__global__ void __launch_bounds__(kBeamThreads) beam_chunk_kernel(BeamParams p) {
    constexpr int W = kBeamThreads / 32;
    __shared__ u64 tmax[kBeamThreads];
    __shared__ u64 cand[kBeamMaxK * kBeamPer];
    __shared__ float wtop[W];
    __shared__ double wsum[W];
    __shared__ u64 s_thr;
    __shared__ int s_cnt;
    const int chunk = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (dead_score(p.scores[row])) return;
    const int t0 = chunk * kBeamChunk, n = min(kBeamChunk, p.vocab - t0);
    const float* x = p.logits + (long long)row * p.stride + t0;
    float v[kBeamPer];
    // thread's element e is token t0 + 4*(tid + 256*(e/4)) + e%4 (16-byte loads where the rows allow them)
#pragma unroll
    for (int e = 0; e < kBeamPer; e += 4) {
        const int i = 4 * (tid + kBeamThreads * (e / 4));
        if (p.vec && i + 4 <= n) {
            const float4 f = *reinterpret_cast<const float4*>(x + i);
            v[e] = f.x;
            v[e + 1] = f.y;
            v[e + 2] = f.z;
            v[e + 3] = f.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[e + j] = i + j < n ? x[i + j] : -INFINITY;
        }
    }
    float top = -INFINITY;
    bool nan = false;
    u64 best = 0;
#pragma unroll
    for (int e = 0; e < kBeamPer; ++e) {
        const int i = 4 * (tid + kBeamThreads * (e / 4)) + (e & 3);
        nan |= v[e] != v[e];
        top = fmaxf(top, v[e]);
        if (i < n) best = max(best, logit_key(v[e], t0 + i));
    }
    if (tid == 0) {
        s_cnt = 0;
        s_thr = 0;
    }
    tmax[tid] = best;
    top = warp_max(top);
    if (lane == 0) wtop[warp] = top;
    __syncthreads();
    top = wtop[0];
#pragma unroll
    for (int w = 1; w < W; ++w) top = fmaxf(top, wtop[w]);
    // Σ exp(x - top): 32 terms a thread in 32 bits, the rest in 64
    float part = 0.f;
    if (top > -INFINITY) {
#pragma unroll
        for (int e = 0; e < kBeamPer; ++e) part += expf(v[e] - top);
    }
    double sum = warp_sum_d(nan ? (double)NAN : (double)part);
    if (lane == 0) wsum[warp] = sum;
    // the K-th largest of the threads' largest
    const int K = min(p.K, n);
    if (best) {
        int rank = 0;
        for (int i = 0; i < kBeamThreads; ++i) rank += tmax[i] > best;
        if (rank == K - 1) s_thr = best;  // fewer than K threads with logits: 0, everything passes
    }
    __syncthreads();
    const u64 thr = s_thr;
#pragma unroll
    for (int e = 0; e < kBeamPer; ++e) {
        const int i = 4 * (tid + kBeamThreads * (e / 4)) + (e & 3);
        if (i < n) {
            const u64 k = logit_key(v[e], t0 + i);
            if (k >= thr) cand[atomicAdd(&s_cnt, 1)] = k;
        }
    }
    __syncthreads();
    const int cnt = s_cnt;
    const long long list = (long long)row * p.chunks + chunk;
    for (int c = tid; c < cnt; c += kBeamThreads) {
        const u64 k = cand[c];
        int rank = 0;
        for (int i = 0; i < cnt; ++i) rank += cand[i] > k;
        if (rank < K) p.keys[list * p.K + rank] = k;
    }
    for (int c = K + tid; c < p.K; c += kBeamThreads) p.keys[list * p.K + c] = 0;
    if (tid == 0) {
        sum = 0.;
        for (int w = 0; w < W; ++w) sum += wsum[w];
        p.sums[list] = sum;
        p.tops[list] = top;
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

// A candidate: ordered score, then the lower (beam, token) first.
struct Cand {
    u64 score;
    unsigned flat;
};
__device__ __forceinline__ bool better(u64 s, unsigned f, u64 s2, unsigned f2) { return s > s2 || (s == s2 && f < f2); }

constexpr int kMergeSmem = kBeamLists * 12 + kBeamMaxK * kBeamMaxK * 12 + 64 * 8 + 64;

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(BeamParams p) {
    extern __shared__ __align__(16) uint8_t sm[];
    u64* hs = reinterpret_cast<u64*>(sm);                        // [lists] heads
    u64* cs = hs + kBeamLists;                                   // [K*K] candidates
    double* base = reinterpret_cast<double*>(cs + kBeamMaxK * kBeamMaxK);  // [beams]
    unsigned* hf = reinterpret_cast<unsigned*>(base + 64);
    unsigned* cf = hf + kBeamLists;
    int* ctl = reinterpret_cast<int*>(cf + kBeamMaxK * kBeamMaxK);  // [0] candidates
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row0 = seq * p.beams, K = p.K;
    // a beam's base: scores[b] - log Σ exp, -inf for a dead one
    for (int b = warp; b < p.beams; b += kMergeThreads / 32) {
        const float s = p.scores[row0 + b];
        double d = -INFINITY;
        if (!dead_score(s)) {
            float top = -INFINITY;
            for (int c = lane; c < p.chunks; c += 32) top = fmaxf(top, p.tops[(long long)(row0 + b) * p.chunks + c]);
            top = warp_max(top);
            double sum = 0.;
            for (int c = lane; c < p.chunks; c += 32) {
                const long long l = (long long)(row0 + b) * p.chunks + c;
                const float t = p.tops[l];
                sum += p.sums[l] * (t == top ? 1. : exp((double)t - (double)top));
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
        const u64 k = p.keys[((long long)(row0 + b) * p.chunks + chunk) * K + c];
        if (!k) return false;
        const double x = (double)ordered_to_float((uint32_t)(k >> 32));
        s = double_ordered(base[b] + x);
        f = (unsigned)b * p.vocab + (0xFFFFFFFFu - (uint32_t)k);
        return true;
    };
    const int lists = p.beams * p.chunks;
    u64 ms = 0;
    unsigned mf = 0;
    bool have = false;
    if (tid < lists) {
        have = entry(tid, 0, ms, mf);
        hs[tid] = have ? ms : 0;
        hf[tid] = have ? mf : UINT_MAX;
    }
    __syncthreads();
    if (have) {
        int rank = 0;
        for (int i = 0; i < lists; ++i) rank += better(hs[i], hf[i], ms, mf);
        // only the K lists with the best heads can hold the K best
        if (rank < K) {
            for (int c = 0; c < K; ++c) {
                u64 s;
                unsigned f;
                if (!entry(tid, c, s, f)) break;
                const int at = atomicAdd(&ctl[0], 1);
                cs[at] = s;
                cf[at] = f;
            }
        }
    }
    __syncthreads();
    const int cnt = ctl[0];
    for (int c = tid; c < cnt; c += kMergeThreads) {
        const u64 s = cs[c];
        const unsigned f = cf[c];
        int rank = 0;
        for (int i = 0; i < cnt; ++i) rank += better(cs[i], cf[i], s, f);
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

size_t beam_ws(const af_beam_select_args& a) {
    const size_t lists = (size_t)a.n_seq * a.n_beams * ((a.vocab + kBeamChunk - 1) / kBeamChunk);
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
    p.chunks = (a->vocab + kBeamChunk - 1) / kBeamChunk;
    p.vec = !(reinterpret_cast<uintptr_t>(a->logits) & 15) && p.stride % 4 == 0;
    p.out_score = a->out_score;
    p.out_beam = a->out_beam;
    p.out_token = a->out_token;
    const size_t lists = (size_t)a->n_seq * a->n_beams * p.chunks;
    p.keys = static_cast<u64*>(a->ws);
    p.sums = reinterpret_cast<double*>(p.keys + lists * p.K);
    p.tops = reinterpret_cast<float*>(p.sums + lists);
    beam_chunk_kernel<<<dim3(p.chunks, p.n_seq * p.beams), kBeamThreads, 0, stream>>>(p);
    AF_CUDA_TRY(cudaGetLastError());
    AF_CUDA_TRY(cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMergeSmem));
    beam_merge_kernel<<<p.n_seq, kMergeThreads, kMergeSmem, stream>>>(p);
    return cudaGetLastError();
}
