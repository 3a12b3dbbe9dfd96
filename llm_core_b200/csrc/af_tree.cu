// af_tree.cu — attention of drafted tokens over a paged cache
// (af_attention_tree_f32): the nodes of every sequence see its cached
// positions and, by a bit mask, one another.
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
            set_err(kErrBadArgs);
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

cudaError_t refuse(const std::string& why) {
    set_last_error("af_attention_tree_f32: " + why);
    return cudaErrorInvalidValue;
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" size_t af_attention_tree_f32_workspace(const af_attention_tree_args*) { return 0; }

extern "C" cudaError_t af_attention_tree_f32(const af_attention_tree_args* a, cudaStream_t stream) {
    if (!a) return refuse("null arguments");
    std::string why = kv_cache_wrong(a->kv);
    if (why.empty()) why = kv_batch_wrong(a->batch, a->kv, true);
    if (!why.empty()) return refuse(why);
    if (a->layer < 0 || a->layer >= a->kv.n_layers) return refuse("layer outside the cache");
    if (a->n_rows < 0 || a->n_heads <= 0 || a->n_heads > 65535 || a->n_heads % a->kv.n_kv_heads)
        return refuse("need n_rows >= 0 and n_heads a multiple of n_kv_heads");
    if (a->max_len < 0) return refuse("max_len must not be negative");
    if (a->n_rows == 0 || a->batch.n_seq == 0) return cudaSuccess;
    if (!a->q || !a->out) return refuse("null q or out");
    if (a->mask && (a->mask_words <= 0 || (long long)a->mask_words * 64 < a->batch.max_nodes))
        return refuse("mask_words must cover max_nodes");
    const long long qd = (long long)a->n_heads * a->kv.head_dim;
    if ((a->q_stride && a->q_stride < qd) || (a->out_stride && a->out_stride < qd))
        return refuse("a row stride is shorter than a row");
    TreeParams p = {};
    p.kv = kv_view(a->kv);
    p.b = kv_batch(a->batch);
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
    const dim3 grid(a->n_rows, a->n_heads);
    switch (a->kv.type) {
        case AF_KV_F32: tree_row_kernel<AF_KV_F32><<<grid, kTreeThreads, 0, stream>>>(p); break;
        case AF_KV_F16: tree_row_kernel<AF_KV_F16><<<grid, kTreeThreads, 0, stream>>>(p); break;
        default: tree_row_kernel<AF_KV_BF16><<<grid, kTreeThreads, 0, stream>>>(p); break;
    }
    return cudaGetLastError();
}
