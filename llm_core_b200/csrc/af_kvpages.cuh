// af_kvpages.cuh — the paged key/value cache as the kernels see it, and the
// host checks that its entry points share (af_kv_cache, af_kv_batch).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <string>

#include "af_common.cuh"

namespace af {

// af_kv_cache with its sizes in bytes and its page size as a shift.
struct KvView {
    uint8_t *k, *v;
    long long layer_bytes;
    int row_bytes;   // one position: n_kv_heads * head_dim values
    int ps_shift;    // page_size = 1 << ps_shift
    int n_layers, n_pages, kv_heads, hd;
};

struct KvBatch {
    const int *table, *len, *first;
    int n_seq, max_blocks, max_nodes;
    int* err;  // the device error word
};

inline int kv_type_bytes(int type) { return type == AF_KV_F32 ? 4 : 2; }

inline KvView kv_view(const af_kv_cache& c) {
    KvView v = {};
    v.k = static_cast<uint8_t*>(c.k);
    v.v = static_cast<uint8_t*>(c.v);
    const int size = kv_type_bytes(c.type);
    v.row_bytes = c.n_kv_heads * c.head_dim * size;
    v.layer_bytes = (c.layer_stride ? (long long)c.layer_stride
                                    : (long long)c.n_pages * c.page_size * c.n_kv_heads * c.head_dim) * size;
    while ((1 << v.ps_shift) < c.page_size) ++v.ps_shift;
    v.n_layers = c.n_layers;
    v.n_pages = c.n_pages;
    v.kv_heads = c.n_kv_heads;
    v.hd = c.head_dim;
    return v;
}

inline KvBatch kv_batch(const af_kv_batch& b, int* err) {
    return {b.block_table, b.len, b.first, b.n_seq, b.max_blocks, b.max_nodes, err};
}

// "" if the cache's shape and pointers can be served, else what is wrong.
std::string kv_cache_wrong(const af_kv_cache& c);
// The same for a batch of `n_rows` node rows (nodes false: a call that has none).
std::string kv_batch_wrong(const af_kv_batch& b, const af_kv_cache& c, bool nodes);

// Page block b of sequence s, or -1 (nothing held, or an id outside the pool).
__device__ __forceinline__ int kv_page(const KvBatch& b, int n_pages, int s, int blk) {
    if (blk < 0 || blk >= b.max_blocks) return -1;
    const long long at = (long long)s * b.max_blocks + blk;
    const long long id = b.table ? (long long)b.table[at] : at;
    return id >= 0 && id < n_pages ? (int)id : -1;
}

// Byte offset of a position's row in a layer of the K or the V pool, -1 where
// the sequence holds no page for it.  64-bit: a layer may pass 4 GB.
__device__ __forceinline__ long long kv_row(const KvView& v, const KvBatch& b, int s, int pos) {
    const int page = kv_page(b, v.n_pages, s, pos >> v.ps_shift);
    if (page < 0) return -1;
    return (((long long)page << v.ps_shift) + (pos & ((1 << v.ps_shift) - 1))) * v.row_bytes;
}

// Rows [r0, r0 + n) of the call's row arrays are sequence s's nodes; a count
// that does not fit the call sets the error word and gives none.
__device__ __forceinline__ void kv_nodes(const KvBatch& b, int n_rows, int s, int& r0, int& n) {
    if (b.first) {
        r0 = b.first[s];
        n = b.first[s + 1] - r0;
        if (r0 < 0 || n < 0 || n > b.max_nodes || r0 > n_rows - n) {
            set_err_at(b.err, kErrBadArgs);
            n = 0;
        }
    } else {
        r0 = s * b.max_nodes;
        n = min(b.max_nodes, max(0, n_rows - r0));
    }
}

// Cached positions of sequence s: its length where it and `n` more fit its
// table, else the error word and -1.
__device__ __forceinline__ int kv_len(const KvView& v, const KvBatch& b, int s, int n) {
    const int len = b.len[s];
    if (len < 0 || (long long)len + n > ((long long)b.max_blocks << v.ps_shift)) {
        set_err_at(b.err, kErrBadArgs);
        return -1;
    }
    return len;
}

template <int TYPE>
struct KvElem;
template <>
struct KvElem<AF_KV_F32> {
    using T = float;
    static __device__ __forceinline__ float load(const float& x) { return x; }
    static __device__ __forceinline__ float round(float x) { return x; }
};
template <>
struct KvElem<AF_KV_F16> {
    using T = __half;
    static __device__ __forceinline__ float load(const __half& x) { return __half2float(x); }
    static __device__ __forceinline__ __half round(float x) { return __float2half_rn(x); }
};
template <>
struct KvElem<AF_KV_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float load(const __nv_bfloat16& x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 round(float x) { return __float2bfloat16_rn(x); }
};

}  // namespace af
