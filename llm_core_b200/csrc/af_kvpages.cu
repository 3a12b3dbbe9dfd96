// af_kvpages.cu — the paged key/value cache: new tokens written into pages
// (af_kv_store_f32), sequences forked, reordered, extended and freed
// (af_kv_fork), accepted rows moved together (af_kv_compact).
#include <climits>
#include <cstdint>
#include <type_traits>

#include "af_kvpages.cuh"
#include "af_ops.cuh"

namespace af {

std::string kv_cache_wrong(const af_kv_cache& c) {
    if (c.type != AF_KV_F32 && c.type != AF_KV_F16 && c.type != AF_KV_BF16) return "unknown cache type";
    if (c.n_layers <= 0 || c.n_pages <= 0 || c.n_kv_heads <= 0) return "n_layers, n_pages and n_kv_heads must be positive";
    if (c.page_size <= 0 || c.page_size > (1 << 20) || (c.page_size & (c.page_size - 1)))
        return "page_size must be a power of two up to 2^20";
    if (c.head_dim <= 0 || c.head_dim > 256 || c.head_dim % 8) return "head_dim must be a multiple of 8 up to 256";
    if (c.n_kv_heads > 65535 || c.n_layers > 32767) return "n_kv_heads must be at most 65535, n_layers at most 32767";
    if ((long long)c.n_pages * c.page_size > INT_MAX) return "n_pages * page_size must be below 2^31";
    const long long dense = (long long)c.n_pages * c.page_size * c.n_kv_heads * c.head_dim;
    if (c.layer_stride < 0 || c.layer_stride % 8 || (c.layer_stride && c.n_layers > 1 && c.layer_stride < dense))
        return "layer_stride must be 0 or a multiple of 8 that holds a layer";
    if (!c.k || !c.v) return "null cache";
    if ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15) return "k and v must be 16-byte aligned";
    return "";
}

std::string kv_batch_wrong(const af_kv_batch& b, const af_kv_cache& c, bool nodes) {
    if (b.n_seq < 0 || b.n_seq > 65535) return "n_seq must be in 0..65535";
    if (b.max_blocks <= 0 || (long long)b.max_blocks * c.page_size > (1ll << 30))
        return "max_blocks must be positive and max_blocks * page_size at most 2^30";
    if (nodes && b.max_nodes <= 0) return "max_nodes must be positive";
    if (nodes && !b.first && (long long)b.n_seq * b.max_nodes > INT_MAX) return "too many rows";
    if (b.n_seq > 0 && !b.len) return "null len";
    return "";
}

namespace {

// ------------------------------------------------------------------- store

constexpr int kStoreThreads = 256;

struct StoreParams {
    KvView kv;
    KvBatch b;
    int layer, n_rows, n_ctx, H, order;
    const float *q, *k, *v;
    float* q_out;
    long long qs, ks, vs, os;
    const int* depth;
    const float *cos_t, *sin_t, *q_norm, *k_norm;
    float eps;
};

// A row's sequence (-1: a row behind the last), node and cached length, found
// by the whole block: every load that does not need another's result goes out
// with it.
struct StorePlace {
    int seq, node, len;
};
__device__ __forceinline__ void store_row(const StoreParams& p, int row, StorePlace* out) {
    const int tid = threadIdx.x;
    if (tid == 0) out->seq = -1;
    __syncthreads();
    if (p.b.first) {
        for (int s = tid; s < p.b.n_seq; s += blockDim.x) {
            const int f = p.b.first[s], e = p.b.first[s + 1], len = p.b.len[s];
            if (f <= row && row < e) *out = {s, row - f, len};
        }
    } else if (tid == 0 && row / p.b.max_nodes < p.b.n_seq) {
        *out = {row / p.b.max_nodes, row % p.b.max_nodes, p.b.len[row / p.b.max_nodes]};
    }
    __syncthreads();
}

// The same by one warp.
__device__ __forceinline__ StorePlace store_row_warp(const StoreParams& p, int row) {
    const int lane = threadIdx.x & 31;
    StorePlace w = {-1, 0, 0};
    if (!p.b.first) {
        const int s = row / p.b.max_nodes;
        if (s < p.b.n_seq) w = {s, row % p.b.max_nodes, p.b.len[s]};
        return w;
    }
    for (int s0 = 0; s0 < p.b.n_seq; s0 += 32) {
        const int s = s0 + lane;
        StorePlace mine = {-1, 0, 0};
        if (s < p.b.n_seq) {
            const int f = p.b.first[s], e = p.b.first[s + 1], len = p.b.len[s];
            if (f <= row && row < e) mine = {s, row - f, len};
        }
        const unsigned hit = __ballot_sync(0xffffffffu, mine.seq >= 0);
        if (hit) {
            const int src = 31 - __clz(hit);  // first[] that does not rise: the last one, as a block takes it or another
            w.seq = __shfl_sync(0xffffffffu, mine.seq, src);
            w.node = __shfl_sync(0xffffffffu, mine.node, src);
            w.len = __shfl_sync(0xffffffffu, mine.len, src);
        }
    }
    return w;
}

// Where the row's rotation and cache position are; false (and the error word) where it has none.
__device__ __forceinline__ bool store_place(const StoreParams& p, const StorePlace& w, int depth, long long& at, long long& slot) {
    at = (long long)w.len + (p.depth ? depth : w.node);
    if (w.len < 0 || at < 0 || at >= p.n_ctx || w.node < 0 || w.node >= p.b.max_nodes) {
        set_err_at(p.b.err, kErrBadArgs);
        return false;
    }
    const long long pos = (long long)w.len + w.node;
    slot = pos < ((long long)p.b.max_blocks << p.kv.ps_shift) ? kv_row(p.kv, p.b, w.seq, (int)pos) : -1;
    return true;
}

// A block per row, its heads (queries, keys, values) over the warps, or, where
// rows are many, a warp per row.  HD 64 and 128 with 16-byte rows: a lane holds 4
// values, HD/4 lanes a head, the partner of a rotation sits HD/8 lanes away; a
// warp's first heads (U) are loaded before the row's place is known.  Bound by
// memory, q, k, v once in, once out, and by a row's chain of loads (counts, then
// table and rotation), hidden behind other rows': 8 sequences of up to 509 rows,
// 16/2 heads of 128, bf16, 17.5 us a warp a row (3.9 TB/s), 20.5 a block of 8 warps,
// 18.3 of 4; one row 2.9 us, a launch.  Measured and not taken: 2 to 8 rows a block with the next row's loads
// ahead, 27 us (64 registers, fewer blocks an SM).
template <int TYPE, int HD, bool WARP>
__global__ void __launch_bounds__(kStoreThreads, WARP ? 4 : 5) kv_store_vec_kernel(StoreParams p) {
    constexpr int LH = HD / 4, HPW = 32 / LH, W = WARP ? 1 : kStoreThreads / 32, U = WARP ? 5 : 3;
    using E = KvElem<TYPE>;
    __shared__ StorePlace shared;
    const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = WARP ? blockIdx.x * (kStoreThreads / 32) + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && row >= p.n_rows) return;
    const int sub = lane / LH, col = lane % LH, KV = p.kv.kv_heads, heads = p.H + 2 * KV;
    const float* q = p.q + (long long)row * p.qs + 4 * col;
    const float* k = p.k + (long long)row * p.ks + 4 * col - p.H * HD;         // by the head's number
    const float* v = p.v + (long long)row * p.vs + 4 * col - (p.H + KV) * HD;
    auto load = [&](int h) -> float4 {
        return __ldcs(reinterpret_cast<const float4*>((h < p.H ? q : h < p.H + KV ? k : v) + h * HD));
    };
    float4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int h = (u * W + warp) * HPW + sub;
        if (h < heads) x[u] = load(h);
    }
    const int depth = p.depth ? p.depth[row] : 0;
    StorePlace where;
    if (WARP) {
        where = store_row_warp(p, row);
    } else {
        store_row(p, row, &shared);
        where = shared;
    }
    if (where.seq < 0) return;
    long long at, slot;
    if (!store_place(p, where, depth, at, slot)) return;
    const float4 c = *reinterpret_cast<const float4*>(p.cos_t + at * (HD / 2) + 4 * (col % (LH / 2)));
    float4 sn = *reinterpret_cast<const float4*>(p.sin_t + at * (HD / 2) + 4 * (col % (LH / 2)));
    if (col < LH / 2) sn = make_float4(-sn.x, -sn.y, -sn.z, -sn.w);
    if (slot < 0 && tid == 0) set_err_at(p.b.err, kErrBadArgs);
    float* qo = p.q_out + (long long)row * p.os + 4 * col;
    typename E::T* ko = reinterpret_cast<typename E::T*>(p.kv.k + (long long)p.layer * p.kv.layer_bytes + slot) + 4 * col - p.H * HD;
    typename E::T* vo = reinterpret_cast<typename E::T*>(p.kv.v + (long long)p.layer * p.kv.layer_bytes + slot) + 4 * col - (p.H + KV) * HD;
    for (int h0 = 0; h0 < heads; h0 += U * W * HPW) {
        if (h0) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + (u * W + warp) * HPW + sub;
                if (h < heads) x[u] = load(h);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (h0 + (u * W + warp) * HPW >= heads) break;  // the same in the whole warp
            const int h = h0 + (u * W + warp) * HPW + sub;
            const bool isv = h >= p.H + KV;
            float4 y = x[u];
            auto norm = [&]() {  // the heads of a warp may differ in kind: all lanes add up
                const float* nw = isv ? nullptr : h < p.H ? p.q_norm : p.k_norm;
                float ss = y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
#pragma unroll
                for (int o = 1; o < LH; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (nw) {
                    const float sc = rsqrtf(ss * (1.f / HD) + p.eps);
                    const float4 w = *reinterpret_cast<const float4*>(nw + 4 * col);
                    y.x = w.x * (y.x * sc), y.y = w.y * (y.y * sc), y.z = w.z * (y.z * sc), y.w = w.w * (y.w * sc);
                }
            };
            if (p.order == 1) norm();
            float4 o;
            o.x = __shfl_xor_sync(0xffffffffu, y.x, LH / 2), o.y = __shfl_xor_sync(0xffffffffu, y.y, LH / 2);
            o.z = __shfl_xor_sync(0xffffffffu, y.z, LH / 2), o.w = __shfl_xor_sync(0xffffffffu, y.w, LH / 2);
            if (!isv) {  // x0·cos - x1·sin in the first half, x1·cos + x0·sin in the second
                y.x = fmaf(y.x, c.x, o.x * sn.x), y.y = fmaf(y.y, c.y, o.y * sn.y);
                y.z = fmaf(y.z, c.z, o.z * sn.z), y.w = fmaf(y.w, c.w, o.w * sn.w);
            }
            if (p.order == 2) norm();
            if (h >= heads) continue;
            if (h < p.H) {
                *reinterpret_cast<float4*>(qo + h * HD) = y;
            } else if (slot >= 0) {
                typename E::T* dst = (isv ? vo : ko) + h * HD;
                if (TYPE == AF_KV_F32) {
                    *reinterpret_cast<float4*>(dst) = y;
                } else {
                    typename E::T r[4] = {E::round(y.x), E::round(y.y), E::round(y.z), E::round(y.w)};
                    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(r);
                }
            }
        }
    }
}

// Any head size and alignment: a warp per head, a lane the pairs (i, i + hd/2) for i = lane, lane + 32, ...
template <int TYPE>
__global__ void __launch_bounds__(kStoreThreads) kv_store_kernel(StoreParams p) {
    using E = KvElem<TYPE>;
    __shared__ StorePlace where;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int depth = p.depth ? p.depth[row] : 0;
    store_row(p, row, &where);
    if (where.seq < 0) return;
    long long at, slot;
    if (!store_place(p, where, depth, at, slot)) return;
    if (slot < 0 && tid == 0) set_err_at(p.b.err, kErrBadArgs);
    const int hd = p.kv.hd, half = hd / 2;
    const float* c = p.cos_t + at * half;
    const float* sn = p.sin_t + at * half;
    for (int h = warp; h < p.H + 2 * p.kv.kv_heads; h += kStoreThreads / 32) {
        const bool isq = h < p.H, isv = h >= p.H + p.kv.kv_heads;
        const int kvh = isv ? h - p.H - p.kv.kv_heads : h - p.H;
        const float* src = isq ? p.q + (long long)row * p.qs + (long long)h * hd
                               : (isv ? p.v + (long long)row * p.vs : p.k + (long long)row * p.ks) + (long long)kvh * hd;
        float a[4], b[4];
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = lane + 32 * j;
            a[j] = i < half ? src[i] : 0.f;
            b[j] = i < half ? src[i + half] : 0.f;
            ss += a[j] * a[j] + b[j] * b[j];
        }
        const float* nw = isv ? nullptr : (isq ? p.q_norm : p.k_norm);
        if (nw && p.order == 1) {
            const float sc = 1.f / sqrtf(warp_sum(ss) / (float)hd + p.eps);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = lane + 32 * j;
                if (i < half) {
                    a[j] = nw[i] * (a[j] * sc);
                    b[j] = nw[i + half] * (b[j] * sc);
                }
            }
        }
        if (!isv) {
            ss = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = lane + 32 * j;
                if (i < half) {
                    const float x = a[j], y = b[j], cc = c[i], s1 = sn[i];
                    a[j] = x * cc - y * s1;
                    b[j] = x * s1 + y * cc;
                    ss += a[j] * a[j] + b[j] * b[j];
                }
            }
        }
        if (nw && p.order == 2) {
            const float sc = 1.f / sqrtf(warp_sum(ss) / (float)hd + p.eps);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = lane + 32 * j;
                if (i < half) {
                    a[j] = nw[i] * (a[j] * sc);
                    b[j] = nw[i + half] * (b[j] * sc);
                }
            }
        }
        if (isq) {
            float* dst = p.q_out + (long long)row * p.os + (long long)h * hd;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = lane + 32 * j;
                if (i < half) {
                    dst[i] = a[j];
                    dst[i + half] = b[j];
                }
            }
        } else if (slot >= 0) {
            uint8_t* pool = (isv ? p.kv.v : p.kv.k) + (long long)p.layer * p.kv.layer_bytes + slot;
            auto* dst = reinterpret_cast<typename E::T*>(pool) + (long long)kvh * hd;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = lane + 32 * j;
                if (i < half) {
                    dst[i] = E::round(a[j]);
                    dst[i + half] = E::round(b[j]);
                }
            }
        }
    }
}

// -------------------------------------------------------------------- fork

constexpr int kForkThreads = 1024;
constexpr int kForkMax = 4096;  // sequences of a call

constexpr int kForkAhead = 4;   // reference counts a thread loads before anything else

struct ForkParams {
    KvView kv;
    KvBatch in;  // table_in, len_in; n_seq = n_in
    const int *ref_in, *parent, *n_new;
    int *table_out, *len_out, *ref_out, *n_short;
    int n_out;
    int4* copies;  // [n_out] source page, destination page, rows
    int* fresh;    // [n_pages] the free pages taken, in order
    int* before;   // [n_pages] the counts as they came, where ref_out is ref_in
};

// What an output needs: pages behind its `full` whole ones up to `need`.
struct ForkNeed {
    int parent, len, need, base;  // base: its first page among those taken
};

constexpr int kForkSmem = kForkMax * (4 + 16);

// The bookkeeping of a fork, one block: which output is a parent's first
// child, how many pages each output takes, which pages are free, and then
// tables, reference counts and the list of pages to copy.  Bound by latency: a
// chain of dependent loads (parent, length; page, count; page again), so what
// does not hang on it is loaded first and the counts go out as reductions.
__global__ void __launch_bounds__(kForkThreads) kv_fork_kernel(ForkParams p) {
    extern __shared__ __align__(16) uint8_t sm[];
    ForkNeed* needs = reinterpret_cast<ForkNeed*>(sm);        // [n_out]
    int* eldest = reinterpret_cast<int*>(needs + kForkMax);  // [n_in]
    __shared__ int wsum[32];
    __shared__ int s_total;
    __shared__ unsigned long long s_missing;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_pages = p.kv.n_pages, nb = p.in.max_blocks;
    const bool in_place = p.ref_out == p.ref_in;
    const int* ref = in_place ? p.before : p.ref_in;  // the counts as they came
    pdl_launch_dependents();                          // the copies may start launching
    int held[kForkAhead];
#pragma unroll
    for (int e = 0; e < kForkAhead; ++e) {
        const int page = e * kForkThreads + tid;
        held[e] = page < n_pages ? p.ref_in[page] : 1;
    }
    for (int j = tid; j < p.in.n_seq; j += kForkThreads) eldest[j] = INT_MAX;
    if (tid == 0) s_missing = 0;
    __syncthreads();
    for (int i = tid; i < p.n_out; i += kForkThreads) {
        const int j = p.parent[i], more = p.n_new ? max(0, p.n_new[i]) : 0;
        ForkNeed n = {j >= 0 && j < p.in.n_seq ? j : -1, 0, 0, 0};
        if (n.parent >= 0) {
            n.len = kv_len(p.kv, p.in, j, 0);
            if (n.len < 0) n.parent = -1, n.len = 0;
        }
        if (n.parent >= 0) atomicMin(&eldest[j], i);
        const long long blocks = ((long long)n.len + more + (1 << p.kv.ps_shift) - 1) >> p.kv.ps_shift;
        n.need = (int)min(blocks, (long long)nb);
        if (blocks > n.need) atomicAdd(&s_missing, (unsigned long long)(blocks - n.need));
        needs[i] = n;
    }
    // the counts, where they go
#pragma unroll
    for (int e = 0; e < kForkAhead; ++e) {
        const int page = e * kForkThreads + tid;
        if (page < n_pages) (in_place ? p.before : p.ref_out)[page] = held[e];
    }
    for (int page = kForkAhead * kForkThreads + tid; page < n_pages; page += kForkThreads)
        (in_place ? p.before : p.ref_out)[page] = p.ref_in[page];
    __syncthreads();
    auto keeps = [&](int parent, int b) {  // whether the first child of `parent` keeps its page of block b
        const int page = kv_page(p.in, n_pages, parent, b);
        return page >= 0 && ref[page] == 1;
    };
    // pages that each output takes
    for (int i = warp; i < p.n_out; i += kForkThreads / 32) {
        const ForkNeed n = needs[i];
        const int full = n.len >> p.kv.ps_shift;
        int cnt = max(0, n.need - full);
        if (n.parent >= 0 && eldest[n.parent] == i) {
            cnt = 0;
            for (int b = full + lane; b < n.need; b += 32) cnt += !keeps(n.parent, b);
            cnt = __reduce_add_sync(0xffffffffu, cnt);
        }
        __syncwarp();
        if (lane == 0) needs[i].base = cnt;
    }
    __syncthreads();
    {  // exclusive prefix sum of base
        constexpr int per = kForkMax / kForkThreads;
        int v[per], sum = 0;
#pragma unroll
        for (int e = 0; e < per; ++e) {
            const int i = tid * per + e;
            v[e] = i < p.n_out ? needs[i].base : 0;
            sum += v[e];
        }
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) wsum[warp] = inc;
        __syncthreads();
        int front = 0;
        for (int w = 0; w < warp; ++w) front += wsum[w];
        int at = front + inc - sum;
#pragma unroll
        for (int e = 0; e < per; ++e) {
            const int i = tid * per + e;
            if (i < p.n_out) needs[i].base = at;
            at += v[e];
        }
        if (tid == kForkThreads - 1) s_total = at;
    }
    __syncthreads();
    // the lowest s_total pages that nobody holds, in order
    const int total = s_total;
    int found = 0;
    for (int e = 0; e * kForkThreads < n_pages && found < total; ++e) {
        const int page = e * kForkThreads + tid;
        int count = 1;
        if (e < kForkAhead) {
#pragma unroll
            for (int k = 0; k < kForkAhead; ++k)
                if (k == e) count = held[k];
        } else if (page < n_pages) {
            count = ref[page];
        }
        const unsigned m = __ballot_sync(0xffffffffu, count == 0);
        if (lane == 0) wsum[warp] = __popc(m);
        __syncthreads();
        const int mine = wsum[lane];
        const int front = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0);
        const int rank = found + front + __popc(m & ((1u << lane) - 1));
        if (count == 0 && rank < total) p.fresh[rank] = page;
        found += __reduce_add_sync(0xffffffffu, mine);
        __syncthreads();
    }
    const int avail = min(found, total);
    // one off for every entry of the inputs
    for (long long e = tid; e < (long long)p.in.n_seq * nb; e += kForkThreads) {
        const int page = p.in.table[e];
        if (page >= 0 && page < n_pages) atomicSub(&p.ref_out[page], 1);
        else if (page != -1) set_err_at(p.in.err, kErrBadArgs);  // nobody's page
    }
    int missing = 0;
    for (int i = warp; i < p.n_out; i += kForkThreads / 32) {
        const ForkNeed n = needs[i];
        const bool first = n.parent >= 0 && eldest[n.parent] == i;
        const int full = n.len >> p.kv.ps_shift, rows = n.len & ((1 << p.kv.ps_shift) - 1);
        int taken = n.base, len = n.len;
        for (int b0 = 0; b0 < nb; b0 += 32) {
            const int b = b0 + lane;
            const int old = n.parent >= 0 && b < n.need ? kv_page(p.in, n_pages, n.parent, b) : -1;
            const bool shared = b < full;
            const bool keep = !shared && b < n.need && first && old >= 0 && ref[old] == 1;
            const bool take = !shared && !keep && b < n.need;
            const unsigned m = __ballot_sync(0xffffffffu, take);
            int page = shared || keep ? old : -1;
            if (take) {
                const int rank = taken + __popc(m & ((1u << lane) - 1));
                if (rank < avail) page = p.fresh[rank];
                else ++missing;
            }
            taken += __popc(m);
            if (b < nb) p.table_out[(long long)i * nb + b] = page;
            if (page >= 0) atomicAdd(&p.ref_out[page], 1);
            // the partly filled page
            if (b == full && b < nb) p.copies[i] = make_int4(old, page, take && page >= 0 && old >= 0 ? rows : 0, 0);
            if (__any_sync(0xffffffffu, b == full && rows > 0 && page < 0)) len = min(len, full << p.kv.ps_shift);
            // a position below the length that the parent holds no page for: the child ends in front of it
            const unsigned hole = __ballot_sync(0xffffffffu, b < full + (rows > 0) && old < 0);
            if (hole) {
                len = min(len, (b0 + __ffs(hole) - 1) << p.kv.ps_shift);
                set_err_at(p.in.err, kErrBadArgs);
            }
        }
        if (lane == 0) {
            if (full >= nb) p.copies[i] = make_int4(-1, -1, 0, 0);
            p.len_out[i] = len;
        }
    }
    missing = __reduce_add_sync(0xffffffffu, missing);
    if (lane == 0 && missing) atomicAdd(&s_missing, (unsigned long long)missing);
    __syncthreads();
    if (tid == 0) *p.n_short = (int)min(s_missing, (unsigned long long)INT_MAX);
}

constexpr int kCopyThreads = 256;

// Block (i, layer, K or V): the rows of output i's partly filled page, one
// contiguous range.  Bound by memory; 4 loads of 16 bytes a thread in flight:
// 4 sequences of 8 beams, 32 layers of 32 heads of 128, bf16, 22.6 us with the
// bookkeeping (110 MB, 4.9 TB/s); 4 beams over 22 layers 6.4 us, two launches.
__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(KvView kv, const int4* copies) {
    pdl_wait();
    const int4 c = copies[blockIdx.x];
    if (c.z <= 0) return;
    uint8_t* pool = (blockIdx.z ? kv.v : kv.k) + (long long)blockIdx.y * kv.layer_bytes;
    const uint4* src = reinterpret_cast<const uint4*>(pool + ((long long)c.x << kv.ps_shift) * kv.row_bytes);
    uint4* dst = reinterpret_cast<uint4*>(pool + ((long long)c.y << kv.ps_shift) * kv.row_bytes);
    const long long n = (long long)c.z * kv.row_bytes / 16;
    for (long long i = threadIdx.x; i < n; i += 4 * kCopyThreads) {
        uint4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * kCopyThreads < n) x[j] = __ldcs(src + i + j * kCopyThreads);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * kCopyThreads < n) dst[i + j * kCopyThreads] = x[j];
    }
}

// ----------------------------------------------------------------- compact

constexpr int kCompactThreads = 128;
constexpr int kCompactVec = 2;    // 16-byte columns of a thread
constexpr int kCompactRows = 8;   // rows read before the first is written
constexpr int kCompactPath = 128; // of a path at a time

// A sequence's path, checked by the whole block.
__device__ __forceinline__ bool path_bad(const KvView& kv, const KvBatch& b, const int* pa, int s, int n, int max_path, int len) {
    bool bad = len < 0 || n < 0 || n > max_path;
    for (int i = threadIdx.x; i < n && !bad; i += blockDim.x) {
        const int x = pa[i];
        bad = x < 0 || (i && x <= pa[i - 1]) || (long long)len + x >= ((long long)b.max_blocks << kv.ps_shift) ||
              kv_row(kv, b, s, len + x) < 0 || kv_row(kv, b, s, len + i) < 0;
    }
    return __syncthreads_or(bad);
}

// Block (columns, layer and K or V, sequence): a thread moves its columns of
// every row of the path, in path order.  A row's source is never in front of
// its destination and destinations rise, so a row is read before it is
// written over: dst i = len + i <= len + path[i'] for every i' >= i.  Bound by
// memory; each block first turns the path into row offsets, side by side: 24
// sequences, paths of up to 6, 32 layers of 32 heads of 128, f16, 25.6 us (126 MB,
// 4.9 TB/s); one path of 4 over 22 layers 3.0 us, a launch.
__global__ void __launch_bounds__(kCompactThreads) kv_compact_kernel(KvView kv, KvBatch b, const int* path,
                                                                     const int* n_path, int max_path, int* len_out) {
    __shared__ long long from[kCompactPath], to[kCompactPath];
    const int s = blockIdx.z, layer = blockIdx.y >> 1, tid = threadIdx.x;
    const int* pa = path + (long long)s * max_path;
    const int n = n_path[s], len = b.len[s];
    const bool bad = path_bad(kv, b, pa, s, n, max_path, len);
    if (tid == 0 && blockIdx.x == 0 && blockIdx.y == 0) {
        if (bad) set_err_at(b.err, kErrBadArgs);
        if (len_out) len_out[s] = bad ? len : len + n;
    }
    if (bad) return;
    const int col = (blockIdx.x * kCompactThreads + tid) * 16, step = gridDim.x * kCompactThreads * 16;
    uint8_t* pool = ((blockIdx.y & 1) ? kv.v : kv.k) + (long long)layer * kv.layer_bytes;
    for (int i0 = 0; i0 < n; i0 += kCompactPath) {
        const int m = min(kCompactPath, n - i0);
        __syncthreads();
        if (tid < m) {
            from[tid] = pa[i0 + tid] == i0 + tid ? -1 : kv_row(kv, b, s, len + pa[i0 + tid]);  // -1: in its place
            to[tid] = kv_row(kv, b, s, len + i0 + tid);
        }
        __syncthreads();
        for (int j0 = 0; j0 < m; j0 += kCompactRows) {
            uint4 x[kCompactRows][kCompactVec];
#pragma unroll
            for (int j = 0; j < kCompactRows; ++j)
#pragma unroll
                for (int v = 0; v < kCompactVec; ++v)
                    if (j0 + j < m && from[j0 + j] >= 0 && col + v * step < kv.row_bytes)
                        x[j][v] = *reinterpret_cast<const uint4*>(pool + from[j0 + j] + col + v * step);
#pragma unroll
            for (int j = 0; j < kCompactRows; ++j)
#pragma unroll
                for (int v = 0; v < kCompactVec; ++v)
                    if (j0 + j < m && from[j0 + j] >= 0 && col + v * step < kv.row_bytes)
                        *reinterpret_cast<uint4*>(pool + to[j0 + j] + col + v * step) = x[j][v];
        }
    }
}

// The new lengths where they replace the old, which the rows' blocks read.
__global__ void kv_compact_len_kernel(KvView kv, KvBatch b, const int* path, const int* n_path, int max_path,
                                      int* len_out) {
    const int s = blockIdx.x, n = n_path[s], len = b.len[s];
    const bool bad = path_bad(kv, b, path + (long long)s * max_path, s, n, max_path, len);
    if (threadIdx.x == 0) len_out[s] = bad ? len : len + n;
}

cudaError_t refuse(const char* what, const std::string& why) {
    set_last_error(std::string(what) + ": " + why);
    return cudaErrorInvalidValue;
}

size_t fork_ws(const af_kv_fork_args& a) {
    return (size_t)a.n_out * sizeof(int4) + 2 * (size_t)a.kv.n_pages * sizeof(int);
}

std::string fork_wrong(const af_kv_fork_args& a) {
    const std::string why = kv_cache_wrong(a.kv);
    if (!why.empty()) return why;
    if (a.n_in < 0 || a.n_in > kForkMax || a.n_out < 0 || a.n_out > kForkMax) return "n_in and n_out must be in 0..4096";
    if (a.max_blocks <= 0 || (long long)a.max_blocks * a.kv.page_size > (1ll << 30))
        return "max_blocks must be positive and max_blocks * page_size at most 2^30";
    if ((long long)a.n_out * a.max_blocks > INT_MAX) return "n_out * max_blocks must be below 2^31";
    if (!a.ref_in || !a.ref_out || !a.n_short) return "null ref_in, ref_out or n_short";
    if (a.n_in > 0 && (!a.table_in || !a.len_in)) return "null table_in or len_in";
    if (a.n_out > 0 && (!a.table_out || !a.len_out || !a.parent)) return "null table_out, len_out or parent";
    auto over = [](const void* x, size_t nx, const void* y, size_t ny) {
        const uintptr_t p = reinterpret_cast<uintptr_t>(x), q = reinterpret_cast<uintptr_t>(y);
        return nx && ny && p < q + ny && q < p + nx;
    };
    const size_t ti = (size_t)a.n_in * a.max_blocks * 4, to = (size_t)a.n_out * a.max_blocks * 4;
    if (over(a.table_in, ti, a.table_out, to) || over(a.len_in, (size_t)a.n_in * 4, a.len_out, (size_t)a.n_out * 4))
        return "table_out and len_out may not overlap the inputs";
    if (a.ref_in != a.ref_out && over(a.ref_in, (size_t)a.kv.n_pages * 4, a.ref_out, (size_t)a.kv.n_pages * 4))
        return "ref_out must be ref_in or apart from it";
    return "";
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" cudaError_t af_kv_store_f32(const af_kv_store_args* a, cudaStream_t stream) {
    const char* me = "af_kv_store_f32";
    if (!a) return refuse(me, "null arguments");
    std::string why = kv_cache_wrong(a->kv);
    if (why.empty()) why = kv_batch_wrong(a->batch, a->kv, true);
    if (!why.empty()) return refuse(me, why);
    if (a->layer < 0 || a->layer >= a->kv.n_layers) return refuse(me, "layer outside the cache");
    if (a->n_rows < 0 || a->n_heads <= 0 || a->n_ctx <= 0) return refuse(me, "need n_rows >= 0, n_heads > 0, n_ctx > 0");
    if (a->qk_norm_order < 0 || a->qk_norm_order > 2) return refuse(me, "qk_norm_order must be 0, 1 or 2");
    if (a->n_rows == 0 || a->batch.n_seq == 0) return cudaSuccess;
    if (!a->q || !a->k || !a->v || !a->q_out || !a->cos || !a->sin) return refuse(me, "null q, k, v, q_out, cos or sin");
    const long long qd = (long long)a->n_heads * a->kv.head_dim, kd = (long long)a->kv.n_kv_heads * a->kv.head_dim;
    if ((a->q_stride && a->q_stride < qd) || (a->q_out_stride && a->q_out_stride < qd) ||
        (a->k_stride && a->k_stride < kd) || (a->v_stride && a->v_stride < kd))
        return refuse(me, "a row stride is shorter than a row");
    if (a->q_out == a->q && (a->q_out_stride ? a->q_out_stride : qd) != (a->q_stride ? a->q_stride : qd))
        return refuse(me, "q_out in place needs q's stride");
    StoreParams p = {};
    int* err = nullptr;
    AF_CUDA_TRY(device_error_word(&err));
    p.kv = kv_view(a->kv);
    p.b = kv_batch(a->batch, err);
    p.layer = a->layer;
    p.n_rows = a->n_rows;
    p.n_ctx = a->n_ctx;
    p.H = a->n_heads;
    p.order = a->qk_norm_order;
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.q_out = a->q_out;
    p.qs = a->q_stride ? a->q_stride : qd;
    p.os = a->q_out_stride ? a->q_out_stride : qd;
    p.ks = a->k_stride ? a->k_stride : kd;
    p.vs = a->v_stride ? a->v_stride : kd;
    p.depth = a->depth;
    p.cos_t = a->cos;
    p.sin_t = a->sin;
    p.q_norm = a->q_norm;
    p.k_norm = a->k_norm;
    p.eps = a->eps;
    const int hd = a->kv.head_dim;
    auto vec = [](const void* x) { return !(reinterpret_cast<uintptr_t>(x) & 15); };
    const bool wide = (hd == 64 || hd == 128) && vec(p.q) && vec(p.k) && vec(p.v) && vec(p.q_out) && vec(p.cos_t) &&
                      vec(p.sin_t) && vec(p.q_norm) && vec(p.k_norm) && !((p.qs | p.ks | p.vs | p.os) & 3);
    auto go = [&](auto type) {
        constexpr int TYPE = decltype(type)::value;
        // A warp a row where rows are so many that a row's chain hides behind others', and short enough: a warp has 5
        // heads of 128 or 10 of 64 in flight and takes a row's heads in turn.  Block a row / warp a row, us:
        //   heads         rows  bf16         f32
        //   16/2 of 128   1,400  8.3 / 10.5   8.7 / 14.6     2,400 13.0 / 12.4  13.9 / 17.6     8,000 39.6 / 33.4  41.9 / 44.6
        //   16/8 of 128   1,400 11.2 / 16.1  12.7 / 25.6     2,400 18.5 / 18.8  20.9 / 30.3     8,000 53.9 / 47.0  59.1 / 68.8
        //   32/8 of 128   1,400 14.8 / 23.6  17.9 / 39.3     2,400 25.4 / 29.8  30.8 / 45.0     8,000 71.0 / 69.0  87.0 / 99.2
        //   32/32 of 128  1,400 25.9 / 45.5  34.3 / 76.9     2,400 43.1 / 52.0  57.8 / 84.4     8,000  124 / 123    168 / 190
        //   32/4 of 64    1,400  8.4 / 10.3   8.4 / 10.5     2,400 13.1 / 12.5  13.4 / 12.7     8,000 40.0 / 33.7  40.4 / 34.4
        const int values = (p.H + 2 * p.kv.kv_heads) * hd;
        const bool many = p.n_rows > 15 * 148 && values <= 4096 && (TYPE != AF_KV_F32 || hd == 64);
        const int packed = (p.n_rows + kStoreThreads / 32 - 1) / (kStoreThreads / 32);
        if (wide && hd == 64 && many) kv_store_vec_kernel<TYPE, 64, true><<<packed, kStoreThreads, 0, stream>>>(p);
        else if (wide && many) kv_store_vec_kernel<TYPE, 128, true><<<packed, kStoreThreads, 0, stream>>>(p);
        else if (wide && hd == 64) kv_store_vec_kernel<TYPE, 64, false><<<p.n_rows, kStoreThreads, 0, stream>>>(p);
        else if (wide) kv_store_vec_kernel<TYPE, 128, false><<<p.n_rows, kStoreThreads, 0, stream>>>(p);
        else kv_store_kernel<TYPE><<<p.n_rows, kStoreThreads, 0, stream>>>(p);
    };
    switch (a->kv.type) {
        case AF_KV_F32: go(std::integral_constant<int, AF_KV_F32>()); break;
        case AF_KV_F16: go(std::integral_constant<int, AF_KV_F16>()); break;
        default: go(std::integral_constant<int, AF_KV_BF16>()); break;
    }
    return cudaGetLastError();
}

extern "C" size_t af_kv_fork_workspace(const af_kv_fork_args* a) {
    if (!a || a->n_out < 0 || a->kv.n_pages < 0) return 0;
    return fork_ws(*a);
}

extern "C" cudaError_t af_kv_fork(const af_kv_fork_args* a, cudaStream_t stream) {
    const char* me = "af_kv_fork";
    if (!a) return refuse(me, "null arguments");
    const std::string why = fork_wrong(*a);
    if (!why.empty()) return refuse(me, why);
    if (!a->ws || a->ws_bytes < fork_ws(*a) || (reinterpret_cast<uintptr_t>(a->ws) & 15))
        return refuse(me, "ws must hold af_kv_fork_workspace bytes, 16-byte aligned");
    ForkParams p = {};
    p.kv = kv_view(a->kv);
    int* err = nullptr;
    AF_CUDA_TRY(device_error_word(&err));
    p.in = {a->table_in, a->len_in, nullptr, a->n_in, a->max_blocks, 0, err};
    p.ref_in = a->ref_in;
    p.parent = a->parent;
    p.n_new = a->n_new;
    p.table_out = a->table_out;
    p.len_out = a->len_out;
    p.ref_out = a->ref_out;
    p.n_short = a->n_short;
    p.n_out = a->n_out;
    p.copies = static_cast<int4*>(a->ws);
    p.fresh = reinterpret_cast<int*>(p.copies + a->n_out);
    p.before = p.fresh + a->kv.n_pages;
    AF_CUDA_TRY(cudaFuncSetAttribute(kv_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kForkSmem));
    kv_fork_kernel<<<1, kForkThreads, kForkSmem, stream>>>(p);
    AF_CUDA_TRY(cudaGetLastError());
    if (a->n_out == 0) return cudaSuccess;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a->n_out, a->kv.n_layers, 2);
    cfg.blockDim = dim3(kCopyThreads);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv_copy_kernel, p.kv, (const int4*)p.copies);
}

extern "C" cudaError_t af_kv_compact(const af_kv_compact_args* a, cudaStream_t stream) {
    const char* me = "af_kv_compact";
    if (!a) return refuse(me, "null arguments");
    std::string why = kv_cache_wrong(a->kv);
    if (why.empty()) why = kv_batch_wrong(a->batch, a->kv, false);
    if (!why.empty()) return refuse(me, why);
    if (a->max_path < 0) return refuse(me, "max_path must not be negative");
    if (a->batch.n_seq == 0) return cudaSuccess;
    if (!a->len_out || !a->n_path || (a->max_path > 0 && !a->path)) return refuse(me, "null path, n_path or len_out");
    const KvView kv = kv_view(a->kv);
    int* err = nullptr;
    AF_CUDA_TRY(device_error_word(&err));
    const KvBatch b = kv_batch(a->batch, err);
    const int per = kCompactThreads * kCompactVec * 16;
    const dim3 grid((kv.row_bytes + per - 1) / per, 2 * kv.n_layers, b.n_seq);
    const bool in_place = a->len_out == a->batch.len;
    kv_compact_kernel<<<grid, kCompactThreads, 0, stream>>>(kv, b, a->path, a->n_path, a->max_path,
                                                           in_place ? nullptr : a->len_out);
    AF_CUDA_TRY(cudaGetLastError());
    if (in_place)
        kv_compact_len_kernel<<<b.n_seq, 32, 0, stream>>>(kv, b, a->path, a->n_path, a->max_path, a->len_out);
    return cudaGetLastError();
}
