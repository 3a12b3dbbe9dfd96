"""af_kv_store_f32 where rows are so many that a warp takes one: against the
same rows stored a few at a time."""
import numpy as np
import pytest
import torch

import kv_helpers as kh
from llm_core_b200 import _lib

pytestmark = pytest.mark.gpu


def store(lib, cache, q, k, v, out, length, first, n_rows, top, cos, sin, order, norms, depth=None):
    a = _lib.KvStoreArgs()
    a.kv, a.batch = cache.struct(), cache.batch(length, first, top)
    a.layer, a.n_rows, a.n_heads, a.n_ctx = 0, n_rows, q.shape[1], cos.shape[0]
    a.q, a.k, a.v, a.q_out = kh.ptr(q), kh.ptr(k), kh.ptr(v), kh.ptr(out)
    a.cos, a.sin, a.depth = kh.ptr(cos), kh.ptr(sin), kh.ptr(depth)
    a.qk_norm_order, a.q_norm, a.k_norm, a.eps = order, kh.ptr(norms[0]), kh.ptr(norms[1]), 1e-5
    a.keep = (q, k, v, out, cos, sin, length, first, depth, norms)
    kh.call(lib, "af_kv_store_f32", a)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 64), (3, 1, 128), (40, 8, 64)])
@pytest.mark.parametrize("order", [0, 1, 2])
def test_many_rows_as_few(gpu, kv, H, KV, hd, order):
    counts = [0, 1, 1500, 37, 700, 11]  # 2,249 rows, and 3 behind the last sequence
    lengths = [5, 0, 20, 300, 1, 63]
    n = sum(counts)
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn((n + 3, h, hd), device="cuda", generator=g) for h in (H, KV, KV))
    cos, sin = (torch.randn((2048, hd // 2), device="cuda", generator=g) for _ in range(2))
    norms = [torch.rand(hd, device="cuda", generator=g) + 0.5 for _ in range(2)]
    depth = torch.randint(0, 40, (n + 3,), device="cuda", dtype=torch.int32, generator=g)
    caches = [kh.Cache(kv, KV, hd, [a + b for a, b in zip(lengths, counts)], fill=7.0, seed=1) for _ in range(2)]
    outs = [torch.full_like(q, 7.0) for _ in range(2)]
    first = np.concatenate([[0], np.cumsum(counts)])
    store(gpu, caches[0], q, k, v, outs[0], kh.ints(lengths), kh.ints(first), n + 3, 1500, cos, sin, order, norms, depth)
    assert kh.device_error(gpu) == 0
    for s, m in enumerate(counts):  # a sequence at a time, at most 500 rows
        for a in range(0, m, 500):
            b = min(m, a + 500)
            lo, hi = int(first[s]) + a, int(first[s]) + b
            f = [0] * (s + 1) + [b - a] * (len(counts) - s)
            at = list(lengths)
            at[s] += a
            dp = depth[lo:hi] - a  # rotated at length + depth
            store(gpu, caches[1], q[lo:hi].contiguous(), k[lo:hi].contiguous(), v[lo:hi].contiguous(),
                  outs[1][lo:hi], kh.ints(at), kh.ints(f), hi - lo, 500, cos, sin, order, norms, dp.contiguous())
    assert torch.equal(outs[0], outs[1])
    assert (outs[0][n:] == 7).all()
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
