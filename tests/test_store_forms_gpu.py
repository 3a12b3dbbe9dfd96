"""af_kv_store_f32 with thousands of rows against the definition in 64 bits: layouts of a few heads, which a warp
takes, and of many, which a block takes."""
import numpy as np
import pytest
import torch

import kv_helpers as kh
from llm_core_b200 import _lib
from test_kvcache_gpu import store_plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", [(16, 2, 128), (16, 8, 128), (17, 8, 128), (32, 32, 64), (32, 4, 64), (3, 1, 64)])
@pytest.mark.parametrize("order", [0, 1, 2])
def test_many_rows(gpu, kv, H, KV, hd, order):
    counts, lengths = [900, 0, 1, 1400], [33, 5, 0, 64]
    n, page = sum(counts), 16
    rng = np.random.default_rng(H + hd)
    c = kh.Cache(kv, KV, hd, [a + b for a, b in zip(lengths, counts)], page=page, seed=2, fill=7.0)
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn((n, h, hd), device="cuda", generator=g) for h in (H, KV, KV))
    depth = rng.integers(0, 300, n).astype(np.int32)
    cos, sin = kh.rope_tables(512, hd)
    qn, kn = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    dev = [torch.from_numpy(x).cuda() for x in (cos, sin, qn, kn)]
    out, lens, first, dep = torch.empty_like(q), kh.ints(lengths), kh.ints(np.concatenate([[0], np.cumsum(counts)])), kh.ints(depth)
    a = _lib.KvStoreArgs()
    a.kv, a.batch, a.n_rows, a.n_heads, a.n_ctx = c.struct(), c.batch(lens, first, max(counts)), n, H, 512
    a.q, a.k, a.v, a.q_out, a.depth = (x.data_ptr() for x in (q, k, v, out, dep))
    a.cos, a.sin, a.q_norm, a.k_norm = (x.data_ptr() for x in dev)
    a.qk_norm_order, a.eps = order, 1e-6
    kh.call(gpu, "af_kv_store_f32", a)
    assert kh.device_error(gpu) == 0
    seq = np.repeat(np.arange(4), counts)
    node = np.arange(n) - np.concatenate([[0], np.cumsum(counts)])[seq]
    pos, at = np.array(lengths)[seq] + node, np.array(lengths)[seq] + depth
    slot = [torch.as_tensor(x.astype(np.int64)).cuda() for x in (c.table_h[seq, pos // page], pos % page)]
    # a rotation is two products and a sum of values up to |x0| + |x1| (3·2^-24 of it); a norm's mean adds hd/32 + 5
    # roundings, its root, quotient and products 4; a root by rsqrtf is good to 2^-22
    step = (3 + (hd / 32 + 9 + 4 if order else 0)) * 2.0 ** -24

    def close(got, want, half):
        big = np.abs(want).max(-1, keepdims=True) * 2
        assert (np.abs(got - want) <= step * big + half * np.abs(want) * (1 + 2.0 ** -10) + (2.0 ** -25 if half == 2.0 ** -11 else 0)).all()
    w = [x.astype(np.float64) if order else None for x in (qn, kn)]
    close(out.cpu().numpy(), store_plain(q.double().cpu().numpy(), order, w[0], cos[at], sin[at], 1e-6), 0)
    r = kh.HALF_STEP[kv]
    close(c.k[0, slot[0], slot[1]].double().cpu().numpy(), store_plain(k.double().cpu().numpy(), order, w[1], cos[at], sin[at], 1e-6), r)
    close(c.v[0, slot[0], slot[1]].double().cpu().numpy(), v.double().cpu().numpy(), r)
    kept = torch.ones(c.k.shape[1:3], dtype=torch.bool, device="cuda")
    kept[slot[0], slot[1]] = False
    assert (c.k[0][kept] == 7).all() and (c.v[0][kept] == 7).all()
