"""Positions that a sequence holds no page for: the error word, and on every kernel of af_attention_tree_f32 the same
result, of keys and values of zeros; no other sequence's page is read."""
import numpy as np
import pytest
import torch

import kv_helpers as kh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kernel,hd", [("tensor", 64), ("tensor", 128), ("small", 64), ("small", 128), ("row", 40)])
@pytest.mark.parametrize("page", [1, 16, 64, 256])
@pytest.mark.parametrize("holes,bad", [([1], -1), ([0, 2], 1 << 30), ([0, 1, 2], -7)])
def test_positions_without_a_page_are_zeros(gpu, kv, kernel, hd, page, holes, bad):
    H, KV, lengths, n = 8, 2, [250, 61], 9
    rng = np.random.default_rng(page)
    c = kh.Cache(kv, KV, hd, [x + n for x in lengths], page=page, seed=4, extra_blocks=4096 if kernel == "tensor" else 1)
    q = torch.from_numpy(rng.standard_normal((2 * n, H, hd)).astype(np.float32)).cuda()
    kv64 = [[c.rows(pool, 0, s, lengths[s] + n) for pool in (c.k, c.v)] for s in range(2)]
    table = c.table_h.copy()
    for b in holes:
        if b * page < lengths[0] + n:
            table[0, b] = bad
            for x in kv64[0]:
                x[b * page:(b + 1) * page] = 0
    # a page of the pool that is read in place of a missing one would show
    held = set(table[(table >= 0) & (table < c.pages)].tolist())
    for i in range(c.pages):
        if i not in held:
            c.k[:, i] = c.v[:, i] = 1e4
    c.table = kh.ints(table)
    out = torch.zeros_like(q)
    a = kh.attention_args(c, q, out, kh.ints(lengths), kh.ints([0, n, 2 * n]), n,
                          max_len=0 if kernel == "tensor" else max(lengths) + n)
    ws = kh.workspace(gpu, "af_attention_tree_f32", a)
    assert a.ws_bytes > 1 << 20 or kernel != "tensor"
    kh.call(gpu, "af_attention_tree_f32", a)
    assert kh.device_error(gpu) != 0
    for s in range(2):
        want, tol = kh.attention_plain(q[s * n:(s + 1) * n].cpu().numpy().astype(np.float64), *kv64[s],
                                       kh.seen_matrix(lengths[s], n), kh.isqrt(hd))
        assert (np.abs(out[s * n:(s + 1) * n].cpu().numpy() - want) <= tol).all(), s
    del ws
