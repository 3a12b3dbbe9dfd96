"""An infinite or NaN value of V reaches the rows that see it, as what it is, also where its weight is far below the
smallest number of 32 bits: in front of and behind larger scores, in other splits and blocks of a cluster."""
import numpy as np
import pytest
import torch

import kv_helpers as kh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kernel,hd,length", [("tensor", 64, 150), ("tensor", 128, 3000), ("small", 64, 200), ("small", 128, 90),
                                              ("row", 40, 100), ("row", 256, 30)])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("where", [0, 40, -1])  # a cached position, or the first node
def test_values_of_vanishing_weight(gpu, kv, kernel, hd, length, bad, where):
    H, KV, n = 4, 2, 3
    rng = np.random.default_rng(hd)
    c = kh.Cache(kv, KV, hd, [length + n], page=16, seed=4, extra_blocks=4096 if kernel == "tensor" else 1)
    p = length if where < 0 else min(where, length - 1)
    page, off = int(c.table_h[0, p // 16]), p % 16
    c.k[..., 0] = 0
    c.k[0, page, off, :, 0] = -300.0  # q's first value and the scale are 1: e^-300 of the others' weight
    clean = c.v.clone()
    c.v[0, page, off, 0, 7] = bad
    q = 0.1 * torch.from_numpy(rng.standard_normal((n, H, hd)).astype(np.float32)).cuda()
    q[..., 0] = 1
    out = torch.zeros_like(q)
    a = kh.attention_args(c, q, out, kh.ints([length]), kh.ints([0, n]), n, scale=1.0,
                          max_len=0 if kernel == "tensor" else length + n)
    ws = kh.workspace(gpu, "af_attention_tree_f32", a)
    assert a.ws_bytes > 1 << 20 or kernel != "tensor"
    kh.call(gpu, "af_attention_tree_f32", a)
    assert kh.device_error(gpu) == 0
    got = out.cpu().numpy()
    np.testing.assert_array_equal(got[:, :H // KV, 7], np.float32(bad))
    clean[0, page, off, 0, 7] = 0
    want, tol = kh.attention_plain(q.cpu().numpy().astype(np.float64), c.rows(c.k, 0, 0, length + n),
                                   c.rows(clean, 0, 0, length + n), kh.seen_matrix(length, n), 1.0)
    rest = np.ones((n, H, hd), bool)
    rest[:, :H // KV, 7] = False
    assert (np.abs(got - want) <= tol)[rest].all()
    del ws
