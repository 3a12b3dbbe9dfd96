"""af_attention_tree_f32 with bounds far above what a call has: max_nodes is a
limit, rows and lengths say how much there is."""
import numpy as np
import pytest
import torch

import kv_helpers as kh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("H,KV,hd,max_nodes", [(32, 32, 64, (1 << 27) + 8), (4, 4, 128, (1 << 30) + 3), (16, 4, 64, 1 << 27),
                                               (4, 4, 64, (1 << 31) - 1)])
def test_any_limit_of_nodes(gpu, kv, H, KV, hd, max_nodes):
    """Rows times heads of such a limit pass 32 bits; two sequences, one of them split."""
    lengths, counts = [4000, 70], [3, 18]
    rng = np.random.default_rng(4)
    c = kh.Cache(kv, KV, hd, [a + b for a, b in zip(lengths, counts)], page=64, seed=5)
    q = torch.from_numpy(rng.standard_normal((sum(counts), H, hd)).astype(np.float32)).cuda()
    outs = []
    for top in (max(counts), max_nodes):
        out = torch.full_like(q, 7.0)
        a = kh.attention_args(c, q, out, kh.ints(lengths), kh.ints([0, 3, 21]), top)
        ws = kh.workspace(gpu, "af_attention_tree_f32", a)
        kh.call(gpu, "af_attention_tree_f32", a)
        assert kh.device_error(gpu) == 0
        outs.append(out.cpu().numpy())
        del ws
    at = 0
    for s, n in enumerate(counts):
        want, tol = kh.attention_plain(q[at:at + n].cpu().numpy().astype(np.float64), c.rows(c.k, 0, s, lengths[s] + n),
                                       c.rows(c.v, 0, s, lengths[s] + n), kh.seen_matrix(lengths[s], n), kh.isqrt(hd))
        for got in outs:
            assert (np.abs(got[at:at + n] - want) <= tol).all()
        at += n
