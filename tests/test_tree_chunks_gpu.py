"""af_attention_tree_f32 on chunks of several hundred tokens and trees of many nodes over long caches, in every type,
with and without max_len, against the definition in 64 bits on the device."""
import numpy as np
import pytest
import torch

import kv_helpers as kh

pytestmark = pytest.mark.gpu


def check(lib, kv, H, KV, hd, lengths, counts, tree, exact_len, page=32, seed=0):
    rng = np.random.default_rng(seed)
    c = kh.Cache(kv, KV, hd, [a + b for a, b in zip(lengths, counts)], page=page, seed=seed, extra_blocks=3)
    first = np.concatenate([[0], np.cumsum(counts)])
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = 1.5 * torch.randn((int(first[-1]), H, hd), device="cuda", generator=g)
    out = torch.full_like(q, 7.0)
    rows = [kh.tree_of(m, rng)[2] for m in counts] if tree else None
    words = -(-max(counts) // 64)
    mask = kh.mask_words([b for r in rows for b in r], words) if tree else None
    most = max(a + b for a, b in zip(lengths, counts))
    a = kh.attention_args(c, q, out, kh.ints(lengths), kh.ints(first), max(counts), mask, max_len=most if exact_len else 0)
    ws = kh.workspace(lib, "af_attention_tree_f32", a)
    kh.call(lib, "af_attention_tree_f32", a)
    assert kh.device_error(lib) == 0
    for s, n in enumerate(counts):
        L = lengths[s] + n
        k, v = (torch.from_numpy(c.rows(x, 0, s, L)).cuda() for x in (c.k, c.v))
        seen = torch.ones((n, L), dtype=torch.bool, device="cuda")
        if tree:
            bits = np.array([[(b >> j) & 1 for j in range(n)] for b in rows[s]], bool)
            seen[:, lengths[s]:] = torch.from_numpy(bits).cuda()
        else:
            seen[:, lengths[s]:] = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        for h in range(H):
            x, kk, vv = q[first[s]:first[s + 1], h].double(), k[:, h // (H // KV)], v[:, h // (H // KV)]
            w = (x @ kk.T * kh.isqrt(hd)).masked_fill(~seen, -torch.inf)
            want = torch.softmax(w, -1) @ vv
            # as attention_plain: scores off by ds, weights, sum and output by L + 8 roundings, of the largest |v|
            ds = (3 * 2.0 ** -22 + hd * 2.0 ** -24) * (x.abs() @ kk.abs().T).amax() * kh.isqrt(hd)
            assert (out[first[s]:first[s + 1], h] - want).abs().max() <= vv.abs().max() * (2 * ds + (L + 8) * 2.0 ** -24)
    del ws


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 64), (6, 2, 128), (4, 4, 128)])
@pytest.mark.parametrize("exact_len", [False, True])
@pytest.mark.parametrize("lengths,counts", [([5000, 3], [509, 260]), ([0], [700]), ([2047, 1, 130, 900], [300, 500, 129, 1])])
def test_chunks(gpu, kv, H, KV, hd, exact_len, lengths, counts):
    check(gpu, kv, H, KV, hd, lengths, counts, False, exact_len)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", [(16, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("exact_len", [False, True])
def test_trees(gpu, kv, H, KV, hd, exact_len):
    check(gpu, kv, H, KV, hd, [6000, 511, 0], [200, 256, 65], True, exact_len, seed=1)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lengths", [[137], [4095], [20] * 24, [3000, 5, 700]])
def test_tokens_with_their_longest_length_given(gpu, kv, hd, lengths):
    """What a decode step calls: one node a sequence."""
    check(gpu, kv, 8, 2, hd, lengths, [1] * len(lengths), False, True, seed=2)
