"""af_attention_tree_f32 over caches whose values differ by as much as the entry allows: V of zeros beside V just
below 2^56, in other tiles, other groups of rows and other splits of the positions, and keys near 2^100."""
import numpy as np
import pytest
import torch

import kv_helpers as kh

pytestmark = pytest.mark.gpu


def run(lib, kv, hd, length, n, change, q_of, scale):
    H, KV = 4, 2
    rng = np.random.default_rng(length + n)
    c = kh.Cache(kv, KV, hd, [length + n], page=16, seed=2, extra_blocks=4096)
    pos = np.arange(length + n)
    page, off = (torch.as_tensor(x).cuda() for x in (c.table_h[0, pos // 16].astype(np.int64), pos % 16))
    k, v = (torch.from_numpy(rng.uniform(-1, 1, (length + n, KV, hd)).astype(np.float32)).cuda() for _ in range(2))
    k, v = change(k, v)
    c.k[0, page, off], c.v[0, page, off] = k.to(c.k.dtype), v.to(c.v.dtype)
    q = torch.from_numpy(q_of(rng.standard_normal((n, H, hd))).astype(np.float32)).cuda()
    out = torch.zeros((n, H, hd), device="cuda")
    a = kh.attention_args(c, q, out, kh.ints([length]), kh.ints([0, n]), n, None, scale=scale)
    ws = kh.workspace(lib, "af_attention_tree_f32", a)
    kh.call(lib, "af_attention_tree_f32", a)
    assert kh.device_error(lib) == 0
    want, tol = kh.attention_plain(q.cpu().numpy().astype(np.float64), c.rows(c.k, 0, 0, length + n),
                                   c.rows(c.v, 0, 0, length + n), kh.seen_matrix(length, n), scale)
    assert (np.abs(out.cpu().numpy() - want) <= tol).all()
    del ws


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("zeros", ["first half", "first tile", "last half", "groups"])
@pytest.mark.parametrize("length,n", [(300, 3), (3000, 20)])
@pytest.mark.parametrize("lift", [0.0, 16.0])  # how much less the zeros' scores are: e^-16 = 2^-23 of the weight
def test_zeros_beside_the_largest_values(gpu, kv, hd, zeros, length, n, lift):
    at = np.arange(length + n)
    mine = torch.from_numpy({"first half": at < length // 2, "first tile": at < 128, "last half": at >= length // 2,
                             "groups": at // 32 % 2 == 0}[zeros]).cuda()[:, None, None]

    def change(k, v):
        v = torch.where(mine, 0.0, v * (2.0 ** 56 * (1 - 2.0 ** -8)))
        k[..., 0] = torch.where(mine[..., 0], 0.0, lift)  # q's first value is 1, the scale 1
        return k, v

    def q_of(q):
        q = 0.05 * q
        q[..., 0] = 1
        return q
    run(gpu, kv, hd, length, n, change, q_of, 1.0)


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_the_largest_keys(gpu, kv, hd):
    """Keys just below 2^100 beside zeros, in groups of 32 and alone."""
    length, n = 400, 5
    at = torch.arange(length + n, device="cuda")
    some = ((at // 32 % 2 == 0) | (at % 7 == 0))[:, None, None]

    def change(k, v):
        return torch.where(some, k * (2.0 ** 100 * (1 - 2.0 ** -8)), 0.0), v
    run(gpu, kv, hd, length, n, change, lambda q: q * 2.0 ** -60, 2.0 ** -40)
