"""af_attention_tree_f32: what a row does not see does not reach it, whatever it
holds.  Nodes of other branches, slots that no row marks and later tokens of a
chain hold very large values, infinities and NaN; the tolerance of each row
follows from what it sees alone."""
import numpy as np
import pytest
import torch

import kv_helpers as kh

pytestmark = pytest.mark.gpu
KERNELS = [("tensor", 64), ("tensor", 128), ("small", 64), ("small", 128), ("row", 40)]


def check(lib, kv, kernel, hd, length, n, rows, change, undefined=(), scale=0.0, H=8, KV=2, seed=0, page=16):
    """`change(k, v, at)` writes into the pools; at(node) gives a node's (page, row).  `rows`: mask rows, None: a chain;
    rows whose number is in `undefined` are not looked at."""
    rng = np.random.default_rng(seed)
    c = kh.Cache(kv, KV, hd, [length + n], page=page, seed=seed, extra_blocks=4096 if kernel == "tensor" else 1)

    def at(node):
        p = length + node
        return int(c.table_h[0, p // page]), p % page
    change(c.k, c.v, at)
    q = torch.from_numpy(rng.standard_normal((n, H, hd)).astype(np.float32)).cuda()
    out = torch.full((n, H, hd), 7.0, device="cuda")
    mask = None if rows is None else kh.mask_words(rows, -(-n // 64))
    a = kh.attention_args(c, q, out, kh.ints([length]), kh.ints([0, n]), n, mask, scale=scale)
    ws = kh.workspace(lib, "af_attention_tree_f32", a)
    assert (a.ws_bytes > 1 << 20) == (kernel == "tensor")
    kh.call(lib, "af_attention_tree_f32", a)
    assert kh.device_error(lib) == 0
    keep = [i for i in range(n) if i not in undefined]
    seen = kh.seen_matrix(length, n, rows)[keep]
    want, tol = kh.attention_plain(q.cpu().numpy().astype(np.float64)[keep], c.rows(c.k, 0, 0, length + n),
                                   c.rows(c.v, 0, 0, length + n), seen, scale or kh.isqrt(hd))
    err = np.abs(out.cpu().numpy()[keep] - want)
    assert (err <= tol).all(), (float((err / np.maximum(tol, 1e-300)).max()), np.argwhere(~(err <= tol))[:5])
    del ws


def big(kv):
    return 6e4 if kv == "f16" else 1e30


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kernel,hd", KERNELS)
@pytest.mark.parametrize("bad", ["large", float("inf"), float("nan")])
@pytest.mark.parametrize("which", ["k", "v", "both"])
@pytest.mark.parametrize("length,n", [(75, 5), (0, 3), (61, 24)])
def test_a_slot_that_no_row_marks(gpu, kv, kernel, hd, bad, which, length, n):
    rows = [(1 << i | 1) & ~2 for i in range(n)]
    bad = big(kv) if bad == "large" else bad

    def change(k, v, at):
        page, off = at(1)
        if which != "v":
            k[:, page, off] = bad
        if which != "k":
            v[:, page, off] = bad
    check(gpu, kv, kernel, hd, length, n, rows, change)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kernel,hd", KERNELS)
@pytest.mark.parametrize("length,n", [(75, 9), (0, 12), (130, 40)])
def test_branches_of_very_different_size(gpu, kv, kernel, hd, length, n):
    """Two branches in turn, which see themselves and the past: V of one is 1e8 times the other's (f16: 1e4), its
    keys 1e3 times."""
    rows, seen = [], [0, 0]
    for i in range(n):
        seen[i % 2] |= 1 << i
        rows.append(seen[i % 2])

    def change(k, v, at):
        for i in range(1, n, 2):
            page, off = at(i)
            v[:, page, off] *= 1e4 if kv == "f16" else 1e8
            k[:, page, off] *= 1e3
    check(gpu, kv, kernel, hd, length, n, rows, change, scale=1e-3)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kernel,hd", KERNELS)
@pytest.mark.parametrize("masked", [False, True])
def test_later_tokens_that_grow(gpu, kv, kernel, hd, masked):
    """Token i's V is 10^(3 i) (f16: 10^(i/2)) times the first one's."""
    n, length = 9, 70

    def change(k, v, at):
        for i in range(n):
            page, off = at(i)
            v[:, page, off] *= 10.0 ** (i / 2 if kv == "f16" else 3 * i)
    rows = [(2 << i) - 1 for i in range(n)] if masked else None
    check(gpu, kv, kernel, hd, length, n, rows, change)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kernel,hd", KERNELS)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("where", [0, 3, 7])
def test_a_key_that_is_not_finite_leaves_its_own_rows_alone_undefined(gpu, kv, kernel, hd, bad, where):
    """One element of token `where`'s key, of a chain whose other keys are small: the tokens before it are right."""
    n, length = 12, 50

    def change(k, v, at):
        page, off = at(where)
        k *= 2.0 ** -12 if kv == "f16" else 2.0 ** -40
        k[:, page, off, 0, 5] = bad
    check(gpu, kv, kernel, hd, length, n, None, change, undefined=range(where, n), scale=2.0 ** 10 if kv == "f16" else 2.0 ** 38)


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_chains_with_outliers(gpu, kv, hd):
    """300 tokens behind 1,000: tiles of nodes only, every 37th token's V 1e12 times the others', seen by those behind."""
    n = 300

    def change(k, v, at):
        for i in range(36, n, 37):
            page, off = at(i)
            v[:, page, off] *= 1e12
    check(gpu, kv, "tensor", hd, 1000, n, None, change, H=4, KV=2)


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [7, 40])
def test_channels_that_are_large_in_every_row(gpu, kv, hd, n):
    """A few channels of K and V are 3e4 times the others, in all rows."""
    def change(k, v, at):
        k[..., 5] *= 3e4
        v[..., 1] *= 3e4
        v[..., hd - 3] *= 3e4
    check(gpu, kv, "tensor", hd, 300, n, None, change, scale=1e-5)
