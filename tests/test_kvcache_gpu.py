"""The paged cache: af_kv_store_f32, af_kv_fork and af_kv_compact against
their definitions."""
import ctypes as C

import numpy as np
import pytest
import torch

import kv_helpers as kh
from llm_core_b200 import _lib

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------- store

def store_plain(x, order, w, cos, sin, eps, rotate=True):
    """[rows][heads][hd] in 64 bits."""
    hd = x.shape[-1]

    def norm(y):
        return w * (y / np.sqrt((y * y).mean(-1, keepdims=True) + eps))
    if order == 1 and w is not None:
        x = norm(x)
    if rotate:
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        x = np.concatenate([a * cos[:, None] - b * sin[:, None], a * sin[:, None] + b * cos[:, None]], -1)
    if order == 2 and w is not None:
        x = norm(x)
    return x


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", [(32, 4, 64), (16, 2, 128), (3, 1, 40), (2, 2, 256), (5, 5, 8), (6, 2, 96)])
@pytest.mark.parametrize("order", [0, 1, 2])
def test_store(gpu, kv, H, KV, hd, order):
    rng = np.random.default_rng(hd + order)
    lengths, counts = [37, 0, 64, 11], [5, 3, 0, 9]
    c = kh.Cache(kv, KV, hd, [a + b for a, b in zip(lengths, counts)], page=8, layers=2, seed=1)
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    n, extra = int(first[-1]), 2
    depth = np.concatenate([kh.tree_of(m, rng)[1] for m in counts if m]).astype(np.int32)
    depth = np.concatenate([depth, np.zeros(extra, np.int32)])
    qkv = torch.from_numpy(rng.standard_normal((n + extra, (H + 2 * KV) * hd)).astype(np.float32)).cuda()
    stride = qkv.shape[1]
    cos, sin = kh.rope_tables(64, hd)
    qn, kn = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    dev = [torch.from_numpy(x).cuda() for x in (cos, sin, qn, kn)]
    q_out = torch.full((n + extra, H, hd), 9.0, device="cuda")
    before = [c.k.clone(), c.v.clone()]
    lens, fst, dep = kh.ints(lengths), kh.ints(first), kh.ints(depth)
    a = _lib.KvStoreArgs()
    a.kv, a.batch, a.layer, a.n_rows = c.struct(), c.batch(lens, fst, max(counts)), 1, n + extra
    a.q, a.k, a.v = qkv.data_ptr(), qkv.data_ptr() + 4 * H * hd, qkv.data_ptr() + 4 * (H + KV) * hd
    a.q_stride = a.k_stride = a.v_stride = stride
    a.q_out, a.depth, a.cos, a.sin = q_out.data_ptr(), dep.data_ptr(), dev[0].data_ptr(), dev[1].data_ptr()
    a.n_ctx, a.n_heads, a.qk_norm_order = cos.shape[0], H, order
    a.q_norm, a.k_norm, a.eps = dev[2].data_ptr(), dev[3].data_ptr(), 1e-6
    kh.call(gpu, "af_kv_store_f32", a)
    assert kh.device_error(gpu) == 0
    x = qkv.cpu().numpy().astype(np.float64)[:n]
    seq = np.repeat(np.arange(4), counts)
    at = np.array(lengths)[seq] + depth[:n]
    want_q = store_plain(x[:, :H * hd].reshape(n, H, hd), order, qn.astype(np.float64) if order else None, cos[at], sin[at], 1e-6)
    want_k = store_plain(x[:, H * hd:(H + KV) * hd].reshape(n, KV, hd), order, kn.astype(np.float64) if order else None,
                         cos[at], sin[at], 1e-6)
    want_v = x[:, (H + KV) * hd:].reshape(n, KV, hd)
    # a rotation is two products and a sum of values up to |x0| + |x1| (3·2^-24 of it); a norm's
    # mean adds hd/32 + 5 roundings, its root, quotient and products 4
    step = (3 + (hd / 32 + 9 if order else 0)) * 2.0 ** -24

    def close(got, want, rounding):
        big = np.abs(want).max(-1, keepdims=True) * 2
        assert (np.abs(got - want) <= step * big + rounding * np.abs(want) * (1 + 2.0 ** -10)
                + (2.0 ** -25 if kv == "f16" and rounding else 0)).all()
    got_q = q_out.cpu().numpy()
    close(got_q[:n], want_q, 0)
    assert (got_q[n:] == 9.0).all()
    r = kh.HALF_STEP[kv]
    touched = torch.zeros(c.k.shape[:3], dtype=torch.bool)
    for s, m in enumerate(counts):
        for i in range(m):
            p = lengths[s] + i
            page, off = int(c.table_h[s, p // c.page]), p % c.page
            touched[1, page, off] = True
            close(c.k[1, page, off].double().cpu().numpy(), want_k[first[s] + i], r)
            close(c.v[1, page, off].double().cpu().numpy(), want_v[first[s] + i], r)
    for pool, old in ((c.k, before[0]), (c.v, before[1])):
        same = (pool == old).flatten(3).all(-1).cpu()
        assert bool(same[~touched].all())


def test_store_in_place_chain_and_values_as_given(gpu):
    """q_out = q, no depth (a chain), no first: 2 sequences of 3 tokens; V in f32 comes through as it is."""
    H, KV, hd, n = 4, 2, 64, 3
    c = kh.Cache("f32", KV, hd, [20, 30], seed=3, contiguous=True)
    rng = np.random.default_rng(0)
    q, k, v = (torch.from_numpy(rng.standard_normal((2 * n, h, hd)).astype(np.float32)).cuda() for h in (H, KV, KV))
    v[0, 0, 0], v[1, 1, 5] = float("inf"), float("nan")
    cos, sin = (torch.from_numpy(x).cuda() for x in kh.rope_tables(64, hd))
    lens = kh.ints([16, 7])
    q0 = q.cpu().numpy().astype(np.float64)
    a = _lib.KvStoreArgs()
    a.kv, a.batch, a.n_rows = c.struct(), c.batch(lens, None, n), 2 * n
    a.q, a.k, a.v, a.q_out, a.cos, a.sin = (t.data_ptr() for t in (q, k, v, q, cos, sin))
    a.n_ctx, a.n_heads = 64, H
    kh.call(gpu, "af_kv_store_f32", a)
    assert kh.device_error(gpu) == 0
    at = np.array([16, 17, 18, 7, 8, 9])
    want = store_plain(q0, 0, None, cos.cpu().numpy()[at], sin.cpu().numpy()[at], 0)
    assert np.abs(q.cpu().numpy() - want).max() <= 6 * 2.0 ** -24 * np.abs(want).max()
    for s in range(2):
        for i in range(n):
            p = at[s * n + i]
            got = c.v[0, int(c.table_h[s, p // c.page]), p % c.page]
            assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(v[s * n + i]))
            assert torch.equal(got.isnan(), v[s * n + i].isnan())


@pytest.mark.parametrize("what", ["page", "context"])
def test_store_refuses_on_the_device(gpu, what):
    H, KV, hd = 4, 2, 64
    c = kh.Cache("f32", KV, hd, [20], seed=3)
    q, k, v = (torch.ones((1, h, hd), device="cuda") for h in (H, KV, KV))
    cos, sin = (torch.from_numpy(x).cuda() for x in kh.rope_tables(32, hd))
    before = c.k.clone()
    length = 20 if what == "page" else 40
    if what == "page":
        t = c.table_h.copy()
        t[0, 20 // c.page] = -1
        c.table = kh.ints(t)
    lens, first = kh.ints([length]), kh.ints([0, 1])
    a = _lib.KvStoreArgs()
    a.kv, a.batch, a.n_rows = c.struct(), c.batch(lens, first, 1), 1
    a.q, a.k, a.v, a.q_out, a.cos, a.sin = (t.data_ptr() for t in (q, k, v, q, cos, sin))
    a.n_ctx, a.n_heads = 32, H
    kh.call(gpu, "af_kv_store_f32", a)
    assert kh.device_error(gpu) != 0
    assert torch.equal(before, c.k)


# -------------------------------------------------------------------- fork

def run_fork(lib, c, table, length, ref, parent, new, in_place=False, twice=True):
    blocks, n_in, n_out = table.shape[1], table.shape[0], len(parent)
    want = kh.fork_plain(c.page, c.pages, table, length, ref, parent, new, blocks)
    pools = [(c.k.clone(), c.k), (c.v.clone(), c.v)]
    for old, _ in pools:
        for src, dst, rows in want[4]:
            old[:, dst, :rows] = old[:, src, :rows]
    t_in, l_in, r_in, par, nw = (kh.ints(x) for x in (table, length, ref, parent, new))
    t_out = torch.full((max(n_out, 1), blocks), -7, dtype=torch.int32, device="cuda")
    l_out = torch.full((max(n_out, 1),), -7, dtype=torch.int32, device="cuda")
    r_out = r_in if in_place else torch.full_like(r_in, -7)
    short = torch.full((1,), -7, dtype=torch.int32, device="cuda")
    a = _lib.KvForkArgs()
    a.kv = c.struct()
    a.table_in, a.len_in, a.ref_in = (x.data_ptr() for x in (t_in, l_in, r_in))
    a.table_out, a.len_out, a.ref_out = (x.data_ptr() for x in (t_out, l_out, r_out))
    a.parent, a.n_new, a.n_short = par.data_ptr(), nw.data_ptr(), short.data_ptr()
    a.n_in, a.n_out, a.max_blocks = n_in, n_out, blocks
    ws = kh.workspace(lib, "af_kv_fork", a)
    for _ in range(1 if in_place else 2):
        kh.call(lib, "af_kv_fork", a)
    assert kh.device_error(lib) == 0
    if n_out:
        np.testing.assert_array_equal(t_out.cpu().numpy(), np.array(want[0], np.int32))
        np.testing.assert_array_equal(l_out.cpu().numpy(), np.array(want[1], np.int32))
    np.testing.assert_array_equal(r_out.cpu().numpy(), np.array(want[2], np.int32))
    assert int(short.item()) == want[3]
    for old, now in pools:
        assert torch.equal(old, now)
    del ws
    return np.array(want[0], np.int32).reshape(n_out, blocks), np.array(want[1], np.int32), np.array(want[2], np.int32)


def counts_of(table, pages):
    ref = np.zeros(pages, np.int32)
    np.add.at(ref, table[table >= 0], 1)
    return ref


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("page", [1, 4, 16])
def test_fork_reorders_beams(gpu, kv, in_place, page):
    """A prompt forked into beams, then steps of reordering and growth, each
    against the definition."""
    rng = np.random.default_rng(page)
    c = kh.Cache(kv, 2, 8, [45], page=page, layers=3, spare=300, seed=2, extra_blocks=40)
    table, length = c.table_h, np.array([45], np.int32)
    ref = counts_of(table, c.pages)
    table, length, ref = run_fork(gpu, c, table, length, ref, [0] * 6, [1] * 6, in_place)
    for step in range(8):
        length = length + 1  # the token was stored
        parent = rng.integers(0, 6, 6).tolist()
        if step == 3:
            parent = [5, 5, 5, 5, 5, 5]
        table, length, ref = run_fork(gpu, c, table, length, ref, parent, [1] * 6, in_place)
    table, length, ref = run_fork(gpu, c, table, length, ref, [2], [0], in_place)
    assert (ref <= 1).all()
    run_fork(gpu, c, table, length, ref, [], [], in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_fork_new_freed_and_continued_sequences(gpu, in_place):
    c = kh.Cache("f16", 1, 16, [10, 16, 3, 0], page=8, spare=12, seed=4, extra_blocks=6)
    ref = counts_of(c.table_h, c.pages)
    length = np.array([10, 16, 3, 0], np.int32)
    out = run_fork(gpu, c, c.table_h, length, ref, [1, -1, 3, 1, 99, 0], [0, 20, 1, 9, 0, 6], in_place)
    # pages that were taken ahead and are no longer wanted are given back
    run_fork(gpu, c, out[0], out[1], out[2], [5, 3, 3, 1], [0, 0, 1, 0], in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_fork_pages_shared_with_another_table(gpu, in_place):
    """A page that an entry outside the call holds is copied, not kept."""
    c = kh.Cache("f32", 2, 8, [21], page=8, spare=9, seed=4, extra_blocks=2)
    ref = counts_of(c.table_h, c.pages)
    ref[c.table_h[0, :3]] += 1
    run_fork(gpu, c, c.table_h, np.array([21], np.int32), ref, [0, 0], [1, 1], in_place)


@pytest.mark.parametrize("spare", [0, 1, 2, 3])
def test_fork_when_pages_run_out(gpu, spare):
    c = kh.Cache("f32", 1, 8, [21, 30], page=8, spare=spare, seed=4, extra_blocks=2)
    ref = counts_of(c.table_h, c.pages)
    run_fork(gpu, c, c.table_h, np.array([21, 30], np.int32), ref, [0, 0, 1, 1, 0], [1, 40, 3, 9, 0])


def test_fork_many_sequences_and_pages(gpu):
    rng = np.random.default_rng(3)
    n = 300
    lens = rng.integers(0, 200, n)
    c = kh.Cache("f16", 1, 8, lens.tolist(), page=4, spare=5000, seed=5, extra_blocks=9)
    ref = counts_of(c.table_h, c.pages)
    parent = rng.integers(-3, n + 3, 500).tolist()
    run_fork(gpu, c, c.table_h, lens.astype(np.int32), ref, parent, rng.integers(0, 30, 500).tolist())


def test_fork_bad_page_ids_set_the_error_word_or_count_as_none(gpu):
    """An id outside the pool is nobody's page: it is not read, counted or passed on."""
    c = kh.Cache("f32", 1, 8, [21], page=8, spare=5, seed=4, extra_blocks=2)
    ref = counts_of(c.table_h, c.pages)
    bad = c.table_h.copy()
    bad[0, 1] = 1 << 30
    want = bad.copy()
    want[0, 1] = -1
    t_in, l_in, r_in, par = kh.ints(bad), kh.ints([21]), kh.ints(ref), kh.ints([0])
    t_out, l_out, r_out, short = (torch.zeros_like(t_in), torch.zeros_like(l_in), torch.zeros_like(r_in),
                                  torch.zeros(1, dtype=torch.int32, device="cuda"))
    a = _lib.KvForkArgs()
    a.kv = c.struct()
    a.table_in, a.len_in, a.ref_in = (x.data_ptr() for x in (t_in, l_in, r_in))
    a.table_out, a.len_out, a.ref_out = (x.data_ptr() for x in (t_out, l_out, r_out))
    a.parent, a.n_short, a.n_in, a.n_out, a.max_blocks = par.data_ptr(), short.data_ptr(), 1, 1, c.blocks
    ws = kh.workspace(gpu, "af_kv_fork", a)
    kh.call(gpu, "af_kv_fork", a)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(t_out.cpu().numpy(), want)
    kh.device_error(gpu)
    del ws


# ----------------------------------------------------------------- compact

@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("KV,hd,page", [(4, 64, 16), (1, 8, 4), (2, 128, 8), (3, 40, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(gpu, kv, KV, hd, page, in_place):
    rng = np.random.default_rng(hd)
    lengths, nodes = [33, 0, 64, 17, 5], 31
    c = kh.Cache(kv, KV, hd, [x + nodes for x in lengths], page=page, layers=2, seed=7)
    paths = [sorted(rng.choice(nodes, n, replace=False).tolist()) for n in (6, 1, 0, 12, 31)]
    top = 31
    pa = np.full((5, top), -5, np.int32)
    for s, x in enumerate(paths):
        pa[s, :len(x)] = x
    want = [c.k.clone(), c.v.clone()]
    for old, pool in zip(want, (c.k, c.v)):
        for s, x in enumerate(paths):
            for i, j in enumerate(x):
                p, d = lengths[s] + j, lengths[s] + i
                old[:, int(c.table_h[s, d // page]), d % page] = pool[:, int(c.table_h[s, p // page]), p % page]
    lens = kh.ints(lengths)
    out = lens if in_place else torch.full_like(lens, -7)
    pd, nd = kh.ints(pa), kh.ints([len(x) for x in paths])
    a = _lib.KvCompactArgs()
    a.kv, a.batch = c.struct(), c.batch(lens)
    a.path, a.n_path, a.max_path, a.len_out = pd.data_ptr(), nd.data_ptr(), top, out.data_ptr()
    kh.call(gpu, "af_kv_compact", a)
    assert kh.device_error(gpu) == 0
    assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[1])
    assert out.tolist() == [x + len(y) for x, y in zip(lengths, paths)]


@pytest.mark.parametrize("path", [[3, 2], [1, 1], [-1, 2], [0, 400], [0, 90]])
def test_compact_refuses_a_bad_path_on_the_device(gpu, path):
    c = kh.Cache("f32", 2, 8, [40, 40], page=8, seed=7)
    lens, out = kh.ints([20, 20]), kh.ints([-1, -1])
    pd, nd = kh.ints([path, [2, 5]]), kh.ints([2, 2])
    before = c.k.clone()
    a = _lib.KvCompactArgs()
    a.kv, a.batch = c.struct(), c.batch(lens)
    a.path, a.n_path, a.max_path, a.len_out = pd.data_ptr(), nd.data_ptr(), 2, out.data_ptr()
    kh.call(gpu, "af_kv_compact", a)
    assert kh.device_error(gpu) != 0
    assert out.tolist() == [20, 22]
    for d, s in ((20, 22), (21, 25)):
        before[:, int(c.table_h[1, d // 8]), d % 8] = before[:, int(c.table_h[1, s // 8]), s % 8].clone()
    assert torch.equal(before, c.k)


# -------------------------------------------------- the operators together

@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 64), (4, 4, 128)])
def test_tree_verified_and_committed(gpu, kv, H, KV, hd):
    """A prompt stored as a chain; a tree stored, attended to and its accepted
    path compacted; the next token then attends as if only the accepted
    tokens had ever been there."""
    rng = np.random.default_rng(3)
    prompt, n, page = 50, 20, 8
    c = kh.Cache(kv, KV, hd, [prompt + n + 1], page=page, seed=1, fill=0.0)
    cos, sin = (torch.from_numpy(x).cuda() for x in kh.rope_tables(128, hd))
    toks = {}

    def rows(name, m):
        toks[name] = [torch.from_numpy(rng.standard_normal((m, h, hd)).astype(np.float32)).cuda() for h in (H, KV, KV)]
        return toks[name]

    def step(length, q, k, v, depth, mask):
        m = q.shape[0]
        lens, first, out, qr = kh.ints([length]), kh.ints([0, m]), torch.empty_like(q), torch.empty_like(q)
        dep = None if depth is None else kh.ints(depth)
        a = _lib.KvStoreArgs()
        a.kv, a.batch, a.n_rows = c.struct(), c.batch(lens, first, m), m
        a.q, a.k, a.v, a.q_out, a.cos, a.sin = (t.data_ptr() for t in (q, k, v, qr, cos, sin))
        a.depth, a.n_ctx, a.n_heads = kh.ptr(dep), 128, H
        kh.call(gpu, "af_kv_store_f32", a)
        t = kh.attention_args(c, qr, out, lens, first, m, mask)
        ws = kh.workspace(gpu, "af_attention_tree_f32", t)
        kh.call(gpu, "af_attention_tree_f32", t)
        assert kh.device_error(gpu) == 0
        del ws
        return out

    step(0, *rows("prompt", prompt), None, None)
    parent, depth, seen = kh.tree_of(n, rng, branch=3)
    tree = step(prompt, *rows("tree", n), depth, kh.mask_words(seen, 1))
    path = [max(i for i in range(n) if depth[i] == max(depth))]
    while parent[path[0]] >= 0:
        path.insert(0, parent[path[0]])
    lens, out, pd, nd = kh.ints([prompt]), kh.ints([0]), kh.ints([path]), kh.ints([len(path)])
    a = _lib.KvCompactArgs()
    a.kv, a.batch = c.struct(), c.batch(lens)
    a.path, a.n_path, a.max_path, a.len_out = pd.data_ptr(), nd.data_ptr(), len(path), out.data_ptr()
    kh.call(gpu, "af_kv_compact", a)
    assert int(out.item()) == prompt + len(path)
    last = step(prompt + len(path), *rows("next", 1), None, None)
    # the same tokens as one chain in another cache
    d = kh.Cache(kv, KV, hd, [prompt + len(path) + 1], page=16, seed=5, fill=0.0)
    tree_c, c = c, d
    chain = [torch.cat([toks["prompt"][i], toks["tree"][i][path], toks["next"][i]]) for i in range(3)]
    whole = step(0, *chain, None, None)
    tol = 2.0 ** -18 * float(chain[2].abs().max())
    assert (whole[-1] - last[0]).abs().max() <= tol
    assert (whole[prompt:-1] - tree[path]).abs().max() <= tol
    del tree_c


def test_beams_decode_on_shared_pages(gpu):
    """A beam search of several steps: select, fork by the selected beams, store,
    attend — each beam's attention equals that of its own tokens in a cache of their own."""
    B, H, KV, hd, V, page, prompt, steps = 4, 4, 2, 64, 1000, 8, 29, 7
    rng = np.random.default_rng(9)
    c = kh.Cache("f32", KV, hd, [prompt], page=page, spare=40, seed=1, extra_blocks=4)
    table, blocks = [c.table, torch.empty((B, c.blocks), dtype=torch.int32, device="cuda")], c.blocks
    table.append(torch.empty_like(table[1]))
    ref = kh.ints(counts_of(c.table_h, c.pages))
    cos, sin = (torch.from_numpy(x).cuda() for x in kh.rope_tables(64, hd))
    kvals = torch.from_numpy(rng.standard_normal((V, KV, hd)).astype(np.float32)).cuda()
    vvals = torch.from_numpy(rng.standard_normal((V, KV, hd)).astype(np.float32)).cuda()
    qvals = torch.from_numpy(rng.standard_normal((V, H, hd)).astype(np.float32)).cuda()
    ids = rng.integers(0, V, prompt)

    def store(cache, tab, lens, toks, first, n):
        b = cache.batch(lens, first, n, n_seq=lens.shape[0])
        b.block_table = tab.data_ptr()
        q, k, v = (x[torch.as_tensor(toks, dtype=torch.int64).cuda()].contiguous() for x in (qvals, kvals, vvals))
        a = _lib.KvStoreArgs()
        a.kv, a.batch, a.n_rows = cache.struct(), b, len(toks)
        qr = torch.empty_like(q)
        a.q, a.k, a.v, a.q_out, a.cos, a.sin = (t.data_ptr() for t in (q, k, v, qr, cos, sin))
        a.n_ctx, a.n_heads = 64, H
        kh.call(gpu, "af_kv_store_f32", a)
        out = torch.empty_like(q)
        t = kh.attention_args(cache, qr, out, lens, first, n)
        t.batch = b
        ws = kh.workspace(gpu, "af_attention_tree_f32", t)
        kh.call(gpu, "af_attention_tree_f32", t)
        torch.cuda.synchronize()
        del ws
        return out

    store(c, table[0], kh.ints([0]), ids, kh.ints([0, prompt]), prompt)
    scores = torch.tensor([[0.0] + [-np.inf] * (B - 1)], device="cuda")
    lens, cur, n_in = kh.ints([prompt]), table[0], 1
    history = [ids.tolist()]
    for step in range(steps):
        logits = torch.from_numpy((3 * rng.standard_normal((B, V))).astype(np.float32)).cuda()
        os_, ob, ot = (torch.zeros((1, B), dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32))
        a = _lib.BeamSelectArgs()
        a.logits, a.scores, a.out_score, a.out_beam, a.out_token = (x.data_ptr() for x in (logits, scores, os_, ob, ot))
        a.n_seq, a.n_beams, a.vocab, a.n_out = 1, B, V, B
        ws = kh.workspace(gpu, "af_beam_select_f32", a)
        kh.call(gpu, "af_beam_select_f32", a)
        nxt = table[1 + step % 2]
        new_lens = torch.zeros(B, dtype=torch.int32, device="cuda")
        one, short = kh.ints([1] * B), kh.ints([0])
        f = _lib.KvForkArgs()
        f.kv = c.struct()
        f.table_in, f.len_in, f.ref_in = cur.data_ptr(), lens.data_ptr(), ref.data_ptr()
        f.table_out, f.len_out, f.ref_out = nxt.data_ptr(), new_lens.data_ptr(), ref.data_ptr()
        f.parent, f.n_new, f.n_short, f.n_in, f.n_out, f.max_blocks = (ob.data_ptr(), one.data_ptr(), short.data_ptr(),
                                                                      n_in, B, blocks)
        ws2 = kh.workspace(gpu, "af_kv_fork", f)
        kh.call(gpu, "af_kv_fork", f)
        assert int(short.item()) == 0
        tok, par = ot[0].tolist(), ob[0].tolist()
        got = store(c, nxt, new_lens, tok, kh.ints(range(B + 1)), 1)
        assert kh.device_error(gpu) == 0
        history = [history[p] + [t] for p, t in zip(par, tok)]
        for b in range(B):
            alone = kh.Cache("f32", KV, hd, [len(history[b])], page=16, seed=2)
            want = store(alone, alone.table, kh.ints([0]), history[b], kh.ints([0, len(history[b])]), len(history[b]))
            assert (got[b] - want[-1]).abs().max() <= 2.0 ** -18 * float(vvals.abs().max()), (step, b)
        scores, lens, cur, n_in = os_.clone(), new_lens + 1, nxt, B
        del ws, ws2
    held = cur.cpu().numpy()
    np.testing.assert_array_equal(ref.cpu().numpy(), counts_of(held, c.pages))
