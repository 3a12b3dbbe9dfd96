"""Cases of the operators that decode several hypotheses over one paged key/value cache.

A cache is a pool of pages; a sequence is a row of page ids and a length.  Five operators work on it:

* ``attention``: drafted tokens ("nodes") of each sequence attend to its cached positions and, by a bit mask,
  to the nodes that they descend from (a chain without a mask).
* ``store``: rotary positions of the nodes' queries and keys, and their K/V rows written into the pages.
* ``beam``: the best (beam, token) continuations of every sequence by cumulative log-probability.
* ``fork``: sequences follow their parents: whole pages are shared, a partly filled page is copied, pages for
  the next tokens are taken, and what nobody holds any more becomes free.
* ``compact``: the rows of the accepted nodes move to the positions behind the cached ones.

``run`` computes them in elementary torch operations, or with the library's calls where ``own`` is set.
"""
import ctypes as C
import math

import torch

own = False

TYPES = {"f32": (torch.float32, 0, 4), "f16": (torch.float16, 1, 2), "bf16": (torch.bfloat16, 2, 2)}
DEV = "cuda"


# ------------------------------------------------------------------ cases

def _attention(name, kv, heads, kv_heads, hd, n_seq, length, nodes, tree, page):
    return dict(name=name, op="attention", kv=kv, heads=heads, kv_heads=kv_heads, hd=hd, n_seq=n_seq, length=length,
                nodes=nodes, tree=tree, page=page)


def _store(name, kv, heads, kv_heads, hd, n_seq, length, nodes, norm, page):
    return dict(name=name, op="store", kv=kv, heads=heads, kv_heads=kv_heads, hd=hd, n_seq=n_seq, length=length,
                nodes=nodes, norm=norm, page=page)


def _beam(name, n_seq, beams, vocab, n_out, alive):
    return dict(name=name, op="beam", n_seq=n_seq, beams=beams, vocab=vocab, n_out=n_out, alive=alive)


def _fork(name, kv, layers, kv_heads, hd, n_seq, beams, length, new, page):
    return dict(name=name, op="fork", kv=kv, layers=layers, kv_heads=kv_heads, hd=hd, n_seq=n_seq, beams=beams,
                length=length, new=new, page=page)


def _compact(name, kv, layers, kv_heads, hd, n_seq, length, nodes, path, page):
    return dict(name=name, op="compact", kv=kv, layers=layers, kv_heads=kv_heads, hd=hd, n_seq=n_seq, length=length,
                nodes=nodes, path=path, page=page)


def listed():
    return [
        # one token of a short TinyLlama chat: the smallest call of a decode loop, all latency
        _attention("attention token 32/4x64", "f32", 32, 4, 64, 1, 137, 1, False, 16),
        # a drafted tree verified late in a Llama-2-7B context, the engine's own cache type
        _attention("attention tree 32/32x128", "f32", 32, 32, 128, 1, 3989, 26, True, 16),
        # a serving batch of Qwen2.5-3B trees, lengths from nothing to long
        _attention("attention batch 16/2x128", "f16", 16, 2, 128, 16, 8190, 31, True, 32),
        # a chunk of a long prompt behind what is cached of it: the arithmetic-bound end
        _attention("attention chunk 32/4x64", "bf16", 32, 4, 64, 2, 16001, 509, False, 64),
        # the token of the first case on its way into the cache
        _store("store token 32/4x64", "f32", 32, 4, 64, 1, 137, 1, False, 16),
        # prompt chunks of a batch, with per-head norms, into a bf16 cache
        _store("store chunk 16/2x128", "bf16", 16, 2, 128, 8, 2001, 509, True, 32),
        # the first step of a beam search: one beam alive, Llama vocabulary
        _beam("beam first 1x4x32000", 1, 4, 32000, 8, 1),
        # a serving batch over the Qwen2.5 vocabulary
        _beam("beam batch 16x8x151936", 16, 8, 151936, 16, 8),
        # four TinyLlama beams reordered between two tokens
        _fork("fork 4 beams", "f32", 22, 4, 64, 1, 4, 137, 1, 16),
        # beams of several Llama-2-7B prompts reordered
        _fork("fork 4x8 beams", "bf16", 32, 32, 128, 4, 8, 523, 1, 16),
        # a tree's accepted path, one TinyLlama sequence
        _compact("compact one", "f32", 22, 4, 64, 1, 137, 16, 4, 16),
        # accepted paths of a batch of Llama-2-7B sequences
        _compact("compact batch", "f16", 32, 32, 128, 24, 251, 31, 6, 16),
    ]


HEADS = ((32, 32, 128), (32, 4, 64), (16, 2, 128), (8, 4, 128), (4, 2, 64), (16, 8, 128))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "store", "beam", "fork", "compact"))
    kv = rng.choice(("f32", "f16", "bf16"))
    heads, kv_heads, hd = rng.choice(HEADS)
    page = rng.choice((8, 16, 32, 64))
    if op == "beam":
        n_seq, beams = _log(rng, 1, 16), rng.randint(1, 8)
        vocab = _log(rng, 500, 151936)
        return dict(op=op, n_seq=n_seq, beams=beams, vocab=vocab, n_out=min(vocab, beams * rng.randint(1, 2)),
                    alive=rng.randint(1, beams))
    if op == "attention":
        nodes, n_seq = _log(rng, 1, 256), _log(rng, 1, 16)
        length = _log(rng, 1, max(2, int(8192 * 16 // (n_seq * max(1, nodes * heads // 512)))))
        length = min(length, 16001)
        return dict(op=op, kv=kv, heads=heads, kv_heads=kv_heads, hd=hd, n_seq=n_seq, length=length, nodes=nodes,
                    tree=rng.random() < 0.7, page=page)
    if op == "store":
        return dict(op=op, kv=kv, heads=heads, kv_heads=kv_heads, hd=hd, n_seq=_log(rng, 1, 8),
                    length=_log(rng, 1, 2001), nodes=_log(rng, 1, 300), norm=rng.random() < 0.5, page=page)
    layers = rng.randint(2, 24)
    if op == "fork":
        return dict(op=op, kv=kv, layers=layers, kv_heads=kv_heads, hd=hd, n_seq=_log(rng, 1, 4),
                    beams=rng.randint(2, 8), length=_log(rng, 1, 250), new=rng.randint(1, 20), page=page)
    nodes = _log(rng, 2, 31)
    return dict(op=op, kv=kv, layers=layers, kv_heads=kv_heads, hd=hd, n_seq=_log(rng, 1, 12),
                length=_log(rng, 1, 250), nodes=nodes, path=rng.randint(1, min(nodes, 6)), page=page)


def _lengths(c):
    """The cached lengths of a case's sequences: from its longest down to nothing, evenly."""
    n = c["n_seq"]
    return [c["length"] * (n - s) // n if s < n - 1 or n == 1 else 0 for s in range(n)]


def _counts(c):
    """The nodes of each sequence: the case's number, and fewer on every other sequence."""
    return [max(1, c["nodes"] - (s % 2) * (c["nodes"] // 3)) for s in range(c["n_seq"])]


def _fork_lengths(c):
    """The lengths of the beams: equal within a prompt."""
    return [max(1, c["length"] - 37 * s % c["length"]) for s in range(c["n_seq"]) for _ in range(c["beams"])]


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    return {"attention": _prepare_rows, "store": _prepare_rows, "beam": _prepare_beam, "fork": _prepare_fork,
            "compact": _prepare_compact}[case["op"]](dict(case), g, h)


def _pool(c, layers, pages, g):
    shape = (layers, pages, c["page"], c["kv_heads"], c["hd"])
    t = TYPES[c["kv"]][0]
    return torch.randn(shape, generator=g, device=DEV, dtype=t), torch.randn(shape, generator=g, device=DEV, dtype=t)


def _tables(lengths, page, h, spare, extra=0):
    """Page ids for sequences of these many positions: pages of a shuffled pool, -1 where none is held."""
    need = [-(-n // page) for n in lengths]
    blocks = max(1, max(need) + extra)
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=h).tolist()
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (blocks - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32), pages


def _tree(n, h):
    """A drafted tree: each node's parent is one of the few nodes before it, or the last cached position."""
    back = torch.randint(1, 6, (n,), generator=h).tolist()
    parent = [max(-1, i - back[i]) for i in range(n)]
    depth, seen = [], []
    for i, p in enumerate(parent):
        depth.append(0 if p < 0 else depth[p] + 1)
        seen.append((seen[p] if p >= 0 else 0) | (1 << i))
    return depth, seen


def _prepare_rows(c, g, h):
    lengths, counts = _lengths(c), _counts(c)
    table, pages = _tables([a + b for a, b in zip(lengths, counts)], c["page"], h, 3)
    k, v = _pool(c, 1, pages, g)
    first = [0]
    for n in counts:
        first.append(first[-1] + n)
    rows = first[-1]
    words = -(-max(counts) // 64)
    depth, mask = [], []
    for n in counts:
        if c["op"] == "attention" and not c["tree"]:
            d, m = list(range(n)), []
        else:
            d, m = _tree(n, h)
        depth += d
        for bits in m:
            w = [(bits >> (64 * i)) & (2 ** 64 - 1) for i in range(words)]
            mask.append([x - 2 ** 64 if x >= 2 ** 63 else x for x in w])
    put = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device=DEV)  # noqa: E731
    s = dict(case=c, k_pool=k, v_pool=v, table=table.to(DEV), length=put(lengths), first=put(first),
             max_length=max(a + b for a, b in zip(lengths, counts)))
    H, KV, hd = c["heads"], c["kv_heads"], c["hd"]
    s["q"] = 1.5 * torch.randn((rows, H, hd), generator=g, device=DEV)
    s["out"] = torch.empty((rows, H, hd), device=DEV)
    if c["op"] == "attention":
        s["mask"] = put(mask, torch.int64) if c["tree"] else None
        return s
    s["k"] = torch.randn((rows, KV, hd), generator=g, device=DEV)
    s["v"] = torch.randn((rows, KV, hd), generator=g, device=DEV)
    s["depth"] = put(depth)
    n_ctx = s["max_length"]
    angle = torch.arange(n_ctx, dtype=torch.float64, device=DEV)[:, None] * (
        10000.0 ** (-torch.arange(hd // 2, dtype=torch.float64, device=DEV) * 2 / hd))
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    for n in ("q_norm", "k_norm"):
        s[n] = 1 + 0.1 * torch.randn(hd, generator=g, device=DEV) if c["norm"] else None
    return s


def _prepare_beam(c, g, h):
    rows = c["n_seq"] * c["beams"]
    logits = 3 * torch.randn((rows, c["vocab"]), generator=g, device=DEV)
    scores = -3 * torch.rand((c["n_seq"], c["beams"]), generator=g, device=DEV)
    scores[:, c["alive"]:] = -math.inf
    n = (c["n_seq"], c["n_out"])
    return dict(case=c, logits=logits, scores=scores, out_score=torch.empty(n, device=DEV),
                out_beam=torch.empty(n, dtype=torch.int32, device=DEV),
                out_token=torch.empty(n, dtype=torch.int32, device=DEV))


def _prepare_fork(c, g, h):
    page, beams, lengths = c["page"], c["beams"], _fork_lengths(c)
    n, new = len(lengths), c["new"]
    blocks = max(-(-(x + 2 * new + page) // page) for x in lengths)
    rows, pages = [], 0
    for i, x in enumerate(lengths):  # whole pages shared by a prompt's beams, the rest a beam's own
        full = x // page
        mine = full + (1 if x % page else 0)
        shared = rows[i - i % beams][:full] if i % beams else list(range(pages, pages + full))
        pages += 0 if i % beams else full
        rows.append(shared + list(range(pages, pages + mine - full)))
        pages += mine - full
    total = pages + 2 * n + n * (-(-new // page)) + 3
    order = torch.randperm(total, generator=h)
    table = torch.full((n, blocks), -1, dtype=torch.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = order[torch.tensor(r, dtype=torch.int64)].to(torch.int32)
    ref = torch.zeros(total, dtype=torch.int32)
    held = table[table >= 0].long()
    ref.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    parent = torch.cat([s * beams + torch.randint(0, beams, (beams,), generator=h) for s in range(c["n_seq"])])
    k, v = _pool(c, c["layers"], total, g)
    put = lambda x: x.to(device=DEV, dtype=torch.int32)  # noqa: E731
    return dict(case=c, k_pool=k, v_pool=v, table=put(table), length=put(torch.tensor(lengths)), ref=put(ref),
                parent=put(parent), new=torch.full((n,), new, dtype=torch.int32, device=DEV),
                table_out=torch.empty((n, blocks), dtype=torch.int32, device=DEV),
                length_out=torch.empty(n, dtype=torch.int32, device=DEV),
                ref_out=torch.empty(total, dtype=torch.int32, device=DEV),
                short=torch.zeros(1, dtype=torch.int32, device=DEV))


def _prepare_compact(c, g, h):
    n = c["n_seq"]
    lengths = [c["length"] - 7 * s % c["length"] for s in range(n)]
    table, pages = _tables([x + c["nodes"] for x in lengths], c["page"], h, 2)
    k, v = _pool(c, c["layers"], pages, g)
    path = torch.stack([torch.randperm(c["nodes"], generator=h)[:c["path"]].sort().values for _ in range(n)])
    count = torch.tensor([max(1, c["path"] - s % 3) for s in range(n)])
    put = lambda x: x.to(device=DEV, dtype=torch.int32)  # noqa: E731
    return dict(case=c, k_pool=k, v_pool=v, table=put(table), length=put(torch.tensor(lengths)), path=put(path),
                count=put(count), length_out=torch.empty(n, dtype=torch.int32, device=DEV))


# ------------------------------------------------------------------ one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    return {"attention": _plain_attention, "store": _plain_store, "beam": _plain_beam, "fork": _plain_fork,
            "compact": _plain_compact}[op](state)


def _rows_of(s):
    """The sequence and the node number of every row."""
    row = torch.arange(s["q"].shape[0], device=DEV)
    seq = (row[:, None] >= s["first"][None, 1:]).sum(1)
    return seq, row - s["first"][seq]


def _slots(s, seq, pos):
    """The pool rows of positions `pos` of sequences `seq`."""
    page = s["case"]["page"]
    return s["table"][seq, pos // page].long() * page + pos % page


def _plain_attention(s):
    c = s["case"]
    H, KV, hd, n, L = c["heads"], c["kv_heads"], c["hd"], c["n_seq"], s["max_length"]
    G, N = H // KV, max(_counts(c))
    seq, node = _rows_of(s)
    pos = torch.arange(L, device=DEV)
    end = s["length"] + s["first"][1:] - s["first"][:-1]
    inside = pos[None, :] < end[:, None]
    slots = torch.where(inside, _slots(s, torch.arange(n, device=DEV)[:, None], pos[None, :]), 0)
    k = s["k_pool"][0].view(-1, KV, hd)[slots].float() * inside[..., None, None]
    v = s["v_pool"][0].view(-1, KV, hd)[slots].float() * inside[..., None, None]
    q = torch.zeros((n, N, H, hd), device=DEV)
    q[seq, node] = s["q"]
    q = q.view(n, N, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(n, KV, G * N, hd)
    w = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(hd)
    past = pos[None, :] - s["length"][:, None]
    if s["mask"] is None:
        seen = past[:, None, :] <= torch.arange(N, device=DEV)[None, :, None]
    else:
        bits = torch.zeros((n, N, s["mask"].shape[1]), dtype=torch.int64, device=DEV)
        bits[seq, node] = s["mask"]
        at = past.clamp(0, N - 1)
        word = torch.gather(bits, 2, (at // 64)[:, None, :].expand(n, N, L))
        seen = (past < 0)[:, None, :] | ((word >> (at % 64)[:, None, :]) & 1).bool()
    seen = seen & inside[:, None, :]
    w = w.view(n, KV, G, N, L).masked_fill_(~seen[:, None, None], -math.inf).view(n, KV, G * N, L)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w, v.permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    o = o.view(n, KV, G, N, hd).permute(0, 3, 1, 2, 4).reshape(n, N, H, hd)
    return o[seq, node]


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _plain_store(s):
    seq, node = _rows_of(s)
    at = (s["length"][seq] + s["depth"]).long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q, k = s["q"], s["k"]
    if s["q_norm"] is not None:
        q = s["q_norm"] * (q / torch.sqrt((q * q).mean(-1, keepdim=True) + 1e-6))
        k = s["k_norm"] * (k / torch.sqrt((k * k).mean(-1, keepdim=True) + 1e-6))
    slots = _slots(s, seq, (s["length"][seq] + node).long())
    c = s["case"]
    s["k_pool"][0].view(-1, c["kv_heads"], c["hd"])[slots] = _rotate(k, cos, sin).to(s["k_pool"].dtype)
    s["v_pool"][0].view(-1, c["kv_heads"], c["hd"])[slots] = s["v"].to(s["v_pool"].dtype)
    return _rotate(q, cos, sin), s["k_pool"], s["v_pool"]


def _plain_beam(s):
    c = s["case"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    total = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    x = (x - total).view(c["n_seq"], c["beams"], c["vocab"]) + s["scores"].double()[..., None]
    x = torch.nan_to_num(x.view(c["n_seq"], -1), nan=-math.inf, neginf=-math.inf)
    best, at = torch.sort(x, dim=-1, descending=True, stable=True)
    best, at = best[:, :c["n_out"]], at[:, :c["n_out"]]
    beam = at // c["vocab"] + torch.arange(c["n_seq"], device=DEV)[:, None] * c["beams"]
    return best.float(), beam.int(), (at % c["vocab"]).int()


def _plain_fork(s):
    page = s["case"]["page"]
    parent, ref, table = s["parent"].long(), s["ref"], s["table"]
    n, blocks = table.shape
    length = s["length"][parent]
    part, full = length % page, (length // page)[:, None]
    need = ((length + s["new"] + page - 1) // page)[:, None]
    b = torch.arange(blocks, device=DEV)[None, :]
    i = torch.arange(n, device=DEV)
    eldest = ~((parent[:, None] == parent[None, :]) & (i[None, :] < i[:, None])).any(1)
    old = table[parent]
    alone = (old >= 0) & (ref[old.clamp(min=0).long()] == 1)
    kept = (b < full) | ((b < need) & eldest[:, None] & alone)
    fresh = (b < need) & ~kept
    order = torch.sort((ref != 0).int(), stable=True).indices
    rank = (torch.cumsum(fresh.view(-1), 0) - 1).view(n, blocks)
    have = fresh & (rank < (ref == 0).sum())
    page_of = order[rank.clamp(0, ref.numel() - 1)].int()
    out = torch.where(kept, old, torch.where(have, page_of, -1))
    count = ref.clone()
    count.index_add_(0, table.clamp(min=0).view(-1).long(), -(table >= 0).view(-1).int())
    count.index_add_(0, out.clamp(min=0).view(-1).long(), (out >= 0).view(-1).int())
    last = (b == full) & (part > 0)[:, None] & fresh
    lost = (last & ~have).any(1)
    new_length = torch.where(lost, (length // page) * page, length)
    seq, blk = torch.nonzero(last & have, as_tuple=True)
    src, dst = old[seq, blk].long(), out[seq, blk].long()
    row = torch.arange(page, device=DEV)[None, :]
    which, at = torch.nonzero(row < part[seq][:, None], as_tuple=True)
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, dst[which], at] = pool[:, src[which], at]
    missing = (fresh & ~have).sum().int().view(1)
    return out, new_length.int(), count, missing, s["k_pool"], s["v_pool"]


def _plain_compact(s):
    c = s["case"]
    i = torch.arange(c["path"], device=DEV)[None, :]
    seq, at = torch.nonzero(i < s["count"][:, None], as_tuple=True)
    src = _slots(s, seq, (s["length"][seq] + s["path"][seq, at]).long())
    dst = _slots(s, seq, (s["length"][seq] + at).long())
    for pool in (s["k_pool"], s["v_pool"]):
        rows = pool.view(c["layers"], -1, c["kv_heads"] * c["hd"])
        rows[:, dst] = rows[:, src]
    return s["k_pool"], s["v_pool"], s["length"] + s["count"]


# ------------------------------------------------------------------ the library's calls

def _ptr(x):
    return None if x is None else x.data_ptr()


def _cache(lib, s):
    k = s["k_pool"]
    c = lib.KvCache()
    c.k, c.v, c.type = _ptr(k), _ptr(s["v_pool"]), TYPES[s["case"]["kv"]][1]
    c.n_layers, c.n_pages, c.page_size, c.n_kv_heads, c.head_dim = k.shape
    return c


def _batch(lib, s):
    b = lib.KvBatch()
    b.block_table, b.len, b.first = _ptr(s["table"]), _ptr(s["length"]), _ptr(s.get("first"))
    b.n_seq, b.max_blocks = s["table"].shape
    b.max_nodes = max(_counts(s["case"])) if "first" in s else 0
    return b


def _args_attention(lib, s):
    a = lib.AttentionTreeArgs()
    a.kv, a.batch = _cache(lib, s), _batch(lib, s)
    a.q, a.out, a.n_heads, a.n_rows, a.max_len = _ptr(s["q"]), _ptr(s["out"]), s["q"].shape[1], s["q"].shape[0], s["max_length"]
    if s["mask"] is not None:
        a.mask, a.mask_words = _ptr(s["mask"]), s["mask"].shape[1]
    return a, "af_attention_tree_f32", s["out"]


def _args_store(lib, s):
    a = lib.KvStoreArgs()
    a.kv, a.batch = _cache(lib, s), _batch(lib, s)
    a.q, a.k, a.v, a.q_out, a.depth = _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(s["out"]), _ptr(s["depth"])
    a.cos, a.sin, a.n_ctx = _ptr(s["cos"]), _ptr(s["sin"]), s["cos"].shape[0]
    a.n_heads, a.n_rows = s["q"].shape[1], s["q"].shape[0]
    a.q_norm, a.k_norm, a.eps = _ptr(s["q_norm"]), _ptr(s["k_norm"]), 1e-6
    a.qk_norm_order = 1 if s["q_norm"] is not None else 0
    return a, "af_kv_store_f32", (s["out"], s["k_pool"], s["v_pool"])


def _args_beam(lib, s):
    c = s["case"]
    a = lib.BeamSelectArgs()
    a.logits, a.scores = _ptr(s["logits"]), _ptr(s["scores"])
    a.out_score, a.out_beam, a.out_token = _ptr(s["out_score"]), _ptr(s["out_beam"]), _ptr(s["out_token"])
    a.n_seq, a.n_beams, a.vocab, a.n_out = c["n_seq"], c["beams"], c["vocab"], c["n_out"]
    return a, "af_beam_select_f32", (s["out_score"], s["out_beam"], s["out_token"])


def _args_fork(lib, s):
    a = lib.KvForkArgs()
    a.kv = _cache(lib, s)
    a.table_in, a.len_in, a.ref_in = _ptr(s["table"]), _ptr(s["length"]), _ptr(s["ref"])
    a.table_out, a.len_out, a.ref_out = _ptr(s["table_out"]), _ptr(s["length_out"]), _ptr(s["ref_out"])
    a.parent, a.n_new, a.n_short = _ptr(s["parent"]), _ptr(s["new"]), _ptr(s["short"])
    a.n_in, a.max_blocks = s["table"].shape
    a.n_out = s["parent"].shape[0]
    return a, "af_kv_fork", (s["table_out"], s["length_out"], s["ref_out"], s["short"], s["k_pool"], s["v_pool"])


def _args_compact(lib, s):
    a = lib.KvCompactArgs()
    a.kv, a.batch = _cache(lib, s), _batch(lib, s)
    a.path, a.n_path, a.max_path, a.len_out = _ptr(s["path"]), _ptr(s["count"]), s["path"].shape[1], _ptr(s["length_out"])
    return a, "af_kv_compact", (s["k_pool"], s["v_pool"], s["length_out"])


def _own(s, op):
    if "call" not in s:  # the argument block and the workspace that a program keeps beside its buffers
        from llm_core_b200 import _lib
        lib = _lib.load()
        a, name, outputs = {"attention": _args_attention, "store": _args_store, "beam": _args_beam,
                            "fork": _args_fork, "compact": _args_compact}[op](_lib, s)
        if op in ("attention", "beam", "fork"):
            size = getattr(lib, name + "_workspace")(C.byref(a))
            s["ws"] = torch.zeros(max(size, 16), dtype=torch.uint8, device=DEV)
            a.ws, a.ws_bytes = s["ws"].data_ptr(), size
        s["call"] = (getattr(lib, name), C.byref(a), _lib.check, name, outputs, a)
    call, a, check, name, outputs, _ = s["call"]
    check(call(a, torch.cuda.current_stream().cuda_stream), name)
    return outputs


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c, op = case, case["op"]
    if op == "beam":
        rows = c["n_seq"] * c["beams"]
        return {"bytes": 4 * rows * c["vocab"] + 4 * rows + 12 * c["n_seq"] * c["n_out"], "flops": 4 * rows * c["vocab"]}
    size = TYPES[c["kv"]][2]
    row = c["kv_heads"] * c["hd"]
    if op in ("attention", "store"):
        lengths, counts = _lengths(c), _counts(c)
        rows, q = sum(counts), c["heads"] * c["hd"]
        if op == "attention":
            pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(lengths, counts))
            return {"bytes": 2 * size * row * (sum(lengths) + rows) + 8 * rows * q, "flops": 4 * pairs * q}
        return {"bytes": rows * (8 * q + (8 + 2 * size) * row + 4 * c["hd"]), "flops": 4 * rows * (q + row)}
    if op == "fork":
        lengths = _fork_lengths(c)
        blocks = sum(-(-x // c["page"]) for x in lengths)
        copied = (c["beams"] - 1) * sum(lengths[s * c["beams"]] % c["page"] for s in range(c["n_seq"])) // 2
        return {"bytes": 4 * size * c["layers"] * row * copied + 12 * blocks, "flops": 0}
    moved = sum(max(1, c["path"] - s % 3) for s in range(c["n_seq"]))
    return {"bytes": 4 * size * c["layers"] * row * moved, "flops": 0}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    op = case["op"]
    if op in ("fork", "compact"):
        return None  # rows are moved and pages counted: nothing is rounded
    s = prepare(case, seed)
    if op == "beam":
        return _exact_beam(s)
    return _exact_attention(s) if op == "attention" else _exact_store(s)


def _exact_attention(s):
    c = s["case"]
    page, G = c["page"], c["heads"] // c["kv_heads"]
    first, lengths, table = s["first"].tolist(), s["length"].tolist(), s["table"].tolist()
    out = []
    for i, past in enumerate(lengths):
        n = first[i + 1] - first[i]
        ids = torch.tensor(table[i][:-(-(past + n) // page)], device=DEV)
        k = s["k_pool"][0, ids].flatten(0, 1)[:past + n].double()
        v = s["v_pool"][0, ids].flatten(0, 1)[:past + n].double()
        seen = torch.ones((n, past + n), dtype=torch.bool, device=DEV)
        if s["mask"] is None:
            seen[:, past:] = torch.ones((n, n), dtype=torch.bool, device=DEV).tril()
        else:
            bits = s["mask"][first[i]:first[i + 1]].cpu().numpy().view("uint64").tolist()
            rows = [[(r[j // 64] >> (j % 64)) & 1 for j in range(n)] for r in bits]
            seen[:, past:] = torch.tensor(rows, dtype=torch.bool, device=DEV)
        q = s["q"][first[i]:first[i + 1]].double()
        heads = []
        for h in range(c["heads"]):
            w = q[:, h] @ k[:, h // G].T * c["hd"] ** -0.5
            heads.append(torch.softmax(w.masked_fill(~seen, -math.inf), -1) @ v[:, h // G])
        out.append(torch.stack(heads, 1))
    return torch.cat(out)


def _exact_store(s):
    c = s["case"]
    page, hd = c["page"], c["hd"]
    first, lengths, table, depth = (s[x].tolist() for x in ("first", "length", "table", "depth"))
    seq = [i for i in range(c["n_seq"]) for _ in range(first[i + 1] - first[i])]
    at = torch.tensor([lengths[i] + depth[r] for r, i in enumerate(seq)], device=DEV)
    slot = torch.tensor([table[i][(lengths[i] + r - first[i]) // page] * page + (lengths[i] + r - first[i]) % page
                         for r, i in enumerate(seq)], device=DEV)
    turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
    done = []
    for x, w in ((s["q"].double(), s["q_norm"]), (s["k"].double(), s["k_norm"])):
        if w is not None:
            x = x * ((x.square().sum(-1, keepdim=True) / hd + 1e-6) ** -0.5) * w.double()
        z = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * turn
        done.append(torch.cat((z.real, z.imag), -1))
    k, v = s["k_pool"].double(), s["v_pool"].double()
    k.view(-1, c["kv_heads"], hd)[slot] = done[1]
    v.view(-1, c["kv_heads"], hd)[slot] = s["v"].double()
    return done[0], k, v


def _exact_beam(s):
    c = s["case"]
    score = []
    for i in range(c["n_seq"]):
        x = torch.log_softmax(s["logits"][i * c["beams"]:(i + 1) * c["beams"]].double(), -1)
        x = (x + s["scores"][i].double()[:, None]).flatten()
        score.append(torch.topk(x, c["n_out"]).values)
    return torch.stack(score), None, None
