"""Paged caches for the tests: argument blocks of the entry points over torch
buffers, and the operators' definitions in plain 64-bit numpy / Python."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from llm_core_b200 import _lib

TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def ptr(x):
    return None if x is None else x.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


def device_error(lib) -> int:
    """Read and clear the device error word."""
    torch.cuda.synchronize()
    code = C.c_int(0)
    _lib.check(lib.af_device_error(C.byref(code), 1), "af_device_error")
    return code.value


class Cache:
    """A pool with a shuffled table for sequences of the given positions."""

    def __init__(self, kv, kv_heads, hd, positions, page=16, layers=1, spare=2, seed=0, extra_blocks=1, fill=None,
                 contiguous=False):
        self.kv, self.kv_heads, self.hd, self.page, self.layers = kv, kv_heads, hd, page, layers
        need = [-(-n // page) for n in positions]
        self.blocks = max(1, max(need, default=1) + extra_blocks)
        rng = np.random.default_rng(seed)
        if contiguous:
            self.pages = len(positions) * self.blocks
            self.table_h = np.arange(self.pages, dtype=np.int32).reshape(len(positions), self.blocks)
            self.table = None
        else:
            self.pages = sum(need) + spare
            order = rng.permutation(self.pages)
            self.table_h = np.full((len(positions), self.blocks), -1, np.int32)
            at = 0
            for s, n in enumerate(need):
                self.table_h[s, :n] = order[at:at + n]
                at += n
            self.table = ints(self.table_h)
        shape = (layers, self.pages, page, kv_heads, hd)
        dt = TYPES[kv][0]
        if fill is None:
            self.k = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dt).cuda()
            self.v = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dt).cuda()
        else:
            self.k = torch.full(shape, fill, dtype=dt, device="cuda")
            self.v = torch.full(shape, fill, dtype=dt, device="cuda")

    def struct(self):
        c = _lib.KvCache()
        c.k, c.v, c.type = ptr(self.k), ptr(self.v), TYPES[self.kv][1]
        c.n_layers, c.n_pages, c.page_size, c.n_kv_heads, c.head_dim = (self.layers, self.pages, self.page,
                                                                        self.kv_heads, self.hd)
        return c

    def batch(self, length, first=None, max_nodes=0, n_seq=None):
        b = _lib.KvBatch()
        b.block_table, b.len, b.first = ptr(self.table), ptr(length), ptr(first)
        b.n_seq, b.max_blocks, b.max_nodes = n_seq or self.table_h.shape[0], self.blocks, max_nodes
        return b

    def rows(self, pool, layer, s, n):
        """Positions 0..n-1 of sequence s in 64 bits: [n][kv_heads][hd]."""
        pos = np.arange(n)
        page = torch.as_tensor(self.table_h[s, pos // self.page].astype(np.int64)).cuda()
        return pool[layer, page, torch.as_tensor(pos % self.page).cuda()].double().cpu().numpy()


def tree_of(n, rng, branch=5):
    """Parents of a random tree of n nodes (-1: a root), depths, and its mask rows as Python ints."""
    parent = [max(-1, i - int(rng.integers(1, branch + 1))) for i in range(n)]
    depth, seen = [], []
    for i, p in enumerate(parent):
        depth.append(0 if p < 0 else depth[p] + 1)
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    return parent, depth, seen


def mask_words(rows, words):
    return torch.as_tensor(np.array([[(b >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for b in rows],
                                    np.uint64).view(np.int64)).cuda()


def attention_args(cache, q, out, length, first, max_nodes, mask=None, layer=0, scale=0.0, max_len=0, q_stride=0,
                   out_stride=0, n_rows=None, heads=None):
    a = _lib.AttentionTreeArgs()
    a.kv, a.batch = cache.struct(), cache.batch(length, first, max_nodes)
    a.layer, a.n_rows, a.n_heads = layer, n_rows if n_rows is not None else q.shape[0], heads or q.shape[1]
    a.q, a.out, a.q_stride, a.out_stride = ptr(q), ptr(out), q_stride, out_stride
    if mask is not None:
        a.mask, a.mask_words = ptr(mask), mask.shape[1]
    a.scale, a.max_len = scale, max_len
    a.keep = (q, out, length, first, mask, cache)  # the buffers live as long as the block that points at them
    return a


def workspace(lib, name, a):
    n = getattr(lib, name + "_workspace")(C.byref(a))
    ws = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda")
    a.ws, a.ws_bytes = ws.data_ptr(), n
    return ws


def call(lib, name, a):
    _lib.check(getattr(lib, name)(C.byref(a), stream()), name)


def attention_plain(q, k, v, seen, scale):
    """q [n][H][hd], k, v [L][KV][hd], seen [n][L] -> out [n][H][hd] and the
    bound of each element's error that fp32 arithmetic leaves: scores off by
    ds = (3·2^-22 + hd·2^-24)·Σ|q||k|·scale (operands held to 2^-22, the dot's hd
    additions), which moves an output by at most 2·ds·max|v|; weights, their sum
    and the output's accumulation add (L + 8)·2^-24 of Σ w|v| <= max|v| (a sum of
    L positive terms, accumulated in any order)."""
    n, H, hd = q.shape
    G = H // k.shape[1]
    out, tol = np.zeros((n, H, hd)), np.zeros((n, H, 1))
    for h in range(H):
        for i in range(n):
            at = np.nonzero(seen[i])[0]
            if not len(at):
                continue
            kk, vv = k[at, h // G], v[at, h // G]
            with np.errstate(all="ignore"):
                s = kk @ q[i, h] * scale
                w = np.exp(s - s.max())
                out[i, h] = w @ vv / w.sum()
                ds = (3 * 2.0 ** -22 + hd * 2.0 ** -24) * (np.abs(kk) @ np.abs(q[i, h])).max() * abs(scale)
                tol[i, h] = np.abs(vv).max() * (2 * ds + (len(at) + 8) * 2.0 ** -24)
    return out, tol


def seen_matrix(length, n, rows=None):
    seen = np.zeros((n, length + n), bool)
    seen[:, :length] = True
    for i in range(n):
        for j in range(n):
            seen[i, length + j] = j <= i if rows is None else bool(rows[i] >> j & 1)
    return seen


def fork_plain(page, pages, table, length, ref, parent, new, blocks):
    """af_kv_fork's definition: tables, lengths, counts, missing pages, and
    the copies (source page, destination page, rows)."""
    n_in = len(length)
    free = [i for i in range(pages) if ref[i] == 0]
    count = list(ref)
    for row in table:
        for x in row:
            if x >= 0:
                count[x] -= 1
    out, out_len, copies, short, done = [], [], [], 0, set()
    for i, j in enumerate(parent):
        j = j if 0 <= j < n_in else -1
        n = int(length[j]) if j >= 0 else 0
        first = j >= 0 and j not in done
        done.add(j)
        need = -(-(n + new[i]) // page)
        short += max(0, need - blocks)
        need = min(need, blocks)
        row = [-1] * blocks
        for b in range(need):
            old = int(table[j][b]) if j >= 0 else -1
            if b < n // page:
                row[b] = old
            elif first and old >= 0 and ref[old] == 1:
                row[b] = old
            elif free:
                row[b] = free.pop(0)
                if b == n // page and n % page and old >= 0:
                    copies.append((old, row[b], n % page))
            else:
                short += 1
                if b == n // page and n % page:
                    n = n // page * page
        for x in row:
            if x >= 0:
                count[x] += 1
        out.append(row)
        out_len.append(n)
    return out, out_len, count, short, copies


def beam_plain(logits, scores, n_out):
    """The best continuations in 64 bits: (score, row, token) lists per sequence."""
    S, B = scores.shape
    V = logits.shape[1]
    with np.errstate(all="ignore"):
        x = logits.astype(np.float64)
        top = x.max(1, keepdims=True)
        x = x - (top + np.log(np.exp(x - top).sum(1, keepdims=True))) + scores.astype(np.float64).reshape(-1, 1)
    x[np.isnan(x)] = -np.inf
    x[~(scores.reshape(-1) > -np.inf)] = -np.inf
    res = []
    for s in range(S):
        f = x[s * B:(s + 1) * B].reshape(-1)
        at = np.argsort(-f, kind="stable")[:n_out]
        res.append((f[at], s * B + at // V, at % V))
    return res


def rope_tables(n_ctx, hd, theta=10000.0):
    ang = np.arange(n_ctx, dtype=np.float64)[:, None] * theta ** (-2.0 * np.arange(hd // 2) / hd)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def isqrt(hd):
    return 1.0 / math.sqrt(hd)
