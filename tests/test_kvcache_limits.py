"""Limits of the cache and tree-attention entries that need no device."""
import ctypes as C

from llm_core_b200 import _lib
from test_kvcache_abi import attention, batch, beam, cache, fork


def test_rows_that_the_merge_cannot_number_are_refused():
    lib = _lib.load()
    big = batch(max_nodes=1 << 30)
    a = attention(kv=cache(n_kv_heads=4), batch=big, n_heads=4, n_rows=1 << 30)
    assert lib.af_attention_tree_f32(C.byref(a), None) != 0
    assert b"2^31" in lib.af_last_error()
    # a limit alone is none: the call has 2 rows, and fails for its workspace only
    a = attention(kv=cache(n_kv_heads=4, n_pages=4096), batch=batch(max_nodes=1 << 30, max_blocks=4096), n_heads=4, n_rows=2)
    size = lib.af_attention_tree_f32_workspace(C.byref(a))
    assert 0 < size < 1 << 28
    assert lib.af_attention_tree_f32(C.byref(a), None) != 0
    assert b"ws must hold" in lib.af_last_error()


def test_the_workspace_does_not_follow_the_rows():
    """One workspace serves calls of fewer rows and of more, up to the limits it was asked for with."""
    lib = _lib.load()
    sizes = {lib.af_attention_tree_f32_workspace(C.byref(attention(
        kv=cache(n_pages=4096), batch=batch(max_nodes=500, max_blocks=4096), n_rows=n))) for n in (0, 1, 7, 500)}
    assert len(sizes) == 1 and sizes.pop() > 0


def test_fork_tables_of_more_entries_than_32_bits_number_are_refused():
    lib = _lib.load()
    a = fork(n_out=4096, max_blocks=1 << 20)
    assert lib.af_kv_fork(C.byref(a), None) != 0
    assert b"n_out * max_blocks" in lib.af_last_error()


def test_a_beam_workspace_serves_every_smaller_call():
    """Also one of fewer rows, which have more segments each: a search whose beams die."""
    lib = _lib.load()

    def size(n_seq, n_beams, vocab, n_out):
        return lib.af_beam_select_f32_workspace(C.byref(beam(n_seq=n_seq, n_beams=n_beams, vocab=vocab, n_out=n_out)))

    for n_seq, n_beams, vocab in ((1, 32, 151936), (1, 64, 100000), (16, 8, 151936), (5, 7, 40000), (500, 2, 30000)):
        most = size(n_seq, n_beams, vocab, 64)
        for s in {1, (n_seq + 1) // 2, n_seq}:
            for b in range(1, n_beams + 1):
                for v in (64, 8192, 8193, vocab // 2, vocab):
                    # as many lists of n_out keys, a sum and a maximum as the rows have segments
                    rows, k = s * b, 64
                    segments = min(-(-v // 8192), max(1, 444 // rows))
                    assert rows * segments * (8 * k + 16) <= size(s, b, v, k) <= most


def test_more_nodes_than_are_kept_apart_are_refused():
    lib = _lib.load()
    for hd, refused in ((64, True), (128, True), (96, False)):
        a = attention(kv=cache(head_dim=hd, n_kv_heads=4), batch=batch(max_nodes=1 << 21), n_heads=4, n_rows=1048449, q=None)
        assert lib.af_attention_tree_f32(C.byref(a), None) != 0
        assert (b"1,048,448 nodes" in lib.af_last_error()) == refused
        a.n_rows = 1048448
        assert lib.af_attention_tree_f32(C.byref(a), None) != 0
        assert b"null q" in lib.af_last_error()
