"""Argument checks of the cache, tree-attention and beam entries, without a device."""
import ctypes as C

import pytest

from llm_core_b200 import _lib


def cache(**kw):
    c = _lib.KvCache()
    c.k, c.v, c.type, c.n_layers, c.n_pages, c.page_size, c.n_kv_heads, c.head_dim = 4096, 8192, 0, 2, 8, 16, 2, 64
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def batch(**kw):
    b = _lib.KvBatch()
    b.block_table, b.len, b.first, b.n_seq, b.max_blocks, b.max_nodes = 256, 512, 768, 1, 4, 2
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def store(**kw):
    a = _lib.KvStoreArgs()
    a.kv, a.batch, a.n_rows, a.n_ctx, a.n_heads = cache(), batch(), 2, 64, 4
    a.q = a.k = a.v = a.q_out = a.cos = a.sin = 4096
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attention(**kw):
    a = _lib.AttentionTreeArgs()
    a.kv, a.batch, a.n_rows, a.n_heads, a.q, a.out = cache(), batch(), 2, 4, 4096, 8192
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def beam(**kw):
    a = _lib.BeamSelectArgs()
    a.logits = a.scores = a.out_score = a.out_beam = a.out_token = 4096
    a.n_seq, a.n_beams, a.vocab, a.n_out = 1, 4, 1000, 8
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def fork(**kw):
    a = _lib.KvForkArgs()
    a.kv = cache()
    a.table_in, a.len_in, a.ref_in, a.table_out, a.len_out, a.ref_out = 4096, 8192, 16384, 32768, 65536, 1 << 20
    a.parent, a.n_new, a.n_short, a.n_in, a.n_out, a.max_blocks = 1 << 21, 0, 1 << 22, 2, 2, 4
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def compact(**kw):
    a = _lib.KvCompactArgs()
    a.kv, a.batch, a.path, a.n_path, a.max_path, a.len_out = cache(), batch(), 4096, 4096, 4, 4096
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_CACHES = [(dict(type=3), b"type"), (dict(type=-1), b"type"), (dict(n_pages=0), b"positive"),
              (dict(n_layers=0), b"positive"), (dict(n_kv_heads=0), b"positive"), (dict(page_size=12), b"power of two"),
              (dict(page_size=0), b"power of two"), (dict(head_dim=12), b"multiple of 8"), (dict(head_dim=264), b"256"),
              (dict(head_dim=0), b"multiple of 8"), (dict(k=None), b"null"), (dict(v=None), b"null"),
              (dict(k=4100), b"aligned"), (dict(layer_stride=12), b"layer_stride"), (dict(layer_stride=64), b"layer_stride"),
              (dict(layer_stride=-8), b"layer_stride")]


@pytest.mark.parametrize("kw,text", BAD_CACHES)
def test_bad_caches(kw, text):
    lib = _lib.load()
    for name, a in (("af_kv_store_f32", store(kv=cache(**kw))), ("af_attention_tree_f32", attention(kv=cache(**kw))),
                    ("af_kv_fork", fork(kv=cache(**kw))), ("af_kv_compact", compact(kv=cache(**kw)))):
        assert getattr(lib, name)(C.byref(a), None) != 0
        assert text in lib.af_last_error() and name.encode() in lib.af_last_error()


@pytest.mark.parametrize("kw,text", [(dict(n_seq=-1), b"n_seq"), (dict(n_seq=70000), b"n_seq"), (dict(max_blocks=0), b"max_blocks"),
                                     (dict(max_blocks=1 << 28), b"max_blocks"), (dict(len=None), b"len")])
def test_bad_batches(kw, text):
    lib = _lib.load()
    for name, a in (("af_kv_store_f32", store(batch=batch(**kw))), ("af_attention_tree_f32", attention(batch=batch(**kw))),
                    ("af_kv_compact", compact(batch=batch(**kw)))):
        assert getattr(lib, name)(C.byref(a), None) != 0
        assert text in lib.af_last_error()


@pytest.mark.parametrize("kw,text", [(dict(layer=2), b"layer"), (dict(layer=-1), b"layer"), (dict(n_rows=-1), b"n_rows"),
                                     (dict(n_heads=0), b"n_heads"), (dict(qk_norm_order=3), b"qk_norm_order"),
                                     (dict(q=None), b"null"), (dict(cos=None), b"null"), (dict(q_stride=100), b"stride"),
                                     (dict(k_stride=100), b"stride"), (dict(q_stride=300), b"in place"),
                                     (dict(n_ctx=0), b"n_ctx")])
def test_bad_store(kw, text):
    lib = _lib.load()
    assert lib.af_kv_store_f32(C.byref(store(**kw)), None) != 0
    assert text in lib.af_last_error()


@pytest.mark.parametrize("kw,text", [(dict(layer=2), b"layer"), (dict(n_rows=-1), b"n_rows"), (dict(n_heads=3), b"multiple"),
                                     (dict(n_heads=0), b"multiple"), (dict(q=None), b"null"), (dict(out=None), b"null"),
                                     (dict(mask=4096, mask_words=0), b"mask_words"), (dict(out_stride=9), b"stride"),
                                     (dict(max_len=-1), b"max_len"),
                                     (dict(mask=4096, mask_words=1, batch=batch(max_nodes=65)), b"mask_words")])
def test_bad_attention(kw, text):
    lib = _lib.load()
    assert lib.af_attention_tree_f32(C.byref(attention(**kw)), None) != 0
    assert text in lib.af_last_error()


@pytest.mark.parametrize("kw,text", [(dict(n_beams=0), b"n_beams"), (dict(n_beams=65), b"n_beams"), (dict(vocab=0), b"vocab"),
                                     (dict(n_out=0), b"n_out"), (dict(n_out=65), b"n_out"), (dict(n_out=9, vocab=2), b"n_out"),
                                     (dict(n_seq=-1), b"n_seq"), (dict(n_seq=20000), b"65535"), (dict(logits_stride=999), b"stride"),
                                     (dict(n_beams=64, vocab=140000), b"1024"), (dict(scores=None), b"null"), (dict(), b"ws")])
def test_bad_beam(kw, text):
    lib = _lib.load()
    assert lib.af_beam_select_f32(C.byref(beam(**kw)), None) != 0
    assert text in lib.af_last_error()


@pytest.mark.parametrize("kw,text", [(dict(n_in=-1), b"n_in"), (dict(n_out=5000), b"n_out"), (dict(max_blocks=0), b"max_blocks"),
                                     (dict(ref_in=None), b"ref_in"), (dict(n_short=None), b"n_short"), (dict(table_in=None), b"table_in"),
                                     (dict(parent=None), b"parent"), (dict(table_out=4096 + 16), b"overlap"),
                                     (dict(len_out=8192 + 4), b"overlap"), (dict(ref_out=16384 + 4), b"ref_out"), (dict(), b"ws")])
def test_bad_fork(kw, text):
    lib = _lib.load()
    assert lib.af_kv_fork(C.byref(fork(**kw)), None) != 0
    assert text in lib.af_last_error()


@pytest.mark.parametrize("kw,text", [(dict(max_path=-1), b"max_path"), (dict(path=None), b"null"), (dict(len_out=None), b"null"),
                                     (dict(n_path=None), b"null")])
def test_bad_compact(kw, text):
    lib = _lib.load()
    assert lib.af_kv_compact(C.byref(compact(**kw)), None) != 0
    assert text in lib.af_last_error()


def test_nothing_to_do_and_null_arguments():
    lib = _lib.load()
    for name in ("af_kv_store_f32", "af_attention_tree_f32", "af_beam_select_f32", "af_kv_fork", "af_kv_compact"):
        assert getattr(lib, name)(None, None) != 0
        assert b"null" in lib.af_last_error()
    assert lib.af_kv_store_f32(C.byref(store(n_rows=0)), None) == 0
    assert lib.af_attention_tree_f32(C.byref(attention(n_rows=0)), None) == 0
    assert lib.af_attention_tree_f32(C.byref(attention(batch=batch(n_seq=0))), None) == 0
    assert lib.af_beam_select_f32(C.byref(beam(n_seq=0)), None) == 0
    assert lib.af_kv_compact(C.byref(compact(batch=batch(n_seq=0))), None) == 0


def test_workspace_sizes():
    lib = _lib.load()
    for name in ("af_attention_tree_f32", "af_beam_select_f32", "af_kv_fork"):
        assert getattr(lib, name + "_workspace")(None) == 0
    assert lib.af_beam_select_f32_workspace(C.byref(beam())) > 0
    assert lib.af_beam_select_f32_workspace(C.byref(beam(n_out=0))) == 0
    assert lib.af_kv_fork_workspace(C.byref(fork())) >= 2 * 16 + 8 * 4


def test_a_cache_of_too_many_layers_is_refused_before_anything_is_launched():
    lib = _lib.load()
    many = cache(n_layers=32768)
    for name, a in (("af_kv_fork", fork(kv=many)), ("af_kv_compact", compact(kv=many))):
        assert getattr(lib, name)(C.byref(a), None) != 0
        assert b"n_layers" in lib.af_last_error()


def test_tree_and_beam_engine_entries_reject_a_null_engine():
    lib = _lib.load()
    i1 = (C.c_int32 * 1)()
    n = C.c_int(0)
    for call in (lambda: lib.af_engine_step_tree(None, i1, i1, 1, 0, None, i1),
                 lambda: lib.af_engine_accept_path(None, i1, 1, 0),
                 lambda: lib.af_engine_generate_beam(None, i1, 1, 1, 1, 1.0, i1, C.byref(n), None)):
        assert call() != 0
        assert b"not finalized" in lib.af_last_error()
