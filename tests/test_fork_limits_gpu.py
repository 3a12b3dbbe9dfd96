"""af_kv_fork at the ends of its ranges."""
import numpy as np
import pytest
import torch

import kv_helpers as kh
from llm_core_b200 import _lib
from test_kvcache_gpu import counts_of, run_fork

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("in_place", [False, True])
def test_missing_pages_are_counted_up_to_the_end_of_the_range(gpu, page, in_place):
    """Outputs that ask for more positions than any table holds: 2^31 - 1 of them
    each, 8 outputs, so that pages of one position pass 32 bits together."""
    most = (1 << 31) - 1
    c = kh.Cache("f32", 1, 8, [21], page=page, spare=9, seed=4, extra_blocks=3)
    ref = counts_of(c.table_h, c.pages)
    length = np.array([21], np.int32)
    plain = kh.fork_plain(page, c.pages, c.table_h, length, ref, [0] * 8, [most] * 8, c.blocks)
    assert (plain[3] > most) == (page == 1)

    def capped(*a, real=kh.fork_plain):
        x = real(*a)
        return (*x[:3], min(x[3], most), x[4])

    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(kh, "fork_plain", capped)
        run_fork(gpu, c, c.table_h, length, ref, [0] * 8, [most] * 8, in_place)


def fork_once(lib, c, table, length, ref, parent, new):
    """Tables, lengths, counts and missing pages of one call, and the error word."""
    t_in, l_in, r_in, par, nw = (kh.ints(x) for x in (table, length, ref, parent, new))
    t_out = torch.full((len(parent), table.shape[1]), -7, dtype=torch.int32, device="cuda")
    l_out, r_out, short = torch.full_like(par, -7), torch.full_like(r_in, -7), kh.ints([-7])
    a = _lib.KvForkArgs()
    a.kv = c.struct()
    a.table_in, a.len_in, a.ref_in = (x.data_ptr() for x in (t_in, l_in, r_in))
    a.table_out, a.len_out, a.ref_out = (x.data_ptr() for x in (t_out, l_out, r_out))
    a.parent, a.n_new, a.n_short = par.data_ptr(), nw.data_ptr(), short.data_ptr()
    a.n_in, a.n_out, a.max_blocks = table.shape[0], len(parent), table.shape[1]
    ws = kh.workspace(lib, "af_kv_fork", a)
    kh.call(lib, "af_kv_fork", a)
    err = kh.device_error(lib)
    del ws
    return t_out.cpu().numpy(), l_out.tolist(), r_out.cpu().numpy(), int(short.item()), err


@pytest.mark.parametrize("at,bad,end", [(1, 1 << 30, 8), (0, -2, 0), (1, -1, 8), (2, -1, 16), (2, 1 << 20, 16),
                                        (40, -1, 8 * 40), (33, -7, 8 * 33)])
def test_a_hole_below_the_length_is_reported_and_ends_the_child(gpu, at, bad, end):
    """Page `at` of a parent is none (-1, or an id outside the pool): its children end in front of it, the pages
    behind stay counted, the other parent's child is whole, and the pool is left as it was."""
    c = kh.Cache("f32", 1, 8, [21 if at < 4 else 8 * 50 + 5, 19], page=8, spare=5, seed=4, extra_blocks=1)
    length = np.array([21 if at < 4 else 8 * 50 + 5, 19], np.int32)
    table = c.table_h.copy()
    table[0, at] = bad
    ref = counts_of(np.where((table >= 0) & (table < c.pages), table, -1), c.pages)
    before = c.k.clone(), c.v.clone()
    t, l, r, short, err = fork_once(gpu, c, table, length, ref, [0, 1], [0, 0])
    assert err != 0
    assert l == [end, 19] and short == 0
    whole = np.arange(table.shape[1]) < length[0] // 8
    np.testing.assert_array_equal(t[0, whole], np.where(table[0] == bad, -1, table[0])[whole])
    np.testing.assert_array_equal(t[1], table[1])
    np.testing.assert_array_equal(r, counts_of(t, c.pages))
    assert torch.equal(c.k, before[0]) and torch.equal(c.v, before[1])


def test_an_id_outside_the_pool_behind_the_length_is_reported(gpu):
    c = kh.Cache("f16", 1, 8, [21], page=8, spare=5, seed=4, extra_blocks=3)
    table = c.table_h.copy()
    table[0, 4] = c.pages
    ref = counts_of(c.table_h, c.pages)
    t, l, r, short, err = fork_once(gpu, c, table, [21], ref, [0], [0])
    assert err != 0 and l == [21] and short == 0
    np.testing.assert_array_equal(t, c.table_h)
    np.testing.assert_array_equal(r, ref)
    t, l, r, short, err = fork_once(gpu, c, c.table_h, [21], ref, [0], [0])
    assert err == 0 and l == [21]
