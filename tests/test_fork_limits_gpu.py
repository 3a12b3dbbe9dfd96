"""af_kv_fork at the ends of its ranges."""
import numpy as np
import pytest

import kv_helpers as kh
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
