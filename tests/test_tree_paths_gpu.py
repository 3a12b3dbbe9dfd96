"""Both kernels of af_attention_tree_f32 on the same calls.  Which one runs
follows from the sizes a call allows; with room for long sequences in the table
the tensor-core kernel takes the short ones too."""
import pytest

import kv_helpers as kh
import test_tree_attention_gpu as ta

pytestmark = pytest.mark.gpu
MMA_WS = 1 << 20  # sums of split items (148 blocks of 128 rows and more): what a call for long sequences asks for


@pytest.fixture
def room(monkeypatch):
    """Tables with 4,096 blocks more than the sequences have; yields the workspaces asked for."""
    make, workspace, asked = kh.Cache.__init__, kh.workspace, []

    def wide(self, *a, **kw):
        make(self, *a, **{"extra_blocks": 4096, **kw})

    def note(lib, name, args):
        asked.append(getattr(lib, name + "_workspace")(args))
        return workspace(lib, name, args)

    monkeypatch.setattr(kh.Cache, "__init__", wide)
    monkeypatch.setattr(kh, "workspace", note)
    yield asked
    assert asked and all(n > MMA_WS for n in asked)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", [(32, 4, 64), (16, 2, 128), (4, 4, 128), (4, 2, 64)])
def test_layouts_and_types(gpu, room, kv, H, KV, hd):
    ta.test_layouts_and_types(gpu, kv, H, KV, hd)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("length,n", [(0, 1), (1, 1), (31, 1), (32, 3), (63, 1), (64, 1), (65, 2), (127, 1), (128, 1),
                                      (129, 7), (300, 2)])
def test_lengths_and_nodes(gpu, room, kv, hd, length, n):
    ta.test_lengths_and_nodes(gpu, kv, hd, length, n)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [1, 2, 8, 64, 256])
def test_page_sizes(gpu, room, kv, page):
    ta.test_page_sizes(gpu, kv, page)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lengths,counts", [([0, 5, 700, 64, 33], [1, 31, 8, 0, 17]), ([10] * 12, [1] * 12),
                                            ([3 * i for i in range(40)], [1 + i % 3 for i in range(40)])])
def test_ragged_batches(gpu, room, kv, hd, lengths, counts):
    ta.test_ragged_batches(gpu, kv, hd, lengths, counts)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_rows_that_see_nothing_are_zero(gpu, room, hd, n):
    ta.test_rows_that_see_nothing_are_zero(gpu, hd, n)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [2, 5, 24])
def test_what_no_row_sees_may_hold_anything(gpu, room, kv, hd, n):
    ta.test_what_no_row_sees_may_hold_anything(gpu, kv, hd, n)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_non_finite_value_reaches_the_rows_that_see_it_alone(gpu, room, hd, bad):
    ta.test_a_non_finite_value_reaches_the_rows_that_see_it_alone(gpu, hd, bad)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [1e-20, 1e-6, 1.0, 1e8, 1e20])
def test_values_of_any_size(gpu, room, hd, scale):
    ta.test_values_of_any_size(gpu, hd, scale)


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [-0.2, 0.01])
@pytest.mark.parametrize("length,n", [(50, 4), (2000, 30)])
def test_a_scale_of_its_own(gpu, kv, scale, length, n):
    ta.run_case(gpu, kv, 8, 2, 64, [length], [n], scale=scale)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lengths,counts", [([33], [1]), ([137], [1]), ([255] * 3, [2] * 3), ([700], [1]),
                                            ([90] * 40, [1] * 40), ([40, 0, 200], [6, 9, 0])])
def test_small_calls(gpu, kv, hd, lengths, counts):
    """Clusters of one block to eight, tiles that end inside, empty sequences."""
    for H, KV in ((8, 8), (12, 4)):
        ta.run_case(gpu, kv, H, KV, hd, lengths, counts, page=8)


def test_a_workspace_for_the_largest_call_serves_smaller_ones(gpu):
    """Sizes on both sides of the choice between the kernels."""
    def bytes_for(n_seq, max_len, hd, H=8, KV=8):
        c = kh.Cache("f32", KV, hd, [1] * n_seq, page=16, extra_blocks=1024)
        q = kh.torch.zeros((n_seq, H, hd), device="cuda")
        a = kh.attention_args(c, q, q, kh.ints([0] * n_seq), kh.ints(range(n_seq + 1)), 1, max_len=max_len)
        return gpu.af_attention_tree_f32_workspace(a)

    for hd in (64, 128):
        most = bytes_for(40, 4000, hd)
        for n_seq in (1, 36, 37, 38, 40):
            for max_len in (1, 100, 256, 1000, 4000):
                assert bytes_for(n_seq, max_len, hd) <= most


@pytest.mark.parametrize("kv,hd", [("f16", 64), ("f32", 128)])
def test_more_items_than_blocks_at_once(gpu, room, kv, hd):
    """640 items and more, some of them long: beyond the blocks of four waves."""
    ta.run_case(gpu, kv, 16, 16, hd, [7 * i for i in range(39)] + [3000], [1 + i % 2 for i in range(40)], seed=3)


@pytest.mark.parametrize("page", [1, 2, 4])
def test_pages_of_few_positions(gpu, room, page):
    for kv in ("f32", "bf16"):
        ta.run_case(gpu, kv, 8, 4, 64, [77, 300], [9, 20], page=page)
