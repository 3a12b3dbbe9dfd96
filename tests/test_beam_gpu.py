"""af_beam_select_f32 against the definition in 64 bits: picks equal, ties to
the lowest beam and token, dead beams, -inf, NaN and +inf logits."""
import numpy as np
import pytest
import torch

import kv_helpers as kh
from llm_core_b200 import _lib

pytestmark = pytest.mark.gpu


def run_beam(lib, logits, scores, n_out, stride=0, shift=0):
    S, B = scores.shape
    V = logits.shape[1]
    if stride:
        buf = torch.full((S * B, stride), 1e30, device="cuda")
        buf[:, :V] = torch.from_numpy(logits).cuda()
    else:
        buf = torch.empty(S * B * V + 4, device="cuda")
        buf = buf[shift:shift + S * B * V].view(S * B, V)
        buf.copy_(torch.from_numpy(logits))
    sc = torch.from_numpy(scores).cuda()
    out = [torch.full((S, n_out), -9, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
    a = _lib.BeamSelectArgs()
    a.logits, a.logits_stride, a.scores = buf.data_ptr(), stride, sc.data_ptr()
    a.n_seq, a.n_beams, a.vocab, a.n_out = S, B, V, n_out
    a.out_score, a.out_beam, a.out_token = (x.data_ptr() for x in out)
    ws = kh.workspace(lib, "af_beam_select_f32", a)
    for _ in range(2):
        kh.call(lib, "af_beam_select_f32", a)
    assert kh.device_error(lib) == 0
    got = [x.cpu().numpy() for x in out]
    for s, (want, beam, token) in enumerate(kh.beam_plain(logits, scores, n_out)):
        np.testing.assert_array_equal(got[1][s], beam)
        np.testing.assert_array_equal(got[2][s], token)
        dead = want == -np.inf
        assert (got[0][s][dead] == -np.inf).all()
        # half a step of f32, and log Σ exp of 32-term f32 sums of exponentials good to 2 ulp
        tol = 2.0 ** -24 * np.abs(want[~dead]) + 40 * 2.0 ** -24
        assert (np.abs(got[0][s][~dead] - want[~dead]) <= tol).all()
    del ws


@pytest.mark.parametrize("S,B,V,n_out", [(1, 1, 1, 1), (1, 1, 7, 7), (1, 4, 3, 12), (2, 3, 1000, 6), (1, 4, 32000, 8),
                                         (3, 8, 8192, 16), (2, 8, 8193, 16), (1, 5, 16385, 64), (2, 2, 151936, 4),
                                         (1, 50, 151936, 64), (4, 64, 500, 64), (70, 2, 333, 3)])
def test_picks(gpu, S, B, V, n_out):
    rng = np.random.default_rng(V + B)
    logits = (3 * rng.standard_normal((S * B, V))).astype(np.float32)
    scores = (-3 * rng.random((S, B))).astype(np.float32)
    run_beam(gpu, logits, scores, n_out)


@pytest.mark.parametrize("stride,shift", [(0, 1), (0, 3), (8204, 0), (8201, 0)])
def test_strides_and_alignment(gpu, stride, shift):
    rng = np.random.default_rng(1)
    logits = rng.standard_normal((6, 8200)).astype(np.float32)
    run_beam(gpu, logits, np.zeros((2, 3), np.float32) - np.arange(3, dtype=np.float32), 7, stride, shift)


@pytest.mark.parametrize("V", [40, 9000])
def test_equal_logits_take_the_lowest(gpu, V):
    logits = np.zeros((4, V), np.float32)
    run_beam(gpu, logits, np.zeros((1, 4), np.float32), 64)
    logits[:, 1::2] = 1.0
    run_beam(gpu, logits, np.array([[0, -1, 0, -0.5]], np.float32), 20)
    logits[:, :] = np.repeat(np.arange(4, dtype=np.float32), V // 4 + 1)[:V]
    run_beam(gpu, logits, np.array([[-2, -1, 0, 0]], np.float32), 33)


def test_first_step_and_dead_beams(gpu):
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((8, 9000)).astype(np.float32)
    scores = np.full((2, 4), -np.inf, np.float32)
    scores[0, 0], scores[1, 2] = 0.0, -1.5
    run_beam(gpu, logits, scores, 8)
    scores[1, 3] = np.nan
    run_beam(gpu, logits, scores, 8)
    run_beam(gpu, logits, np.full((2, 4), -np.inf, np.float32), 8)


def test_masked_vocabulary(gpu):
    """Constrained decoding: all but a few tokens at -inf, or a whole row."""
    rng = np.random.default_rng(3)
    logits = np.full((3, 9000), -np.inf, np.float32)
    logits[0, [5, 8191, 8192, 8999]] = rng.standard_normal(4)
    logits[1, 17] = 2.0
    run_beam(gpu, logits, np.array([[-1, -0.5, 0]], np.float32), 9)
    run_beam(gpu, logits[:1], np.zeros((1, 1), np.float32), 12)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_bad_row_is_dead(gpu, bad):
    rng = np.random.default_rng(4)
    logits = rng.standard_normal((4, 20000)).astype(np.float32)
    logits[2, 12345] = bad
    run_beam(gpu, logits, np.array([[-2, -1, 0, -3]], np.float32), 16)


@pytest.mark.parametrize("off", [0.0, 5e4, -5e4, 3e37])
def test_large_logits(gpu, off):
    rng = np.random.default_rng(5)
    logits = (rng.standard_normal((2, 5000)) * 10 + off).astype(np.float32)
    run_beam(gpu, logits, np.array([[0, -1e-3]], np.float32), 6)


def test_graph_replay(gpu):
    rng = np.random.default_rng(6)
    S, B, V, n = 2, 4, 10000, 8
    x = torch.zeros((S * B, V), device="cuda")
    sc = torch.zeros((S, B), device="cuda")
    out = [torch.zeros((S, n), dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
    a = _lib.BeamSelectArgs()
    a.logits, a.scores, a.out_score, a.out_beam, a.out_token = (t.data_ptr() for t in (x, sc, *out))
    a.n_seq, a.n_beams, a.vocab, a.n_out = S, B, V, n
    ws = kh.workspace(gpu, "af_beam_select_f32", a)
    kh.call(gpu, "af_beam_select_f32", a)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kh.call(gpu, "af_beam_select_f32", a)
    for _ in range(3):
        lg = (3 * rng.standard_normal((S * B, V))).astype(np.float32)
        s = -rng.random((S, B)).astype(np.float32)
        x.copy_(torch.from_numpy(lg))
        sc.copy_(torch.from_numpy(s))
        g.replay()
        torch.cuda.synchronize()
        for i, (w, b, t) in enumerate(kh.beam_plain(lg, s, n)):
            np.testing.assert_array_equal(out[1][i].cpu().numpy(), b)
            np.testing.assert_array_equal(out[2][i].cpu().numpy(), t)
    del ws
