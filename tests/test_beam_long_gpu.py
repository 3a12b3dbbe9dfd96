"""af_beam_select_f32 where a segment has many steps of 4,096 logits: what is
kept is cut back, raised and carried over from step to step."""
import ctypes as C

import numpy as np
import pytest

from llm_core_b200 import _lib
from test_beam_gpu import run_beam
from test_beam_paths_gpu import shaped

pytestmark = pytest.mark.gpu
STEP = 4096


def steps_of(lib, S, B, V, n_out):
    """The fewest steps that a segment can have: the workspace holds n_out keys, a sum and a maximum for each."""
    a = _lib.BeamSelectArgs()
    a.n_seq, a.n_beams, a.vocab, a.n_out = S, B, V, n_out
    segments = lib.af_beam_select_f32_workspace(C.byref(a)) // (n_out * 8 + 16) // (S * B)
    return -(-(V // segments) // STEP)


def scores_of(S, B, rng):
    """Far apart, so that no two beams' continuations nearly tie."""
    return -50 * np.arange(S * B, dtype=np.float32).reshape(S, B) + rng.random((S, B)).astype(np.float32)


@pytest.mark.parametrize("kind", ["zeros of both signs", "few values", "rising", "falling", "few allowed", "few finite"])
@pytest.mark.parametrize("S,B,V,n_out,shift", [(16, 8, 60000, 64, 0), (16, 8, 60003, 8, 1)])
def test_logits_of_a_kind_over_many_steps(gpu, kind, S, B, V, n_out, shift):
    assert steps_of(gpu, S, B, V, n_out) >= 5
    rng = np.random.default_rng(V + n_out)
    run_beam(gpu, shaped(kind, rng, S * B, V), scores_of(S, B, rng), n_out, shift=shift)


@pytest.mark.parametrize("kind", ["rising", "few values", "few allowed"])
def test_whole_vocabularies(gpu, kind):
    S, B, V, n_out = 16, 8, 151936, 16
    assert steps_of(gpu, S, B, V, n_out) >= 12
    rng = np.random.default_rng(7)
    run_beam(gpu, shaped(kind, rng, S * B, V), scores_of(S, B, rng), n_out)


@pytest.mark.parametrize("n_out", [5, 64])
@pytest.mark.parametrize("step", [3, 5, 6])
def test_allowed_tokens_behind_an_equal_prefix(gpu, step, n_out):
    """Every segment begins with equal logits; at one of its later steps, and the
    one behind it, every logit is above all before it."""
    S, B, per = 12, 8, 12 * STEP
    V = 4 * per
    assert steps_of(gpu, S, B, V, n_out) == per // STEP
    rng = np.random.default_rng(step)
    x = np.full((S * B, V), np.float32(-1e4))
    for at in range(0, V, per):
        lo, hi = at + (step - 1) * STEP, at + (step + 1) * STEP
        x[:, lo:hi] = np.sort(rng.standard_normal((S * B, hi - lo)).astype(np.float32), axis=1)
    run_beam(gpu, x, scores_of(S, B, rng), n_out)
