"""af_beam_select_f32 on logits that stress its thresholds: few distinct values,
zeros of both signs, rising and falling rows, few finite ones."""
import numpy as np
import pytest

from test_beam_gpu import run_beam

pytestmark = pytest.mark.gpu


def shaped(kind, rng, rows, V):
    if kind == "zeros of both signs":
        return np.where(rng.random((rows, V)) < 0.5, np.float32(-0.0), np.float32(0.0))
    if kind == "few values":
        return np.round(rng.standard_normal((rows, V))).astype(np.float32)
    if kind == "rising":
        return np.sort(rng.standard_normal((rows, V)).astype(np.float32), axis=1)
    if kind == "falling":
        return -np.sort(-rng.standard_normal((rows, V)).astype(np.float32), axis=1)
    if kind == "few allowed":  # a constrained step: all others far below, and equal
        x = np.full((rows, V), np.float32(-1e4))
        for r in x:
            r[rng.integers(0, V, 5)] = rng.standard_normal(5)
        return x
    x = np.full((rows, V), -np.inf, np.float32)  # "few finite"
    for r in x:
        r[rng.integers(0, V, 3)] = rng.standard_normal(3)
    return x


@pytest.mark.parametrize("kind", ["zeros of both signs", "few values", "rising", "falling", "few allowed", "few finite"])
@pytest.mark.parametrize("S,B,V,n_out", [(1, 1, 5000, 8), (2, 3, 20000, 16), (1, 2, 151936, 64), (3, 1, 37000, 33)])
def test_logits_of_a_kind(gpu, kind, S, B, V, n_out):
    """Beams far apart in score, so that no two beams' continuations nearly tie."""
    rng = np.random.default_rng(V + n_out)
    scores = -50 * np.arange(S * B, dtype=np.float32).reshape(S, B) + rng.random((S, B)).astype(np.float32)
    run_beam(gpu, shaped(kind, rng, S * B, V), scores, n_out)
