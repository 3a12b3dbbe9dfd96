"""af_beam_select_f32 with scores that are not finite: such beams are dead, whatever their logits."""
import numpy as np
import pytest

import kv_helpers as kh
from test_beam_gpu import run_beam

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,n_out", [(50, 7), (9000, 16), (50, 64)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("masked", [False, True])
def test_beams_of_no_finite_score_are_dead(gpu, monkeypatch, V, n_out, bad, masked):
    plain = kh.beam_plain
    monkeypatch.setattr(kh, "beam_plain", lambda x, s, n: plain(x, np.where(np.isfinite(s), s, -np.inf).astype(np.float32), n))
    rng = np.random.default_rng(V)
    logits = rng.standard_normal((6, V)).astype(np.float32)
    if masked:  # a score of +inf and a logit of -inf would be NaN
        logits[:, ::3] = -np.inf
    scores = np.array([[-1, bad, -60], [bad, bad, -0.5]], np.float32)
    run_beam(gpu, logits, scores, n_out)
