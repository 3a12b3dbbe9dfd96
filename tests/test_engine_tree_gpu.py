"""Drafted trees and beam search through the engine: every node and every beam
against the same tokens stepped one at a time."""
import numpy as np
import pytest

from helpers import LOGITS_TOL, model_path, rel_l2
from llm_core_b200.engine import LlamaConfig, LlamaCudaModel, read_config

pytestmark = pytest.mark.gpu
PRESETS = [("tiny", 1), ("tiny-qwen", 4), ("tiny-qwen3", 8), ("tiny-hunyuan", 8), ("small", 5)]


def ancestors(parents, i):
    path = []
    while i >= 0:
        path.append(i)
        i = parents[i]
    return path[::-1]


def random_tree(rng, n):
    return [-1] + [int(rng.integers(max(i - 7, -1), i)) for i in range(1, n)]


@pytest.mark.parametrize("preset,seed", PRESETS)
@pytest.mark.parametrize("n", [1, 6, 32, 45])
def test_tree_nodes_match_stepped_paths(gpu, preset, seed, n):
    path = model_path(preset, seed)
    rng = np.random.default_rng(1000 * seed + n)
    vocab = read_config(path).vocab
    prompt = [1] + rng.integers(0, vocab, 20).tolist()
    tokens = rng.integers(0, vocab, n).tolist()
    parents = random_tree(rng, n)
    m, ref = LlamaCudaModel(path), LlamaCudaModel(path)
    m.prefill(prompt, 0)
    ref.prefill(prompt, 0)
    nxt, lg = m.step_tree(tokens, parents, len(prompt), want_logits=True)
    assert (nxt == lg.argmax(1)).all()
    leaves = [i for i in range(n) if i not in parents]
    for leaf in leaves[:6]:
        for d, node in enumerate(ancestors(parents, leaf)):
            _, want = ref.step(tokens[node], len(prompt) + d)
            assert rel_l2(lg[node], want) < LOGITS_TOL, (leaf, node)
    m.close()
    ref.close()


@pytest.mark.parametrize("preset,seed", [("tiny", 1), ("tiny-hunyuan", 8), ("small", 5)])
def test_accepted_path_continues_as_if_stepped(gpu, preset, seed):
    path = model_path(preset, seed)
    rng = np.random.default_rng(seed)
    cfg = read_config(path)
    prompt = [1] + rng.integers(0, cfg.vocab, 30).tolist()
    tokens = rng.integers(0, cfg.vocab, 24).tolist()
    parents = random_tree(rng, 24)
    accepted = ancestors(parents, 23)
    assert len(accepted) > 1
    m, ref = LlamaCudaModel(path), LlamaCudaModel(path)
    m.prefill(prompt, 0)
    m.step_tree(tokens, parents, len(prompt))
    before = [[m.kv(l, w, len(prompt) + 24) for w in (False, True)] for l in range(cfg.n_layer)]
    m.accept_path(accepted, len(prompt))
    keep = list(range(len(prompt))) + [len(prompt) + a for a in accepted]
    for l in range(cfg.n_layer):
        for w in (False, True):
            assert (m.kv(l, w, len(keep)) == before[l][w][keep]).all()
    seq = prompt + [tokens[a] for a in accepted]
    ref.prefill(seq, 0)
    pos = len(seq)
    for tok in rng.integers(0, cfg.vocab, 3).tolist():
        _, got = m.step(tok, pos)
        _, want = ref.step(tok, pos)
        assert rel_l2(got, want) < LOGITS_TOL
        pos += 1
    # a second tree behind the accepted tokens
    chain = rng.integers(0, cfg.vocab, 5).tolist()
    _, lg = m.step_tree(chain, [-1, 0, 1, 2, 3], pos, want_logits=True)
    for i, tok in enumerate(chain):
        _, want = ref.step(tok, pos + i)
        assert rel_l2(lg[i], want) < LOGITS_TOL
    m.close()
    ref.close()


def test_tree_up_to_the_end_of_the_context(gpu):
    path = model_path("tiny", 1)
    m, ref = LlamaCudaModel(path, max_context_len=50), LlamaCudaModel(path, max_context_len=50)
    prompt = [1] + list(range(7, 47))
    m.prefill(prompt, 0)
    ref.prefill(prompt, 0)
    chain = list(range(100, 109))
    _, lg = m.step_tree(chain, list(range(-1, 8)), 41, want_logits=True)
    for i, tok in enumerate(chain):
        assert rel_l2(lg[i], ref.step(tok, 41 + i)[1]) < LOGITS_TOL
    with pytest.raises(RuntimeError, match="outside the context"):
        m.step_tree(chain, list(range(-1, 8)), 42)
    with pytest.raises(RuntimeError, match="outside the context"):
        m.accept_path([0, 9], 41)
    m.close()
    ref.close()


def test_tree_and_path_refusals(gpu):
    m = LlamaCudaModel(model_path("tiny", 1))
    m.prefill([1, 5, 6], 0)
    for tokens, parents, what in ([[5, 6], [-1, 1], "parent"], [[5, 6], [-1, -2], "parent"], [[5], [0], "parent"],
                                  [[-1], [-1], "vocabulary"], [[m.cfg.vocab], [-1], "vocabulary"],
                                  [[], [], "1..256"], [[5] * 257, list(range(-1, 256)), "1..256"]):
        with pytest.raises(RuntimeError, match=what):
            m.step_tree(tokens, parents, 3)
    with pytest.raises(RuntimeError, match="outside the context"):
        m.step_tree([5], [-1], -1)
    for bad in ([1, 1], [2, 1], [-1], [256]):
        with pytest.raises(RuntimeError, match="rising order"):
            m.accept_path(bad, 3)
    m.accept_path([], 3)
    for args in (([], 2, 4), ([1], 0, 4), ([1], 33, 4)):
        with pytest.raises(RuntimeError):
            m.generate_beam(*args)
    assert m.generate_beam([1, 5], 4, 0) == ([], 0.0)
    m.close()


def plain_beams(ref, cfg, prompt, n_beams, max_new, penalty, stepped):
    """The search by its description, in float64 over logits of stepped sequences."""
    ids = prompt if prompt[0] == cfg.bos_id else [cfg.bos_id] + prompt
    budget = min(max_new, cfg.n_ctx - len(ids))
    live, best = [([], 0.0)], []

    def logp(h):
        key = tuple(h)
        if key not in stepped:
            lg = ref.prefill(ids + h, 0)[1].astype(np.float64)
            stepped[key] = lg - lg.max() - np.log(np.exp(lg - lg.max()).sum())
        return stepped[key]

    for step in range(1, budget + 1):
        cand = np.concatenate([s + logp(h) for h, s in live])
        order = np.argsort(-cand, kind="stable")[:2 * n_beams]
        nxt = []
        for rank, c in enumerate(order):
            row, tok = divmod(int(c), cfg.vocab)
            if len(nxt) == n_beams:
                break
            if tok == cfg.eos_id:
                if rank < n_beams:
                    best.append((cand[c] / step**penalty, live[row][0]))
            else:
                nxt.append((live[row][0] + [tok], cand[c]))
        live = nxt
        best = sorted(best, key=lambda b: -b[0])[:n_beams]
        if step == budget or (len(best) == n_beams and best[-1][0] >= live[0][1] / step**penalty):
            best += [(s / step**penalty, h) for h, s in live]
            break
    return max(best, key=lambda b: b[0])


@pytest.mark.parametrize("preset,seed,n_beams,max_new,penalty", [
    ("tiny", 1, 4, 12, 1.0), ("tiny", 1, 1, 5, 0.0), ("tiny-qwen", 4, 3, 20, 0.0), ("tiny-hunyuan", 8, 5, 9, 2.0),
    ("small", 5, 2, 18, 1.0)])
@pytest.mark.parametrize("with_eos", [False, True])
def test_beam_search_matches_plain_search(gpu, preset, seed, n_beams, max_new, penalty, with_eos):
    """The same hypothesis and rating as a search over sequences stepped from
    their start.  Beams go through the linear layers as rows, whose rounding is
    not that of single steps, and a layer behind another amplifies it: on the
    random qwen2 preset 2e-5 in the first layer's values is 2e-3 in the logits,
    with either attention kernel.  So the rating's tolerance follows from the
    logits: two rows of logits that differ by at most d give log-probabilities
    that differ by at most 2 d, d being what step_tree's rows of the winning
    hypothesis differ by from its steps, and the beams' rows by as much again."""
    path = model_path(preset, seed)
    cfg = read_config(path)
    rng = np.random.default_rng(seed)
    prompt = rng.integers(5, cfg.vocab, 14).tolist()
    ref = LlamaCudaModel(path)
    stepped = {}
    score, ids = plain_beams(ref, cfg, prompt, n_beams, max_new, penalty, stepped)
    if with_eos:  # a token that the search takes ends hypotheses instead
        cfg.eos_id = ids[len(ids) // 2]
        score, ids = plain_beams(ref, cfg, prompt, n_beams, max_new, penalty, stepped)
    m = LlamaCudaModel(path, config=cfg)
    got, rating = m.generate_beam(prompt, n_beams, max_new, penalty)
    assert got == ids
    start = prompt if prompt[0] == cfg.bos_id else [cfg.bos_id] + prompt
    ended = len(ids) < min(max_new, cfg.n_ctx - len(start))  # one log-probability more, of the end
    length = len(ids) + ended
    row, fed = ref.prefill(start, 0)[1], ids[:length - 1]
    rows = [row]
    if fed:
        rows += list(ref.step_tree(fed, list(range(-1, len(fed) - 1)), len(start), want_logits=True)[1])
    steps = [row] + [ref.step(t, len(start) + i)[1] for i, t in enumerate(fed)]
    apart = sum(float(np.abs(r - s).max()) for r, s in zip(rows, steps))
    assert abs(rating - score) <= (2 * 2 * apart + 1e-5 * abs(score)) / length ** penalty + 1e-5
    # and the engine generates as before afterwards
    again = m.generate(prompt, LlamaConfig(max_new_tokens=6, temperature=0))
    fresh = LlamaCudaModel(path, config=cfg)
    assert again == fresh.generate(prompt, LlamaConfig(max_new_tokens=6, temperature=0))
    for x in (m, ref, fresh):
        x.close()


def test_beam_search_at_the_context_cap_and_without_room(gpu):
    path = model_path("tiny", 1)
    cfg = read_config(path, 64)
    m, ref = LlamaCudaModel(path, config=cfg), LlamaCudaModel(path, config=cfg)
    prompt = list(range(7, 45))  # 39 with BOS: 3 of the 4 pages hold it, the last one 7 positions
    # one beam fits and goes to the cap
    score, ids = plain_beams(ref, cfg, prompt, 1, 100, 1.0, {})
    got, rating = m.generate_beam(prompt, 1, 100)
    assert got == ids and len(got) <= 25 and abs(rating - score) < 2e-3
    # eight beams need a last page each
    with pytest.raises(RuntimeError, match="no room"):
        m.generate_beam(prompt, 8, 20)
    assert m.generate(prompt, LlamaConfig(max_new_tokens=4, temperature=0)) == \
        ref.generate(prompt, LlamaConfig(max_new_tokens=4, temperature=0))
    m.close()
    ref.close()
