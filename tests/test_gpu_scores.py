"""Model.score and the scores of generated tokens on the GPU, on a small seeded model:
log probabilities, entropies and alternatives against float64 softmaxes of the model's
own normalised rows (score) and of its own logits (generation), to the bars of
test_gpu_logprobs."""
import numpy as np
import pytest

import obsidian_hip as oh
from obsidian_hip import decoder as D
from obsidian_hip import synth
from test_gpu_logprobs import U, _f64, _logits64, _near, _reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(exe):
    cfg = D.DecoderConfig(n_layers=2, hidden=2048, n_heads=16, n_kv=2, head_dim=128, n_exp=8, top_k=2, inter=256, vocab=700, max_len=160)
    layers, glob = synth.decoder_weights(5, cfg.n_layers, cfg.hidden, cfg.n_heads, cfg.n_kv, cfg.head_dim, cfg.n_exp, cfg.inter, cfg.vocab)
    m = D.Model(exe, cfg, *D.upload_weights(exe, layers, glob))
    yield m, glob
    m.close()


def _check_rows(got, logits, off, tokens, k):
    lp, ent, ids, tlp, bs, be = _reference(logits, tokens, k)
    worst = off.max(1)
    assert _near(got.logprob, lp, bs + 4 * U * np.abs(lp) + 2 * worst)
    logp = logits - (logits.max(1) + np.log(np.sum(np.exp(logits - logits.max(1)[:, None]), 1)))[:, None]
    move = np.sum(np.exp(logp) * np.abs(logp + ent[:, None]), 1)
    assert _near(got.entropy, ent, be + 1.01 * move * worst)
    t = np.arange(len(tokens))[:, None]
    assert np.all(np.abs(logits[t, got.top_ids] - logits[t, ids]) <= 2 * worst[:, None])
    assert _near(got.top_logprobs, tlp, bs[:, None] + 4 * U * np.abs(tlp) + 4 * worst[:, None])


@pytest.mark.parametrize("T,pos0,k", [(1, 0, 3), (9, 0, 0), (33, 5, 5), (130, 0, 2), (30, 130, 20)])
def test_score(exe, model, T, pos0, k):
    m, glob = model
    tokens = [int(t) for t in np.random.default_rng(T).integers(0, m.cfg.vocab, T)]
    state = m.state.download()
    got = m.score(tokens, pos0, k)
    assert np.array_equal(state, m.state.download())
    xn = m._pf["xn"].download()[:T]
    logits, off = _logits64(_f64(xn), glob["lm_w"], glob["lm_s"], glob["lm_b"])
    assert got.logprob.shape == got.entropy.shape == (T,) and got.top_ids.shape == got.top_logprobs.shape == (T, k)
    _check_rows(got, logits, off, np.array(tokens[1:] + [-1]), k)
    assert got.logprob[-1] == 0.0
    again = m.score(tokens, pos0, k)
    for a, b in zip(vars(got).values(), vars(again).values()):
        assert np.array_equal(a, b)


def test_score_then_a_turn(exe, model):
    """A scored prefix is reused by the next turn, and an overwritten one is not."""
    m, _ = model
    a, b, c = ([int(t) for t in np.random.default_rng(s).integers(0, m.cfg.vocab, 30)] for s in (1, 2, 3))
    m.last_seq = []
    fresh = m.run_turn(a + b, 4, -1)
    assert m.last_reused == 0
    m.score(a)
    assert m.run_turn(a + b, 4, -1) == fresh and m.last_reused == 30
    m.score(c, pos0=5)
    m.run_turn(a + b, 4, -1)
    assert m.last_reused == 5


@pytest.mark.parametrize("graph", [False, True])
def test_generated_tokens_have_scores(exe, model, graph):
    m, _ = model
    scores, rows = [], []
    real = m.last_scores
    def keep(top_k):
        rows.append(m.logits.download())
        return real(top_k)
    m.last_scores = keep
    try:
        got = m.generate(7, 0, 6, graph=graph, scores=scores, top_k=4)
    finally:
        del m.last_scores
    assert got == m.generate(7, 0, 6, graph=graph)
    for tok, s, row in zip(got, scores, rows):
        _check_rows(s, row[None, :].astype(np.float64), np.zeros((1, m.cfg.vocab)), np.array([tok]), 4)
        assert s.top_ids[0, 0] == tok and s.top_logprobs[0, 0] == s.logprob[0]


def test_turns_have_scores(exe, model):
    m, _ = model
    prompt = [int(t) for t in np.random.default_rng(8).integers(0, m.cfg.vocab, 40)]
    m.last_seq = []
    scores = []
    got = m.run_turn(prompt, 5, -1, scores=scores, top_k=2)
    assert len(scores) == len(got) == 5 and [int(s.top_ids[0, 0]) for s in scores] == got
    assert all(s.logprob[0] == s.top_logprobs[0, 0] <= 0 < s.entropy[0] for s in scores)
