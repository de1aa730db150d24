"""Host logic of Model.score and of the scores of a turn on the CPU: which tokens the
caches are taken to hold afterwards, and one score a generated token."""
import numpy as np
import pytest

import obsidian_hip as oh
from obsidian_hip import decoder as D


class Rec(D.Model):
    """No device: prefill_layers fails or is passed, the scores' calls are recorded."""

    def __init__(self, max_len=64):
        self.cfg = D.DecoderConfig(max_len=max_len)
        self.last_seq, self.last_reused, self.last_prefilled = [], 0, 0
        self.calls, self.fail, self.exe, self.glob = [], False, None, None

    def prefill_layers(self, tokens, pos0, trace=None):
        if not tokens:
            raise ValueError("empty prompt")
        if self.fail:
            raise oh.ObsError(oh.OBS_E_NOMEM, "no room")
        raise StopIteration  # as far as the host goes

    def prefill(self, tokens, pos0):
        return 3

    def run_one_token(self, tok, pos):
        return 3

    def fill_kv(self, tok, pos):
        pass

    def set_state(self, pos, tok):
        pass

    def replay(self, n=1):
        pass

    def read_state(self):
        return 0, 3

    def last_scores(self, top_k=0):
        self.calls.append(top_k)
        return len(self.calls)


@pytest.mark.parametrize("fail", [False, True])
def test_an_unfinished_score_leaves_no_prefix_behind_its_start(fail):
    m = Rec()
    m.last_seq, m.fail = [1, 2, 3, 4], fail
    with pytest.raises((StopIteration, oh.ObsError)):
        m.score([9, 9], pos0=2)
    assert m.last_seq == [1, 2]


def test_score_of_nothing():
    with pytest.raises(ValueError):
        Rec().score([])


@pytest.mark.parametrize("n,eos,want", [(4, -1, 4), (4, 3, 1), (1, -1, 1)])
def test_a_turn_scores_every_generated_token(n, eos, want):
    m, got = Rec(), []
    gen = m.run_turn(list(range(30)), n, eos, scores=got, top_k=7)
    assert len(gen) == want and got == list(range(1, want + 1)) and m.calls == [7] * want
