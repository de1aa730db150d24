"""The device buffers of Model.score and last_scores on the CPU, over an executor that
counts what is allocated: an outgrown set is freed, also where its successor cannot be had,
and a call brings back its own rows alone."""
import numpy as np
import pytest

import obsidian_hip as oh
from obsidian_hip import decoder as D


class Buffer:
    def __init__(self, exe, n, dtype):
        self.exe, self.dtype, self.nbytes = exe, np.dtype(dtype), n * np.dtype(dtype).itemsize
        self.ptr = exe.next
        exe.next += self.nbytes + 256
        exe.live[self.ptr] = self

    def free(self):
        if self.ptr:
            del self.exe.live[self.ptr]
        self.ptr = 0

    def upload(self, a):
        assert a.nbytes == self.nbytes

    def download(self):
        self.exe.brought += self.nbytes
        return np.zeros(self.nbytes // self.dtype.itemsize, self.dtype)


class Exe:
    def __init__(self):
        self.next, self.live, self.brought, self.fail_at = 4096, {}, 0, None

    def alloc(self, n, dtype):
        if self.fail_at is not None:
            self.fail_at -= 1
            if self.fail_at < 0:
                raise oh.ObsError(oh.OBS_E_NOMEM, "no room")
        return Buffer(self, int(n), dtype)

    def download_raw(self, ptr, shape, dtype):
        out = np.zeros(shape, dtype)
        if out.nbytes:
            assert any(p <= ptr and ptr + out.nbytes <= p + b.nbytes for p, b in self.live.items())
        self.brought += out.nbytes
        return out

    def token_logprobs_workspace(self, T, vocab, top_k=0):
        return 1000

    def lm_logprobs_workspace(self, T, hidden, vocab, top_k=0):
        return 5000 * T

    def token_logprobs(self, *a, **kw):
        pass

    lm_logprobs = rmsnorm_raw = device_status = token_logprobs


class Model(D.Model):
    def __init__(self):
        self.cfg = D.DecoderConfig(max_len=4096)
        self.exe, self._sc, self._pf = Exe(), None, {"xn": None}
        self.glob = dict.fromkeys(D.GLOBAL_KEYS)
        self.last_seq, self.logits, self.state = [], None, Buffer(self.exe, 2, np.int32)

    def prefill_layers(self, tokens, pos0, trace=None):
        return None


def _held(m):
    return sum(b.nbytes for b in m.exe.live.values())


def test_an_outgrown_set_is_freed():
    m = Model()
    for T in range(1, 200, 7):
        m.score([1] * T, top_k=T % 5)
    grown, m = _held(m), Model()
    m.score([1] * 197, top_k=4)
    assert grown == _held(m)


@pytest.mark.parametrize("at", range(6))
def test_a_set_that_cannot_be_had(at):
    """No room for the successor: nothing that was given stays behind the next call's set."""
    m = Model()
    m.score([1, 2])
    m.exe.fail_at = at
    with pytest.raises(oh.ObsError):
        m.score([1] * 50, top_k=3)
    m.exe.fail_at = None
    got = m.score([1, 2], top_k=1)
    assert got.logprob.shape == (2,) and got.top_ids.shape == (2, 1)
    m.score([1] * 50, top_k=3)
    held, m = _held(m), Model()
    m.score([1] * 50, top_k=3)
    assert held == _held(m)


@pytest.mark.parametrize("top_k", [0, 3])
def test_a_token_brings_back_one_row(top_k):
    """After a long scored prompt the scores of a generated token cost no more than before it."""
    m = Model()
    m.score([1] * 500, top_k=20)
    for call, rows in ((lambda: m.last_scores(top_k), 1), (lambda: m.score([1] * 7, top_k=top_k), 7)):
        m.exe.brought = 0
        got = call()
        assert m.exe.brought == 8 * rows * (1 + top_k)
        assert got.logprob.shape == got.entropy.shape == (rows,)
        assert got.top_ids.shape == got.top_logprobs.shape == (rows, top_k)
        assert got.top_ids.dtype == np.int32 and got.top_logprobs.dtype == np.float32
