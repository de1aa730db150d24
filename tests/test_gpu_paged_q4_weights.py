"""Softmax weights of prompts over a cache of 4 bits: scores of all sizes."""
import numpy as np
import pytest

from obsidian_hip import synth
from test_gpu_paged import FILL16, _f64
from test_gpu_paged_q4 import Pool, _f16

pytestmark = pytest.mark.gpu


def _run(exe, pool, q, rows, window=0, sinks=0):
    nh = q.shape[1]
    out = exe.upload(np.full(q.shape, FILL16, np.uint16))
    seqs = pool.seqs(rows)
    ws = exe.upload(np.full(exe.sdpa_paged_workspace(pool.kv, seqs, nh, None, window, sinks), 0xFF, np.uint8))
    exe.sdpa_paged_prefill(pool.kv, seqs, exe.upload(q), out, nh, ws, window=window, sinks=sinks)
    exe.device_status()
    return _f64(out.download())


@pytest.mark.parametrize("k_std", [1.0, 30.0, 1000.0])
@pytest.mark.parametrize("q_std", [300.0, 3e4, 1e7, 1e20])
def test_scores_of_any_size(exe, q_std, k_std):
    """Where a score's own rounding passes one, an output is still a mean of values."""
    nh, nkv, hd, page, n = 8, 2, 128, 16, 900
    rng = np.random.default_rng(73)
    pool = Pool(exe, rng, [n], nkv, hd, page, k_std=k_std)
    q = synth.bf16_normal(rng, (n, nh, hd), q_std)
    got = _run(exe, pool, q, [0, n])
    assert np.all(np.isfinite(got))
    x = pool.parts(0, "v")
    v = np.repeat(_f16(x[0] * x[1] + x[2]), nh // nkv, 1)
    top, low = np.maximum.accumulate(v, 0), np.minimum.accumulate(v, 0)
    slack = (2.0 ** -8 + 2.0 ** -9) * np.maximum(np.abs(top), np.abs(low))
    assert np.all(got <= top + slack) and np.all(got >= low - slack)
