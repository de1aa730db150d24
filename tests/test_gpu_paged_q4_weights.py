"""Softmax weights of prompts over a cache of 4 bits: entries far below a row's largest,
and scores of all sizes.

Bars. P is fp16 of the weights times 2^7 at the running maximum (which a row's largest
passes by 2^8 at most): 2^-11 of each, and half the least step, 2^-25, where that is more,
so 2^-32 of the row's largest weight or less. Both enter numerator and sum. Scores as in
test_gpu_paged_q4; numerator and sum are fp32 sums of n terms of one sign here (2^-24 an
addition each), and the output is rounded once (2^-8)."""
import numpy as np
import pytest

from obsidian_hip import synth
from test_gpu_paged import FILL16, _f64, _visible
from test_gpu_paged_q4 import Pool, _f16

pytestmark = pytest.mark.gpu


def _attend(q, k, v, vis):
    """q [nh, hd] over k, v [n, nkv, hd] of which `vis` are seen -> (out, bound)."""
    nh, hd = q.shape
    per = nh // k.shape[1]
    out, bound = np.zeros((nh, hd)), np.zeros((nh, hd))
    idx = np.flatnonzero(vis)
    n = len(idx)
    for h in range(nh):
        kk, vv = k[idx, h // per], v[idx, h // per]
        s = kk @ q[h] / np.sqrt(hd)
        p = np.exp(s - s.max())
        p /= p.sum()
        mag = np.max(np.abs(kk) @ np.abs(q[h])) / np.sqrt(hd)
        err = 2 * (hd * 2.0 ** -24 * mag + 2.0 ** -21 * np.max(np.abs(s)) + 2.0 ** -20)
        out[h], A = p @ vv, p @ np.abs(vv)
        bound[h] = 1.01 * (2 * 2.0 ** -11 + err + 2 * (n + 40) * 2.0 ** -24) * A + \
            2.0 ** -32 * p.max() * (np.sum(np.abs(vv), 0) + n * A) + 2.0 ** -8 * np.abs(out[h]) + 1e-30
    return out, bound


def _run(exe, pool, q, rows, window=0, sinks=0):
    nh = q.shape[1]
    out = exe.upload(np.full(q.shape, FILL16, np.uint16))
    seqs = pool.seqs(rows)
    ws = exe.upload(np.full(exe.sdpa_paged_workspace(pool.kv, seqs, nh, None, window, sinks), 0xFF, np.uint8))
    exe.sdpa_paged_prefill(pool.kv, seqs, exe.upload(q), out, nh, ws, window=window, sinks=sinks)
    exe.device_status()
    return _f64(out.download())


@pytest.mark.parametrize("gap", [10.0, 16.0, 18.0, 20.0])
@pytest.mark.parametrize("shape,n,t,at,window", [((32, 4, 128, 32), 5000, 40, 0, 0), ((32, 4, 128, 64), 3500, 3500, 0, 0),
                                                 ((16, 1, 64, 16), 6001, 7, 2, 4096), ((8, 2, 128, 16), 4000, 33, 3900, 0)])
def test_one_entry_far_above_thousands(exe, shape, n, t, at, window, gap):
    """An entry `gap` above all others in the exponent whose value is zero: the others' weights, each a
    millionth of its and less, are the output."""
    nh, nkv, hd, page = shape
    rng = np.random.default_rng(71)
    pool = Pool(exe, rng, [n], nkv, hd, page)
    j = np.arange(n)
    k = np.zeros((n, nkv, hd))
    k[at] = gap / np.sqrt(hd)  # queries of one: a score of gap
    v = np.abs(rng.standard_normal((n, nkv, hd))) + 0.5
    v[at] = 0
    pool.k.put(pool.table[0, j // page], j % page, k)
    pool.v.put(pool.table[0, j // page], j % page, v)
    pool.up()
    q = synth.f32_to_bf16_bits(np.ones((t, nh, hd), np.float32))
    got = _run(exe, pool, q, [0, t], window, 4)
    k, v = (_f16(x[0] * x[1] + x[2]) for x in (pool.parts(0, "k"), pool.parts(0, "v")))
    for r in sorted({0, 1, t // 2, t - 1}):
        i = n - t + r
        ref, bound = _attend(_f64(q[r]), k, v, _visible(i, n, window, 4))
        assert np.all(np.abs(got[r] - ref) <= bound), (r, np.max(np.abs(got[r] - ref)), np.max(bound))


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
