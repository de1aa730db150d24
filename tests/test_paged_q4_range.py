"""The range of a cache of 4 bits. Prompts take q * scale + bias in fp16, so up to 65,519
in magnitude (to nearest, 65,504 the largest). Of appended values up to A the bias is
off by 128 (bf16 has steps of 256 from 32,768 on), the scale, below 8,739, by 32 (steps of
64): what is stored passes A by 128 + 15 * 32 = 608 at most. So A is 64,900."""
import numpy as np
import pytest

from obsidian_hip import synth
from test_gpu_paged import FILL16, _f64
from test_gpu_paged_q4 import GROUP, Pool, _attend4, _attend16, _f16, quantize

A = 64900.0


def _ends(a):
    """Groups of all ranges within -a .. a that reach one end of it, or nearly."""
    lo = np.concatenate([-np.linspace(0, a, 4001), [-a] * 4001, a - np.linspace(0, 4000, 4001)])
    hi = np.concatenate([[a] * 4001, np.linspace(-a, a, 4001), [a] * 4001])
    lo, hi = np.minimum(lo, hi), np.maximum(lo, hi)
    x = np.repeat(lo[:, None], GROUP, 1)
    x[:, 1::2] = hi[:, None]
    return x


def test_what_appended_values_become():
    q, s, b = quantize(_ends(A))
    assert np.abs(np.repeat(s, GROUP, -1) * q + np.repeat(b, GROUP, -1)).max() < 65520
    q, s, b = quantize(_ends(65504.0))
    assert np.abs(np.repeat(s, GROUP, -1) * q + np.repeat(b, GROUP, -1)).max() >= 65520  # why the limit lies below fp16's


@pytest.mark.gpu
def test_the_ends_of_the_range(exe):
    """Keys and values at the stated end in prompts and steps; beyond it, steps alone."""
    nh, nkv, hd, page, n, t = 8, 2, 128, 32, 96, 70
    rng = np.random.default_rng(79)
    ends = _ends(A)
    q, s, b = quantize(ends)
    most = np.argsort(np.abs(np.repeat(s, GROUP, -1) * q + np.repeat(b, GROUP, -1)).max(1))[-n * nkv * hd // GROUP:]
    q = synth.bf16_normal(rng, (t, nh, hd), 1e-5)
    for beyond in (False, True):
        pool = Pool(exe, rng, [n], nkv, hd, page)
        j = np.arange(n)
        for side in (pool.k, pool.v):
            x = ends[rng.permutation(most)].reshape(n, nkv, hd)
            side.put(pool.table[0, j // page], j % page, x * (2.0 ** 100 if beyond and side.values else 1.0))
        pool.up()
        dq, out = exe.upload(q), exe.upload(np.full((t, nh, hd), FILL16, np.uint16))
        if not beyond:
            seqs = pool.seqs([0, t])
            ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, seqs, nh), np.uint8)
            exe.sdpa_paged_prefill(pool.kv, seqs, dq, out, nh, ws)
            got = _f64(out.download())
            k, v = (_f16(x[0] * x[1] + x[2]) for x in (pool.parts(0, "k"), pool.parts(0, "v")))
            assert np.all(np.isfinite(k)) and np.all(np.isfinite(v))
            for r in range(t):
                ref, bound = _attend16(_f64(q[r]), k, v, np.arange(n) <= n - t + r)
                assert np.all(np.abs(got[r] - ref) <= bound), r
        seqs = pool.seqs()
        ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, seqs, nh), np.uint8)
        exe.sdpa_paged_decode(pool.kv, seqs, dq, out, nh, ws)
        ref, bound, _, _ = _attend4(_f64(q[0]), pool.parts(0, "k"), pool.parts(0, "v"), np.ones(n, bool))
        assert np.all(np.abs(_f64(out.download())[0] - ref) <= bound)
