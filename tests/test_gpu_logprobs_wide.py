"""obs_lm_logprobs on sizes that take each of its larger workgroups, 64 x 128 to 128 x 256
(rows x columns), where scales, biases and hidden values are of all sizes: vocabulary
rows beside each other, in both of a wave's blocks of columns, have other powers of two.

Bars, with u = 2^-24: a logit is off by its fp32 sums, (64 + in / 64 + 8) u of what they add
(s (16 + q) |x| and |b - 16 s| |x|), by 2^-39 of a row's largest hidden value times
s |q - 8| where a value lies below 2^-29 of that, and by 2^-15 of the largest scale of
a vocabulary row times |x| where a group's lies below 2^-8 of that. A log probability is
off by its own logit's and by the mean of all, weighted by their probabilities, and by
the bars of test_gpu_logprobs."""
import numpy as np
import pytest

from obsidian_hip import synth
from test_gpu_logprobs import U, _f64, _matrix, _near, _reference, _run

pytestmark = pytest.mark.gpu

H = 512
# rows, columns; the workgroup that they take by the rule at present
SIZES = [(64, 40001, "64 x 128"), (96, 40001, "96 x 128"), (128, 39997, "128 x 128"), (150, 60000, "96 x 256"), (200, 40130, "128 x 256")]


def _logits(x, w, s, b):
    """x float64 [T, H] -> logits and what they may be off."""
    top = np.abs(x).max(1, keepdims=True)
    small = np.where((np.abs(x) < 2.0 ** -29 * top) & (x != 0), 2.0 ** -39 * top, 0)
    out, off = np.empty((len(x), len(w))), np.empty((len(x), len(w)))
    for v in range(0, len(w), 4096):
        q = ((w[v:v + 4096, :, None] >> np.arange(0, 32, 4, dtype=np.uint32)) & 15).reshape(-1, H).astype(np.float64)
        s0, b0 = _f64(s[v:v + 4096]), _f64(b[v:v + 4096])
        most = s0.max(1, keepdims=True)
        rough = np.repeat(np.where(s0 < most * 2.0 ** -8, most * 2.0 ** -15, 0), 64, 1)
        ss, bb = np.repeat(s0, 64, 1), np.repeat(b0, 64, 1)
        out[:, v:v + 4096] = x @ (q * ss + bb).T
        off[:, v:v + 4096] = np.abs(x) @ ((ss * (16 + q) + np.abs(bb - 16 * ss)) * ((64 + H // 64 + 8) * U) + rough).T + \
            small @ (ss * np.abs(q - 8)).T
    return out, off


def _check(exe, x, w, s, b, k, tokens):
    T, V = len(x), len(w)
    args = [exe.upload(a) for a in (x, w, s, b)]
    got = _run(exe, T, k, tokens, lambda **kw: exe.lm_logprobs(*args, T, H, V, **kw), exe.lm_logprobs_workspace(T, H, V, k))
    for a in args:
        a.free()
    logits, off = _logits(_f64(x), w, s, b)
    lp, ent, ids, tlp, bs, be = _reference(logits, tokens, k)
    t = np.arange(T)
    logp = logits - (logits.max(1) + np.log(np.sum(np.exp(logits - logits.max(1)[:, None]), 1)))[:, None]
    p = np.exp(logp)
    mean = 1.01 * np.sum(p * off, 1)
    assert _near(got[0], lp, bs + 4 * U * np.abs(lp) + off[t, tokens] + mean), np.max(np.abs(got[0] - lp))
    # an entropy moves by p |log p + H| of each logit's change
    assert _near(got[1], ent, be + 1.01 * np.sum(p * np.abs(logp + ent[:, None]) * off, 1))
    for i in range(k):
        have = got[2][:, i]
        assert np.all(np.abs(logits[t, have] - logits[t, ids[:, i]]) <= off[t, have] + off.max(1))
        assert _near(got[3][:, i], logp[t, have], bs + 4 * U * np.abs(logp[t, have]) + off[t, have] + mean)


@pytest.mark.parametrize("T,V,_", SIZES, ids=lambda v: str(v))
def test_scales_of_all_sizes(exe, T, V, _):
    """A power of two a vocabulary row, others a group in every second one, zeros, biases alone and far above."""
    rng = np.random.default_rng(T)
    w, s, b = _matrix(rng, V, H)
    e = rng.integers(-12, 4, V)[:, None] + rng.integers(-14, 3, s.shape) * (np.arange(V) % 2)[:, None]
    s, b = _f64(s) * np.exp2(e), _f64(b) * np.exp2(e)
    s[7::50, ::3] = 0
    s[9::50] = 0
    b[9::50] = np.exp2(rng.integers(-30, -5, b[9::50].shape))
    b[11::50] *= 2.0 ** 6
    s[13::50] *= 2.0 ** -60
    s, b = (synth.f32_to_bf16_bits(y.astype(np.float32)) for y in (s, b))
    x = synth.bf16_normal(rng, (T, H), 1.0)
    x[T - 1, H // 2:] = 0
    _check(exe, x, w, s, b, 5, rng.integers(0, V, T))


@pytest.mark.parametrize("T,V,_", SIZES, ids=lambda v: str(v))
def test_columns_of_all_sizes(exe, T, V, _):
    """Hidden values to 2^-40 of their row's largest, rows of one value, of zeros, of the least numbers."""
    rng = np.random.default_rng(T + 1)
    w, s, b = _matrix(rng, V, H)
    e = rng.integers(-3, 4, V)[:, None]
    s, b = (synth.f32_to_bf16_bits((_f64(y) * np.exp2(e)).astype(np.float32)) for y in (s, b))
    x = rng.standard_normal((T, H)) * np.exp2(rng.integers(-40, 3, (T, H)))
    x[::5] = rng.standard_normal((len(x[::5]), H)) * np.exp2(np.repeat(rng.integers(-36, 3, (len(x[::5]), H // 32)), 32, 1))
    x[3::7] *= np.exp2(rng.integers(-100, 1, len(x[3::7])))[:, None]
    x[1] = 0
    x[2] = 0
    x[2, 300] = 5.0
    x[T - 1] = 2.0 ** -133  # the least numbers
    _check(exe, synth.f32_to_bf16_bits(x.astype(np.float32)), w, s, b, 3, rng.integers(0, V, T))


@pytest.mark.parametrize("T,V,_", SIZES[3:], ids=lambda v: str(v))
def test_rows_not_finite_stay_their_own(exe, T, V, _):
    rng = np.random.default_rng(T + 2)
    w, s, b = _matrix(rng, V, H)
    x, k = synth.bf16_normal(rng, (T, H), 1.0), 3
    tokens = rng.integers(0, V, T)
    args, dx = [exe.upload(a) for a in (w, s, b)], exe.upload(x)
    n = exe.lm_logprobs_workspace(T, H, V, k)
    clean = _run(exe, T, k, tokens, lambda **kw: exe.lm_logprobs(dx, *args, T, H, V, **kw), n)
    rows = [1, 40, T - 2]
    x[rows, 77] = [0x7FC0, 0x7F80, 0xFFC1]
    dx.upload(x)
    got = _run(exe, T, k, tokens, lambda **kw: exe.lm_logprobs(dx, *args, T, H, V, **kw), n)
    for a, c in zip(got, clean):
        assert np.array_equal(np.delete(a, rows, 0), np.delete(c, rows, 0))
    assert np.all(np.isnan(got[0][rows])) and np.all(np.isnan(got[1][rows]))


@pytest.mark.parametrize("col", [5, 40, 130])
def test_a_vocabulary_row_not_finite_stays_its_own_column(exe, col):
    """A scale of NaN is one token's: every row's log probabilities are NaN, the alternatives are the others'."""
    T, V, k = 200, 40130, 5
    rng = np.random.default_rng(col)
    w, s, b = _matrix(rng, V, H)
    x = synth.bf16_normal(rng, (T, H), 1.0)
    logits, off = _logits(_f64(x), w, s, b)
    s[col, 3] = 0x7FC0
    args = [exe.upload(a) for a in (x, w, s, b)]
    got = _run(exe, T, k, rng.integers(0, V, T), lambda **kw: exe.lm_logprobs(*args, T, H, V, **kw), exe.lm_logprobs_workspace(T, H, V, k))
    assert np.all(np.isnan(got[0])) and np.all(np.isnan(got[1])) and not np.any(got[2] == col)
    logits[:, col] = -np.inf
    off[:, col] = 0
    want = np.sort(logits, 1)[:, ::-1][:, :k]
    t = np.arange(T)[:, None]
    assert np.all(np.abs(logits[t, got[2]] - want) <= 2 * off.max(1)[:, None])
