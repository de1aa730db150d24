"""Log probabilities of tokens, entropies and alternatives on the GPU
(obs_token_logprobs, obs_lm_logprobs) against float64.

Bars, with u = 2^-24, d = m - x below a row's maximum m, W = sum p d and Q = sum p d^2.
exp(-d) is v_exp_f32 (2 u) of d (u of it) times log2 e (2 u): off by (2 + 3 d) u of
itself. A term passes at most ADDS = 112 additions and rescalings (32 in a thread, the
wave's and workgroup's trees, the parts or tiles of a row, five a thread, again a tree).
So log s is off by (ADDS + 2 + 3 W) u and its own rounding, w / s by (2 ADDS + 4) u W +
3 u Q, and log p = (x - m) - log s by what its terms have and round. From hidden rows a
logit is off by the fp32 sums of a group, 64 additions of s (16 + q) |x| and
|b - 16 s| |x|, and of the groups: (64 + in / 64 + 8) u of the sum of those; beyond 32 rows
an x below 2^-24 of its row's largest is held to within 2^-35 of that, a weight whose
scale is below 2^-8 of its vocabulary row's largest to within 2^-15 of that (the sums run over
all columns there, and are held to the same bar); log p by
twice the worst of them, an entropy by that times sum p |log p + H|."""
import ctypes as C

import numpy as np
import pytest

import obsidian_hip as oh
from obsidian_hip import synth

pytestmark = pytest.mark.gpu


def _f64(bits):
    return synth.bf16_bits_to_f32(np.asarray(bits)).astype(np.float64)


ADDS, U = 112, 2.0 ** -24


def _reference(x, tokens, k):
    """x float64 [T, V] -> log probabilities, entropies, ids, their log probabilities; bars of log s and of an entropy [T]."""
    T, V = x.shape
    lp, ent = np.zeros(T), np.zeros(T)
    bs, be = np.zeros(T), np.zeros(T)
    ids, tlp = np.full((T, k), -1), np.full((T, k), -np.inf)
    for t in range(T):
        row = x[t]
        order = np.lexsort((np.arange(V), -np.where(np.isnan(row), -np.inf, row)))[:k]
        order = [i for i in order if row[i] > -np.inf]
        ids[t, :len(order)] = order
        there = 0 <= tokens[t] < V
        if np.any(np.isnan(row)) or np.any(row == np.inf):
            ent[t] = np.nan
            lp[t] = np.nan if there else 0.0
            tlp[t, :len(order)] = np.nan
            continue
        m = row.max()
        if m == -np.inf:
            lp[t] = -np.inf if there else 0.0
            continue
        ls = np.log(np.sum(np.exp(row - m)))
        row = (row - m) - ls  # (not row - (m + ls): m may be 10^38)
        p = np.exp(row)
        d = np.where(p > 0, -ls - row, 0)
        W, Q = p @ d, p @ (d * d)
        bs[t] = (ADDS + 4 + 3 * W + 4 * ls) * U
        be[t] = bs[t] + ((2 * ADDS + 6) * W + 3 * Q) * U
        ent[t] = -np.sum(np.where(p > 0, p * np.where(p > 0, row, 0), 0))
        lp[t] = row[tokens[t]] if there else 0.0
        tlp[t, :len(order)] = row[order]
    return lp, ent, ids, tlp, bs, be


def _near(got, want, bar):
    got, want = got.astype(np.float64), np.asarray(want)
    want = np.where(np.abs(want) > 3.4029e38, np.copysign(np.inf, want), want)  # past fp32's range
    same = (np.isnan(got) & np.isnan(want)) | (got == want)
    with np.errstate(invalid="ignore"):
        return np.all(same | (np.abs(got - want) <= bar))


def _run(exe, T, k, tokens, call, size):
    lp, ent = exe.upload(np.full(T + 1, 77.0, np.float32)), exe.upload(np.full(T + 1, 77.0, np.float32))
    ids, tlp = exe.upload(np.full((T + 1, max(k, 1)), 77, np.int32)), exe.upload(np.full((T + 1, max(k, 1)), 77.0, np.float32))
    ws = exe.upload(np.full(max(size, 1), 0xFF, np.uint8))
    again = lambda: call(ws=ws, ws_bytes=size, tokens=exe_tok, logprob=lp, entropy=ent, top_k=k, top_ids=ids if k else None,
                         top_logprobs=tlp if k else None)
    exe_tok = exe.upload(np.asarray(tokens, np.int32))
    again()
    out = [b.download() for b in (lp, ent, ids, tlp)]
    again()
    for a, b in zip(out, (lp, ent, ids, tlp)):
        assert np.array_equal(a, b.download(), equal_nan=True)  # the same call, the same bits
    assert out[0][T] == 77 and out[1][T] == 77 and np.all(out[2].reshape(-1)[T * k:] == 77)
    return out[0][:T], out[1][:T], out[2].reshape(-1)[:T * k].reshape(T, k), out[3].reshape(-1)[:T * k].reshape(T, k)


def _logits_case(exe, x, tokens, k, bf16, pad=0, shift=0):
    """x float32 [T, V] of values that the type holds; pad: columns behind a row; shift: elements before the first."""
    T, V = x.shape
    raw = synth.f32_to_bf16_bits(x) if bf16 else x
    ld = V + pad
    buf = np.full(shift + T * ld + 8, 0x7F80 if bf16 else np.inf, raw.dtype)
    view = buf[shift:shift + T * ld].reshape(T, ld)
    view[:, :V] = raw
    d = exe.upload(buf)
    dt = oh.LOGITS_BF16 if bf16 else oh.LOGITS_F32
    got = _run(exe, T, k, tokens, lambda **kw: exe.token_logprobs(d.ptr + shift * raw.itemsize, T, V, dtype=dt, ld=ld, **kw),
               exe.token_logprobs_workspace(T, V, k, dt))
    x64 = _f64(raw) if bf16 else x.astype(np.float64)
    lp, ent, ids, tlp, bs, be = _reference(x64, tokens, k)
    size = lambda v: 4 * U * np.where(np.isfinite(v), np.abs(v), 0)
    assert _near(got[0], lp, bs + size(lp)), np.nanmax(np.abs(got[0] - lp))
    assert _near(got[1], ent, be), np.nanmax(np.abs(got[1] - ent))
    assert np.array_equal(got[2], ids)
    assert _near(got[3], tlp, bs[:, None] + size(tlp))
    return got


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,V,k,pad,shift", [(1, 1, 1, 0, 0), (3, 2, 2, 0, 0), (2, 63, 5, 1, 0), (5, 255, 64, 0, 3), (4, 256, 20, 0, 0),
                                             (3, 257, 7, 0, 1), (2, 1023, 0, 0, 0), (6, 5000, 20, 3, 0), (1, 151936, 5, 0, 0),
                                             (70, 151669, 20, 267, 0), (2, 40000, 64, 0, 0), (300, 4097, 1, 0, 0)])
def test_logits(exe, T, V, k, pad, shift, bf16):
    rng = np.random.default_rng(T + V + k)
    x = (rng.standard_normal((T, V)) * 3 - 1).astype(np.float32)
    if V > 60:
        x[:, rng.integers(0, V, V // 50)] = -np.inf
        x[:, rng.integers(0, V, 3)] += 9
    x[:, 0] = 1.0  # something is left
    tokens = rng.integers(0, V, T)
    if T > 2:
        tokens[1], tokens[2] = -1, V
    _logits_case(exe, x, tokens, k, bf16, pad, shift)


def test_logits_of_the_kinds_that_go_wrong(exe):
    """Equal logits, all forbidden, one left, fewer left than asked for, huge and tiny ones, NaN, infinities."""
    V, k = 9000, 10
    x = np.zeros((14, V), np.float32)
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, 8191] = -3.0
    x[3] = -np.inf
    x[3, [8999, 5, 700]] = [1.0, 1.0, 2.0]
    x[4] = np.where(np.arange(V) % 2, 3e38, -3e38)
    x[5] = np.arange(V)  # the largest last
    x[6] = -np.arange(V)
    x[7] = 1e-40 * (np.arange(V) % 7)
    x[8, 4000] = np.nan
    x[9, 17] = np.inf
    x[10] = np.nan
    x[11] = np.where(np.arange(V) % 2, 0.0, -0.0)
    x[12, :4096] = np.nan
    x[13] = np.float32(np.finfo(np.float32).min)  # a mask of the type's lowest value
    x[13, 123] = 0.5
    _logits_case(exe, x, np.array([5, 5, 8191, 700, 1, 8998, 3, 6, 4000, 3, 0, 1, 8000, 123]), k, False)
    _logits_case(exe, x, np.arange(14) - 1, 64, False, pad=1)
    y = np.where(np.isfinite(x), np.clip(x, -3e38, 3e38), x).astype(np.float32)
    _logits_case(exe, synth.bf16_bits_to_f32(synth.f32_to_bf16_bits(y)), np.arange(14), k, True)


@pytest.mark.parametrize("bf16", [False, True])
def test_logits_equal_in_masses(exe, bf16):
    """More equal tiles and logits than the lists hold; the lowest ids win, also where the last tile is cut."""
    V = 700001
    x = np.zeros((3, V), np.float32)
    x[1, V - 1] = 1.0
    x[2] = np.where(np.arange(V) < 300000, -np.inf, -2.0)
    _logits_case(exe, x, np.array([V - 1, 7, 300000]), 64, bf16, pad=3)
    _logits_case(exe, x, np.array([V - 1, 7, 299999]), 1, bf16, pad=0)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,V,k,kinds", [(40, 984, 15, 0), (6, 2000, 20, 0), (3, 5000, 64, 0), (3, 16000, 64, 0), (2, 16200, 63, 0), (5, 700, 64, 9),
                                         (3, 5000, 30, 3), (2, 129, 64, 0)])
def test_logits_more_alternatives_than_tiles(exe, T, V, k, kinds, bf16):
    """All tiles are looked through; `kinds` different values, or all different."""
    rng = np.random.default_rng(V + k)
    x = rng.integers(0, kinds, (T, V)).astype(np.float32) if kinds else (rng.standard_normal((T, V)) * 3).astype(np.float32)
    if bf16:
        x = synth.bf16_bits_to_f32(synth.f32_to_bf16_bits(x))
    _logits_case(exe, x, rng.integers(0, V, T), k, bf16)


def test_logits_every_row_its_own_offset(exe):
    """Rows of a long prompt whose tensor passes 4 GiB."""
    T, V, ld = 2100, 151936, 520000
    d = exe.zeros(T * ld, np.float32)
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, V)).astype(np.float32) * 2
    for i, t in enumerate((0, T - 1)):
        exe._check(oh.lib().obs_upload(exe.ctx, d.ptr + 4 * t * ld, x[i].ctypes.data, x[i].nbytes))
    tokens = np.zeros(T, np.int32)
    tokens[0], tokens[-1] = 5, V - 1
    lp, ids = exe.alloc(T, np.float32), exe.alloc((T, 3), np.int32)
    tl = exe.alloc((T, 3), np.float32)
    ws = exe.alloc(exe.token_logprobs_workspace(T, V, 3), np.uint8)
    exe.token_logprobs(d, T, V, ws, tokens=exe.upload(tokens), logprob=lp, top_k=3, top_ids=ids, top_logprobs=tl, ld=ld)
    got, gi = lp.download(), ids.download()
    d.free()
    ref = _reference(x.astype(np.float64), tokens[[0, -1]], 3)
    assert np.all(np.abs(got[[0, -1]] - ref[0]) <= ref[4] + 4 * U * np.abs(ref[0])) and np.array_equal(gi[[0, -1]], ref[2])
    assert np.all(np.abs(got[1:-1] + np.log(V)) <= (ADDS + 4 + 8 * np.log(V)) * U) and np.all(gi[1:-1] == np.arange(3))


# ---- from hidden rows -----------------------------------------------------------

def _matrix(rng, V, H):
    w = rng.integers(0, 2 ** 32, (V, H // 8), dtype=np.uint32)
    s = synth.f32_to_bf16_bits((0.006 + 0.004 * rng.random((V, H // 64))).astype(np.float32))
    b = synth.f32_to_bf16_bits((_f64(s) * (-7.5 + 0.5 * rng.standard_normal(s.shape))).astype(np.float32))
    return w, s, b


def _logits64(x, w, s, b):
    """Logits and what their fp32 sums may be off."""
    H = x.shape[1]
    out, off = np.empty((x.shape[0], w.shape[0])), np.empty((x.shape[0], w.shape[0]))
    top = np.abs(x).max(1, keepdims=True)
    small = np.where((np.abs(x) < 2.0 ** -24 * top) & (x != 0) & (x.shape[0] > 32), 2.0 ** -35 * top, 0)
    for v in range(0, w.shape[0], 4096):
        q = ((w[v:v + 4096, :, None] >> np.arange(0, 32, 4, dtype=np.uint32)) & 15).reshape(-1, H).astype(np.float64)
        ss, bb = (np.repeat(_f64(y[v:v + 4096]), 64, 1) for y in (s, b))
        out[:, v:v + 4096] = x @ (q * ss + bb).T
        off[:, v:v + 4096] = np.abs(x) @ (ss * (16 + q) + np.abs(bb - 16 * ss)).T * ((64 + H // 64 + 8) * U) + small @ (q * ss).T
    return out, off


def _lm_case(exe, T, H, V, k, seed, scale=1.0, tokens=None):
    rng = np.random.default_rng(seed)
    w, s, b = _matrix(rng, V, H)
    x = synth.bf16_normal(rng, (T, H), scale)
    tokens = rng.integers(0, V, T) if tokens is None else tokens
    if T > 2:
        tokens[1], tokens[2] = -1, V
    dx, dw, ds, db = (exe.upload(a) for a in (x, w, s, b))
    got = _run(exe, T, k, tokens, lambda **kw: exe.lm_logprobs(dx, dw, ds, db, T, H, V, **kw), exe.lm_logprobs_workspace(T, H, V, k))
    logits, off = _logits64(_f64(x), w, s, b)
    lp, ent, ids, tlp, bs, be = _reference(logits, tokens, k)
    worst = off.max(1)
    size = lambda v: 4 * U * np.abs(v)
    assert _near(got[0], lp, bs + size(lp) + 2 * worst), np.max(np.abs(got[0] - lp))
    logp = logits - (logits.max(1) + np.log(np.sum(np.exp(logits - logits.max(1)[:, None]), 1)))[:, None]
    move = np.sum(np.exp(logp) * np.abs(logp + ent[:, None]), 1)
    assert _near(got[1], ent, be + 1.01 * move * worst), np.max(np.abs(got[1] - ent))
    for t in range(T):
        if k:
            assert len(set(got[2][t])) == k and np.all((got[2][t] >= 0) & (got[2][t] < V))
            # the alternatives are the largest but for the order of those as near as the sums are exact
            assert np.all(np.abs(logits[t, got[2][t]] - logits[t, ids[t]]) <= 2 * worst[t])
            assert np.all(np.diff(got[3][t]) <= 0)
            have = logits[t, got[2][t]] - logits[t, ids[t, 0]] + tlp[t, 0]
            assert np.all(np.abs(got[3][t] - have) <= bs[t] + size(have) + 2 * worst[t])
    return got


@pytest.mark.parametrize("T", [1, 2, 8, 9, 16, 17, 32, 33, 64, 65, 127, 128, 129, 300])
def test_lm_rows(exe, T):
    _lm_case(exe, T, 1024, 1000, 5, T)


@pytest.mark.parametrize("T,H,V,k", [(1, 512, 1, 1), (3, 512, 255, 3), (40, 512, 256, 64), (5, 2048, 257, 0), (70, 4096, 777, 20), (20, 4096, 3001, 9),
                                     (600, 512, 5003, 2), (260, 1536, 513, 0), (1, 2048, 40000, 5), (24, 2048, 40001, 20), (200, 2048, 20000, 3),
                                     (1000, 512, 5003, 0), (1500, 512, 20000, 0), (4100, 512, 300, 0), (33, 16384, 600, 2), (2, 16384, 600, 2),
                                     (160, 512, 30000, 3), (64, 512, 40000, 2), (150, 512, 60000, 0), (600, 4096, 3000, 0)])
def test_lm_shapes(exe, T, H, V, k):
    _lm_case(exe, T, H, V, k, T + H + V)


@pytest.mark.parametrize("T", [5, 40])
def test_lm_columns_of_all_sizes(exe, T):
    """Columns from 2^-40 to 2^40 of the others', whole blocks of them, zeros, and rows at the ends of bf16's range."""
    rng = np.random.default_rng(6)
    H, V = 1024, 999
    w, s, b = _matrix(rng, V, H)
    x = rng.standard_normal((T, H)) * np.exp2(rng.integers(-14, 15, (T, H)))
    x[0, ::2] = 0
    x[1] = 0
    x[2] *= np.exp2(np.repeat(rng.integers(-40, 41, H // 32), 32))
    x[3] *= 2.0 ** -120
    x[4] *= 2.0 ** 90 * (np.arange(H) < 32)
    xb = synth.f32_to_bf16_bits(x.astype(np.float32))
    args = [exe.upload(a) for a in (xb, w, s, b)]
    tokens = rng.integers(0, V, T)
    got = _run(exe, T, 1, tokens, lambda **kw: exe.lm_logprobs(*args, T, H, V, **kw), exe.lm_logprobs_workspace(T, H, V, 1))
    logits, off = _logits64(_f64(xb), w, s, b)
    lp, ent, ids, tlp, bs, be = _reference(logits, tokens, 1)
    assert np.all(np.abs(got[0] - lp) <= bs + 4 * U * np.abs(lp) + 2 * off.max(1))
    t = np.arange(T)
    assert np.all(logits[t, got[2][:, 0]] >= logits[t, ids[:, 0]] - 2 * off.max(1))


@pytest.mark.parametrize("T", [5, 40, 100])
def test_lm_scales_of_all_sizes(exe, T):
    """Groups' scales from 2^-20 to 2^20 of each other in a vocabulary row, zeros, rows of zeros alone, biases far above them."""
    rng = np.random.default_rng(16)
    H, V = 1024, 530
    w, s, b = _matrix(rng, V, H)
    s64, b64 = _f64(s), _f64(b)
    f = np.exp2(rng.integers(-10, 11, s.shape) * (np.arange(V) % 2)[:, None])
    s64, b64 = s64 * f, b64 * f
    s64[7::50, ::3] = 0
    s64[9::50] = 0
    b64[9::50] = np.exp2(rng.integers(-30, 3, b64[9::50].shape))
    b64[11::50] *= 2.0 ** 6
    s64[13::50] *= 2.0 ** -60
    s, b = (synth.f32_to_bf16_bits(y.astype(np.float32)) for y in (s64, b64))
    x = synth.bf16_normal(rng, (T, H), 0.02)
    x[T - 1, H // 2:] = 0
    args = [exe.upload(a) for a in (x, w, s, b)]
    tokens = rng.integers(0, V, T)
    got = _run(exe, T, 2, tokens, lambda **kw: exe.lm_logprobs(*args, T, H, V, **kw), exe.lm_logprobs_workspace(T, H, V, 2))
    logits, off = _logits64(_f64(x), w, s, b)
    if T > 32:
        most = _f64(s).max(1, keepdims=True)
        rough = np.repeat(np.where(_f64(s) < most * 2.0 ** -8, most * 2.0 ** -15, 0), 64, 1)
        off += np.abs(_f64(x)) @ rough.T
    lp, ent, ids, tlp, bs, be = _reference(logits, tokens, 2)
    assert _near(got[0], lp, bs + 4 * U * np.abs(lp) + 2 * off.max(1))
    t = np.arange(T)
    assert np.all(logits[t, got[2][:, 0]] >= logits[t, ids[:, 0]] - 2 * off.max(1))


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("e", [-110, -60, 60, 110])
def test_lm_scales_and_rows_of_opposite_sizes(exe, T, e):
    """Scales and biases 2^e of the usual, hidden rows 2^-e."""
    rng = np.random.default_rng(17)
    H, V = 512, 300
    w, s, b = _matrix(rng, V, H)
    s, b = (synth.f32_to_bf16_bits((_f64(y) * 2.0 ** e).astype(np.float32)) for y in (s, b))
    x = synth.f32_to_bf16_bits((rng.standard_normal((T, H)) * 2.0 ** -e).astype(np.float32))
    args = [exe.upload(a) for a in (x, w, s, b)]
    tokens = rng.integers(0, V, T)
    got = _run(exe, T, 1, tokens, lambda **kw: exe.lm_logprobs(*args, T, H, V, **kw), exe.lm_logprobs_workspace(T, H, V, 1))
    logits, off = _logits64(_f64(x), w, s, b)
    lp, ent, ids, tlp, bs, be = _reference(logits, tokens, 1)
    assert _near(got[0], lp, bs + 4 * U * np.abs(lp) + 2 * off.max(1))
    t = np.arange(T)
    assert np.all(logits[t, got[2][:, 0]] >= logits[t, ids[:, 0]] - 2 * off.max(1))


def test_lm_large_rows(exe):
    """Hidden rows of large magnitude: one token takes all."""
    _lm_case(exe, 7, 1024, 2000, 4, 1, scale=200.0)
    _lm_case(exe, 77, 1024, 2000, 4, 2, scale=200.0)


@pytest.mark.parametrize("T", [3, 50])
def test_lm_rows_not_finite_stay_their_own(exe, T):
    """A row with NaN has none but its own results NaN."""
    rng = np.random.default_rng(9)
    H, V, k = 512, 700, 3
    w, s, b = _matrix(rng, V, H)
    x = synth.bf16_normal(rng, (T, H), 1.0)
    tokens = rng.integers(0, V, T)
    args = [exe.upload(a) for a in (w, s, b)]
    n = exe.lm_logprobs_workspace(T, H, V, k)
    clean = _run(exe, T, k, tokens, lambda **kw: exe.lm_logprobs(exe.upload(x), *args, T, H, V, **kw), n)
    x[1, 77] = 0x7FC0
    dx = exe.upload(x)
    got = _run(exe, T, k, tokens, lambda **kw: exe.lm_logprobs(dx, *args, T, H, V, **kw), n)
    for a, c in zip(got, clean):
        assert np.array_equal(np.delete(a, 1, 0), np.delete(c, 1, 0))
    assert np.isnan(got[0][1]) and np.isnan(got[1][1]) and np.all(got[2][1] == -1)


def test_lm_equals_the_gemv_and_logits(exe):
    """One token: the log probabilities of obs_q4_gemv's logits, but for the order of the sums."""
    rng = np.random.default_rng(4)
    H, V, k = 2048, 30000, 8
    w, s, b = _matrix(rng, V, H)
    x = synth.bf16_normal(rng, (1, H), 1.0)
    dx, dw, ds, db = (exe.upload(a) for a in (x, w, s, b))
    lg = exe.alloc(V, np.float32)
    exe.q4_gemv(dx, H, [(dw, ds, db, V, lg, None, None)])
    tokens = [int(np.argmax(lg.download()))]
    a = _run(exe, 1, k, tokens, lambda **kw: exe.token_logprobs(lg, 1, V, **kw), exe.token_logprobs_workspace(1, V, k))
    c = _run(exe, 1, k, tokens, lambda **kw: exe.lm_logprobs(dx, dw, ds, db, 1, H, V, **kw), exe.lm_logprobs_workspace(1, H, V, k))
    off = _logits64(_f64(x), w, s, b)[1].max() * 2
    assert np.all(np.abs(a[0] - c[0]) <= 2 * off + 2.0 ** -19) and a[2][0, 0] == c[2][0, 0] == tokens[0]


def test_captured_calls_follow_the_device_arrays(exe):
    rng = np.random.default_rng(5)
    T, H, V, k = 40, 512, 3000, 4
    with oh.ObsidianExecutor(0) as e:
        mats = [_matrix(rng, V, H) for _ in range(2)]
        x = [synth.bf16_normal(rng, (T, H), 1.0) for _ in range(2)]
        tok = [rng.integers(0, V, T).astype(np.int32) for _ in range(2)]
        d = [e.upload(a) for a in mats[0]]
        dx, dt = e.upload(x[0]), e.upload(tok[0])
        out = [[e.alloc(T, np.float32), e.alloc(T, np.float32), e.alloc((T, k), np.int32), e.alloc((T, k), np.float32)] for _ in range(3)]
        lg = e.upload(rng.standard_normal((T, V)).astype(np.float32))
        ws = e.alloc(e.lm_logprobs_workspace(T, H, V, k), np.uint8)
        ws1 = e.alloc(e.lm_logprobs_workspace(1, H, V, k), np.uint8)
        ws2 = e.alloc(e.token_logprobs_workspace(T, V, k), np.uint8)

        def calls():
            e.lm_logprobs(dx, *d, T, H, V, ws, tokens=dt, logprob=out[0][0], entropy=out[0][1], top_k=k, top_ids=out[0][2],
                          top_logprobs=out[0][3])
            e.lm_logprobs(dx, *d, 1, H, V, ws1, tokens=dt, logprob=out[1][0], entropy=out[1][1], top_k=k, top_ids=out[1][2],
                          top_logprobs=out[1][3])
            e.token_logprobs(lg, T, V, ws2, tokens=dt, logprob=out[2][0], entropy=out[2][1], top_k=k, top_ids=out[2][2],
                             top_logprobs=out[2][3])

        for o in out[1]:
            e._check(oh.lib().obs_memset(e.ctx, o.ptr, 0, o.nbytes))
        calls()
        e.sync()
        e.capture_begin()
        calls()
        g = e.capture_end()
        for i in (1, 0, 1):
            for buf, a in zip(d, mats[i]):
                buf.upload(a)
            dx.upload(x[i])
            dt.upload(tok[i])
            e.graph_launch(g)
            replayed = [[o.download() for o in r] for r in out]
            calls()
            for r, o in zip(replayed, out):
                for a, b in zip(r, o):
                    assert np.array_equal(a, b.download())
        e.graph_destroy(g)
