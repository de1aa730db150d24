"""The paged key/value cache on the GPU (obs_attn_prep_paged, obs_sdpa_paged_decode,
obs_sdpa_paged_prefill, obs_kv_evict) against plain float64 restatements.

Every pool is filled with NaN but for the entries that a call may see, tables
hold -1 behind a sequence's pages, and outputs start from a pattern, so a read or
a write outside what the call owns shows.

Bars. A bf16 rounding is off by at most 2^-8 of its value, an e4m3 one by 2^-4
(2^-10 of the scale below the normal range). Attention: P enters the value product
in bf16 (2^-8 of sum p|v|), the output is rounded once (2^-8 of it), and a score's
fp32 sum of d exact products is off by at most d 2^-24 sum|q k| / sqrt(d), which
moves p by that factor in numerator and denominator (twice); exp2 and the scale
factors are a few units of 2^-23 |s|. Gathered weights: the same score terms and
the fp32 addition."""
import numpy as np
import pytest

import obsidian_hip as oh
from obsidian_hip import synth

pytestmark = pytest.mark.gpu

EPS, THETA = 1e-6, 1e7
NAN16, FILL16 = 0x7FC1, 0x4B4B


def _f64(bits):
    return synth.bf16_bits_to_f32(np.asarray(bits)).astype(np.float64)


def _bf16(x):
    return synth.f32_to_bf16_bits(np.asarray(x, np.float32))


def _e4m3_values():
    v = np.empty(256)
    for i in range(256):
        s, e, m = i >> 7, (i >> 3) & 15, i & 7
        x = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[i] = np.nan if e == 15 and m == 7 else (-x if s else x)
    return v


E4M3 = _e4m3_values()
_POS = np.sort(E4M3[:127])  # 0 .. 448


def _e4m3_bytes(x):
    """Nearest e4m3, ties to even, saturating."""
    x = np.asarray(x, np.float64)
    mag = np.minimum(np.abs(x), 448.0)
    i = np.clip(np.searchsorted(_POS, mag), 1, 126)
    lo, hi = _POS[i - 1], _POS[i]
    up = (mag - lo > hi - mag) | ((mag - lo == hi - mag) & (i % 2 == 0))
    b = np.where(up, i, i - 1).astype(np.uint8)
    return np.where(np.signbit(x), b | 0x80, b).astype(np.uint8)


class Pool:
    """A pool with sequences of lengths `lens` in shuffled pages; hidden[b]: entries of b that hold NaN."""

    def __init__(self, exe, rng, lens, nkv, hd, page, f8, extra=3, hidden=None, k_std=1.0, max_pages=None):
        self.exe, self.lens, self.nkv, self.hd, self.page, self.f8 = exe, list(lens), nkv, hd, page, f8
        B = len(lens)
        need = [-(-max(n, 0) // page) for n in lens]
        self.n_pages = sum(need) + extra
        self.max_pages = max_pages or max(max(need), 1) + 1
        ids = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((B, self.max_pages), -1, np.int32)
        at = 0
        for b in range(B):
            self.table[b, :need[b]] = ids[at:at + need[b]]
            at += need[b]
        self.free = ids[at:]
        T, nan = (np.uint8, 0x7F) if f8 else (np.uint16, NAN16)
        self.k = np.full((self.n_pages, nkv, page, hd), nan, T)
        self.v = np.full((self.n_pages, nkv, hd, page), nan, T)
        self.ks = (0.01 + 0.01 * rng.random(nkv)).astype(np.float32) if f8 else None
        self.vs = (0.01 + 0.01 * rng.random(nkv)).astype(np.float32) if f8 else None
        for b in range(B):
            n = max(lens[b], 0)
            j = np.arange(n)
            if hidden is not None:
                j = j[~np.isin(j, hidden[b])]
            k = rng.standard_normal((len(j), nkv, hd)) * k_std
            v = rng.standard_normal((len(j), nkv, hd))
            kb = _e4m3_bytes(k / self.ks[:, None]) if f8 else _bf16(k)
            vb = _e4m3_bytes(v / self.vs[:, None]) if f8 else _bf16(v)
            p, o = self.table[b, j // page], j % page
            self.k[p, :, o] = kb
            self.v[p, :, :, o] = vb
        self.up()

    def up(self):
        e = self.exe
        self.dk, self.dv, self.dt = e.upload(self.k), e.upload(self.v), e.upload(self.table)
        self.dl = e.upload(np.array(self.lens, np.int32))
        self.kv = oh.PagedKv(self.dk, self.dv, self.n_pages, self.page, self.nkv, self.hd,
                             oh.KV_E4M3 if self.f8 else oh.KV_BF16, e.upload(self.ks) if self.f8 else None,
                             e.upload(self.vs) if self.f8 else None)

    def seqs(self, rows=None, n_rows=None):
        B = len(self.lens)
        if rows is None:
            return oh.PagedSeqs(self.dt, self.dl, B, self.max_pages)
        return oh.PagedSeqs(self.dt, self.dl, B, self.max_pages, n_rows or int(rows[-1]),
                            self.exe.upload(np.array(rows, np.int32)))

    def entries(self, b, what):
        """[n, nkv, hd] float64 keys or values of sequence b."""
        j = np.arange(max(self.lens[b], 0))
        p, o = self.table[b, j // self.page], j % self.page
        x = self.k[p, :, o] if what == "k" else self.v[p, :, :, o]
        if not self.f8:
            return _f64(x)
        return E4M3[x] * (self.ks if what == "k" else self.vs).astype(np.float64)[:, None]


def _visible(i, n, window, sinks):
    j = np.arange(n)
    return (j <= i) & ((window == 0) | (j > i - window) | (j < sinks))


def _attend(q, k, v, vis):
    """q [nh, hd], k, v [n, nkv, hd] -> (out [nh, hd], bound, p [nh, n], score error [nh])."""
    nh, hd = q.shape
    nkv = k.shape[1]
    per = nh // nkv
    out, bound = np.zeros((nh, hd)), np.zeros((nh, hd))
    p_all, err_all = np.zeros((nh, len(vis))), np.zeros(nh)
    idx = np.flatnonzero(vis)
    if len(idx) == 0:
        return out, bound, p_all, err_all
    for h in range(nh):
        kk, vv = k[idx, h // per], v[idx, h // per]
        s = kk @ q[h] / np.sqrt(hd)
        e = np.exp(s - s.max())
        p = e / e.sum()
        mag = np.max(np.abs(kk) @ np.abs(q[h])) / np.sqrt(hd)
        err = 2 * (hd * 2.0 ** -24 * mag + 2.0 ** -21 * np.max(np.abs(s)) + 2.0 ** -20)
        out[h] = p @ vv
        A = p @ np.abs(vv)
        bound[h] = (2.0 ** -8 + err) * A * 1.01 + 2.0 ** -8 * np.abs(out[h]) + 1e-30
        p_all[h, idx], err_all[h] = p, err
    return out, bound, p_all, err_all


SHAPES = [(32, 4, 128, 16, False), (32, 4, 128, 64, True), (16, 16, 64, 32, False), (12, 2, 128, 32, False),
          (16, 1, 64, 256, True), (8, 8, 128, 128, False), (10, 2, 64, 16, True)]
LENS = [[1], [0, 5, 16, 17, 0], [31, 32, 33, 255, 256, 257, 1], [1500, 3, 700]]
WINDOWS = [(0, 0), (1, 0), (40, 3), (33, 32), (300, 100)]


def _decode_case(exe, shape, lens, window, sinks, weight, seed, k_std=1.0, q_ld=0):
    nh, nkv, hd, page, f8 = shape
    rng = np.random.default_rng(seed)
    hidden = [np.flatnonzero(~_visible(n - 1, max(n, 0), window, sinks)) for n in lens]
    pool = Pool(exe, rng, lens, nkv, hd, page, f8, hidden=hidden, k_std=k_std)
    B, ld = len(lens), q_ld or nh * hd
    q = np.full((B, ld), NAN16, np.uint16)
    q[:, :nh * hd] = synth.bf16_normal(rng, (B, nh * hd), 2.0)
    out = exe.upload(np.full((B, nh, hd), FILL16, np.uint16))
    cap = pool.max_pages * page
    w0 = rng.random((B + 2, nkv, cap + 5)).astype(np.float32)
    slot = rng.permutation(B + 2)[:B].astype(np.int32)
    dw = exe.upload(w0)
    wt = oh.KvWeight(dw, B + 2, cap + 5, exe.upload(slot)) if weight else None
    seqs = pool.seqs()
    ws = exe.upload(np.full(exe.sdpa_paged_workspace(pool.kv, seqs, nh, wt, window, sinks), 0xFF, np.uint8))
    call = lambda: exe.sdpa_paged_decode(pool.kv, seqs, exe_q, out, nh, ws, window=window, sinks=sinks, weight=wt, q_ld=ld)
    exe_q = exe.upload(q)
    call()
    exe.device_status()
    got, wgot = _f64(out.download()), dw.download().astype(np.float64)
    wref, werr = w0.astype(np.float64), np.zeros(w0.shape)
    for b, n in enumerate(lens):
        n = max(n, 0)
        k, v = pool.entries(b, "k"), pool.entries(b, "v")
        ref, bound, p, err = _attend(_f64(q[b, :nh * hd]).reshape(nh, hd), k, v, _visible(n - 1, n, window, sinks))
        bad = np.abs(got[b] - ref) > bound
        assert not np.any(bad) and np.all(np.isfinite(got[b])), (b, n, np.max(np.abs(got[b] - ref)))
        if weight and n:
            g = p.reshape(nkv, nh // nkv, n)
            wref[slot[b], :, :n] += g.sum(1)
            werr[slot[b], :, :n] = (g * err.reshape(nkv, -1, 1)).sum(1) + 2.0 ** -22 * wref[slot[b], :, :n]
    assert np.all(np.abs(wgot - wref) <= werr)
    return call, out, dw


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("lens", LENS, ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_decode(exe, shape, lens, window, sinks):
    _decode_case(exe, shape, lens, window, sinks, (len(lens) + window) % 2 == 0, 7)


@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("shape,lens", [((32, 4, 128, 32, False), [9000]), ((8, 1, 128, 16, True), [20001, 40]),
                                        ((32, 8, 64, 64, False), [1 + 37 * i for i in range(130)])])
def test_decode_split(exe, shape, lens, weight):
    """Long sequences over many workgroups, and more sequences than a wave has lanes."""
    call, out, _ = _decode_case(exe, shape, lens, 0, 0, weight, 11)
    first = out.download()
    call()
    assert np.array_equal(first, out.download())  # the same call, the same bits


@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("shape", [(32, 4, 128, 32, False), (32, 4, 128, 64, True), (32, 8, 64, 16, False)], ids=str)
@pytest.mark.parametrize("lens", [[1700, 3, 900, 0, 64, 33, 1300, 100, 5], [40, 512, 1, 300] * 8, [1000, 7, 250, 500] * 16],
                         ids=["joined", "16 blocks", "32 blocks"])
def test_decode_many_rows(exe, shape, lens, weight):
    """Enough rows for one join workgroup each, and batches whose sequences are one part each."""
    _decode_case(exe, shape, lens, 0, 0, weight, 20)


def test_decode_peaked_scores_and_strides(exe):
    """Scores of several hundred (one entry takes all), a q row stride of its own."""
    _decode_case(exe, (32, 4, 128, 32, False), [777, 64], 0, 0, True, 13, k_std=30.0, q_ld=32 * 128 + 64)
    _decode_case(exe, (32, 4, 128, 32, False), [777, 64], 100, 2, False, 17, k_std=30.0, q_ld=32 * 128 + 8)


def test_decode_offsets_past_32_bits(exe):
    """A pool of more than 4 GiB a side, the sequence in its last pages."""
    nh, nkv, hd, page = 32, 4, 128, 256
    n_pages = (1 << 32) // (nkv * page * hd * 2) + 40
    rng = np.random.default_rng(19)
    dk, dv = exe.alloc((n_pages, nkv, page, hd), np.uint16), exe.alloc((n_pages, nkv, hd, page), np.uint16)
    n, per = 1000, nkv * page * hd * 2
    ids = np.array([n_pages - 1, n_pages - 3, n_pages - 2, n_pages - 7], np.int32)
    k, v = synth.bf16_normal(rng, (4, nkv, page, hd)), synth.bf16_normal(rng, (4, nkv, hd, page))
    for i, p in enumerate(ids):
        for d, x in ((dk, k), (dv, v)):
            a = np.ascontiguousarray(x[i])
            exe._check(oh.lib().obs_upload(exe.ctx, d.ptr + int(p) * per, a.ctypes.data, a.nbytes))
    kv = oh.PagedKv(dk, dv, n_pages, page, nkv, hd)
    seqs = oh.PagedSeqs(exe.upload(ids), exe.upload(np.array([n], np.int32)), 1, 4)
    q = synth.bf16_normal(rng, (nh, hd), 2.0)
    out = exe.alloc((nh, hd), np.uint16)
    ws = exe.alloc(exe.sdpa_paged_workspace(kv, seqs, nh), np.uint8)
    exe.sdpa_paged_decode(kv, seqs, exe.upload(q), out, nh, ws)
    kk = _f64(k).transpose(0, 2, 1, 3).reshape(-1, nkv, hd)[:n]
    vv = _f64(v).transpose(0, 3, 1, 2).reshape(-1, nkv, hd)[:n]
    ref, bound, _, _ = _attend(_f64(q), kk, vv, np.ones(n, bool))
    got = _f64(out.download())
    dk.free()
    dv.free()
    assert np.all(np.abs(got - ref) <= bound)


@pytest.mark.parametrize("page", [16, 64])
def test_bad_ids_lengths_and_slots_are_reported(exe, page):
    """A page id out of range hides its entries, a length past the table is cut, a
    slot out of range gathers nothing; each is reported once."""
    nh, nkv, hd = 32, 4, 128
    rng = np.random.default_rng(23)
    pool = Pool(exe, rng, [5 * page, 3 * page], nkv, hd, page, False, max_pages=5)
    q, q0 = synth.bf16_normal(rng, (2, nh, hd), 2.0), None
    exe_q, out = exe.upload(q), exe.alloc((2, nh, hd), np.uint16)
    seqs = pool.seqs()
    w = np.zeros((2, nkv, 5 * page), np.float32)
    dw = exe.upload(w)
    wt = oh.KvWeight(dw, 2, 5 * page, exe.upload(np.array([0, 9], np.int32)))
    ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, seqs, nh, wt), np.uint8)

    def run(weight=None):
        exe.sdpa_paged_decode(pool.kv, seqs, exe_q, out, nh, ws, weight=weight)
        with pytest.raises(oh.ObsError, match="paged cache") as ei:
            exe.device_status()
        assert ei.value.code == oh.OBS_E_INVALID
        exe.device_status()  # cleared

    run(wt)
    assert np.any(dw.download()[0] != 0) and not np.any(dw.download()[1] != 0)
    for bad in (-1, pool.n_pages, 2**31 - 1):
        table = pool.table.copy()
        table[0, 1] = bad
        pool.dt.upload(table)
        run()
        n = 5 * page
        vis = np.ones(n, bool)
        vis[page:2 * page] = False
        ref, bound, _, _ = _attend(_f64(q[0]), pool.entries(0, "k"), pool.entries(0, "v"), vis)
        assert np.all(np.abs(_f64(out.download())[0] - ref) <= bound)
    pool.dt.upload(pool.table)
    pool.dl.upload(np.array([5 * page + 100, 3 * page], np.int32))
    run()
    ref, bound, _, _ = _attend(_f64(q[0]), pool.entries(0, "k"), pool.entries(0, "v"), np.ones(5 * page, bool))
    assert np.all(np.abs(_f64(out.download())[0] - ref) <= bound)


# ---- prefill ----------------------------------------------------------------

PREFILL = [([1], [1]), ([5, 16, 0, 300], [5, 3, 0, 70]), ([257, 31, 64], [200, 31, 1]), ([0, 3], [2, 9])]


def _prefill_case(exe, shape, lens, new, window, sinks, seed, pad_rows=0, check_rows=None, k_std=1.0):
    nh, nkv, hd, page, f8 = shape
    rng = np.random.default_rng(seed)
    pool = Pool(exe, rng, lens, nkv, hd, page, f8, k_std=k_std)
    rows = np.concatenate([[0], np.cumsum(new)]).astype(int)
    R = int(rows[-1])
    q = synth.bf16_normal(rng, (R + pad_rows, nh, hd), 2.0)
    out = exe.upload(np.full((R + pad_rows, nh, hd), FILL16, np.uint16))
    seqs = pool.seqs(rows, R + pad_rows)
    ws = exe.upload(np.full(exe.sdpa_paged_workspace(pool.kv, seqs, nh, None, window, sinks), 0xFF, np.uint8))
    dq = exe.upload(q)
    call = lambda: exe.sdpa_paged_prefill(pool.kv, seqs, dq, out, nh, ws, window=window, sinks=sinks)
    call()
    exe.device_status()
    raw = out.download()
    got = _f64(raw)
    assert np.all(raw[R:] == FILL16)  # rows behind the last sequence
    for b, (n, t) in enumerate(zip(lens, new)):
        k, v = pool.entries(b, "k"), pool.entries(b, "v")
        for r in (range(t) if check_rows is None else sorted({min(r, t - 1) for r in check_rows})):
            i = n - t + r
            vis = _visible(i, n, window, sinks) if i >= 0 else np.zeros(n, bool)
            ref, bound, _, _ = _attend(_f64(q[rows[b] + r]), k, v, vis)
            g = got[rows[b] + r]
            assert np.all(np.abs(g - ref) <= bound), (b, r, i, np.max(np.abs(g - ref)))
    return call, out, pool


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("lens,new", PREFILL, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_prefill(exe, shape, lens, new, window, sinks):
    """Ragged batches, empty sequences, and sequences shorter than their tokens (zeros)."""
    _prefill_case(exe, shape, lens, new, window, sinks, 29, pad_rows=3)


@pytest.mark.parametrize("shape,lens,new,window", [((32, 4, 128, 32, False), [5000], [40], 0),
                                                   ((32, 4, 128, 16, True), [700, 6000, 90], [130, 5, 90], 0),
                                                   ((32, 8, 64, 64, False), [2000, 1500], [1700, 900], 500),
                                                   ((12, 2, 128, 64, False), [1300], [1300], 0)])
def test_prefill_long(exe, shape, lens, new, window):
    """Few rows over long caches (split and joined) and many rows, at rows of every kind of tile."""
    call, out, _ = _prefill_case(exe, shape, lens, new, window, 4, 31, check_rows=[0, 1, 31, 32, 63, 64, 127, 600, 10**9])
    first = out.download()
    call()
    assert np.array_equal(first, out.download())


@pytest.mark.parametrize("shape", [(32, 4, 128, 16, False), (6, 2, 64, 32, True)], ids=str)
def test_prefill_many_short_prompts_in_parts(exe, shape):
    """More sequences than a wave has lanes, some without rows, some of several tiles, over caches
    long enough to be cut into parts."""
    r = np.random.default_rng(95)
    new = [int(x) for x in r.choice([0, 1, 2, 3, 60], 150, p=[0.3, 0.3, 0.2, 0.15, 0.05])]
    lens = [max(t, int(x)) for t, x in zip(new, r.integers(0, 900, 150))]
    _prefill_case(exe, shape, lens, new, 0, 0, 97, pad_rows=2)
    _prefill_case(exe, shape, lens, new, 200, 3, 99)


@pytest.mark.parametrize("shape,lens", [((32, 4, 128, 32, False), [2000]), ((32, 8, 64, 64, True), [1100]),
                                        ((16, 1, 128, 32, False), [2900]), ((32, 4, 128, 16, True), [900, 1, 650])], ids=str)
def test_prefill_whole_prompts_in_parts(exe, shape, lens):
    """Prompts into an empty cache whose tiles have all lengths: the last ones in parts, the first whole."""
    _prefill_case(exe, shape, lens, lens, 0, 0, 101, check_rows=[0, 30, 47, 48, 300, 511, 700, 1000, 1500, 10**9])


def test_prefill_peaked_scores(exe):
    _prefill_case(exe, (32, 4, 128, 32, False), [300, 65], [129, 65], 0, 0, 37, k_std=30.0)


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2), (90, 40)])
@pytest.mark.parametrize("shape", [(32, 4, 128, 16, False), (16, 16, 64, 32, True), (12, 2, 128, 32, False)], ids=str)
def test_prefill_rows_do_not_meet_hidden_nan(exe, shape, window, sinks):
    """NaN keys and NaN (in bf16 also infinite) values in some entries: rows that do
    not see them are as if they were not there, rows that do are not finite."""
    nh, nkv, hd, page, f8 = shape
    lens, new = [150, 40], [120, 40]
    rows = [0, 120, 160]
    nan_k, nan_v, inf_v = [35, 100], [3, 77, 110], [] if f8 else [60]
    for what in ("k", "v"):
        rng = np.random.default_rng(83)
        pool = Pool(exe, rng, lens, nkv, hd, page, f8)
        clean = {b: (pool.entries(b, "k"), pool.entries(b, "v")) for b in range(2)}
        bad = nan_k if what == "k" else nan_v + inf_v
        for j in bad:
            p, o = pool.table[0, j // page], j % page
            if what == "k":
                pool.k[p, :, o, 5] = 0x7F if f8 else NAN16
            else:
                pool.v[p, :, :, o] = 0x7F if f8 else (0x7F80 if j in inf_v else NAN16)
        pool.up()
        q = synth.bf16_normal(rng, (160, nh, hd), 2.0)
        out = exe.upload(np.full((160, nh, hd), FILL16, np.uint16))
        seqs = pool.seqs(rows)
        ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, seqs, nh, None, window, sinks), np.uint8)
        exe.sdpa_paged_prefill(pool.kv, seqs, exe.upload(q), out, nh, ws, window=window, sinks=sinks)
        exe.device_status()
        got = _f64(out.download())
        for b in range(2):
            k, v = clean[b]
            for r in range(new[b]):
                n, i = lens[b], lens[b] - new[b] + r
                vis = _visible(i, n, window, sinks)
                g = got[rows[b] + r]
                if b == 0 and any(vis[j] for j in bad):
                    assert not np.any(np.isfinite(g)), (what, r)
                    continue
                ref, bound, _, _ = _attend(_f64(q[rows[b] + r]), k, v, vis)
                assert np.all(np.abs(g - ref) <= bound), (what, b, r)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("rows", [[0, 90, 0, 90, 0, 90], [90, 0, 90, 0, 90, 0], [-5, 40, 30, 1000, 7, 2**31 - 1],
                                  [50, 40, 30, 20, 10, -2**31]], ids=str)
def test_prefill_rows_out_of_order_stay_in_the_buffers(exe, rows, long):
    """Row arrays that decrease or leave [0, n_rows] are not a batch: what the rows get is open, but
    the call ends, and nothing beside the output and the workspace changes (in parts and whole)."""
    nh, nkv, hd, page = 32, 4, 128, 16
    rng = np.random.default_rng(57)
    n = 900 if long else 300
    pool = Pool(exe, rng, [n, n - 7, 20, n, 100], nkv, hd, page, False)
    R, guard = 90, 4096
    seqs = pool.seqs(rows, R)
    need = exe.sdpa_paged_workspace(pool.kv, seqs, nh)
    ws = exe.upload(np.full(need + guard, 0xFF, np.uint8))
    q = exe.upload(synth.bf16_normal(rng, (R, nh, hd), 2.0))
    out = exe.upload(np.full((R + 2, nh, hd), FILL16, np.uint16))
    exe.sdpa_paged_prefill(pool.kv, seqs, q, out, nh, ws, ws_bytes=need)
    exe.device_status()
    assert np.all(out.download()[R:] == FILL16) and np.all(ws.download()[need:] == 0xFF)


# ---- append -------------------------------------------------------------------

def _prep_case(exe, shape, lens, new, seed, pos=None, rope_len=9000, pad_rows=0, weight=True, one=False):
    nh, nkv, hd, page, f8 = shape
    rng = np.random.default_rng(seed)
    pool = Pool(exe, rng, lens, nkv, hd, page, f8)
    rows = np.concatenate([[0], np.cumsum(new)]).astype(int)
    R, qd, kd = int(rows[-1]), nh * hd, nkv * hd
    ld = qd + 2 * kd + 8
    x = synth.bf16_normal(rng, (R + pad_rows, ld), 2.0)
    qn, kn = synth.norm_weight(rng, hd), synth.norm_weight(rng, hd)
    dx = exe.upload(x)
    q_out = exe.upload(np.full((R + pad_rows, nh, hd), FILL16, np.uint16))
    cap = pool.max_pages * page
    w0 = rng.random((len(lens), nkv, cap)).astype(np.float32) + 1.0
    dw = exe.upload(w0)
    wt = oh.KvWeight(dw, len(lens), cap) if weight else None
    seqs = pool.seqs(None if one else rows, None if one else R + pad_rows)
    exe.attn_prep_paged(pool.kv, seqs, dx.ptr, dx.ptr + 2 * qd, dx.ptr + 2 * (qd + kd), exe.upload(qn), exe.upload(kn),
                        q_out, nh, EPS, THETA, rope_len, pos=None if pos is None else exe.upload(np.array(pos, np.int32)),
                        weight=wt, q_ld=ld, kv_ld=ld)
    return pool, rows, x, qn, kn, q_out, w0, dw


def _rope64(x, w, pos):
    """(value, bound of the two bf16 roundings and the fp32 angle) of [..., hd] rows."""
    hd = x.shape[-1]
    y = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + EPS) * w
    ang = pos * THETA ** (-np.arange(hd // 2) / (hd // 2))
    c, s = np.cos(ang), np.sin(ang)
    a, b = y[..., :hd // 2], y[..., hd // 2:]
    r = np.concatenate([a * c - b * s, b * c + a * s], -1)
    mix = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)], -1)
    turn = np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)
    pre = 2.0 ** -8 * mix + (2.0 ** -22 * max(pos, 1)) * turn + 2.0 ** -20 * mix  # before the last rounding
    return r, pre


def _check_prep(pool, rows, x, qn, kn, q_out, w0, dw, lens, new, pos=None, rope_len=9000, weight=True):
    nkv, hd, page = pool.nkv, pool.hd, pool.page
    raw = q_out.download()
    nh = raw.shape[1]
    got = _f64(raw)
    k, v, w = pool.dk.download(), pool.dv.download(), dw.download()
    k_ref, v_ref, w_ref = pool.k.copy(), pool.v.copy(), w0.copy()
    R = int(rows[-1])
    assert np.all(raw[R:] == FILL16)
    f = _f64(x)
    for b, (n, t) in enumerate(zip(lens, new)):
        for r in range(t):
            row, e = rows[b] + r, max(n, 0) - t + r
            p = e if pos is None else pos[row]
            if not 0 <= p < rope_len:
                assert np.all(raw[row] == FILL16)
                continue
            ref, pre = _rope64(f[row, :nh * hd].reshape(nh, hd), _f64(qn), p)
            assert np.all(np.abs(got[row] - ref) <= pre + 2.0 ** -8 * (np.abs(ref) + pre)), (b, r)
            if e < 0:
                continue
            pg, o = pool.table[b, e // page], e % page
            ref, pre = _rope64(f[row, nh * hd:(nh + nkv) * hd].reshape(nkv, hd), _f64(kn), p)
            vv = x[row, (nh + nkv) * hd:(nh + 2 * nkv) * hd].reshape(nkv, hd)
            if pool.f8:
                s = pool.ks.astype(np.float64)[:, None]
                lim = pre + 2.0 ** -4 * (np.abs(ref) + pre) + 2.0 ** -10 * s
                val, ref = E4M3[k[pg, :, o]] * s, np.clip(ref, -448 * s, 448 * s)
                assert np.all(np.abs(val - ref) <= lim)
                q = _f64(vv).astype(np.float32) / pool.vs[:, None]  # IEEE division, as the kernel's
                assert np.array_equal(v[pg, :, :, o], _e4m3_bytes(q))
            else:
                assert np.all(np.abs(_f64(k[pg, :, o]) - ref) <= pre + 2.0 ** -8 * (np.abs(ref) + pre))
                assert np.array_equal(v[pg, :, :, o], vv)
            k_ref[pg, :, o], v_ref[pg, :, :, o] = k[pg, :, o], v[pg, :, :, o]
            if weight:
                w_ref[b, :, e] = 0.0
    assert np.array_equal(k, k_ref) and np.array_equal(v, v_ref)  # nothing else was written
    assert np.array_equal(w, w_ref)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_prep(exe, shape):
    lens, new = [40, 3, 0, 17, 200], [40, 3, 0, 1, 130]
    a = _prep_case(exe, shape, lens, new, 41, pad_rows=2)
    exe.device_status()
    _check_prep(*a, lens, new)


@pytest.mark.parametrize("shape", [(32, 4, 128, 16, False), (16, 16, 64, 32, True)], ids=str)
def test_prep_one_token_and_positions(exe, shape):
    """A decode step's rows with positions of their own, one of them outside the
    table's range, an empty sequence among them."""
    lens, new = [1, 0, 33, 500, 16], [1] * 5
    pos = [8999, 7, 9000, 0, 4321]
    a = _prep_case(exe, shape, lens, new, 43, pos=pos, one=True)
    exe.device_status()
    _check_prep(*a, lens, new, pos=pos)


def test_prep_many_sequences(exe):
    """More sequences than a wave has lanes, empty ones between them."""
    rng = np.random.default_rng(47)
    new = rng.integers(0, 4, 150)
    lens = [int(t + rng.integers(0, 40)) for t in new]
    a = _prep_case(exe, (8, 1, 64, 16, False), lens, new, 47, weight=False)
    exe.device_status()
    _check_prep(*a, lens, new, weight=False)


@pytest.mark.parametrize("shape", [(32, 4, 64, 16, False), (8, 1, 128, 32, True), (12, 2, 64, 64, True)], ids=str)
def test_prep_many_rows_of_few_heads(exe, shape):
    """Rows that take one wave each: a count that is no multiple of four, sequences without rows,
    rows behind the last one."""
    lens, new = [700, 5, 0, 480, 9], [600, 3, 0, 480, 9]
    a = _prep_case(exe, shape, lens, new, 103, pad_rows=3)
    exe.device_status()
    _check_prep(*a, lens, new)


def test_prep_equals_the_contiguous_cache(exe):
    """bf16 at head_dim 128: q, keys and values are obs_attn_prep_rows' bit for bit."""
    nh, nkv, hd, page, T, pos0 = 32, 4, 128, 32, 75, 60
    a = _prep_case(exe, (nh, nkv, hd, page, False), [pos0 + T], [T], 53, weight=False)
    pool, _, x, qn, kn, q_out = a[:6]
    ld, ml = x.shape[1], 160
    dx = exe.upload(x)
    kc, vc = exe.zeros((nkv, ml, hd), np.uint16), exe.zeros((nkv, hd, ml), np.uint16)
    exe.attn_prep_rows(dx.ptr, dx.ptr + 2 * nh * hd, dx.ptr + 2 * (nh + nkv) * hd, exe.upload(qn), exe.upload(kn), kc, vc, nh,
                       nkv, hd, ml, EPS, THETA, pos0, T, ld, ld)
    assert np.array_equal(dx.download()[:, :nh * hd].reshape(T, nh, hd), q_out.download())
    j = np.arange(pos0, pos0 + T)
    p, o = pool.table[0, j // page], j % page
    assert np.array_equal(kc.download()[:, j].transpose(1, 0, 2), pool.dk.download()[p, :, o])
    assert np.array_equal(vc.download()[:, :, j].transpose(2, 0, 1), pool.dv.download()[p, :, :, o])


def test_prep_in_place_and_bad_pages(exe):
    """q_out may be q; a row whose page id is out of range appends nothing and is reported."""
    nh, nkv, hd, page = 32, 4, 128, 16
    rng = np.random.default_rng(59)
    pool = Pool(exe, rng, [20, 20], nkv, hd, page, False)
    table = pool.table.copy()
    table[1, 1] = pool.n_pages + 5
    pool.dt.upload(table)
    q, k, v = (synth.bf16_normal(rng, (2, h, hd), 2.0) for h in (nh, nkv, nkv))
    qn, kn = synth.norm_weight(rng, hd), synth.norm_weight(rng, hd)
    dq = exe.upload(q)
    exe.attn_prep_paged(pool.kv, pool.seqs(), dq, exe.upload(k), exe.upload(v), exe.upload(qn), exe.upload(kn), dq, nh, EPS,
                        THETA, 64)
    with pytest.raises(oh.ObsError, match="paged cache"):
        exe.device_status()
    got, after = _f64(dq.download()), pool.dk.download()
    for b in range(2):
        ref, pre = _rope64(_f64(q[b]), _f64(qn), 19)
        assert np.all(np.abs(got[b] - ref) <= pre + 2.0 ** -8 * (np.abs(ref) + pre))
    want = pool.k.copy()
    want[pool.table[0, 1], :, 3] = after[pool.table[0, 1], :, 3]
    assert not np.array_equal(after[pool.table[0, 1], :, 3], pool.k[pool.table[0, 1], :, 3])
    assert np.array_equal(after, want)


@pytest.mark.parametrize("rows", [200, 1101])
@pytest.mark.parametrize("shape", [(32, 4, 64, 16, False), (32, 4, 128, 32, True), (8, 1, 128, 32, False)], ids=str)
def test_prep_of_prompts_in_place(exe, shape, rows):
    """q_out is q, inside one projection's rows: what the call gives with a q_out of its own."""
    nh, nkv, hd, page, f8 = shape
    rng = np.random.default_rng(107)
    lens, ld = [rows + 13], (nh + 2 * nkv) * hd
    x, qn, kn = synth.bf16_normal(rng, (rows, ld), 2.0), synth.norm_weight(rng, hd), synth.norm_weight(rng, hd)
    results = []
    for own in (False, True):
        pool = Pool(exe, np.random.default_rng(109), lens, nkv, hd, page, f8)
        dx, out = exe.upload(x), exe.alloc((rows, ld), np.uint16)
        to = out if own else dx
        exe.attn_prep_paged(pool.kv, pool.seqs([0, rows]), dx.ptr, dx.ptr + 2 * nh * hd, dx.ptr + 2 * (nh + nkv) * hd,
                            exe.upload(qn), exe.upload(kn), to.ptr, nh, EPS, THETA, 2048, q_ld=ld, kv_ld=ld, q_out_ld=ld)
        exe.device_status()
        results.append([to.download()[:, :nh * hd], pool.dk.download(), pool.dv.download()])
    for a, b in zip(*results):
        assert np.array_equal(a, b)
    assert not np.array_equal(results[0][0], x[:, :nh * hd])


# ---- eviction -------------------------------------------------------------------

def _kept(w, n, sinks, recent, budget):
    if n <= budget:
        return np.arange(n)
    j = np.arange(sinks, n - recent)
    x = np.where(np.isnan(w[j]), -np.inf, w[j].astype(np.float64) + 0.0)
    rank = np.lexsort((j, np.isnan(w[j]), -x))  # weight, then NaN behind -inf, then the lowest entry
    mid = np.sort(j[rank[:budget - sinks - recent]])
    return np.concatenate([np.arange(sinks), mid, np.arange(n - recent, n)])


def _evict_case(exe, shape, lens, sinks, recent, budget, seed, weights="normal"):
    nh, nkv, hd, page, f8 = shape
    rng = np.random.default_rng(seed)
    B, dmax = len(lens), -(-budget // page)
    pool = Pool(exe, rng, lens, nkv, hd, page, f8, extra=B * dmax + 2)
    cap = pool.max_pages * page
    w = rng.random((B + 1, nkv, cap)).astype(np.float32)
    if weights == "ties":
        w = rng.integers(0, 3, w.shape).astype(np.float32) * rng.choice([0.0, 1.0, -1.0], w.shape).astype(np.float32)
    elif weights == "wild":
        w = rng.choice(np.array([0.0, -0.0, np.nan, np.inf, -np.inf, 1e-42, -1e-42, 3e38, 1.0], np.float32), w.shape)
    slot = rng.permutation(B + 1)[:B].astype(np.int32)
    dst = pool.free[:B * dmax].reshape(B, dmax).copy()
    dw, kept, new_len = exe.upload(w), exe.upload(np.full((B, nkv, budget), 77, np.int32)), exe.upload(np.full(B, 77, np.int32))
    wd0 = np.full((B, nkv, budget + 3), 5.5, np.float32)
    dwd = exe.upload(wd0)
    exe.kv_evict(pool.kv, pool.seqs(), oh.KvWeight(dw, B + 1, cap, exe.upload(slot)), exe.upload(dst), dmax,
                 oh.KvWeight(dwd, B, budget + 3), sinks, recent, budget, kept, new_len)
    exe.device_status()
    gk, gl, k, v, gw = kept.download(), new_len.download(), pool.dk.download(), pool.dv.download(), dwd.download()
    k_ref, v_ref, w_ref = pool.k.copy(), pool.v.copy(), wd0.copy()
    for b, n in enumerate(lens):
        assert gl[b] == min(n, budget)
        for h in range(nkv):
            ref = _kept(w[slot[b], h], n, sinks, recent, budget)
            m = len(ref)
            assert np.array_equal(gk[b, h, :m], ref), (b, h)
            assert np.all(gk[b, h, m:] == -1)
            e = np.arange(m)
            sp, so, dp, do = pool.table[b, ref // page], ref % page, dst[b, e // page], e % page
            k_ref[dp, h, do] = pool.k[sp, h, so]
            v_ref[dp, h, :, do] = pool.v[sp, h, :, so]
            w_ref[b, h, :m] = w[slot[b], h, ref]
    assert np.array_equal(k, k_ref) and np.array_equal(v, v_ref)
    assert np.array_equal(gw.view(np.uint32), w_ref.view(np.uint32))


@pytest.mark.parametrize("weights", ["normal", "ties", "wild"])
@pytest.mark.parametrize("sinks,recent,budget", [(4, 20, 50), (0, 0, 33), (10, 54, 64), (0, 1, 1), (3, 0, 257)])
@pytest.mark.parametrize("shape", [(32, 4, 128, 16, False), (16, 2, 64, 64, True)], ids=str)
def test_evict(exe, shape, sinks, recent, budget, weights):
    lens = [0, 1, budget - 1, budget, budget + 1, 300, 1024, 2500]
    _evict_case(exe, shape, lens, sinks, recent, budget, 61, weights)


def test_evict_long(exe):
    _evict_case(exe, (8, 2, 128, 32, False), [70001, 33000], 4, 500, 3000, 67)
    _evict_case(exe, (8, 2, 64, 256, True), [50000], 0, 0, 25000, 71, "ties")


@pytest.mark.parametrize("weights", ["normal", "ties"])
@pytest.mark.parametrize("shape", [(32, 4, 128, 16, False), (32, 4, 128, 32, True), (16, 4, 64, 64, False), (16, 4, 64, 16, True)],
                         ids=str)
def test_evict_many(exe, shape, weights):
    """Enough entries for the copy's large groups."""
    _evict_case(exe, shape, [2500, 1101, 1100, 60, 1900, 2048, 1333, 0], 4, 100, 1100, 83, weights)


def test_weight_rows_of_odd_strides(exe):
    """Weight rows that begin at any 4-byte address: gathered, cleared and evicted as in aligned ones."""
    nh, nkv, hd, page, lens = 32, 4, 128, 32, [900, 37, 500]
    B, budget = len(lens), 130
    results = []
    for pad, off in ((0, 0), (3, 1)):
        rng = np.random.default_rng(113)
        pool = Pool(exe, rng, lens, nkv, hd, page, False, extra=B * 5)
        cap = pool.max_pages * page
        w = rng.random((B, nkv, cap)).astype(np.float32)
        flat = np.zeros(off + B * nkv * (cap + pad), np.float32)
        flat[off:].reshape(B, nkv, cap + pad)[:, :, :cap] = w
        dw = exe.upload(flat)
        wt = oh.KvWeight(dw.ptr + 4 * off, B, cap + pad)
        q, out = exe.upload(synth.bf16_normal(rng, (B, nh, hd), 2.0)), exe.alloc((B, nh, hd), np.uint16)
        ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, pool.seqs(), nh, wt), np.uint8)
        exe.sdpa_paged_decode(pool.kv, pool.seqs(), q, out, nh, ws, weight=wt)
        kept, new_len = exe.alloc((B, nkv, budget), np.int32), exe.alloc(B, np.int32)
        dwd = exe.alloc(off + B * nkv * (budget + pad), np.float32)
        exe.kv_evict(pool.kv, pool.seqs(), wt, exe.upload(pool.free[:B * 5].reshape(B, 5).copy()), 5,
                     oh.KvWeight(dwd.ptr + 4 * off, B, budget + pad), 2, 30, budget, kept, new_len)
        exe.device_status()
        after = dw.download()[off:].reshape(B, nkv, cap + pad)
        assert not np.any(after[:, :, cap:]) and not np.any(after[1, :, 37:cap] != w[1, :, 37:])
        gw = dwd.download()[off:].reshape(B, nkv, budget + pad)
        results.append([out.download(), after[:, :, :cap], kept.download(), gw[[0, 2], :, :budget], gw[1, :, :37], pool.dk.download()])
    for x, y in zip(*results):
        assert np.array_equal(x, y)


def test_more_kv_heads_than_threads(exe):
    """300 kv heads: loops over heads go round more than once."""
    shape = (300, 300, 64, 16, False)
    _decode_case(exe, shape, [40, 0, 17], 0, 0, True, 87)
    _prefill_case(exe, shape, [40, 9], [11, 9], 0, 0, 87)
    args = _prep_case(exe, shape, [40, 9], [11, 9], 87)
    _check_prep(*args, [40, 9], [11, 9])
    _evict_case(exe, shape, [70, 20], 2, 3, 30, 87)


def test_evict_reports_bad_pages_and_slots(exe):
    nkv, hd, page, n, budget = 2, 64, 16, 64, 32
    rng = np.random.default_rng(73)
    pool = Pool(exe, rng, [n, n], nkv, hd, page, False, extra=6)
    w = np.zeros((2, nkv, pool.max_pages * page), np.float32)
    kept, new_len = exe.alloc((2, nkv, budget), np.int32), exe.alloc(2, np.int32)
    dst = pool.free[:4].reshape(2, 2).copy()
    dst[1, 0] = -5
    table = pool.table.copy()
    table[0, 0] = 10**6
    pool.dt.upload(table)
    dw, dwd = exe.upload(w), exe.upload(np.full((2, nkv, budget), 5.5, np.float32))
    exe.kv_evict(pool.kv, pool.seqs(), oh.KvWeight(dw, 2, w.shape[2]), exe.upload(dst), 2,
                 oh.KvWeight(dwd, 2, budget, exe.upload(np.array([0, 2], np.int32))), 0, 0, budget, kept, new_len)
    with pytest.raises(oh.ObsError, match="paged cache"):
        exe.device_status()
    assert np.array_equal(kept.download(), np.tile(np.arange(budget, dtype=np.int32), (2, nkv, 1)))  # all tied: the first
    k, ref = pool.dk.download(), pool.k.copy()
    ref[dst[0, 0]] = 0  # the source page that is not there
    ref[dst[0, 1]] = pool.k[pool.table[0, 1]]
    ref[dst[1, 1]] = pool.k[pool.table[1, 1]]  # and the destination one is skipped
    assert np.array_equal(k, ref)
    gw = dwd.download()
    assert np.all(gw[0] == 0.0) and np.all(gw[1] == 5.5)
