"""The paged cache in 4 bits (OBS_KV_Q4) on the GPU: append, decode, prompts and
eviction against plain float64 restatements.

Pools are filled with a pattern whose scales and biases are NaN but for the entries
that a call may see, so a read outside shows.

Bars. Decode takes the nibbles as they are: a score's products are exact, its fp32
sums are off by 2^-24 of what they add, once an addition (64 dims, and a few steps
to join the groups), and what they add is s (16 + q) |Q| and |b - 16 s| |Q|. P s
enters the value product in bf16 (2^-8 of sum p s |q - 8|, the middle being split
off), the rest of an output is fp32, off by 2^-24 of sum p s (40 + q) + p |b + 8 s| an
addition; the output is rounded once (2^-8 of it). Prompts take entries rounded to
fp16, which the reference does too, and P in fp16 (2^-11 of sum p |v|, and half its
least step, 2^-25, of every |v| where that is more); scores and the output as above."""
import numpy as np
import pytest

import obsidian_hip as oh
from obsidian_hip import synth
from test_gpu_paged import (EPS, FILL16, LENS, NAN16, PREFILL, THETA, WINDOWS, _f64, _kept, _visible)

pytestmark = pytest.mark.gpu

NAN_PAR = 0x7FC17FC1
GROUP = 64


def _bf(x):
    """float64 -> nearest float32 -> nearest bf16, as float64."""
    return synth.bf16_bits_to_f32(synth.f32_to_bf16_bits(np.asarray(x, np.float32))).astype(np.float64)


def quantize(x):
    """x [..., hd] -> nibbles [..., hd], scale and bias (bf16 values) [..., hd / 64]."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    s, b = _bf((g.max(-1) - g.min(-1)) / 15), _bf(g.min(-1))
    q = np.clip(np.rint((g - b[..., None]) / np.where(s > 0, s, 1)[..., None]), 0, 15)
    return np.where(s[..., None] > 0, q, 0).reshape(x.shape).astype(np.uint8), s, b


def par_words(s, b):
    return synth.f32_to_bf16_bits(s.astype(np.float32)).astype(np.uint32) | \
        synth.f32_to_bf16_bits(b.astype(np.float32)).astype(np.uint32) << 16


class Side:
    """Keys or values of a pool on the host, in the layout of the header: bytes [n_pages, nkv, page * 9 hd / 16]."""

    def __init__(self, n_pages, nkv, hd, page, values):
        self.hd, self.page, self.values = hd, page, values
        self.raw = np.full((n_pages, nkv, page * (hd // 2 + hd // 16)), 0xA5, np.uint8)
        cut = page * hd // 2
        self.data = self.raw[..., :cut].reshape(n_pages, nkv, *((hd // 2, page) if values else (page, hd // 2)))
        if values:
            self.data = self.data.swapaxes(2, 3)
        assert np.shares_memory(self.data, self.raw)
        self.par = self.raw.view(np.uint32)[..., cut // 4:].reshape(n_pages, nkv, hd // GROUP, page).swapaxes(2, 3)
        assert np.shares_memory(self.par, self.raw)
        self.par[...] = NAN_PAR

    def put(self, p, o, x):
        """Entries x [n, nkv, hd] to pages p at o."""
        q, s, b = quantize(x)
        self.data[p, :, o] = q[..., :self.hd // 2] | q[..., self.hd // 2:] << 4
        self.par[p, :, o] = par_words(s, b)

    def get(self, p, o, raw=None):
        """(q, s, b) of entries, q [n, nkv, hd] and s, b spread over the dims; float64."""
        if raw is not None:
            other = Side.__new__(Side)
            other.hd, other.page, other.values = self.hd, self.page, self.values
            n_pages, nkv = raw.shape[:2]
            cut = self.page * self.hd // 2
            other.data = raw[..., :cut].reshape(n_pages, nkv, *((self.hd // 2, self.page) if self.values else (self.page, self.hd // 2)))
            other.data = other.data.swapaxes(2, 3) if self.values else other.data
            other.par = np.ascontiguousarray(raw[..., cut:]).view(np.uint32).reshape(n_pages, nkv, self.hd // GROUP, self.page).swapaxes(2, 3)
            return other.get(p, o)
        by, w = self.data[p, :, o], self.par[p, :, o]
        q = np.concatenate([by & 15, by >> 4], -1).astype(np.float64)
        s, b = _f64((w & 0xFFFF).astype(np.uint16)), _f64((w >> 16).astype(np.uint16))
        return q, np.repeat(s, GROUP, -1), np.repeat(b, GROUP, -1)


class Pool:
    """Sequences of lengths `lens` in shuffled pages; hidden[b]: entries of b that hold the pattern."""

    def __init__(self, exe, rng, lens, nkv, hd, page, extra=3, hidden=None, k_std=1.0, max_pages=None):
        self.exe, self.lens, self.nkv, self.hd, self.page = exe, list(lens), nkv, hd, page
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
        self.k, self.v = Side(self.n_pages, nkv, hd, page, False), Side(self.n_pages, nkv, hd, page, True)
        gain = np.exp(0.5 * rng.standard_normal((nkv, hd)))
        for b in range(B):
            j = np.arange(max(lens[b], 0))
            if hidden is not None:
                j = j[~np.isin(j, hidden[b])]
            p, o = self.table[b, j // page], j % page
            self.k.put(p, o, rng.standard_normal((len(j), nkv, hd)) * gain * k_std)
            self.v.put(p, o, rng.standard_normal((len(j), nkv, hd)) + 0.5)
        self.up()

    def up(self):
        e = self.exe
        self.dk, self.dv, self.dt = e.upload(self.k.raw), e.upload(self.v.raw), e.upload(self.table)
        self.dl = e.upload(np.array(self.lens, np.int32))
        self.kv = oh.PagedKv(self.dk, self.dv, self.n_pages, self.page, self.nkv, self.hd, oh.KV_Q4)

    def seqs(self, rows=None, n_rows=None):
        B = len(self.lens)
        if rows is None:
            return oh.PagedSeqs(self.dt, self.dl, B, self.max_pages)
        return oh.PagedSeqs(self.dt, self.dl, B, self.max_pages, n_rows or int(rows[-1]),
                            self.exe.upload(np.array(rows, np.int32)))

    def parts(self, b, what):
        j = np.arange(max(self.lens[b], 0))
        return (self.k if what == "k" else self.v).get(self.table[b, j // self.page], j % self.page)


def _attend4(q, kparts, vparts, vis):
    """q [nh, hd] over entries of (nibbles, scales, biases) -> (out, bound, p, relative error of p)."""
    nh, hd = q.shape
    nkv = kparts[0].shape[1]
    per = nh // nkv
    out, bound = np.zeros((nh, hd)), np.zeros((nh, hd))
    p_all, err_all = np.zeros((nh, len(vis))), np.zeros(nh)
    idx = np.flatnonzero(vis)
    if len(idx) == 0:
        return out, bound, p_all, err_all
    n = len(idx)
    for h in range(nh):
        kq, ks, kb = (x[idx, h // per] for x in kparts)
        vq, vs, vb = (x[idx, h // per] for x in vparts)
        s = (kq * ks + kb) @ q[h] / np.sqrt(hd)
        e = np.exp(s - s.max())
        p = e / e.sum()
        mag = np.max((ks * (16 + kq) + np.abs(kb - 16 * ks)) @ np.abs(q[h])) / np.sqrt(hd)
        err = 2 * (72 * 2.0 ** -24 * mag + 2.0 ** -21 * np.max(np.abs(s)) + 2.0 ** -20)
        v = vq * vs + vb
        out[h] = p @ v
        fp32 = (n + 16) * 2.0 ** -24 * (p @ (vs * (40 + vq) + np.abs(vb + 8 * vs)))
        bound[h] = 1.01 * 2.0 ** -8 * (p @ (vs * np.abs(vq - 8))) + err * (p @ np.abs(v)) + fp32 + \
            2.0 ** -8 * np.abs(out[h]) + 1e-30
        p_all[h, idx], err_all[h] = p, err
    return out, bound, p_all, err_all


# n_heads, n_kv, head_dim, page
SHAPES = [(32, 4, 128, 16), (32, 4, 128, 64), (16, 16, 64, 32), (12, 2, 128, 32), (16, 1, 64, 256), (8, 8, 128, 128),
          (10, 2, 64, 16)]


def _decode_case(exe, shape, lens, window, sinks, weight, seed, k_std=1.0, q_ld=0):
    nh, nkv, hd, page = shape
    rng = np.random.default_rng(seed)
    hidden = [np.flatnonzero(~_visible(n - 1, max(n, 0), window, sinks)) for n in lens]
    pool = Pool(exe, rng, lens, nkv, hd, page, hidden=hidden, k_std=k_std)
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
    dq = exe.upload(q)
    call = lambda: exe.sdpa_paged_decode(pool.kv, seqs, dq, out, nh, ws, window=window, sinks=sinks, weight=wt, q_ld=ld)
    call()
    exe.device_status()
    got, wgot = _f64(out.download()), dw.download().astype(np.float64)
    wref, werr = w0.astype(np.float64), np.zeros(w0.shape)
    for b, n in enumerate(lens):
        n = max(n, 0)
        ref, bound, p, err = _attend4(_f64(q[b, :nh * hd]).reshape(nh, hd), pool.parts(b, "k"), pool.parts(b, "v"),
                                      _visible(n - 1, n, window, sinks))
        bad = ~(np.abs(got[b] - ref) <= bound)
        assert not np.any(bad), (b, n, np.max(np.abs(got[b] - ref)), np.max(bound))
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
@pytest.mark.parametrize("shape,lens", [((32, 4, 128, 32), [9000]), ((8, 1, 128, 16), [20001, 40]),
                                        ((32, 8, 64, 64), [1 + 37 * i for i in range(130)]),
                                        ((32, 4, 128, 16), [1700, 3, 900, 0, 64, 33, 1300, 100, 5]),
                                        ((32, 4, 128, 64), [40, 512, 1, 300] * 8)])
def test_decode_split(exe, shape, lens, weight):
    """Long sequences over many workgroups, and more sequences than a wave has lanes."""
    call, out, _ = _decode_case(exe, shape, lens, 0, 0, weight, 11)
    first = out.download()
    call()
    assert np.array_equal(first, out.download())  # the same call, the same bits


def test_decode_peaked_scores_and_strides(exe):
    _decode_case(exe, (32, 4, 128, 32), [777, 64], 0, 0, True, 13, k_std=30.0, q_ld=32 * 128 + 64)
    _decode_case(exe, (16, 4, 64, 32), [777, 64], 100, 2, False, 17, k_std=30.0, q_ld=16 * 64 + 8)


def test_decode_offsets_past_32_bits(exe):
    """A pool of more than 4 GiB a side, the sequence in its last pages."""
    nh, nkv, hd, page = 32, 4, 128, 256
    per = nkv * page * 72
    n_pages = (1 << 32) // per + 40
    rng = np.random.default_rng(19)
    dk, dv = exe.alloc(n_pages * per, np.uint8), exe.alloc(n_pages * per, np.uint8)
    n = 1000
    ids = np.array([n_pages - 1, n_pages - 3, n_pages - 2, n_pages - 7], np.int32)
    small = Pool(exe, rng, [n], nkv, hd, page, extra=0)
    for i, p in enumerate(ids):
        for d, side in ((dk, small.k), (dv, small.v)):
            a = np.ascontiguousarray(side.raw[small.table[0, i]])
            exe._check(oh.lib().obs_upload(exe.ctx, d.ptr + int(p) * per, a.ctypes.data, a.nbytes))
    kv = oh.PagedKv(dk, dv, n_pages, page, nkv, hd, oh.KV_Q4)
    seqs = oh.PagedSeqs(exe.upload(ids), exe.upload(np.array([n], np.int32)), 1, 4)
    q = synth.bf16_normal(rng, (nh, hd), 2.0)
    out = exe.alloc((nh, hd), np.uint16)
    ws = exe.alloc(exe.sdpa_paged_workspace(kv, seqs, nh), np.uint8)
    exe.sdpa_paged_decode(kv, seqs, exe.upload(q), out, nh, ws)
    ref, bound, _, _ = _attend4(_f64(q), small.parts(0, "k"), small.parts(0, "v"), np.ones(n, bool))
    got = _f64(out.download())
    dk.free()
    dv.free()
    assert np.all(np.abs(got - ref) <= bound)


@pytest.mark.parametrize("page", [16, 32, 64])
def test_decode_parts_of_many_blocks(exe, page):
    """So many entries in all that a wave takes more than 64 blocks of a part: 600 sequences over the same pages."""
    nh, nkv, hd, n, B = 8, 1, 64, 30011, 600
    rng = np.random.default_rng(47)
    pool = Pool(exe, rng, [n], nkv, hd, page)
    table = exe.upload(np.repeat(pool.table, B, 0))
    seqs = oh.PagedSeqs(table, exe.upload(np.full(B, n, np.int32)), B, pool.max_pages)
    q = synth.bf16_normal(rng, (B, nh, hd), 2.0)
    dq, out = exe.upload(q), exe.upload(np.full((B, nh, hd), FILL16, np.uint16))
    ws = exe.upload(np.full(exe.sdpa_paged_workspace(pool.kv, seqs, nh), 0xFF, np.uint8))
    exe.sdpa_paged_decode(pool.kv, seqs, dq, out, nh, ws)
    exe.device_status()
    got = _f64(out.download())
    assert np.all(np.isfinite(got))
    for b in (0, 1, 299, B - 1):
        ref, bound, _, _ = _attend4(_f64(q[b]), pool.parts(0, "k"), pool.parts(0, "v"), np.ones(n, bool))
        assert np.all(np.abs(got[b] - ref) <= bound), b


@pytest.mark.parametrize("page", [16, 64])
def test_decode_bad_pages(exe, page):
    nh, nkv, hd = 32, 4, 128
    rng = np.random.default_rng(23)
    pool = Pool(exe, rng, [5 * page, 3 * page], nkv, hd, page, max_pages=5)
    q = synth.bf16_normal(rng, (2, nh, hd), 2.0)
    dq, out = exe.upload(q), exe.alloc((2, nh, hd), np.uint16)
    seqs = pool.seqs()
    ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, seqs, nh), np.uint8)
    for bad in (-1, pool.n_pages):
        table = pool.table.copy()
        table[0, 1] = bad
        pool.dt.upload(table)
        exe.sdpa_paged_decode(pool.kv, seqs, dq, out, nh, ws)
        with pytest.raises(oh.ObsError, match="paged cache"):
            exe.device_status()
        vis = np.ones(5 * page, bool)
        vis[page:2 * page] = False
        ref, bound, _, _ = _attend4(_f64(q[0]), pool.parts(0, "k"), pool.parts(0, "v"), vis)
        assert np.all(np.abs(_f64(out.download())[0] - ref) <= bound)


# ---- prompts ------------------------------------------------------------------

def _f16(x):
    """float64 -> nearest float32 -> nearest fp16, as float64."""
    with np.errstate(over="ignore"):
        return np.asarray(x, np.float32).astype(np.float16).astype(np.float64)


def _attend16(q, k, v, vis):
    """q [nh, hd], k, v [n, nkv, hd] -> (out, bound)."""
    nh, hd = q.shape
    per = nh // k.shape[1]
    out, bound = np.zeros((nh, hd)), np.zeros((nh, hd))
    idx = np.flatnonzero(vis)
    if len(idx) == 0:
        return out, bound
    for h in range(nh):
        kk, vv = k[idx, h // per], v[idx, h // per]
        s = kk @ q[h] / np.sqrt(hd)
        e = np.exp(s - s.max())
        p = e / e.sum()
        mag = np.max(np.abs(kk) @ np.abs(q[h])) / np.sqrt(hd)
        err = 2 * (hd * 2.0 ** -24 * mag + 2.0 ** -21 * np.max(np.abs(s)) + 2.0 ** -20)
        out[h] = p @ vv
        A = p @ np.abs(vv)
        # p is at least 1 / n of its largest: the least step is taken of that, in numerator and sum
        bound[h] = 1.01 * (2 * 2.0 ** -11 + err) * A + 2.0 ** -24 * p.max() * (np.sum(np.abs(vv), 0) + len(idx) * A) + \
            2.0 ** -8 * np.abs(out[h]) + 1e-30
    return out, bound


def _prefill_case(exe, shape, lens, new, window, sinks, seed, pad_rows=0, check_rows=None, k_std=1.0, q_std=2.0):
    nh, nkv, hd, page = shape
    rng = np.random.default_rng(seed)
    pool = Pool(exe, rng, lens, nkv, hd, page, k_std=k_std)
    rows = np.concatenate([[0], np.cumsum(new)]).astype(int)
    R = int(rows[-1])
    q = synth.bf16_normal(rng, (R + pad_rows, nh, hd), q_std)
    out = exe.upload(np.full((R + pad_rows, nh, hd), FILL16, np.uint16))
    seqs = pool.seqs(rows, R + pad_rows)
    ws = exe.upload(np.full(exe.sdpa_paged_workspace(pool.kv, seqs, nh, None, window, sinks), 0xFF, np.uint8))
    dq = exe.upload(q)
    call = lambda: exe.sdpa_paged_prefill(pool.kv, seqs, dq, out, nh, ws, window=window, sinks=sinks)
    call()
    exe.device_status()
    raw = out.download()
    got = _f64(raw)
    assert np.all(raw[R:] == FILL16)
    for b, (n, t) in enumerate(zip(lens, new)):
        k, v = (_f16(x[0] * x[1] + x[2]) for x in (pool.parts(b, "k"), pool.parts(b, "v")))
        for r in (range(t) if check_rows is None else sorted({min(r, t - 1) for r in check_rows})):
            i = n - t + r
            vis = _visible(i, n, window, sinks) if i >= 0 else np.zeros(n, bool)
            ref, bound = _attend16(_f64(q[rows[b] + r]), k, v, vis)
            g = got[rows[b] + r]
            assert np.all(np.abs(g - ref) <= bound), (b, r, i, np.max(np.abs(g - ref)))
    return call, out, pool


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("lens,new", PREFILL, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_prefill(exe, shape, lens, new, window, sinks):
    _prefill_case(exe, shape, lens, new, window, sinks, 29, pad_rows=3)


@pytest.mark.parametrize("shape,lens,new,window", [((32, 4, 128, 32), [5000], [40], 0), ((8, 1, 128, 16), [2500], [2500], 0),
                                                   ((32, 8, 64, 64), [3000, 70], [1500, 70], 900),
                                                   ((32, 4, 128, 128), [600, 1], [600, 1], 0),
                                                   ((16, 1, 64, 16), [4000, 333, 1200], [5, 333, 400], 0)])
def test_prefill_long(exe, shape, lens, new, window):
    call, out, _ = _prefill_case(exe, shape, lens, new, window, 4, 31, check_rows=[0, 1, 37, 200, 599, 1100, 2499])
    first = out.download()
    call()
    assert np.array_equal(first, out.download())


def test_prefill_peaked_scores(exe):
    _prefill_case(exe, (32, 4, 128, 32), [300], [300], 0, 0, 33, k_std=30.0)


@pytest.mark.parametrize("q_std", [1e-30, 3e4, 1e30])
def test_prefill_queries_of_any_size(exe, q_std):
    """Queries keep bf16's range (they are brought into fp16's by a power of two a head)."""
    _prefill_case(exe, (8, 2, 128, 16), [70], [70], 0, 0, 35, q_std=q_std, k_std=min(1.0, 1.0 / q_std))


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2), (90, 40)])
@pytest.mark.parametrize("shape", [(32, 4, 128, 16), (16, 16, 64, 32), (12, 2, 128, 32)], ids=str)
def test_hidden_entries_that_are_not_finite(exe, shape, window, sinks):
    """Values whose scale is NaN or infinite reach the rows that see them, and no others, in prompts and steps."""
    nh, nkv, hd, page = shape
    rng = np.random.default_rng(37)
    n, t = 200, 130
    pool = Pool(exe, rng, [n], nkv, hd, page)
    bad = {90: 0x00007FC1, 140: 0x3F807F80, 171: 0x7F803F80}  # NaN scale; infinite scale; infinite bias
    j = np.array(list(bad))
    for e, word in bad.items():
        pool.v.par[pool.table[0, e // page], :, e % page] = word
    pool.up()
    q = synth.bf16_normal(rng, (t, nh, hd), 2.0)
    out = exe.alloc((t, nh, hd), np.uint16)
    seqs = pool.seqs([0, t])
    ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, seqs, nh, None, window, sinks), np.uint8)
    exe.sdpa_paged_prefill(pool.kv, seqs, exe.upload(q), out, nh, ws, window=window, sinks=sinks)
    got = _f64(out.download())
    one = pool.seqs()
    out1 = exe.alloc((1, nh, hd), np.uint16)
    ws1 = exe.alloc(exe.sdpa_paged_workspace(pool.kv, one, nh, None, window, sinks), np.uint8)
    exe.sdpa_paged_decode(pool.kv, one, exe.upload(q[-1:]), out1, nh, ws1, window=window, sinks=sinks)
    step = _f64(out1.download())
    with np.errstate(invalid="ignore"):
        k, v = (_f16(x[0] * x[1] + x[2]) for x in (pool.parts(0, "k"), pool.parts(0, "v")))
    v[j] = 0.0
    for r in range(t):
        vis = _visible(n - t + r, n, window, sinks)
        if np.any(vis[j]):
            assert not np.any(np.isfinite(got[r])), r
        else:
            ref, bound = _attend16(_f64(q[r]), k, v, vis)
            assert np.all(np.abs(got[r] - ref) <= bound), r
    assert np.any(np.isfinite(step)) != np.any(_visible(n - 1, n, window, sinks)[j])


# ---- append -------------------------------------------------------------------

def _rope(x, w, pos):
    """Normed and rotated x, and what fp32 may be off (the norm and a few products; angles are formed in double)."""
    hd = x.shape[-1]
    y = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + EPS) * w
    ang = pos * THETA ** (-np.arange(hd // 2) / (hd // 2))
    c, s = np.cos(ang), np.sin(ang)
    a, b = y[..., :hd // 2], y[..., hd // 2:]
    r = np.concatenate([a * c - b * s, b * c + a * s], -1)
    turn = np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)
    return r, 2.0 ** -20 * turn


def _check_appended(side, raw, p, o, ref, off):
    """Stored entries against values ref [n, nkv, hd] that the kernel knows to within off."""
    q, s, b = side.get(p, o, raw)
    g = ref.reshape(*ref.shape[:-1], -1, GROUP)
    e = np.max(off.reshape(g.shape), -1)
    lo, hi = g.min(-1), g.max(-1)
    sg, bg = s[..., ::GROUP], b[..., ::GROUP]
    assert np.all(np.abs(bg - lo) <= 2.0 ** -8 * np.abs(lo) + e)
    assert np.all(np.abs(sg - (hi - lo) / 15) <= 2.0 ** -8 * (hi - lo) / 15 + e)
    want = (ref - b) / np.where(s > 0, s, 1)
    slack = 0.5 + off / np.where(s > 0, s, 1) + 2.0 ** -20 * np.abs(want)
    near = np.abs(q - np.clip(want, 0, 15)) <= slack
    assert np.all(near | (s == 0)) and np.all(q[s == 0] == 0)


def _append_case(exe, shape, lens, new, seed, one=False, weight=True, pad_rows=0, pos=None):
    nh, nkv, hd, page = shape
    rng = np.random.default_rng(seed)
    pool = Pool(exe, rng, lens, nkv, hd, page)
    rows = np.concatenate([[0], np.cumsum(new)]).astype(int)
    R = int(rows[-1])
    qd, kd = nh * hd, nkv * hd
    ld = qd + 2 * kd
    x = synth.bf16_normal(rng, (R + pad_rows, ld), 2.0)
    qn, kn = synth.norm_weight(rng, hd), synth.norm_weight(rng, hd)
    dx, q = exe.upload(x), exe.upload(np.full((R + pad_rows, nh, hd), FILL16, np.uint16))
    cap = pool.max_pages * page
    dw = exe.upload(np.ones((len(lens), nkv, cap), np.float32))
    seqs = pool.seqs() if one else pool.seqs(rows, R + pad_rows)
    exe.attn_prep_paged(pool.kv, seqs, dx.ptr, dx.ptr + 2 * qd, dx.ptr + 2 * (qd + kd), exe.upload(qn), exe.upload(kn), q, nh,
                        EPS, THETA, 9000, weight=oh.KvWeight(dw, len(lens), cap) if weight else None, q_ld=ld, kv_ld=ld,
                        pos=None if pos is None else exe.upload(np.array(pos, np.int32)))
    exe.device_status()
    raw_k, raw_v, w, got_q = pool.dk.download(), pool.dv.download(), dw.download(), q.download()
    assert np.all(got_q[R:] == FILL16)
    xf = _f64(x)
    keep_k, keep_v = np.ones(raw_k.shape, bool), np.ones(raw_v.shape, bool)
    for b, (n, t) in enumerate(zip(lens, new)):
        for r in range(t):
            i = n - t + r
            if i < 0:
                continue
            row = rows[b] + r
            at = i if pos is None else pos[row]
            k, off = _rope(xf[row, qd:qd + kd].reshape(nkv, hd), _f64(kn), at)
            want, qoff = _rope(xf[row, :qd].reshape(nh, hd), _f64(qn), at)
            assert np.all(np.abs(_f64(got_q[row]) - want) <= 2.0 ** -8 * np.abs(want) + 1.01 * qoff)  # rounded once
            v = xf[row, qd + kd:].reshape(nkv, hd)
            p, o = pool.table[b, i // page:i // page + 1], np.array([i % page])
            _check_appended(pool.k, raw_k, p, o, k[None], off[None])
            _check_appended(pool.v, raw_v, p, o, v[None], np.zeros((1, nkv, hd)))
            if weight:
                assert np.all(w[b, :, i] == 0.0)
            for keep, side in ((keep_k, pool.k), (keep_v, pool.v)):
                d = keep[p[0], :, :page * hd // 2].reshape(nkv, *((hd // 2, page) if side.values else (page, hd // 2)))
                (d[:, :, o[0]] if side.values else d[:, o[0]])[...] = False
                g = keep[p[0], :, page * hd // 2:].reshape(nkv, hd // GROUP, page, 4)
                g[:, :, o[0]] = False
                keep[p[0], :, :page * hd // 2] = d.reshape(nkv, -1)
                keep[p[0], :, page * hd // 2:] = g.reshape(nkv, -1)
    assert np.array_equal(raw_k[keep_k], pool.k.raw[keep_k]) and np.array_equal(raw_v[keep_v], pool.v.raw[keep_v])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_append(exe, shape):
    """Ragged prompts into pages that hold other entries; every other byte stays."""
    _append_case(exe, shape, [5, 16, 0, 300, 2, 70], [5, 3, 0, 70, 4, 65], 41, pad_rows=2)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_append_one_token(exe, shape):
    _append_case(exe, shape, [1, 300, 17, 0, 64], [1, 1, 1, 1, 1], 43, one=True)


@pytest.mark.parametrize("shape", [(32, 4, 64, 16), (8, 1, 128, 32), (12, 2, 64, 64)], ids=str)
def test_append_many_rows_of_few_heads(exe, shape):
    """From 1,024 rows on few heads take a wave a row."""
    _append_case(exe, shape, [900, 333], [800, 333], 47, weight=False)


def test_append_positions(exe):
    """Keys at positions of the caller's own."""
    _append_case(exe, (32, 4, 128, 32), [40, 7], [9, 7], 53, pos=[100 + 3 * i for i in range(16)])


@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("nkv,hd", [(4, 128), (3, 64)])
def test_append_odd_groups(exe, nkv, hd, one):
    """Groups of one value, of zeros, with NaN or infinities, at the ends of the range."""
    nh, page, cases = nkv, 16, 7
    rng = np.random.default_rng(59)
    pool = Pool(exe, rng, [1] * cases, nkv, hd, page)
    v = rng.standard_normal((cases, nkv, hd)).astype(np.float32)
    v[0] = 3.0
    v[1] = 0.0
    v[2, :, 5] = np.nan
    v[3, :, 7] = np.inf
    v[4, :, 9] = -np.inf
    v[5] = np.where(np.arange(hd) % 2, 3e38, -3e38)
    v[6] *= 1e-38
    x = np.zeros((cases, 3 * nkv * hd), np.uint16)
    x[:, :2 * nkv * hd] = synth.bf16_normal(rng, (cases, 2 * nkv * hd), 1.0)
    x[:, 2 * nkv * hd:] = synth.f32_to_bf16_bits(v.reshape(cases, -1))
    dx, q = exe.upload(x), exe.alloc((cases, nh, hd), np.uint16)
    seqs = pool.seqs() if one else pool.seqs(np.arange(cases + 1))
    w = exe.upload(synth.norm_weight(rng, hd))
    exe.attn_prep_paged(pool.kv, seqs, dx.ptr, dx.ptr + 2 * nkv * hd, dx.ptr + 4 * nkv * hd, w, w, q, nh, EPS, THETA, 64,
                        q_ld=3 * nkv * hd, kv_ld=3 * nkv * hd)
    exe.device_status()
    qq, s, b = pool.v.get(pool.table[:, 0], np.zeros(cases, int), pool.dv.download())
    got, want = qq * s + b, _f64(x[:, 2 * nkv * hd:]).reshape(cases, nkv, hd)
    assert np.array_equal(got[0], want[0]) and np.all(qq[0] == 0) and not np.any(got[1])
    hit = np.zeros((3, hd // GROUP), bool)
    for c, d in ((2, 5), (3, 7), (4, 9)):
        hit[c - 2, d // GROUP] = True
        g = got[c].reshape(nkv, -1, GROUP)
        assert np.all(np.isnan(g[:, hit[c - 2]])) and np.all(np.isfinite(g[:, ~hit[c - 2]]))
    # half a step, the bias's and (fifteen times) the scale's rounding
    for c in (5, 6):
        span = want[c].max() - want[c].min()
        assert np.all(np.abs(got[c] - want[c]) <= span / 30 + 2.0 ** -8 * (np.abs(want[c]).max() + span) + 1e-40)


# ---- eviction -------------------------------------------------------------------

@pytest.mark.parametrize("sinks,recent,budget", [(4, 20, 50), (0, 0, 33), (10, 54, 64), (3, 0, 257), (2, 9, 700)])
@pytest.mark.parametrize("shape", [(32, 4, 128, 16), (16, 2, 64, 64), (16, 1, 128, 64), (16, 3, 64, 16)], ids=str)
def test_evict(exe, shape, sinks, recent, budget):
    nh, nkv, hd, page = shape
    rng = np.random.default_rng(61)
    lens = [300, 0, 40, 65, 1, 1500]
    B = len(lens)
    dst_pages = -(-budget // page)
    pool = Pool(exe, rng, lens, nkv, hd, page, extra=B * dst_pages + 2)
    cap = pool.max_pages * page
    to = pool.free[:B * dst_pages].reshape(B, dst_pages).astype(np.int32)
    w = rng.standard_normal((B, nkv, cap)).astype(np.float32)
    wd = exe.upload(np.full((B, nkv, dst_pages * page), 7.0, np.float32))
    kept, new_len = exe.alloc((B, nkv, budget), np.int32), exe.alloc(B, np.int32)
    exe.kv_evict(pool.kv, pool.seqs(), oh.KvWeight(exe.upload(w), B, cap), exe.upload(to), dst_pages,
                 oh.KvWeight(wd, B, dst_pages * page), sinks, recent, budget, kept, new_len)
    exe.device_status()
    raw = {"k": pool.dk.download(), "v": pool.dv.download()}
    got, n_new = kept.download(), new_len.download()
    touched = np.zeros(pool.n_pages, bool)
    for b, n in enumerate(lens):
        m = min(n, budget)
        assert n_new[b] == m
        touched[to[b, :-(-m // page)]] = True
        for h in range(nkv):
            want = _kept(w[b, h, :n], n, sinks, recent, budget)
            assert np.array_equal(got[b, h, :m], want) and np.all(got[b, h, m:] == -1)
            e = np.arange(m)
            for name, side in (("k", pool.k), ("v", pool.v)):
                have = side.get(to[b, e // page], e % page, raw[name])
                src = side.get(pool.table[b, want // page], want % page)
                assert all(np.array_equal(x[:, h], y[:, h]) for x, y in zip(have, src)), (b, h, name)
    for name, side in (("k", pool.k), ("v", pool.v)):
        assert np.array_equal(raw[name][~touched], side.raw[~touched])


def test_evict_copies_zeros_of_a_page_that_is_not_there(exe):
    nkv, hd, page = 2, 128, 16
    rng = np.random.default_rng(67)
    pool = Pool(exe, rng, [48], nkv, hd, page, extra=4)
    pool.table[0, 1] = -1
    pool.dt.upload(pool.table)
    to = pool.free[:3].reshape(1, 3).astype(np.int32)
    wd, kept, new_len = exe.zeros((1, nkv, 48), np.float32), exe.alloc((1, nkv, 48), np.int32), exe.alloc(1, np.int32)
    exe.kv_evict(pool.kv, pool.seqs(), oh.KvWeight(exe.zeros((1, nkv, 64), np.float32), 1, 64), exe.upload(to), 3,
                 oh.KvWeight(wd, 1, 48), 0, 0, 48, kept, new_len)
    with pytest.raises(oh.ObsError, match="paged cache"):
        exe.device_status()
    q, s, b = pool.v.get(to[0, [1]], np.array([3]), pool.dv.download())
    assert not np.any(q) and not np.any(s) and not np.any(b)
    assert all(np.array_equal(x, y) for x, y in zip(pool.v.get(to[0, [0, 2]], np.array([5, 7]), pool.dv.download()),
                                                    pool.v.get(pool.table[0, [0, 2]], np.array([5, 7]))))
