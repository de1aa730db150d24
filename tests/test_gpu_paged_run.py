"""The paged cache's operators together, as a server would run them: prompts in
two chunks of a ragged batch, decode steps that gather attention weight (eager and
as a replayed graph), an eviction, and decode steps over what is left, each
against a float64 simulation that keeps every sequence's entries in plain arrays;
and the calls that share something: a context's stream, a page, a sequence, a
workspace of their own on two streams at once.

Bars as in test_gpu_paged.py: the simulation takes the stored entries and the
rotated queries from the device, so each call is judged by its own roundings."""
import numpy as np
import pytest

import obsidian_hip as oh
from obsidian_hip import synth
from test_gpu_paged import (E4M3, EPS, FILL16, NAN16, THETA, Pool, _attend, _f64, _kept, _rope64, _visible)

pytestmark = pytest.mark.gpu


class Server:
    """Pages, tables and slots of a few sequences, handed out as they grow."""

    def __init__(self, exe, rng, B, nh, nkv, hd, page, f8, cap, n_pages):
        self.exe, self.rng, self.B, self.nh, self.nkv, self.hd, self.page, self.f8 = exe, rng, B, nh, nkv, hd, page, f8
        self.max_pages = cap // page
        T, nan = (np.uint8, 0x7F) if f8 else (np.uint16, NAN16)
        self.dk = exe.upload(np.full((n_pages, nkv, page, hd), nan, T))
        self.dv = exe.upload(np.full((n_pages, nkv, hd, page), nan, T))
        self.ks = (0.02 + 0.01 * rng.random(nkv)).astype(np.float32)
        self.vs = (0.02 + 0.01 * rng.random(nkv)).astype(np.float32)
        self.kv = oh.PagedKv(self.dk, self.dv, n_pages, page, nkv, hd, oh.KV_E4M3 if f8 else oh.KV_BF16,
                             exe.upload(self.ks), exe.upload(self.vs))
        self.free = list(rng.permutation(n_pages).astype(np.int32))
        self.table = np.full((B, self.max_pages), -1, np.int32)
        self.len, self.pos = np.zeros(B, np.int32), np.zeros(B, np.int32)  # entries held; tokens ever seen
        self.dt, self.dl = exe.upload(self.table), exe.upload(self.len)
        self.qn, self.kn = synth.norm_weight(rng, hd), synth.norm_weight(rng, hd)
        self.dqn, self.dkn = exe.upload(self.qn), exe.upload(self.kn)
        self.w = [exe.upload(np.full((B + 1, nkv, cap), np.nan, np.float32)) for _ in range(2)]
        self.slot = rng.permutation(B + 1)[:B].astype(np.int32)
        dslot = exe.upload(self.slot)
        self.wt = [oh.KvWeight(w, B + 1, cap, dslot) for w in self.w]
        self.cur = 0
        ws = oh.PagedSeqs(self.dt, self.dl, B, self.max_pages)
        need = exe.sdpa_paged_workspace(self.kv, ws, nh, self.wt[0])
        self.row = exe.upload(np.zeros(B + 1, np.int32))
        need = max(need, exe.sdpa_paged_workspace(self.kv, oh.PagedSeqs(self.dt, self.dl, B, self.max_pages, 600, self.row), nh))
        self.ws = exe.upload(np.full(need, 0xFF, np.uint8))

    def grow(self, new):
        for b, t in enumerate(new):
            have = -(-int(self.len[b]) // self.page)
            self.len[b] += t
            for p in range(have, -(-int(self.len[b]) // self.page)):
                self.table[b, p] = self.free.pop()
        self.dt.upload(self.table)
        self.dl.upload(self.len)

    def entries(self, what):
        x = (self.dk if what == "k" else self.dv).download()
        s = self.ks if what == "k" else self.vs
        out = []
        for b in range(self.B):
            j = np.arange(self.len[b])
            p, o = self.table[b, j // self.page], j % self.page
            y = x[p, :, o] if what == "k" else x[p, :, :, o]
            out.append(E4M3[y] * s.astype(np.float64)[:, None] if self.f8 else _f64(y))
        return out

    def prep(self, x, seqs, R, pos=None):
        nh, nkv, hd = self.nh, self.nkv, self.hd
        qd, kd = nh * hd, nkv * hd
        ld = qd + 2 * kd
        dx = self.exe.upload(x)
        q = self.exe.alloc((R, nh, hd), np.uint16)
        self.exe.attn_prep_paged(self.kv, seqs, dx.ptr, dx.ptr + 2 * qd, dx.ptr + 2 * (qd + kd), self.dqn, self.dkn, q, nh,
                                 EPS, THETA, 4096, pos=None if pos is None else self.exe.upload(np.array(pos, np.int32)),
                                 weight=self.wt[self.cur], q_ld=ld, kv_ld=ld)
        return q

    def check(self, q, out, rows, window, sinks):
        """out against attention of the device's own entries; rows: (row, sequence, entry)."""
        k, v = self.entries("k"), self.entries("v")
        q, out = _f64(q.download()), _f64(out.download())
        P = []
        for row, b, i in rows:
            n = len(k[b])
            ref, bound, p, err = _attend(q[row], k[b], v[b], _visible(i, n, window, sinks))
            assert np.all(np.abs(out[row] - ref) <= bound), (row, b, i)
            P.append((b, p, err))
        return P


@pytest.mark.parametrize("nh,nkv,hd,page,f8", [(32, 4, 128, 16, False), (12, 2, 64, 32, True)], ids=str)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
def test_serve_and_evict(exe, nh, nkv, hd, page, f8, window, sinks):
    rng = np.random.default_rng(101)
    B, cap = 3, 256
    s = Server(exe, rng, B, nh, nkv, hd, page, f8, cap, 3 * cap // page + 40)
    ld = (nh + 2 * nkv) * hd
    for chunk in ([70, 1, 33], [41, 90, 0]):  # prompts, in two ragged chunks
        s.grow(chunk)
        rows = np.concatenate([[0], np.cumsum(chunk)]).astype(np.int32)
        R = int(rows[-1])
        s.row.upload(rows)
        seqs = oh.PagedSeqs(s.dt, s.dl, B, s.max_pages, R, s.row)
        x = synth.bf16_normal(rng, (R, ld), 2.0)
        q = s.prep(x, seqs, R)
        out = exe.alloc((R, nh, hd), np.uint16)
        exe.sdpa_paged_prefill(s.kv, seqs, q, out, nh, s.ws, window=window, sinks=sinks)
        exe.device_status()
        where = [(int(rows[b]) + t, b, int(s.len[b]) - chunk[b] + t) for b in range(B) for t in range(chunk[b])]
        s.check(q, out, where, window, sinks)
        s.pos += np.array(chunk, np.int32)
    k0 = [e.copy() for e in s.entries("k")]
    ref, pre = _rope64(_f64(x[-1, nh * hd:(nh + nkv) * hd]).reshape(nkv, hd), _f64(s.kn), int(s.len[1]) - 1)
    step = 2.0 ** -4 if f8 else 2.0 ** -8
    assert np.all(np.abs(k0[1][-1] - ref) <= pre + step * (np.abs(ref) + pre) + (2.0 ** -10 * s.ks[:, None] if f8 else 0))

    def decode(n):
        got = s.w[s.cur].download().astype(np.float64)
        for _ in range(n):
            s.grow([1] * B)
            seqs = oh.PagedSeqs(s.dt, s.dl, B, s.max_pages)
            q = s.prep(synth.bf16_normal(rng, (B, ld), 2.0), seqs, B, pos=s.pos)
            out = exe.alloc((B, nh, hd), np.uint16)
            exe.sdpa_paged_decode(s.kv, seqs, q, out, nh, s.ws, window=window, sinks=sinks, weight=s.wt[s.cur])
            exe.device_status()
            P = s.check(q, out, [(b, b, int(s.len[b]) - 1) for b in range(B)], window, sinks)
            now = s.w[s.cur].download().astype(np.float64)
            for b, p, err in P:
                m = p.shape[1]
                got[s.slot[b], :, m - 1] = 0.0  # the new entry's weight starts at 0
                g = p.reshape(nkv, -1, m)
                ref = got[s.slot[b], :, :m] + g.sum(1)
                lim = (g * err.reshape(nkv, -1, 1)).sum(1) + 2.0 ** -22 * np.abs(ref)
                assert np.all(np.abs(now[s.slot[b], :, :m] - ref) <= lim)
            got = now
            s.pos += 1

    decode(6)
    budget, recent, first = 40, 12, 4
    dst = np.full((B, -(-budget // page)), -1, np.int32)
    for b in range(B):
        for p in range(-(-min(budget, int(s.len[b])) // page)):
            dst[b, p] = s.free.pop()
    k, v, w = s.entries("k"), s.entries("v"), s.w[s.cur].download()
    kept, new_len = exe.alloc((B, nkv, budget), np.int32), exe.alloc(B, np.int32)
    exe.kv_evict(s.kv, oh.PagedSeqs(s.dt, s.dl, B, s.max_pages), s.wt[s.cur], exe.upload(dst), dst.shape[1], s.wt[1 - s.cur],
                 first, recent, budget, kept, new_len)
    exe.device_status()
    gk = kept.download()
    assert np.array_equal(new_len.download(), np.minimum(s.len, budget))
    old_len = s.len.copy()
    s.table[:] = -1
    s.table[:, :dst.shape[1]] = dst
    s.len = np.minimum(s.len, budget).astype(np.int32)
    s.cur = 1 - s.cur
    s.dt.upload(s.table)
    s.dl.upload(s.len)
    k2, v2, w2 = s.entries("k"), s.entries("v"), s.w[s.cur].download()
    for b in range(B):
        for h in range(nkv):
            ref = _kept(w[s.slot[b], h], int(old_len[b]), first, recent, budget)
            assert np.array_equal(gk[b, h, :len(ref)], ref)
            assert np.array_equal(k2[b][:, h], k[b][ref, h]) and np.array_equal(v2[b][:, h], v[b][ref, h])
            assert np.array_equal(w2[s.slot[b], h, :len(ref)], w[s.slot[b], h, ref])
    decode(4)  # positions go on from all tokens ever seen


def _step(exe, pool, nh, seqs, x, qn, kn, q, out, ws, wt=None):
    hd, nkv = pool.hd, pool.nkv
    qd, kd = nh * hd, nkv * hd
    ld = qd + 2 * kd
    exe.attn_prep_paged(pool.kv, seqs, x.ptr, x.ptr + 2 * qd, x.ptr + 2 * (qd + kd), qn, kn, q, nh, EPS, THETA, 4096,
                        weight=wt, q_ld=ld, kv_ld=ld)
    exe.sdpa_paged_decode(pool.kv, seqs, q, out, nh, ws, weight=wt)


def test_captured_step_follows_the_device_arrays():
    """A decode step, an eviction and a prompt's attention recorded once: each
    replay, with eager work and other lengths between them, gives what the eager
    calls give, bit for bit."""
    nh, nkv, hd, page, lens = 32, 4, 128, 16, [300, 45, 2000]
    with oh.ObsidianExecutor(0) as exe:
        rng = np.random.default_rng(107)
        B, budget = len(lens), 100
        pool = Pool(exe, rng, lens, nkv, hd, page, False, extra=B * 8, max_pages=130)
        seqs = pool.seqs()
        ld = (nh + 2 * nkv) * hd
        x = exe.upload(synth.bf16_normal(rng, (B, ld), 2.0))
        qn, kn = exe.upload(synth.norm_weight(rng, hd)), exe.upload(synth.norm_weight(rng, hd))
        q, out = exe.alloc((B, nh, hd), np.uint16), exe.alloc((B, nh, hd), np.uint16)
        cap = 130 * page
        w0 = rng.random((B, nkv, cap)).astype(np.float32)
        dw, dw2 = exe.upload(w0), exe.upload(np.zeros((B, nkv, budget), np.float32))
        wt, wt2 = oh.KvWeight(dw, B, cap), oh.KvWeight(dw2, B, budget)
        ws = exe.upload(np.full(exe.sdpa_paged_workspace(pool.kv, seqs, nh, wt), 0xFF, np.uint8))
        dst = exe.upload(pool.free[:B * 7].reshape(B, 7).copy())
        kept, new_len = exe.alloc((B, nkv, budget), np.int32), exe.alloc(B, np.int32)
        rows = [0, 20, 25, 90]
        pseqs = pool.seqs(rows)
        pq = exe.upload(synth.bf16_normal(rng, (90, nh, hd), 2.0))
        pout = exe.alloc((90, nh, hd), np.uint16)
        pws = exe.upload(np.full(exe.sdpa_paged_workspace(pool.kv, pseqs, nh, None, 200, 4), 0xFF, np.uint8))

        def all_calls():
            _step(exe, pool, nh, seqs, x, qn, kn, q, out, ws, wt)
            exe.kv_evict(pool.kv, seqs, wt, dst, 7, wt2, 4, 20, budget, kept, new_len)
            exe.sdpa_paged_prefill(pool.kv, pseqs, pq, pout, nh, pws, window=200, sinks=4)

        def results():
            exe.device_status()
            return [b.download() for b in (q, out, dw, dw2, kept, new_len, pout, pool.dk, pool.dv)]

        def reset():
            pool.dk.upload(pool.k)
            pool.dv.upload(pool.v)
            dw.upload(w0)
            dw2.upload(np.zeros((B, nkv, budget), np.float32))
            for b in (q, out, pout):
                b.upload(np.full(b.shape, FILL16, np.uint16))

        all_calls()  # the RoPE table exists from here on
        exe.sync()
        exe.capture_begin()
        all_calls()
        g = exe.capture_end()
        try:
            for ln in (lens, [299, 45, 1999], lens, [90, 40, 100]):
                pool.dl.upload(np.array(ln, np.int32))
                reset()
                all_calls()
                want = results()
                reset()
                exe.graph_launch(g)
                got = results()
                for a, b in zip(got, want):
                    assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
                all_calls()  # eager work before the next replay
        finally:
            exe.graph_destroy(g)


def test_two_contexts_at_once(exe):
    """The same cache read by two contexts, each with its stream and workspace, calls in flight together."""
    nh, nkv, hd, page, lens = 32, 4, 128, 32, [4000, 700, 90, 2500]
    rng = np.random.default_rng(109)
    pool = Pool(exe, rng, lens, nkv, hd, page, False)
    seqs, B = pool.seqs(), len(lens)
    rows = [0, 30, 60, 90, 120]
    pseqs = pool.seqs(rows)
    with oh.ObsidianExecutor(0) as other:
        sets = []
        for e in (exe, other):
            q, pq = e.upload(synth.bf16_normal(rng, (B, nh, hd), 2.0)), e.upload(synth.bf16_normal(rng, (120, nh, hd), 2.0))
            sets.append((e, q, e.alloc((B, nh, hd), np.uint16), pq, e.alloc((120, nh, hd), np.uint16),
                         e.alloc(e.sdpa_paged_workspace(pool.kv, seqs, nh), np.uint8),
                         e.alloc(e.sdpa_paged_workspace(pool.kv, pseqs, nh), np.uint8)))

        def call(e, q, out, pq, pout, ws, pws):
            e.sdpa_paged_decode(pool.kv, seqs, q, out, nh, ws)
            e.sdpa_paged_prefill(pool.kv, pseqs, pq, pout, nh, pws)

        want = []
        for s in sets:
            call(*s)
            s[0].device_status()
            want.append((s[2].download(), s[4].download()))
        for _ in range(20):
            for s in sets:
                call(*s)
        for s, w in zip(sets, want):
            s[0].device_status()
            assert np.array_equal(s[2].download(), w[0]) and np.array_equal(s[4].download(), w[1])


def test_a_callers_stream(exe):
    """Calls on a stream of the caller's (another context's) are ordered with its other
    work: queries and entries written there are read with no wait between."""
    nh, nkv, hd, page, n = 32, 4, 128, 32, 500
    rng = np.random.default_rng(113)
    pool = Pool(exe, rng, [n], nkv, hd, page, False)
    seqs, ld = pool.seqs(), (nh + 2 * nkv) * hd
    x = exe.upload(synth.bf16_normal(rng, (1, ld), 2.0))
    qn, kn = exe.upload(synth.norm_weight(rng, hd)), exe.upload(synth.norm_weight(rng, hd))
    q, out = exe.zeros((1, nh, hd), np.uint16), exe.zeros((1, nh, hd), np.uint16)
    ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, seqs, nh), np.uint8)
    exe.sync()
    with oh.ObsidianExecutor(0) as other:
        exe.set_stream(oh.lib().obs_get_stream(other.ctx))
        try:
            other.stream_hold(2000)
            other.attn_prep_paged(pool.kv, seqs, x.ptr, x.ptr + 2 * nh * hd, x.ptr + 2 * (nh + nkv) * hd, qn, kn, q, nh, EPS,
                                  THETA, 512, q_ld=ld, kv_ld=ld)
            exe.sdpa_paged_decode(pool.kv, seqs, q, out, nh, ws)
            other.sync()
        finally:
            exe.set_stream(None)
    pool.k, pool.v = pool.dk.download(), pool.dv.download()
    ref, bound, _, _ = _attend(_f64(q.download()[0]), pool.entries(0, "k"), pool.entries(0, "v"), np.ones(n, bool))
    assert np.any(ref != 0) and np.all(np.abs(_f64(out.download()[0]) - ref) <= bound)


def test_shared_pages_and_one_sequence_twice(exe):
    """Sequences with a common prefix in the same pages, and a sequence that is in the
    batch twice: each row and each slot as if it were alone."""
    nh, nkv, hd, page = 32, 4, 128, 16
    rng = np.random.default_rng(127)
    pool = Pool(exe, rng, [100, 70, 100], nkv, hd, page, False)
    table = pool.table.copy()
    table[1, :4] = table[0, :4]   # 64 entries in common
    table[2] = table[0]
    pool.table = table
    pool.dt.upload(table)
    q = synth.bf16_normal(rng, (3, nh, hd), 2.0)
    q[2] = q[0]
    cap = pool.max_pages * page
    dw = exe.zeros((3, nkv, cap), np.float32)
    out, seqs = exe.alloc((3, nh, hd), np.uint16), pool.seqs()
    wt = oh.KvWeight(dw, 3, cap)
    ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, seqs, nh, wt), np.uint8)
    exe.sdpa_paged_decode(pool.kv, seqs, exe.upload(q), out, nh, ws, weight=wt)
    exe.device_status()
    got, w = _f64(out.download()), dw.download().astype(np.float64)
    for b, n in enumerate(pool.lens):
        ref, bound, p, err = _attend(_f64(q[b]), pool.entries(b, "k"), pool.entries(b, "v"), np.ones(n, bool))
        assert np.all(np.abs(got[b] - ref) <= bound)
        g = p.reshape(nkv, -1, n)
        assert np.all(np.abs(w[b, :, :n] - g.sum(1)) <= (g * err.reshape(nkv, -1, 1)).sum(1) + 2.0 ** -22 * g.sum(1))
        assert not np.any(w[b, :, n:])
    assert np.array_equal(got[0], got[2]) and np.array_equal(w[0], w[2])


@pytest.mark.parametrize("window,sinks", [(0xffffffff, 0xffffffff), (0x80000000, 7), (5, 0xffffffff)])
def test_largest_windows(exe, window, sinks):
    nh, nkv, hd, page, lens = 16, 2, 128, 16, [700, 31]
    rng = np.random.default_rng(131)
    pool = Pool(exe, rng, lens, nkv, hd, page, False)
    rows = [0, 50, 81]
    q, pq = synth.bf16_normal(rng, (2, nh, hd), 2.0), synth.bf16_normal(rng, (81, nh, hd), 2.0)
    out, pout = exe.alloc((2, nh, hd), np.uint16), exe.alloc((81, nh, hd), np.uint16)
    for s, qq, o, fn in ((pool.seqs(), q, out, exe.sdpa_paged_decode), (pool.seqs(rows), pq, pout, exe.sdpa_paged_prefill)):
        ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, s, nh, None, window, sinks), np.uint8)
        fn(pool.kv, s, exe.upload(qq), o, nh, ws, window=window, sinks=sinks)
    exe.device_status()
    got, pgot = _f64(out.download()), _f64(pout.download())
    for b, n in enumerate(lens):
        k, v = pool.entries(b, "k"), pool.entries(b, "v")
        ref, bound, _, _ = _attend(_f64(q[b]), k, v, _visible(n - 1, n, window, sinks))
        assert np.all(np.abs(got[b] - ref) <= bound)
        new = rows[b + 1] - rows[b]
        for r in range(new):
            ref, bound, _, _ = _attend(_f64(pq[rows[b] + r]), k, v, _visible(n - new + r, n, window, sinks))
            assert np.all(np.abs(pgot[rows[b] + r] - ref) <= bound)


def test_rows_before_the_first_sequence_are_left_alone(exe):
    nh, nkv, hd, page = 32, 4, 128, 16
    rng = np.random.default_rng(137)
    pool = Pool(exe, rng, [40, 20], nkv, hd, page, False)
    rows = [5, 45, 65]
    seqs = pool.seqs(rows, 70)
    ld = (nh + 2 * nkv) * hd
    x = exe.upload(synth.bf16_normal(rng, (70, ld), 2.0))
    q = exe.upload(np.full((70, nh, hd), FILL16, np.uint16))
    out = exe.upload(np.full((70, nh, hd), FILL16, np.uint16))
    exe.attn_prep_paged(pool.kv, seqs, x.ptr, x.ptr + 2 * nh * hd, x.ptr + 2 * (nh + nkv) * hd,
                        exe.upload(synth.norm_weight(rng, hd)), exe.upload(synth.norm_weight(rng, hd)), q, nh, EPS, THETA, 64,
                        q_ld=ld, kv_ld=ld)
    ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, seqs, nh), np.uint8)
    exe.sdpa_paged_prefill(pool.kv, seqs, q, out, nh, ws)
    exe.device_status()
    pool.k, pool.v = pool.dk.download(), pool.dv.download()
    qf, got = q.download(), out.download()
    assert np.all(qf[:5] == FILL16) and np.all(qf[65:] == FILL16)
    assert np.all(got[:5] == FILL16) and np.all(got[65:] == FILL16)
    for b, n in enumerate((40, 20)):
        for r in range(n):
            ref, bound, _, _ = _attend(_f64(qf[rows[b] + r]), pool.entries(b, "k"), pool.entries(b, "v"), np.arange(n) <= r)
            assert np.all(np.abs(_f64(got[rows[b] + r]) - ref) <= bound)


def test_many_sequences_at_the_limit(exe):
    """4,096 sequences of no to three entries, in every operator."""
    nh, nkv, hd, page, B = 4, 1, 64, 16, 4096
    rng = np.random.default_rng(139)
    lens = rng.integers(0, 4, B)
    pool = Pool(exe, rng, [int(n) for n in lens], nkv, hd, page, False, extra=B + 2, max_pages=1)
    seqs = pool.seqs()
    q = synth.bf16_normal(rng, (B, nh, hd), 2.0)
    out = exe.upload(np.full((B, nh, hd), FILL16, np.uint16))
    w = exe.zeros((B, nkv, page), np.float32)
    wt = oh.KvWeight(w, B, page)
    ws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, seqs, nh, wt), np.uint8)
    exe.sdpa_paged_decode(pool.kv, seqs, exe.upload(q), out, nh, ws, weight=wt)
    rows = np.concatenate([[0], np.cumsum(lens)]).astype(int)
    R = int(rows[-1])
    pseqs = pool.seqs(rows)
    pq = synth.bf16_normal(rng, (R, nh, hd), 2.0)
    pout = exe.alloc((R, nh, hd), np.uint16)
    pws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, pseqs, nh), np.uint8)
    exe.sdpa_paged_prefill(pool.kv, pseqs, exe.upload(pq), pout, nh, pws)
    dst = pool.free[:B].reshape(B, 1).copy()
    w2 = exe.zeros((B, nkv, 2), np.float32)
    kept, new_len = exe.alloc((B, nkv, 2), np.int32), exe.alloc(B, np.int32)
    exe.kv_evict(pool.kv, seqs, wt, exe.upload(dst), 1, oh.KvWeight(w2, B, 2), 0, 1, 2, kept, new_len)
    exe.device_status()
    got, pgot, gw, gk = _f64(out.download()), _f64(pout.download()), w.download(), kept.download()
    assert np.array_equal(new_len.download(), np.minimum(lens, 2))
    for b in range(B):
        n = int(lens[b])
        k, v = pool.entries(b, "k"), pool.entries(b, "v")
        ref, bound, p, _ = _attend(_f64(q[b]), k, v, np.ones(n, bool))
        assert np.all(np.abs(got[b] - ref) <= bound)
        assert abs(gw[b].sum() - (nh if n else 0)) < 1e-4
        ref = _kept(gw[b, 0], n, 0, 1, 2)
        assert np.array_equal(gk[b, 0], np.concatenate([ref, [-1] * (2 - len(ref))]))
        for r in range(n):
            ref, bound, _, _ = _attend(_f64(pq[rows[b] + r]), k, v, np.arange(n) <= r)
            assert np.all(np.abs(pgot[rows[b] + r] - ref) <= bound)


def test_offsets_past_32_bits(exe):
    """Append, prompt attention and eviction in pages behind 4 GiB of keys and of values: bit for
    bit what the same calls give in a small pool."""
    nh, nkv, hd, page, n, R = 32, 8, 128, 256, 1000, 700
    rng = np.random.default_rng(91)
    n_pages = 8300  # 4.05 GiB of keys
    per = nkv * page * hd
    ld = (nh + 2 * nkv) * hd
    x = exe.upload(synth.bf16_normal(rng, (R, ld), 2.0))
    qn, kn = exe.upload(synth.bf16_normal(rng, hd)), exe.upload(synth.bf16_normal(rng, hd))
    old = [synth.bf16_normal(rng, (8, per)) for _ in range(2)]
    w = rng.random((1, nkv, 4 * page)).astype(np.float32)
    results = []
    for total in (8, n_pages):
        dk, dv = exe.alloc((total, per), np.uint16), exe.alloc((total, per), np.uint16)
        at = total - 8  # the last eight pages
        for d, o in ((dk, old[0]), (dv, old[1])):
            exe._check(oh.lib().obs_upload(exe.ctx, d.ptr + at * per * 2, o.ctypes.data, o.nbytes))
        kv = oh.PagedKv(dk, dv, total, page, nkv, hd)
        ids = exe.upload(np.array([at + 7, at + 2, at + 5, at], np.int32))
        seqs = oh.PagedSeqs(ids, exe.upload(np.array([n], np.int32)), 1, 4, R, exe.upload(np.array([0, R], np.int32)))
        q, out = exe.alloc((R, nh, hd), np.uint16), exe.alloc((R, nh, hd), np.uint16)
        exe.attn_prep_paged(kv, seqs, x.ptr, x.ptr + 2 * nh * hd, x.ptr + 2 * (nh + nkv) * hd, qn, kn, q, nh, 1e-6, 1e7, 2048,
                            q_ld=ld, kv_ld=ld)
        ws = exe.alloc(exe.sdpa_paged_workspace(kv, seqs, nh), np.uint8)
        exe.sdpa_paged_prefill(kv, seqs, q, out, nh, ws)
        dw, dwd = exe.upload(w), exe.alloc((1, nkv, 400), np.float32)
        kept, new_len = exe.alloc((1, nkv, 400), np.int32), exe.alloc(1, np.int32)
        exe.kv_evict(kv, seqs, oh.KvWeight(dw, 1, 4 * page), exe.upload(np.array([at + 6, at + 1], np.int32)), 2,
                     oh.KvWeight(dwd, 1, 400), 4, 50, 400, kept, new_len)
        exe.device_status()
        results.append([out.download(), kept.download(), dwd.download()] +
                       [exe.download_raw(d.ptr + at * per * 2, (8, per), np.uint16) for d in (dk, dv)])
        dk.free()
        dv.free()
    for a, b in zip(*results):
        assert np.array_equal(a, b)
    keys = results[0][3]  # entries 300 on were appended (pages 2, 5 and 0), kept ones copied to pages 6 and 1
    assert np.array_equal(keys[7], old[0][7]) and not any(np.array_equal(keys[i], old[0][i]) for i in (2, 5, 0, 6, 1))
