"""The cache in 4 bits and the log probabilities together, as a server would run them:
prompts in ragged chunks, decode steps that gather attention weight, an eviction, decode
steps over what is left, and a distribution over tokens from every step's rows; eager, as
replayed graphs that share a workspace, on two contexts at once and on a caller's stream.

Bars as in test_gpu_paged_q4.py and test_gpu_logprobs.py: every call is judged on what the
device holds before it."""
import numpy as np
import pytest

import obsidian_hip as oh
from obsidian_hip import synth
from test_gpu_logprobs import U, _logits64, _matrix, _near, _reference
from test_gpu_paged import EPS, FILL16, THETA, _f64, _kept, _visible
from test_gpu_paged_q4 import Pool, Side, _attend16, _attend4, _f16, _rope

pytestmark = pytest.mark.gpu


class Server:
    """Pages, tables and slots of a few sequences, handed out as they grow."""

    def __init__(self, exe, rng, B, nh, nkv, hd, page, cap, n_pages):
        self.exe, self.rng, self.B, self.nh, self.nkv, self.hd, self.page = exe, rng, B, nh, nkv, hd, page
        self.max_pages = cap // page
        self.k, self.v = Side(n_pages, nkv, hd, page, False), Side(n_pages, nkv, hd, page, True)
        self.dk, self.dv = exe.upload(self.k.raw), exe.upload(self.v.raw)  # scales and biases NaN where nothing is written
        self.kv = oh.PagedKv(self.dk, self.dv, n_pages, page, nkv, hd, oh.KV_Q4)
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
        self.row = exe.upload(np.zeros(B + 1, np.int32))
        # the matrix that makes logits of the rows; one workspace for every call
        self.vocab, self.top = 900, 5
        self.lm = _matrix(rng, self.vocab, nh * hd)
        self.dlm = [exe.upload(a) for a in self.lm]
        need = [exe.sdpa_paged_workspace(self.kv, oh.PagedSeqs(self.dt, self.dl, B, self.max_pages), nh, self.wt[0]),
                exe.sdpa_paged_workspace(self.kv, oh.PagedSeqs(self.dt, self.dl, B, self.max_pages, 600, self.row), nh),
                exe.lm_logprobs_workspace(300, nh * hd, self.vocab, self.top)]
        self.ws = exe.upload(np.full(max(need), 0xFF, np.uint8))

    def grow(self, new):
        for b, t in enumerate(new):
            have = -(-int(self.len[b]) // self.page)
            self.len[b] += t
            for p in range(have, -(-int(self.len[b]) // self.page)):
                self.table[b, p] = self.free.pop()
        self.dt.upload(self.table)
        self.dl.upload(self.len)

    def parts(self, what):
        side, raw = (self.k, self.dk.download()) if what == "k" else (self.v, self.dv.download())
        j = [np.arange(n) for n in self.len]
        return [side.get(self.table[b, j[b] // self.page], j[b] % self.page, raw) for b in range(self.B)]

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

    def tell(self, out, R):
        """Log probabilities from the rows out [R, nh hd], checked."""
        exe, V, k, H = self.exe, self.vocab, self.top, self.nh * self.hd
        tokens = self.rng.integers(0, V, R)
        lp, ent = exe.alloc(R, np.float32), exe.alloc(R, np.float32)
        ids, tl = exe.alloc((R, k), np.int32), exe.alloc((R, k), np.float32)
        exe.lm_logprobs(out, *self.dlm, R, H, V, self.ws, tokens=exe.upload(tokens.astype(np.int32)), logprob=lp, entropy=ent,
                        top_k=k, top_ids=ids, top_logprobs=tl)
        exe.device_status()
        logits, off = _logits64(_f64(out.download()).reshape(-1, H)[:R], *self.lm)
        want, ent64, ids64, tl64, bs, be = _reference(logits, tokens, k)
        worst = off.max(1)
        assert _near(lp.download(), want, bs + 4 * U * np.abs(want) + 2 * worst)
        t = np.arange(R)[:, None]
        assert np.all(np.abs(logits[t, ids.download()] - logits[t, ids64]) <= 2 * worst[:, None])
        assert _near(tl.download(), tl64, bs[:, None] + 4 * U * np.abs(tl64) + 4 * worst[:, None])


@pytest.mark.parametrize("nh,nkv,hd,page", [(32, 4, 128, 32), (16, 1, 64, 16), (16, 4, 128, 64)], ids=str)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
def test_serve_and_evict(exe, nh, nkv, hd, page, window, sinks):
    rng = np.random.default_rng(201)
    B, cap = 3, 256
    s = Server(exe, rng, B, nh, nkv, hd, page, cap, 3 * cap // page + 40)
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
        k, v = ([_f16(y[0] * y[1] + y[2]) for y in s.parts(n)] for n in "kv")
        qf, got = _f64(q.download()), _f64(out.download())
        for b in range(B):
            for t in range(chunk[b]):
                n = int(s.len[b])
                ref, bound = _attend16(qf[rows[b] + t], k[b], v[b], _visible(n - chunk[b] + t, n, window, sinks))
                assert np.all(np.abs(got[rows[b] + t] - ref) <= bound), (b, t)
        s.tell(out, R)
        s.pos += np.array(chunk, np.int32)

    def decode(n):
        gathered = s.w[s.cur].download().astype(np.float64)
        for _ in range(n):
            s.grow([1] * B)
            seqs = oh.PagedSeqs(s.dt, s.dl, B, s.max_pages)
            x = synth.bf16_normal(rng, (B, ld), 2.0)
            q = s.prep(x, seqs, B, pos=s.pos)
            out = exe.alloc((B, nh, hd), np.uint16)
            exe.sdpa_paged_decode(s.kv, seqs, q, out, nh, s.ws, window=window, sinks=sinks, weight=s.wt[s.cur])
            exe.device_status()
            k, v, qf, got = s.parts("k"), s.parts("v"), _f64(q.download()), _f64(out.download())
            now = s.w[s.cur].download().astype(np.float64)
            for b in range(B):
                m = int(s.len[b])
                # the new key is the token's, turned to its position among all ever seen
                key, off = _rope(_f64(x[b, nh * hd:(nh + nkv) * hd]).reshape(nkv, hd), _f64(s.kn), int(s.pos[b]))
                new = k[b][0][-1] * k[b][1][-1] + k[b][2][-1]
                span = 15 * k[b][1][-1]  # its group's: half a step, and what rounding of the scale and bias leaves out at the ends
                assert np.all(np.abs(new - key) <= span / 30 + 2.0 ** -7 * (span + np.abs(k[b][2][-1])) + 2 * off)
                ref, bound, p, err = _attend4(qf[b], k[b], v[b], _visible(m - 1, m, window, sinks))
                assert np.all(np.abs(got[b] - ref) <= bound), b
                gathered[s.slot[b], :, m - 1] = 0.0  # the new entry's weight starts at 0
                g = p.reshape(nkv, -1, m)
                ref = gathered[s.slot[b], :, :m] + g.sum(1)
                lim = (g * err.reshape(nkv, -1, 1)).sum(1) + 2.0 ** -22 * np.abs(ref)
                assert np.all(np.abs(now[s.slot[b], :, :m] - ref) <= lim)
            gathered = now
            s.tell(out, B)
            s.pos += 1

    decode(5)
    budget, recent, first = 40, 12, 4
    dst = np.full((B, -(-budget // page)), -1, np.int32)
    for b in range(B):
        for p in range(-(-min(budget, int(s.len[b])) // page)):
            dst[b, p] = s.free.pop()
    k, v, w = s.parts("k"), s.parts("v"), s.w[s.cur].download()
    kept, new_len = exe.alloc((B, nkv, budget), np.int32), exe.alloc(B, np.int32)
    exe.kv_evict(s.kv, oh.PagedSeqs(s.dt, s.dl, B, s.max_pages), s.wt[s.cur], exe.upload(dst), dst.shape[1], s.wt[1 - s.cur],
                 first, recent, budget, kept, new_len)
    exe.device_status()
    gk, old_len = kept.download(), s.len.copy()
    s.table[:] = -1
    s.table[:, :dst.shape[1]] = dst
    s.len = np.minimum(s.len, budget).astype(np.int32)
    s.cur = 1 - s.cur
    s.dt.upload(s.table)
    s.dl.upload(s.len)
    assert np.array_equal(new_len.download(), s.len)
    k2, v2, w2 = s.parts("k"), s.parts("v"), s.w[s.cur].download()
    for b in range(B):
        for h in range(nkv):
            ref = _kept(w[s.slot[b], h], int(old_len[b]), first, recent, budget)
            assert np.array_equal(gk[b, h, :len(ref)], ref)
            for old, new in ((k, k2), (v, v2)):
                assert all(np.array_equal(y[:, h], x[ref, h]) for x, y in zip(old[b], new[b]))
            assert np.array_equal(w2[s.slot[b], h, :len(ref)], w[s.slot[b], h, ref])
    decode(3)  # positions go on from all tokens ever seen


class Step:
    """A decode step with its log probabilities, and a prompt's, over device arrays that stay where they are."""

    def __init__(self, e, rng, pool, nh, cap, ws=None):
        self.e, self.pool, self.nh = e, pool, nh
        B, hd, nkv = len(pool.lens), pool.hd, pool.nkv
        self.B, self.ld, self.V = B, (nh + 2 * nkv) * hd, 1300
        self.seqs = pool.seqs()
        self.x = e.upload(synth.bf16_normal(rng, (B, self.ld), 2.0))
        self.qn, self.kn = e.upload(synth.norm_weight(rng, hd)), e.upload(synth.norm_weight(rng, hd))
        self.q, self.out = e.alloc((B, nh, hd), np.uint16), e.alloc((B, nh, hd), np.uint16)
        self.w0 = rng.random((B, nkv, cap)).astype(np.float32)
        self.dw = e.upload(self.w0)
        self.wt = oh.KvWeight(self.dw, B, cap)
        rows = [0, 20, 25, 90]
        self.pseqs = pool.seqs(rows)
        self.pq, self.pout = e.upload(synth.bf16_normal(rng, (90, nh, hd), 2.0)), e.alloc((90, nh, hd), np.uint16)
        self.lm = [e.upload(a) for a in _matrix(rng, self.V, nh * hd)]
        self.tok = e.upload(rng.integers(0, self.V, 90).astype(np.int32))
        self.res = [[e.alloc(n, np.float32), e.alloc(n, np.float32), e.alloc((n, 3), np.int32), e.alloc((n, 3), np.float32)] for n in (B, 90, B)]
        self.logits = e.upload((3 * rng.standard_normal((B, 40000))).astype(np.float32))
        need = max(e.sdpa_paged_workspace(pool.kv, self.seqs, nh, self.wt), e.sdpa_paged_workspace(pool.kv, self.pseqs, nh, None, 200, 4),
                   e.lm_logprobs_workspace(90, nh * hd, self.V, 3), e.lm_logprobs_workspace(B, nh * hd, self.V, 3),
                   e.token_logprobs_workspace(B, 40000, 3))
        self.ws = ws if ws is not None else e.upload(np.full(need, 0xFF, np.uint8))
        assert self.ws.nbytes >= need

    def call(self, first=None):
        e, nh, kv, p = self.e, self.nh, self.pool.kv, self.x.ptr
        qd, kd = nh * self.pool.hd, self.pool.nkv * self.pool.hd
        (first or e).attn_prep_paged(kv, self.seqs, p, p + 2 * qd, p + 2 * (qd + kd), self.qn, self.kn, self.q, nh, EPS, THETA, 4096,
                          weight=self.wt, q_ld=self.ld, kv_ld=self.ld)
        e.sdpa_paged_decode(kv, self.seqs, self.q, self.out, nh, self.ws, weight=self.wt)
        kw = lambda r: dict(tokens=self.tok, logprob=r[0], entropy=r[1], top_k=3, top_ids=r[2], top_logprobs=r[3])
        e.lm_logprobs(self.out, *self.lm, self.B, qd, self.V, self.ws, **kw(self.res[0]))
        e.sdpa_paged_prefill(kv, self.pseqs, self.pq, self.pout, nh, self.ws, window=200, sinks=4)
        e.lm_logprobs(self.pout, *self.lm, 90, qd, self.V, self.ws, **kw(self.res[1]))
        e.token_logprobs(self.logits, self.B, 40000, self.ws, **kw(self.res[2]))

    def buffers(self):
        return [self.q, self.out, self.pout, self.dw, self.pool.dk, self.pool.dv] + [b for r in self.res for b in r]

    def reset(self):
        self.pool.dk.upload(self.pool.k.raw)
        self.pool.dv.upload(self.pool.v.raw)
        self.dw.upload(self.w0)
        for b in (self.q, self.out, self.pout):
            b.upload(np.full(b.shape, FILL16, np.uint16))
        for r in self.res:
            for b in r:
                b.upload(np.full(b.shape, 77, b.dtype))

    def results(self):
        self.e.device_status()
        return [b.download() for b in self.buffers()]


def _same(got, want):
    for a, b in zip(got, want):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("nh,nkv,hd,page", [(32, 4, 128, 16), (16, 1, 64, 64)], ids=str)
def test_captured_steps_share_a_workspace(nh, nkv, hd, page):
    """Two steps recorded once each over one workspace: each replay, with the other's, eager work
    and other lengths between, gives what the eager calls give, bit for bit."""
    lens = [300, 45, 2000]
    with oh.ObsidianExecutor(0) as exe:
        rng = np.random.default_rng(207)
        cap = 2080 // page + 1
        steps = [Step(exe, rng, Pool(exe, rng, lens, nkv, hd, page, max_pages=cap), nh, cap * page)]
        steps.append(Step(exe, rng, Pool(exe, rng, lens, nkv, hd, page, max_pages=cap), nh, cap * page, ws=steps[0].ws))
        graphs = []
        try:
            for s in steps:
                s.call()  # the RoPE table exists from here on
                exe.sync()
                exe.capture_begin()
                s.call()
                graphs.append(exe.capture_end())
            for ln in (lens, [299, 45, 1999], lens, [90, 40, 100]):
                want = []
                for s in steps:
                    s.pool.dl.upload(np.array(ln, np.int32))
                    s.reset()
                    s.call()
                    want.append(s.results())
                    s.reset()
                exe.graph_launch(graphs[0])
                exe.graph_launch(graphs[1])
                for s, w in zip(steps, want):
                    _same(s.results(), w)
                    s.call()  # eager work before the next replays
        finally:
            for g in graphs:
                exe.graph_destroy(g)


def test_two_contexts_at_once(exe):
    """Two contexts, each with its stream, workspace and cache, calls in flight together."""
    nh, nkv, hd, page, lens = 32, 4, 128, 32, [1700, 700, 90]
    rng = np.random.default_rng(209)
    cap = 1700 // page + 2
    with oh.ObsidianExecutor(0) as other:
        steps = [Step(e, rng, Pool(e, rng, lens, nkv, hd, page, max_pages=cap), nh, cap * page) for e in (exe, other)]
        want = []
        for s in steps:
            s.call()
            s.results()
            s.reset()
            s.call()
            want.append(s.results())
            s.reset()
        for s in steps:
            s.e.sync()
        for s in steps:
            s.call()
        for s, w in zip(steps, want):
            _same(s.results(), w)


def test_a_callers_stream(exe):
    """Calls on a stream of another context's are ordered with its other work: queries and entries
    written there are read with no wait between."""
    nh, nkv, hd, page = 32, 4, 128, 64
    rng = np.random.default_rng(213)
    step = Step(exe, rng, Pool(exe, rng, [500, 3, 1], nkv, hd, page, max_pages=9), nh, 9 * page)
    step.call()
    step.results()
    step.reset()
    step.call()
    want = step.results()
    step.reset()
    exe.sync()
    with oh.ObsidianExecutor(0) as other:
        exe.set_stream(oh.lib().obs_get_stream(other.ctx))
        try:
            other.stream_hold(2000)
            step.call(other)  # the queries and entries
            other.sync()
        finally:
            exe.set_stream(None)
        _same(step.results(), want)
