"""Calls on the paged cache (obs_attn_prep_paged, obs_sdpa_paged_prefill, obs_kv_evict,
obs_device_status) that the documentation allows and that are easily answered
wrongly: positions past the RoPE table's, far positions, tables that grow,
padded batches, several device failures at once. Helpers, pools and bars as in
test_gpu_paged.py; a test that needs another bar derives it beside it."""
import numpy as np
import pytest

import obsidian_hip as oh
from obsidian_hip import synth
from test_gpu_paged import (E4M3, EPS, FILL16, NAN16, SHAPES, THETA, Pool, _attend, _check_prep, _e4m3_bytes, _f64, _kept,
                            _prep_case, _rope64, _visible)

pytestmark = pytest.mark.gpu


# ---- positions ------------------------------------------------------------------

@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("shape", [(32, 4, 128, 16, False), (8, 1, 128, 32, True), (12, 2, 64, 64, True)], ids=str)
def test_entries_past_the_positions_are_reported(exe, shape, one):
    """pos NULL: a row whose entry lies at or past rope_len writes nothing, as one whose length
    is out of range, and that is reported once; a batch that ends right at rope_len is clean."""
    lens = [40, 64, 65, 0] if one else [40, 64, 70, 0]
    new = [1] * 4 if one else [40, 10, 12, 0]
    a = _prep_case(exe, shape, lens, new, 151, rope_len=64, one=one)
    with pytest.raises(oh.ObsError, match="paged cache") as ei:
        exe.device_status()
    assert ei.value.code == oh.OBS_E_INVALID
    exe.device_status()
    _check_prep(*a, lens, new, rope_len=64)
    lens[2] = 64
    a = _prep_case(exe, shape, lens, new, 151, rope_len=64, one=one)
    exe.device_status()
    _check_prep(*a, lens, new, rope_len=64)


def test_many_rows_past_the_positions_are_reported(exe):
    """The same in the form that takes one wave a row."""
    lens, new = [1100, 30], [1100, 30]
    a = _prep_case(exe, (32, 4, 64, 16, False), lens, new, 153, rope_len=1099)
    with pytest.raises(oh.ObsError, match="paged cache"):
        exe.device_status()
    _check_prep(*a, lens, new, rope_len=1099)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_prompt_rows_with_positions_of_their_own(exe, shape):
    """Ragged prompts behind an eviction: positions ahead of the entries, and rows whose own position
    is outside [0, rope_len) write nothing (that is how a caller leaves rows out; not reported)."""
    lens, new = [40, 3, 0, 17, 200], [40, 3, 0, 1, 130]
    rng = np.random.default_rng(157)
    pos = rng.integers(0, 9000, sum(new))
    pos[[0, 5, 70]], pos[[41, 100]] = [9000, 2**31 - 1, 9001], [-1, -2**31]
    a = _prep_case(exe, shape, lens, new, 157, pos=pos, pad_rows=1)
    exe.device_status()
    _check_prep(*a, lens, new, pos=[int(p) for p in pos])


@pytest.mark.parametrize("shape", [(32, 4, 128, 16, True), (16, 16, 64, 32, True), (12, 2, 64, 64, True)], ids=str)
@pytest.mark.parametrize("rows", [60, 1030])
def test_e4m3_keys_are_rounded_once(exe, shape, rows):
    """A key in e4m3 is the nearest to the exact value over the scale, but where the fp32
    arithmetic's own error reaches over the middle between two. That error: at most 32 roundings
    of 2^-24 behind each of the two products (the sum of squares as a tree of 11 levels, root,
    quotient, two products; cosine, product, difference, division), and the angle's 2^-23 p."""
    nh, nkv, hd, page, _ = shape
    pos = np.arange(rows) % 61
    pool, _, x, _, kn, _, _, _ = _prep_case(exe, shape, [rows], [rows], 163, pos=pos)
    exe.device_status()
    k, f, s = pool.dk.download(), _f64(x), pool.ks.astype(np.float64)[:, None]
    for r in range(rows):
        y = f[r, nh * hd:(nh + nkv) * hd].reshape(nkv, hd)
        ref, _ = _rope64(y, _f64(kn), int(pos[r]))
        y = y / np.sqrt(np.mean(y * y, -1, keepdims=True) + EPS) * _f64(kn)
        turn = np.concatenate([np.abs(y[:, :hd // 2]) + np.abs(y[:, hd // 2:])] * 2, -1)
        err = (2.0 ** -19 + 2.0 ** -23 * pos[r]) * turn
        got = E4M3[k[pool.table[0, r // page], :, r % page]]
        lo, hi = E4M3[_e4m3_bytes((ref - err) / s)], E4M3[_e4m3_bytes((ref + err) / s)]
        assert np.all((lo <= got) & (got <= hi)), (r, np.sum((lo > got) | (got > hi)))


# ---- the RoPE table ---------------------------------------------------------------

def test_a_growing_rope_len_needs_no_new_table():
    """A caller that passes its present longest position as rope_len: no call up to the next
    power of two builds a table, so the calls can be captured (building one cannot be)."""
    nh, nkv, hd, page = 32, 4, 128, 16
    with oh.ObsidianExecutor(0) as exe:
        rng = np.random.default_rng(167)
        pool = Pool(exe, rng, [60], nkv, hd, page, False)
        ld = (nh + 2 * nkv) * hd
        x, q = exe.upload(synth.bf16_normal(rng, (1, ld), 2.0)), exe.alloc((1, nh, hd), np.uint16)
        qn, kn = exe.upload(synth.norm_weight(rng, hd)), exe.upload(synth.norm_weight(rng, hd))

        def step(rope_len):
            exe.attn_prep_paged(pool.kv, pool.seqs(), x.ptr, x.ptr + 2 * nh * hd, x.ptr + 2 * (nh + nkv) * hd, qn, kn, q, nh, EPS,
                                THETA, rope_len, q_ld=ld, kv_ld=ld)

        for first, later in ((100, (101, 4000, 8192)), (8193, (8194, 16384, 100))):
            step(first)
            want = q.download()
            for n in later:
                q.upload(np.full((1, nh, hd), FILL16, np.uint16))
                exe.sync()
                exe.capture_begin()
                try:
                    step(n)
                finally:
                    g = exe.capture_end()
                exe.graph_launch(g)
                exe.device_status()
                exe.graph_destroy(g)
                assert np.array_equal(q.download(), want)


def test_a_table_that_is_long_enough_is_taken():
    """A context that has a table for a call's positions, from the contiguous cache or the other way
    round, needs no other one: such a first call can be captured."""
    nh, nkv, hd, page, ml = 32, 4, 128, 16, 160
    rng = np.random.default_rng(197)
    ld = (nh + 2 * nkv) * hd
    x0 = synth.bf16_normal(rng, (1, ld), 2.0)
    norms = [synth.norm_weight(rng, hd) for _ in range(2)]
    results = []
    for order in ("paged last", "paged first"):
        with oh.ObsidianExecutor(0) as exe:
            pool = Pool(exe, np.random.default_rng(199), [60], nkv, hd, page, False)
            seqs, q = pool.seqs(), exe.alloc((1, nh, hd), np.uint16)
            qn, kn = (exe.upload(w) for w in norms)
            kc, vc = exe.zeros((nkv, ml, hd), np.uint16), exe.zeros((nkv, hd, ml), np.uint16)
            x, y = exe.upload(x0), exe.upload(x0)  # the contiguous call norms q in place

            def paged():
                exe.attn_prep_paged(pool.kv, seqs, x.ptr, x.ptr + 2 * nh * hd, x.ptr + 2 * (nh + nkv) * hd, qn, kn, q, nh, EPS, THETA,
                                    100, q_ld=ld, kv_ld=ld)

            def contiguous():
                exe.attn_prep_rows(y.ptr, y.ptr + 2 * nh * hd, y.ptr + 2 * (nh + nkv) * hd, qn, kn, kc, vc, nh, nkv, hd, ml, EPS, THETA,
                                   59, 1, ld, ld)

            first, later = (contiguous, paged) if order == "paged last" else (paged, contiguous)
            first()
            exe.sync()
            exe.capture_begin()
            try:
                later()
            finally:
                g = exe.capture_end()
            exe.graph_launch(g)
            exe.device_status()
            exe.graph_destroy(g)
            results += [q.download().reshape(-1), y.download()[0, :nh * hd]]
    for r in results[1:]:
        assert np.array_equal(r, results[0])


FAR = [8191, 8192, 8193, 100_003, 1_000_000, (1 << 20) - 1]


@pytest.mark.parametrize("shape", [(32, 4, 128, 16, False), (16, 16, 64, 32, False), (8, 1, 128, 16, True)], ids=str)
@pytest.mark.parametrize("one", [True, False])
def test_far_positions(exe, shape, one):
    """Rotations at positions up to 2^20 against 64 bits, with a bar that does not grow with the
    position: below 8,192 the angle is an fp32 product of two fp32 factors, the largest of which
    with a rounding is 0.78: 2^13 0.78 2^-23 < 2^-10; from there on it is formed in double, and the
    rounded cosine and sine (2^-24 of each) are within 2^-20 like the other fp32 steps."""
    nh, nkv, hd, page, f8 = shape
    new = [1] * len(FAR) if one else [1, 30, 1, 2, 40, 1]
    lens = [20, 33, 1, 500, 64, 17]
    rows = np.concatenate([[0], np.cumsum(new)]).astype(int)
    pos = np.concatenate([p + 1 - np.arange(t, 0, -1) for p, t in zip(FAR, new)])
    pool, rows, x, qn, kn, q_out, w0, dw = _prep_case(exe, shape, lens, new, 173, pos=pos, rope_len=1 << 20, one=one)
    exe.device_status()
    got, k, f = _f64(q_out.download()), pool.dk.download(), _f64(x)
    for b, (n, t) in enumerate(zip(lens, new)):
        for r in range(t):
            row, e = rows[b] + r, n - t + r
            turn_err = 2.0 ** -10 if pos[row] < 8192 else 0.0
            for y, w, g in ((f[row, :nh * hd].reshape(nh, hd), qn, got[row]),
                            (f[row, nh * hd:(nh + nkv) * hd].reshape(nkv, hd), kn, k[pool.table[b, e // page], :, e % page])):
                ref, _ = _rope64(y, _f64(w), int(pos[row]))
                y = y / np.sqrt(np.mean(y * y, -1, keepdims=True) + EPS) * _f64(w)
                turn = np.concatenate([np.abs(y[:, :hd // 2]) + np.abs(y[:, hd // 2:])] * 2, -1)
                pre = (2.0 ** -8 + 2.0 ** -20 + turn_err) * turn  # the normed value's rounding, the fp32 steps
                lim = pre + 2.0 ** -8 * (np.abs(ref) + pre)
                if w is kn and f8:
                    s = pool.ks.astype(np.float64)[:, None]
                    g, ref = E4M3[g] * s, np.clip(ref, -448 * s, 448 * s)
                    lim = pre + 2.0 ** -4 * (np.abs(ref) + pre) + 2.0 ** -10 * s
                elif w is kn:
                    g = _f64(g)
                assert np.all(np.abs(g - ref) <= lim), (b, r, int(pos[row]), np.max(np.abs(g - ref)))


@pytest.mark.parametrize("rope_len", [8192, 1 << 20])
def test_near_positions_equal_the_contiguous_cache(exe, rope_len):
    """Below 8,192 q and keys are obs_attn_prep_rows' bit for bit, whatever rope_len."""
    nh, nkv, hd, page, T, ml = 32, 4, 128, 32, 60, 8192
    pos0 = ml - T
    a = _prep_case(exe, (nh, nkv, hd, page, False), [T], [T], 179, pos=np.arange(pos0, ml), rope_len=rope_len, weight=False)
    pool, _, x, qn, kn, q_out = a[:6]
    ld, dx = x.shape[1], exe.upload(x)
    kc, vc = exe.zeros((nkv, ml, hd), np.uint16), exe.zeros((nkv, hd, ml), np.uint16)
    exe.attn_prep_rows(dx.ptr, dx.ptr + 2 * nh * hd, dx.ptr + 2 * (nh + nkv) * hd, exe.upload(qn), exe.upload(kn), kc, vc, nh,
                       nkv, hd, ml, EPS, THETA, pos0, T, ld, ld)
    assert np.array_equal(dx.download()[:, :nh * hd].reshape(T, nh, hd), q_out.download())
    j = np.arange(T)
    p, o = pool.table[0, j // page], j % page
    assert np.array_equal(kc.download()[:, pos0 + j].transpose(1, 0, 2), pool.dk.download()[p, :, o])


# ---- padded batches and several reports --------------------------------------------

@pytest.mark.parametrize("slots", [[-1, 0, 1, 9], None], ids=["slots", "no slots"])
def test_evict_of_a_padded_batch(exe, slots):
    """Sequences without entries keep nothing and need no slot, in the eviction as in the append
    and the attention: nothing is reported. One with entries and no slot is."""
    nkv, hd, page, budget = 2, 64, 16, 50
    rng = np.random.default_rng(181)
    lens = [0, 300, 40, -3] if slots else [300, 40, 0, -3]
    pool = Pool(exe, rng, lens, nkv, hd, page, False, extra=4 * 4)
    cap = pool.max_pages * page
    w = rng.random((2, nkv, cap)).astype(np.float32)
    kept, new_len = exe.upload(np.full((4, nkv, budget), 77, np.int32)), exe.upload(np.full(4, 77, np.int32))
    dwd = exe.upload(np.full((2, nkv, budget), 5.5, np.float32))
    ds = None if slots is None else exe.upload(np.array(slots, np.int32))
    dst = exe.upload(pool.free[:16].reshape(4, 4).copy())

    def call():
        exe.kv_evict(pool.kv, pool.seqs(), oh.KvWeight(exe.upload(w), 2, cap, ds), dst, 4, oh.KvWeight(dwd, 2, budget, ds), 4, 10,
                     budget, kept, new_len)

    call()
    exe.device_status()
    gk = kept.download()
    assert list(new_len.download()) == [min(max(n, 0), budget) for n in lens]
    for b, n in enumerate(lens):
        for h in range(nkv):
            ref = _kept(w[b if slots is None else slots[b], h], n, 4, 10, budget) if n > 0 else np.arange(0)
            assert np.array_equal(gk[b, h], np.concatenate([ref, np.full(budget - len(ref), -1)]))
    pool.dl.upload(np.array([1] * 4, np.int32))  # now all have an entry
    call()
    with pytest.raises(oh.ObsError, match="paged cache"):
        exe.device_status()


def test_two_failures_are_reported_one_after_the_other():
    """A time-out of the grouped prefill (forced by its test hook) and a bad page id in one stretch of
    work: each has its own report, code and message together, and neither takes the other away."""
    E, H, I, K, T = 128, 2048, 768, 8, 64
    rng = np.random.default_rng(191)
    with oh.ObsidianExecutor(0) as exe:
        layer = oh.MoeLayer.upload(exe, synth.moe_layer(41, E, H, I, 64))
        cfg = oh.MoeConfig(E, K, H, I, 64, True)
        ids, w = synth.zipf_routing(T, E, K, 1.1, seed=5)
        ws_bytes = exe.moe_prefill_workspace(cfg, T)
        ws, Y = exe.alloc(ws_bytes, np.uint8), exe.alloc((T, H), np.uint16)
        exe.debug_ffn_wait(1, 200)
        exe.moe_prefill(cfg, layer, exe.upload(synth.bf16_normal(rng, (T, H))), Y, T, ids=exe.upload(ids), weights=exe.upload(w),
                        ws=ws, ws_bytes=ws_bytes)
        pool = Pool(exe, rng, [40], 4, 128, 16, False)
        pool.dt.upload(np.full_like(pool.table, -1))
        q, out = exe.upload(synth.bf16_normal(rng, (1, 32, 128))), exe.alloc((1, 32, 128), np.uint16)
        pws = exe.alloc(exe.sdpa_paged_workspace(pool.kv, pool.seqs(), 32), np.uint8)
        exe.sdpa_paged_decode(pool.kv, pool.seqs(), q, out, 32, pws)
        with pytest.raises(oh.ObsError, match="timed out") as ei:
            exe.device_status()
        assert ei.value.code == oh.OBS_E_HIP
        with pytest.raises(oh.ObsError, match="paged cache") as ei:
            exe.device_status()
        assert ei.value.code == oh.OBS_E_INVALID
        exe.device_status()
        assert not np.any(out.download())  # nothing visible: zeros


# ---- values that are not finite, in parts ------------------------------------------

@pytest.mark.parametrize("shape,n,new,window,bad", [
    # a window whose low edge and whose diagonal lie in different parts
    ((32, 4, 128, 32, False), 3000, 100, 1000, [1910, 1920, 2970, 2990]),
    ((16, 2, 64, 64, True), 3000, 100, 1000, [1910, 1920, 2970, 2990]),
    # parts of more than 64 blocks: page ids are fetched twice
    ((64, 64, 64, 16, False), 9000, 100, 0, [8905, 8950, 8999])], ids=str)
def test_prefill_values_not_finite_in_parts(exe, shape, n, new, window, bad):
    nh, nkv, hd, page, f8 = shape
    rng = np.random.default_rng(193)
    pool = Pool(exe, rng, [n], nkv, hd, page, f8)
    k, v = pool.entries(0, "k"), pool.entries(0, "v")
    for j in bad:
        pool.v[pool.table[0, j // page], :, :, j % page] = 0x7F if f8 else (0x7F80 if j % 4 else NAN16)
    pool.up()
    q = synth.bf16_normal(rng, (new, nh, hd), 2.0)
    out = exe.upload(np.full((new, nh, hd), FILL16, np.uint16))
    seqs = pool.seqs([0, new])
    ws = exe.upload(np.full(exe.sdpa_paged_workspace(pool.kv, seqs, nh, None, window, 0), 0xFF, np.uint8))
    exe.sdpa_paged_prefill(pool.kv, seqs, exe.upload(q), out, nh, ws, window=window)
    exe.device_status()
    got = _f64(out.download())
    clean = 0
    for r in range(new):
        vis = _visible(n - new + r, n, window, 0)
        if any(vis[j] for j in bad):
            assert not np.any(np.isfinite(got[r])), r
            continue
        clean += 1
        if r % 5 and r not in (0, new - 1):
            assert np.all(np.isfinite(got[r])), r
            continue
        ref, bound, _, _ = _attend(_f64(q[r]), k, v, vis)
        assert np.all(np.abs(got[r] - ref) <= bound), r
    assert clean == (50 if window else 5)  # the rows between the edges, or before the first bad entry
