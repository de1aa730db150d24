"""Calls on the paged cache (obs_attn_prep_paged, obs_sdpa_paged_prefill, obs_kv_evict,
obs_device_status) that the documentation allows and that are easily answered
wrongly: positions past the RoPE table's, far positions, tables that grow,
padded batches, several device failures at once. Helpers, pools and bars as in
test_gpu_paged.py; a test that needs another bar derives it beside it."""
import numpy as np
import pytest

import obsidian_hip as oh
from obsidian_hip import synth
from test_gpu_paged import (E4M3, EPS, FILL16, NAN16, SHAPES, THETA, Pool, _attend, _bf16, _check_prep, _e4m3_bytes, _f64, _kept,
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
