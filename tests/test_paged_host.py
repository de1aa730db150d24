"""The paged cache's host side without a GPU: every refusal (they come before any
device work, so a context that owns no device gives them), the workspace sizes,
and the functions that turn lengths, rows, page ids and windows into what a
kernel reads, at their edges and with garbage in the device arrays.

No counterpart in the reference, whose KvCache holds one sequence
(src/kv_cache.rs:5-24)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import obsidian_hip as oh

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 0x10000  # an aligned address that is never followed


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("paged") / "paged_host.so")
    subprocess.run(["/opt/rocm/bin/hipcc", "-O1", "-std=c++17", "-x", "hip", "--offload-host-only", "-fPIC", "-shared", "-w",
                    os.path.join(ROOT, "tests", "paged_host.cpp"), "-o", so], check=True)
    h = C.CDLL(so)
    h.bare_ctx.restype = C.c_void_p
    h.bare_free.argtypes = [C.c_void_p]
    return h


@pytest.fixture
def ctx(host):
    c = host.bare_ctx()
    yield c
    host.bare_free(c)


def _kv(**kw):
    d = dict(k_pages=A, v_pages=A, k_scale=None, v_scale=None, n_pages=8, page=16, n_kv=4, head_dim=128, dtype=0)
    d.update(kw)
    return oh.ObsPagedKv(**d)


def _seqs(**kw):
    d = dict(pages=A, len=A, row=None, n_seqs=2, max_pages=4, n_rows=2)
    d.update(kw)
    return oh.ObsPagedSeqs(**d)


def _weight(**kw):
    d = dict(w=A, slot=None, n_slots=2, ld=64)
    d.update(kw)
    return oh.ObsKvWeight(**d)


def _prep(ctx, kv, seqs, weight=None, **kw):
    d = dict(q=A, k=A, v=A, qn=A, kn=A, qo=A, nh=32, eps=1e-6, theta=1e7, pos=None, rope=64, q_ld=0, kv_ld=0, o_ld=0)
    d.update(kw)
    return oh.lib().obs_attn_prep_paged(ctx, kv, seqs, weight, d["q"], d["k"], d["v"], d["qn"], d["kn"], d["qo"], d["nh"],
                                        d["eps"], d["theta"], d["pos"], d["rope"], d["q_ld"], d["kv_ld"], d["o_ld"])


def _decode(ctx, kv, seqs, weight=None, **kw):
    d = dict(q=A, out=A, nh=32, window=0, sinks=0, q_ld=0, ws=A, n=1 << 40)
    d.update(kw)
    return oh.lib().obs_sdpa_paged_decode(ctx, kv, seqs, weight, d["q"], d["out"], d["nh"], d["window"], d["sinks"],
                                          d["q_ld"], d["ws"], d["n"])


def _prefill(ctx, kv, seqs, weight=None, **kw):
    d = dict(q=A, out=A, nh=32, window=0, sinks=0, q_ld=0, ws=A, n=1 << 40)
    d.update(kw)
    if seqs is not None and not d.pop("no_row", False):
        seqs.row = A
    return oh.lib().obs_sdpa_paged_prefill(ctx, kv, seqs, d["q"], d["out"], d["nh"], d["window"], d["sinks"], d["q_ld"],
                                           d["ws"], d["n"])


def _evict(ctx, kv, seqs, weight="own", **kw):
    d = dict(dst=A, dmax=2, dw=_weight(ld=32), sinks=4, recent=8, budget=32, kept=A, new_len=A)
    d.update(kw)
    return oh.lib().obs_kv_evict(ctx, kv, seqs, _weight() if weight == "own" else weight, d["dst"], d["dmax"], d["dw"],
                                 d["sinks"], d["recent"], d["budget"], d["kept"], d["new_len"])


CALLS = {"prep": _prep, "decode": _decode, "prefill": _prefill, "evict": _evict}
INV, SHAPE, ALIGN, NOMEM = oh.OBS_E_INVALID, oh.OBS_E_SHAPE, oh.OBS_E_ALIGN, oh.OBS_E_NOMEM


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("kv,seqs,code", [
    (dict(k_pages=None), {}, INV), (dict(v_pages=None), {}, INV), ({}, dict(pages=None), INV), ({}, dict(len=None), INV),
    (dict(dtype=2), {}, INV), (dict(dtype=1), {}, INV), (dict(dtype=1, k_scale=A), {}, INV),
    (dict(k_pages=A + 8), {}, ALIGN), (dict(v_pages=A + 2), {}, ALIGN),
    (dict(page=8), {}, SHAPE), (dict(page=48), {}, SHAPE), (dict(page=512), {}, SHAPE), (dict(head_dim=96), {}, SHAPE),
    (dict(n_kv=0), {}, SHAPE), (dict(n_kv=1025), {}, SHAPE), (dict(n_pages=0), {}, SHAPE),
    (dict(n_pages=1 << 31), {}, SHAPE), ({}, dict(n_seqs=4097), SHAPE), ({}, dict(max_pages=0), SHAPE),
    ({}, dict(max_pages=1 << 27), SHAPE), ({}, dict(n_rows=(1 << 24) + 1), SHAPE)])
def test_bad_pool_and_sequences(ctx, call, kv, seqs, code):
    assert CALLS[call](ctx, _kv(**kv), _seqs(**seqs)) == code
    assert oh.lib().obs_last_error(ctx).startswith(b"obs_")


@pytest.mark.parametrize("call", CALLS)
def test_null_structures(ctx, call):
    assert CALLS[call](ctx, None, _seqs()) == INV
    assert CALLS[call](ctx, _kv(), None) == INV


@pytest.mark.parametrize("call", ["prep", "decode", "prefill"])
@pytest.mark.parametrize("kw,code", [(dict(nh=30), SHAPE), (dict(nh=0), SHAPE), (dict(nh=68), SHAPE), (dict(q=None), INV),
                                     (dict(q=A + 8), ALIGN), (dict(q_ld=4088), SHAPE), (dict(q_ld=4100), SHAPE)])
def test_bad_heads_and_queries(ctx, call, kw, code):
    assert CALLS[call](ctx, _kv(), _seqs(), **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), INV), (dict(v=None), INV), (dict(qn=None), INV), (dict(kn=None), INV), (dict(qo=None), INV),
    (dict(k=A + 4), ALIGN), (dict(v=A + 2), ALIGN), (dict(qn=A + 8), ALIGN), (dict(kn=A + 8), ALIGN),
    (dict(qo=A + 8), ALIGN), (dict(kv_ld=504), SHAPE), (dict(o_ld=4090), SHAPE), (dict(q_ld=5120, qo=A), INV),
    (dict(rope=0), SHAPE), (dict(rope=(1 << 24) + 1), SHAPE)])
def test_prep_refusals(ctx, kw, code):
    assert _prep(ctx, _kv(), _seqs(), **kw) == code


def test_rows_have_to_fit_the_call(ctx):
    assert _prep(ctx, _kv(), _seqs(n_rows=3)) == SHAPE      # no row array: one token a sequence
    assert _decode(ctx, _kv(), _seqs(n_rows=3)) == SHAPE
    assert _decode(ctx, _kv(), _seqs(row=A)) == SHAPE
    assert _prefill(ctx, _kv(), _seqs(), no_row=True) == INV


@pytest.mark.parametrize("call", ["prep", "decode"])
@pytest.mark.parametrize("w,code", [(dict(w=None), INV), (dict(w=A + 2), ALIGN), (dict(n_slots=0), SHAPE), (dict(ld=63), SHAPE)])
def test_bad_weight(ctx, call, w, code):
    assert CALLS[call](ctx, _kv(), _seqs(), _weight(**w)) == code


@pytest.mark.parametrize("call", ["decode", "prefill"])
def test_workspace_refusals(ctx, call):
    kv, seqs = _kv(), _seqs()
    seqs.row = A if call == "prefill" else None
    n = C.c_size_t()
    assert oh.lib().obs_sdpa_paged_workspace(ctx, kv, seqs, None, 32, 0, 0, C.byref(n)) == oh.OBS_OK
    assert 0 < n.value < 1 << 30
    assert CALLS[call](ctx, kv, seqs, n=n.value - 1) == NOMEM
    assert CALLS[call](ctx, kv, seqs, ws=None) == INV
    assert CALLS[call](ctx, kv, seqs, ws=A + 8) == ALIGN
    assert CALLS[call](ctx, kv, seqs, out=None) == INV
    assert CALLS[call](ctx, kv, seqs, out=A + 8) == ALIGN


def test_workspace_by_sizes_alone(ctx):
    def need(kv, seqs, weight=None, nh=32, window=0, sinks=0):
        n = C.c_size_t(7)
        rc = oh.lib().obs_sdpa_paged_workspace(ctx, kv, seqs, weight, nh, window, sinks, C.byref(n))
        return n.value if rc == oh.OBS_OK else rc

    bare = dict(k_pages=None, v_pages=None)
    seqs = dict(pages=None, len=None)
    assert need(_kv(**bare), _seqs(**seqs)) > 0  # pointers are not read
    assert need(_kv(page=17), _seqs()) == SHAPE and need(_kv(), _seqs(), nh=31) == SHAPE
    assert need(None, _seqs()) == INV and need(_kv(), None) == INV
    assert oh.lib().obs_sdpa_paged_workspace(ctx, _kv(), _seqs(), None, 32, 0, 0, None) == INV
    # gathering weights holds every visible score of every head; a window bounds them
    long = _seqs(max_pages=4096)
    plain, gathers = need(_kv(), long), need(_kv(), long, _weight(ld=1 << 16))
    assert gathers - plain >= 2 * 32 * 65536 * 4
    assert need(_kv(), long, _weight(ld=1 << 16), window=1000, sinks=4) < plain + 2 * 32 * 1200 * 4 + 4096


@pytest.mark.parametrize("kw,code", [
    (dict(dst=None), INV), (dict(kept=None), INV), (dict(new_len=None), INV), (dict(weight=None), INV),
    (dict(dw=None), INV), (dict(dw=_weight(ld=31)), SHAPE), (dict(weight=_weight(ld=63)), SHAPE),
    (dict(budget=0, sinks=0, recent=0), SHAPE), (dict(sinks=25), SHAPE), (dict(sinks=0xffffffff, recent=0xffffffff), SHAPE),
    (dict(budget=33, dw=_weight(ld=64)), SHAPE), (dict(dmax=0), SHAPE), (dict(dmax=1 << 27), SHAPE)])
def test_evict_refusals(ctx, kw, code):
    assert _evict(ctx, _kv(), _seqs(), **kw) == code


def test_evict_refuses_arrays_it_reads_and_writes(ctx):
    B = A + 4096
    own = dict(dst=B, new_len=B, dw=_weight(w=B, ld=32))
    for kw in (dict(dst=A), dict(new_len=A), dict(dw=_weight(ld=32))):
        assert _evict(ctx, _kv(), _seqs(), **{**own, **kw}) == INV


def test_more_than_a_launch_holds(ctx):
    """2^32 threads and more are refused before any device work."""
    rows = dict(n_seqs=4096, n_rows=1 << 24)
    assert _prep(ctx, _kv(), _seqs(row=A, **rows)) == SHAPE
    assert _prefill(ctx, _kv(n_kv=1024), _seqs(**rows), nh=16 * 1024) == SHAPE
    assert _decode(ctx, _kv(n_kv=1024), _seqs(n_seqs=4096, n_rows=4096), nh=16 * 1024) == SHAPE
    wide = _seqs(n_seqs=512, n_rows=512, max_pages=1 << 26)
    assert _decode(ctx, _kv(), wide, _weight(n_slots=512, ld=1 << 30), nh=32, n=1 << 60) == SHAPE
    B = A + 4096
    assert _evict(ctx, _kv(n_kv=1024), _seqs(n_seqs=4096, n_rows=4096), dst=B, new_len=B, dw=_weight(w=B, ld=32)) == SHAPE
    assert _evict(ctx, _kv(), wide, _weight(n_slots=512, ld=1 << 30), dst=B, new_len=B, dmax=1 << 26,
                  dw=_weight(w=B, ld=1 << 30), budget=1 << 30) == SHAPE


def test_nothing_to_do(ctx):
    """No sequences: success without a launch (this context has no device)."""
    empty = dict(n_seqs=0, n_rows=0)
    assert _prep(ctx, _kv(), _seqs(**empty)) == oh.OBS_OK
    assert _decode(ctx, _kv(), _seqs(**empty)) == oh.OBS_OK
    assert _prefill(ctx, _kv(), _seqs(**empty)) == oh.OBS_OK
    assert _evict(ctx, _kv(), _seqs(**empty)) == oh.OBS_OK


# ---- what a kernel reads ----------------------------------------------------

def _span(host, i0, hi, window, sinks):
    out = (C.c_uint32 * (5 + 4096))()
    host.span(i0, hi, window, sinks, out, 4096)
    return list(out[:5]), list(out[5:5 + out[4]])


@pytest.mark.parametrize("sinks", [0, 1, 4, 31, 32, 33, 100, 5000, 0xffffffff])
@pytest.mark.parametrize("window", [0, 1, 2, 31, 32, 33, 64, 100, 4000, 0xffffffff])
@pytest.mark.parametrize("rows", [1, 2, 16, 40])
def test_span_lists_every_visible_block_once(host, rows, window, sinks):
    """The listed blocks hold every entry that a row of the tile sees, none twice,
    in order, and none past the last entry."""
    for hi in (1, 2, 16, 31, 32, 33, 63, 64, 65, 100, 129, 1000, 2049):
        i0 = max(0, hi - rows)
        (h, lo, sb, wb, nblk), starts = _span(host, i0, hi, window, sinks)
        seen = {j // 32 for i in range(i0, hi) for j in range(i + 1)
                if window == 0 or j > i - window or j < sinks}
        assert h == hi and starts == sorted(set(starts)) and all(t % 32 == 0 and t < hi for t in starts)
        assert seen <= {t // 32 for t in starts}
        if rows == 1:
            assert seen == {t // 32 for t in starts}


def test_span_of_nothing(host):
    assert _span(host, 0, 0, 0, 0)[0][4] == 0 and _span(host, 0, 0, 16, 4)[0][4] == 0


def test_garbage_in_the_device_arrays_stays_in_bounds(host):
    """Lengths, rows and page ids of any value give an entry of the pool, rows of
    the call and table words of the sequence's own row."""
    rng = np.random.default_rng(7)
    big = np.array([-2**31, -1, 0, 1, 5, 7, 8, 9, 63, 64, 65, 2**30, 2**31 - 1], np.int32)
    out = np.zeros(6, np.int64)
    for _ in range(400):
        B, mp, lp = int(rng.integers(1, 4)), int(rng.integers(1, 5)), int(rng.integers(4, 9))
        n_pages, n_rows = int(rng.integers(1, 10)), int(rng.integers(0, 9))
        table, ln, row = (rng.choice(big, n).astype(np.int32) for n in (B * mp, B, B + 1))
        b, j = int(rng.integers(0, B)), int(rng.integers(0, 2**31))
        host.entry(table.ctypes.data_as(C.c_void_p), ln.ctypes.data_as(C.c_void_p), row.ctypes.data_as(C.c_void_p),
                   n_pages, lp, B, mp, n_rows, b, j, out.ctypes.data_as(C.c_void_p))
        idx = min(j >> lp, mp - 1)
        want = int(table[b * mp + idx])
        ok = 0 <= want < n_pages
        assert bool(out[1]) == ok and out[0] == (want if ok else 0)
        assert out[2] == min(max(int(ln[b]), 0), mp << lp) and bool(out[3]) == (int(ln[b]) > mp << lp)
        assert 0 <= out[4] <= out[5] <= n_rows


@pytest.mark.parametrize("t", [0, 32, 64, (1 << 30) - 32])
def test_masks_of_a_block(host, t):
    """A bit each for the entries below hi that are at or above lo or among the first tokens."""
    edges = [0, 1, 31, 32, 33, 50, 63, 64, 65, 96, 1000, t, t + 1, t + 16, t + 31, t + 32, t + 33, 1 << 30]
    host.seen.restype = C.c_uint32
    for hi in edges:
        for lo in edges:
            for sinks in [*edges, 0xffffffff]:
                ref = sum(1 << j for j in range(32) if t + j < hi and (t + j >= lo or t + j < sinks))
                assert host.seen(C.c_uint32(t), C.c_uint32(hi), C.c_uint32(lo), C.c_uint32(sinks)) == ref, (hi, lo, sinks)


def test_rope_tables_grow_by_doubling(host):
    """Whatever lengths a caller goes through, it meets few tables, each holding all of its positions."""
    host.rope_rows.restype = C.c_uint32
    assert [host.rope_rows(n) for n in (1, 8191, 8192, 8193, 16384, 16385)] == [8192, 8192, 8192, 16384, 16384, 32768]
    sizes = {host.rope_rows(n) for n in [*range(1, 70000, 13), 1 << 20, (1 << 24) - 1, 1 << 24]}
    assert sizes == {1 << i for i in (13, 14, 15, 16, 17, 20, 24)}
    for n in (1, 4097, 8193, 100_003, (1 << 23) + 1, 1 << 24):
        assert n <= host.rope_rows(n) <= max(8192, 2 * n - 1)


def test_a_batch_with_rows_names_their_number():
    """PagedSeqs takes one row a sequence only where there is no row array: with one, the rows behind
    the first n_seqs would be left out without a word."""
    with pytest.raises(ValueError, match="n_rows"):
        oh.PagedSeqs(A, A, 3, 4, row=A)
    assert oh.PagedSeqs(A, A, 3, 4, 17, A).c.n_rows == 17 and oh.PagedSeqs(A, A, 3, 4).c.n_rows == 3


def test_an_empty_batch_needs_no_workspace(ctx):
    """A call gets by with exactly what obs_sdpa_paged_workspace names, which for no sequences may be nothing."""
    n, none = C.c_size_t(7), _seqs(n_seqs=0, n_rows=0)
    assert oh.lib().obs_sdpa_paged_workspace(ctx, _kv(), none, None, 32, 0, 0, C.byref(n)) == oh.OBS_OK
    assert n.value == 0 and _decode(ctx, _kv(), none, ws=None, n=0) == oh.OBS_OK
    assert _decode(ctx, _kv(), _seqs(), ws=None, n=0) == INV
