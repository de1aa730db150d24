"""The paged cache in 4 bits without a GPU: the calls take it without scales of the
pool, refuse what they refuse of the other types, and its neighbours' numbers."""
import ctypes as C

import pytest

import obsidian_hip as oh
from test_paged_host import ALIGN, CALLS, INV, NOMEM, SHAPE, A, _evict, _kv, _seqs, _weight, ctx, host  # noqa: F401


@pytest.mark.parametrize("call", CALLS)
def test_taken_without_scales(ctx, call):  # noqa: F811
    empty = _seqs(n_seqs=0, n_rows=0)
    for scales in ({}, dict(k_scale=A, v_scale=A)):
        assert CALLS[call](ctx, _kv(dtype=oh.KV_Q4, **scales), empty) == oh.OBS_OK


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("kv,seqs,code", [
    (dict(dtype=2), {}, INV), (dict(dtype=3), {}, INV), (dict(dtype=5), {}, INV), (dict(dtype=-4), {}, INV),
    (dict(k_pages=None), {}, INV), (dict(v_pages=None), {}, INV), ({}, dict(pages=None), INV), ({}, dict(len=None), INV),
    (dict(k_pages=A + 8), {}, ALIGN), (dict(v_pages=A + 4), {}, ALIGN), (dict(page=8), {}, SHAPE), (dict(page=24), {}, SHAPE),
    (dict(page=512), {}, SHAPE), (dict(head_dim=32), {}, SHAPE), (dict(head_dim=192), {}, SHAPE), (dict(n_kv=0), {}, SHAPE),
    (dict(n_pages=1 << 31), {}, SHAPE), ({}, dict(max_pages=1 << 27), SHAPE)], ids=str)
def test_refusals(ctx, call, kv, seqs, code):  # noqa: F811
    assert CALLS[call](ctx, _kv(**{"dtype": oh.KV_Q4, **kv}), _seqs(**seqs)) == code
    assert oh.lib().obs_last_error(ctx).startswith(b"obs_")


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("nh,nkv", [(32, 4), (16, 1)])
@pytest.mark.parametrize("call", ["decode", "prefill"])
def test_workspaces(ctx, call, nh, nkv, page):  # noqa: F811
    kv = _kv(dtype=oh.KV_Q4, page=page, n_kv=nkv)
    for seqs in (_seqs(), _seqs(n_seqs=64, n_rows=64, max_pages=1024)):
        seqs.row = A if call == "prefill" else None
        n = C.c_size_t()
        assert oh.lib().obs_sdpa_paged_workspace(ctx, kv, seqs, None, nh, 0, 0, C.byref(n)) == oh.OBS_OK
        assert n.value < 1 << 31
        if n.value:
            assert CALLS[call](ctx, kv, seqs, nh=nh, n=n.value - 1) == NOMEM


def test_evict_refuses_arrays_it_reads_and_writes(ctx):  # noqa: F811
    kv, B = _kv(dtype=oh.KV_Q4), A + 4096
    own = dict(dst=B, new_len=B, dw=_weight(w=B, ld=32))
    for kw in (dict(dst=A), dict(new_len=A), dict(dw=_weight(ld=32))):
        assert _evict(ctx, kv, _seqs(), **{**own, **kw}) == INV
