"""Refusals and workspace sizes of the log probability calls without a GPU (they come
before any device work, so a context that owns no device gives them)."""
import ctypes as C

import pytest

import obsidian_hip as oh
from test_paged_host import ctx, host  # noqa: F401

A = 0x10000  # an aligned address that is never followed
INV, SHAPE, ALIGN, NOMEM = oh.OBS_E_INVALID, oh.OBS_E_SHAPE, oh.OBS_E_ALIGN, oh.OBS_E_NOMEM


def _logits(ctx, **kw):
    d = dict(x=A, dtype=0, T=2, V=1000, ld=0, tok=A, lp=A, ent=A, k=3, ids=A, tlp=A, ws=A, n=1 << 40)
    d.update(kw)
    return oh.lib().obs_token_logprobs(ctx, d["x"], d["dtype"], d["T"], d["V"], d["ld"], d["tok"], d["lp"], d["ent"], d["k"],
                                       d["ids"], d["tlp"], d["ws"], d["n"])


def _lm(ctx, **kw):
    d = dict(x=A, w=A, s=A, b=A, T=2, H=512, V=1000, group=64, tok=A, lp=A, ent=A, k=3, ids=A, tlp=A, ws=A, n=1 << 40)
    d.update(kw)
    return oh.lib().obs_lm_logprobs(ctx, d["x"], d["w"], d["s"], d["b"], d["T"], d["H"], d["V"], d["group"], d["tok"], d["lp"],
                                    d["ent"], d["k"], d["ids"], d["tlp"], d["ws"], d["n"])


BOTH = [(dict(ws=None), INV), (dict(tok=None), INV), (dict(lp=None), INV), (dict(ids=None), INV), (dict(tlp=None), INV),
        (dict(k=65), SHAPE), (dict(V=2), SHAPE), (dict(V=0), SHAPE), (dict(V=(1 << 24) + 1), SHAPE), (dict(T=(1 << 24) + 1), SHAPE),
        (dict(ws=A + 8), ALIGN), (dict(n=15), NOMEM), (dict(x=None), INV)]


@pytest.mark.parametrize("kw,code", BOTH + [(dict(dtype=2), INV), (dict(dtype=-1), INV), (dict(ld=999), SHAPE), (dict(x=A + 2), ALIGN),
                                            (dict(dtype=1, x=A + 1), ALIGN)], ids=str)
def test_logits_refusals(ctx, kw, code):  # noqa: F811
    assert _logits(ctx, **kw) == code
    assert oh.lib().obs_last_error(ctx)


@pytest.mark.parametrize("kw,code", BOTH + [(dict(H=0), SHAPE), (dict(H=256), SHAPE), (dict(H=520), SHAPE), (dict(H=16896), SHAPE),
                                            (dict(group=32), SHAPE), (dict(w=None), INV), (dict(s=None), INV), (dict(b=None), INV),
                                            (dict(x=A + 8), ALIGN), (dict(w=A + 4), ALIGN), (dict(s=A + 2), ALIGN), (dict(b=A + 8), ALIGN)],
                         ids=str)
def test_lm_refusals(ctx, kw, code):  # noqa: F811
    assert _lm(ctx, **kw) == code
    assert oh.lib().obs_last_error(ctx)


def test_empty_calls_need_nothing(ctx):  # noqa: F811
    assert _logits(ctx, T=0, x=None, ws=None, n=0) == oh.OBS_OK
    assert _lm(ctx, T=0, x=None, w=None, s=None, b=None, ws=None, n=0) == oh.OBS_OK


def test_workspaces(ctx):  # noqa: F811
    n = C.c_size_t()
    L = oh.lib()
    sizes = []
    for T in (0, 1, 7, 700, 5000):
        assert L.obs_token_logprobs_workspace(ctx, T, 151936, 0, 5, C.byref(n)) == oh.OBS_OK
        sizes.append(n.value)
        assert _logits(ctx, T=T, V=151936, k=5, n=n.value - 1 if T else 0) == (NOMEM if T else oh.OBS_OK)
    assert sizes == sorted(sizes) and sizes[0] == 0
    assert L.obs_token_logprobs_workspace(ctx, 1, 0, 0, 0, C.byref(n)) == SHAPE and n.value == 0
    assert L.obs_token_logprobs_workspace(ctx, 1, 10, 3, 0, C.byref(n)) == INV
    assert L.obs_token_logprobs_workspace(ctx, 1, 10, 0, 0, None) == INV
    for T in (1, 32, 33, 300, 100000):
        for k in (0, 5):
            assert L.obs_lm_logprobs_workspace(ctx, T, 2048, 151936, k, C.byref(n)) == oh.OBS_OK
            # the sums of a pass at most, and the logits of no more than 256 rows
            assert 0 < n.value < (4096 if k == 0 else 256) * (594 * 16 + 2048 * 2 + 4096) + (256 * 151936 * 4 if k else 0) + (1 << 22)
            assert _lm(ctx, T=T, H=2048, V=151936, k=k, n=n.value - 1) == NOMEM
    assert L.obs_lm_logprobs_workspace(ctx, 1, 100, 10, 0, C.byref(n)) == SHAPE
