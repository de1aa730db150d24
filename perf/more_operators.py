"""Operators around a cache of 4 bits and around what a model answers with, as
cases that can be timed and checked: attention over a paged key/value cache whose
entries are held in 4 bits (one new token a sequence, or a batch of prompt tokens;
with the new entries appended first or there already), and the log probabilities
of given tokens with the entropy and the most likely alternatives, from logits or
from hidden rows and the 4-bit output matrix.

The cache is a pool of pages; a sequence is a row of page ids and a length. A
group of 64 dims of an entry is q * scale + bias with q in 0 .. 15 and scale and
bias in bf16. A (page, kv head) of keys is [entry][dim / 2] bytes, byte i holding
dim i (low) and dim i + dim / 2 (high), then uint32 [group][entry]: the scale
(low half) and the bias. Values are [dim / 2][entry] bytes and then the same.

`run` has every operator in its plain form (torch, 32 bits); with `own` set it
calls the library. Lengths go by the case alone, everything else by the seed.
"""
import math
import random

import torch

own = False

EPS, THETA, GROUP = 1e-6, 1e7, 64


def listed():
    qwen = {"heads": 32, "kv": 4, "dim": 128}
    whole = {"window": 0, "sinks": 0, "weight": False, "append": False}
    lm = {"hidden": 2048, "vocab": 151936}
    return [
        # one user, early in a conversation: latency
        {"name": "decode_one_short", "kind": "decode", **qwen, "page": 16, "seqs": 1, "len": 517, **whole},
        # one user with a very long document
        {"name": "decode_one_long", "kind": "decode", **qwen, "page": 64, "seqs": 1, "len": 100003, **whole},
        # a layer's step of a batch of conversations of all lengths: the new entries in, then attention
        {"name": "decode_batch", "kind": "decode", **qwen, "page": 32, "seqs": 48, "len": 16000, **whole, "append": True},
        # streams under a window whose cache is evicted from: the weights are gathered
        {"name": "decode_window", "kind": "decode", **qwen, "page": 32, "seqs": 16, "len": 24001, "window": 8192,
         "sinks": 4, "weight": True, "append": False},
        # short follow-up messages over long conversations, appended and attended
        {"name": "prefill_follow_ups", "kind": "prefill", **qwen, "page": 32, "seqs": 5, "len": 6000, "tokens": 150,
         **whole, "append": True},
        # a prompt into an empty cache
        {"name": "prefill_prompt", "kind": "prefill", **qwen, "page": 64, "seqs": 1, "len": 5001, "tokens": 5001, **whole},
        # one sampled token: its log probability and five alternatives
        {"name": "logprobs_one", "kind": "logprobs", "rows": 1, "vocab": 151936, "dtype": "fp32", "top": 5, "pad": 0},
        # a decode step of a batch, with the twenty alternatives that an API offers at most
        {"name": "logprobs_step", "kind": "logprobs", "rows": 48, "vocab": 151936, "dtype": "fp32", "top": 20, "pad": 0},
        # the logits of a prompt, kept in bf16 in rows of a padded vocabulary
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 777, "vocab": 151669, "dtype": "bf16", "top": 1, "pad": 267},
        # the same from the hidden row: one token, a decode step of a batch, and the scoring of a prompt
        {"name": "lm_one", "kind": "lm", "rows": 1, **lm, "top": 5},
        {"name": "lm_step", "kind": "lm", "rows": 24, **lm, "top": 5},
        {"name": "lm_prompt", "kind": "lm", "rows": 2000, **lm, "top": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prefill", "prefill", "logprobs", "lm", "lm"])
    if kind == "logprobs":
        vocab = _log(rng, 300, 151936)
        return {"kind": kind, "rows": _log(rng, 1, max(1, min(4000, 110_000_000 // vocab))), "vocab": vocab,
                "dtype": rng.choice(["fp32", "bf16"]), "top": rng.choice([0, 1, 5, rng.randint(2, 20)]),
                "pad": rng.choice([0, 0, rng.randint(1, 300)])}
    if kind == "lm":
        hidden, vocab = rng.choice([2048, 2048, 1024, 4096]), rng.choice([151936, _log(rng, 2000, 151936)])
        rows = _log(rng, 1, min(2000, 600_000_000_000 // (hidden * vocab)))
        # (alternatives of few rows: the order of near-equal logits of many is not settled in 32 bits)
        return {"kind": kind, "rows": rows, "hidden": hidden, "vocab": vocab, "top": rng.randint(0, 5) if rows <= 24 else 0}
    heads, kv = rng.choice([(32, 4), (32, 4), (32, 8), (16, 16), (8, 1), (12, 2), (16, 1)])
    windowed = rng.random() < 0.4
    case = {"kind": kind, "heads": heads, "kv": kv, "dim": rng.choice([128, 128, 64]),
            "page": rng.choice([16, 32, 64, 128]), "window": _log(rng, 16, 8000) if windowed else 0,
            "sinks": rng.choice([0, 4, rng.randint(1, 200)]) if windowed else 0, "weight": False,
            "append": rng.random() < 0.5}
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        return {**case, "seqs": seqs, "len": _log(rng, 1, min(60000, 400000 // seqs)), "weight": rng.random() < 0.3}
    tokens = _log(rng, 1, 4000)
    seqs = _log(rng, 1, max(1, min(16, 4000 // tokens)))
    return {**case, "seqs": seqs, "len": tokens + rng.choice([0, _log(rng, 1, 8000)]), "tokens": tokens}


# ---- sizes, by the case alone ----------------------------------------------

def _spread(case, most, least, salt):
    """One size a sequence, from `least` to `most`, log-uniform; the first is `most`."""
    r = random.Random("%s %d %d %d" % (salt, case["seqs"], most, case["page"]))
    return [most] + [_log(r, least, most) for _ in range(case["seqs"] - 1)]


def _tokens(case):
    """New tokens of each sequence."""
    n = case.get("tokens", 1)
    return _spread(case, n, max(1, n // 8), "tokens")


def _lens(case):
    """Entries of each sequence, its new tokens included."""
    lens = _spread(case, case["len"], max(1, case["len"] // 8), "len")
    return [max(n, t) for n, t in zip(lens, _tokens(case))]


def _seen(n, window, sinks):
    """Entries that the token at the end of n entries attends to."""
    return n if window == 0 or n <= window else window + min(sinks, n - window)


# ---- 4 bits ------------------------------------------------------------------

def _quantized(x):
    """q (0 .. 15, as x), scale and bias (bf16 values, as x [..., groups]) of x [..., dim]."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    s, b = ((hi - lo) / 15.0).bfloat16().to(x.dtype), lo.bfloat16().to(x.dtype)
    step = torch.where(s > 0, s, 1.0).unsqueeze(-1)
    q = ((g - b.unsqueeze(-1)) / step).round_().clamp_(0.0, 15.0)
    return torch.where(s.unsqueeze(-1) > 0, q, 0.0).flatten(-2), s, b


def _bytes_of(q):
    """[..., dim] whole numbers 0 .. 15 -> [..., dim / 2] bytes."""
    low, high = q.to(torch.uint8).chunk(2, -1)
    return low | high << 4


def _params(s, b):
    """Scales and biases -> int32 [..., groups]."""
    word = torch.stack([s.bfloat16(), b.bfloat16()], -1).contiguous()
    return word.view(torch.int32).squeeze(-1)


class _Side:
    """The keys (or values) of a pool: bytes [page, kv head, ...], and views of its nibbles and of its parameters."""

    def __init__(self, pool, case, values):
        page, half, groups = case["page"], case["dim"] // 2, case["dim"] // GROUP
        self.pool, self.values = pool, values
        data = pool[..., :page * half]
        # [pages, kv, entry, byte] and [pages, kv, entry, group, (scale, bias)]
        self.data = data.unflatten(-1, (half, page)).transpose(-1, -2) if values else data.unflatten(-1, (page, half))
        self.params = pool.view(torch.bfloat16)[..., page * half // 2:].unflatten(-1, (groups, page, 2)).transpose(2, 3)

    def entries(self, ids, dtype):
        """[..., kv, page, dim] values of pages `ids`."""
        x, p = self.data[ids], self.params[ids].to(dtype)
        q = torch.cat([x & 15, x >> 4], -1).to(dtype).unflatten(-1, (-1, GROUP))
        return torch.addcmul(p[..., 1:], q, p[..., :1]).flatten(-2)

    def put(self, page, off, x):
        """Rows x [R, kv, dim] at entry off of each page."""
        q, s, b = _quantized(x)
        self.data[page, :, off] = _bytes_of(q)
        self.params[page, :, off] = torch.stack([s, b], -1).bfloat16()


# ---- inputs -----------------------------------------------------------------

class _State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def _q4_matrix(rows, cols, g):
    """A 4-bit affine matrix: uint32-packed weight, scales and biases, as a quantised normal one has them."""
    dev = "cuda"
    w = torch.randint(-2**31, 2**31, (rows, cols // 8), generator=g, device=dev, dtype=torch.int64).to(torch.int32)
    s = ((0.8 + 0.4 * torch.rand((rows, cols // GROUP), generator=g, device=dev)) * 0.009).bfloat16()
    b = (s.float() * (-7.5 + 0.5 * torch.randn((rows, cols // GROUP), generator=g, device=dev))).bfloat16()
    return w, s, b


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dev, kind = "cuda", case["kind"]
    if kind in ("logprobs", "lm"):
        R, V, top = case["rows"], case["vocab"], case["top"]
        st = _State(case=case, tokens=torch.randint(0, V, (R,), generator=g, device=dev, dtype=torch.int32),
                    logprob=torch.empty(R, device=dev), entropy=torch.empty(R, device=dev),
                    top_ids=torch.empty((R, top), dtype=torch.int32, device=dev) if top else None,
                    top_lp=torch.empty((R, top), device=dev) if top else None)
        if R > 3:  # a padded row has no token
            st.tokens[torch.randint(0, R, (1,), generator=g, device=dev)] = -1
        if kind == "lm":
            st.w, st.s, st.b = _q4_matrix(V, case["hidden"], g)
            st.x = torch.randn((R, case["hidden"]), generator=g, device=dev).bfloat16()
        else:
            t = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
            st.logits = (torch.randn((R, V + case["pad"]), generator=g, device=dev) * 2.5 - 1.0).to(t)
            likely = torch.randint(0, V, (R, 4), generator=g, device=dev)  # a few likely tokens, some forbidden ones
            st.logits.scatter_add_(1, likely, (6.0 + 6.0 * torch.rand((R, 4), generator=g, device=dev)).to(t))
            st.logits[:, torch.randint(0, V, (max(1, V // 500),), generator=g, device=dev)] = -math.inf
        torch.cuda.synchronize()
        return st
    kv, dim, page, heads, B = case["kv"], case["dim"], case["page"], case["heads"], case["seqs"]
    lens, toks = _lens(case), _tokens(case)
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + 3
    ids = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32).cpu()
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = ids[at:at + need[b]]
        at += need[b]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16) * scale

    # a pool of entries that were quantised; some dims of keys are larger than others
    gain = torch.exp(0.5 * torch.randn((kv, 1, dim), generator=g, device=dev))
    pools = []
    for values in (False, True):
        parts = []
        for first in range(0, n_pages, 4096 // page * 16):
            x = torch.randn((min(4096 // page * 16, n_pages - first), kv, page, dim), generator=g, device=dev)
            q, s, b = _quantized(x if values else x * gain)
            data, words = _bytes_of(q), _params(s, b).transpose(2, 3).contiguous().view(torch.uint8)
            data = data.transpose(2, 3) if values else data
            parts.append(torch.cat([data.flatten(2), words.flatten(2)], -1))
        pools.append(torch.cat(parts))
    rows = [0]
    for t in toks:
        rows.append(rows[-1] + t)
    R = rows[-1]
    st = _State(case=case, k=_Side(pools[0], case, False), v=_Side(pools[1], case, True), table=table.to(dev),
                n_pages=n_pages, len=torch.tensor(lens, dtype=torch.int32, device=dev), rows=R, most=max(toks),
                row=torch.tensor(rows, dtype=torch.int32, device=dev) if kind == "prefill" else None, weight=None)
    cap = table.shape[1] * page
    if case["weight"]:
        st.slot = torch.randperm(B + 1, generator=g, device=dev)[:B].to(torch.int32)
        st.weight = torch.rand((B + 1, kv, cap), generator=g, device=dev) ** 6 * 4.0
    if case["append"]:  # q, k and v as column ranges of one projection's output rows
        st.qkv = normal(R, (heads + 2 * kv) * dim, scale=2.0)
        st.q_norm, st.k_norm = 1.0 + normal(dim, scale=0.1), 1.0 + normal(dim, scale=0.1)
        st.q = torch.empty((R, heads, dim), dtype=torch.bfloat16, device=dev)
    else:
        st.q = normal(R, heads, dim, scale=2.0)
    st.out = torch.empty((R, heads, dim), dtype=torch.bfloat16, device=dev)
    torch.cuda.synchronize()
    return st


# ---- one pass ---------------------------------------------------------------

def run(st):
    if own:
        return _call(st)
    return {"decode": _attend, "prefill": _attend, "logprobs": _logprobs, "lm": _lm}[st.case["kind"]](st)


def _outputs(st):
    """An appended nibble next to a border of its rounding may fall to either side: nibbles are compared by what the
    attention reads from them, the entries' scales and biases by themselves."""
    out = {"out": st.out, "weight": st.weight}
    if st.case["append"]:
        out.update(q=st.q, k_params=st.k.params, v_params=st.v.params)
    return out


def _scores(st):
    return {"logprob": st.logprob, "entropy": st.entropy, "top_ids": st.top_ids, "top_logprobs": st.top_lp}


def _call(st):
    """The library's calls, as a program with an executor, a workspace and a handle a cache makes them."""
    c, exe = st.case, _executor()
    if c["kind"] in ("logprobs", "lm"):
        args = dict(tokens=_at(st.tokens), logprob=_at(st.logprob), entropy=_at(st.entropy), top_k=c["top"],
                    top_ids=_at(st.top_ids), top_logprobs=_at(st.top_lp))
        if c["kind"] == "lm":
            ws = _workspace(exe.lm_logprobs_workspace(c["rows"], c["hidden"], c["vocab"], c["top"]))
            exe.lm_logprobs(st.x.data_ptr(), st.w.data_ptr(), st.s.data_ptr(), st.b.data_ptr(), c["rows"], c["hidden"],
                            c["vocab"], ws=ws.data_ptr(), ws_bytes=ws.numel(), **args)
        else:
            oh = _library()
            ws = _workspace(exe.token_logprobs_workspace(c["rows"], c["vocab"], c["top"]))
            exe.token_logprobs(st.logits.data_ptr(), c["rows"], c["vocab"], ws=ws.data_ptr(), ws_bytes=ws.numel(),
                               dtype=oh.LOGITS_F32 if c["dtype"] == "fp32" else oh.LOGITS_BF16, ld=c["vocab"] + c["pad"],
                               **args)
        return _scores(st)
    if not hasattr(st, "handle"):
        st.handle = _handle(st)
    kv, seqs, weight = st.handle
    if c["append"]:
        q, nq, nk = st.qkv.data_ptr(), 2 * c["heads"] * c["dim"], 2 * c["kv"] * c["dim"]
        ld = st.qkv.shape[1]
        exe.attn_prep_paged(kv, seqs, q, q + nq, q + nq + nk, st.q_norm.data_ptr(), st.k_norm.data_ptr(),
                            st.q.data_ptr(), c["heads"], EPS, THETA, st.table.shape[1] * c["page"], weight=weight,
                            q_ld=ld, kv_ld=ld)
    ws = _workspace(exe.sdpa_paged_workspace(kv, seqs, c["heads"], weight=weight, window=c["window"], sinks=c["sinks"]))
    if c["kind"] == "decode":
        exe.sdpa_paged_decode(kv, seqs, st.q.data_ptr(), st.out.data_ptr(), c["heads"], ws.data_ptr(), ws.numel(),
                              window=c["window"], sinks=c["sinks"], weight=weight)
    else:
        exe.sdpa_paged_prefill(kv, seqs, st.q.data_ptr(), st.out.data_ptr(), c["heads"], ws.data_ptr(), ws.numel(),
                               window=c["window"], sinks=c["sinks"])
    return _outputs(st)


_KEPT = {}


def _at(t):
    return None if t is None else t.data_ptr()


def _executor():
    """The program's executor: one context and one stream for all of its work."""
    if "exe" not in _KEPT:
        _KEPT["exe"] = _library().ObsidianExecutor(torch.cuda.current_device())
    return _KEPT["exe"]


def _library():
    import os
    import sys
    folder = os.path.join(os.getcwd(), "project-obsidian_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import obsidian_hip
    return obsidian_hip


def _workspace(nbytes):
    """The program's one workspace, as large as its largest call needs."""
    ws = _KEPT.get("ws")
    if ws is None or ws.numel() < nbytes:
        torch.cuda.synchronize()
        ws = _KEPT["ws"] = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device="cuda")
    return ws


def _handle(st):
    oh, c = _library(), st.case
    kv = oh.PagedKv(st.k.pool.data_ptr(), st.v.pool.data_ptr(), st.n_pages, c["page"], c["kv"], c["dim"], dtype=oh.KV_Q4)
    seqs = oh.PagedSeqs(_at(st.table), _at(st.len), c["seqs"], st.table.shape[1], st.rows, row=_at(st.row))
    weight = None
    if st.weight is not None:
        weight = oh.KvWeight(_at(st.weight), st.weight.shape[0], st.weight.shape[2], slot=_at(st.slot))
    return kv, seqs, weight


# ---- the plain forms: torch in 32 bits --------------------------------------

def _rows(st):
    """(sequence, place among its new tokens, entry) of every token row."""
    c = st.case
    if st.row is None:
        b = torch.arange(c["seqs"], device=st.len.device)
        return b, torch.zeros_like(b), st.len.long() - 1
    at = torch.arange(st.rows, device=st.row.device)
    b = torch.bucketize(at, st.row.long(), right=True) - 1
    t = at - st.row.long()[b]
    new = (st.row[1:] - st.row[:-1]).long()
    return b, t, st.len.long()[b] - new[b] + t


def _normed(x, w):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _rotated(x, pos):
    half = x.shape[-1] // 2
    angle = pos.double()[:, None] * THETA ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _appended(st, b, entry):
    c = st.case
    qd, kd = c["heads"] * c["dim"], c["kv"] * c["dim"]
    q, k, v = (x.reshape(st.rows, -1, c["dim"]) for x in st.qkv.split([qd, kd, kd], 1))
    st.q.copy_(_rotated(_normed(q, st.q_norm), entry))
    page, off = st.table[b, entry // c["page"]].long(), entry % c["page"]
    st.k.put(page, off, _rotated(_normed(k, st.k_norm), entry))
    st.v.put(page, off, v.float())
    if st.weight is not None:
        st.weight[st.slot.long()[b], :, entry] = 0.0


def _entries(st, side):
    """Every sequence's keys or values, fp32 [seqs, kv, entries, dim]; what lies behind a sequence is zero."""
    x = side.entries(st.table.long().clamp(min=0), torch.float32).permute(0, 2, 1, 3, 4).flatten(2, 3)
    there = (torch.arange(x.shape[2], device=x.device) < st.len[:, None])[:, None, :, None]
    return torch.where(there, x, 0.0)


def _attend(st):
    c = st.case
    b, t, entry = _rows(st)
    if c["append"]:
        _appended(st, b, entry)
    B, T, per = c["seqs"], st.most, c["heads"] // c["kv"]
    q = torch.zeros((B, T, c["heads"], c["dim"]), device=st.q.device)
    last = torch.full((B, T), -1, device=st.q.device)
    q[b, t], last[b, t] = st.q.float(), entry
    q = q.view(B, T, c["kv"], per, c["dim"]).permute(0, 2, 1, 3, 4).reshape(B, c["kv"], T * per, c["dim"])
    s = torch.matmul(q, _entries(st, st.k).transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(c["dim"]))
    s = s.view(B, c["kv"], T, per, -1)
    at, i = torch.arange(s.shape[-1], device=s.device), last[:, :, None]
    seen = at <= i
    if c["window"]:
        seen &= (at > i - c["window"]) | (at < c["sinks"])
    s.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    s.div_(torch.where(total == 0.0, 1.0, total))
    out = torch.matmul(s.view(B, c["kv"], T * per, -1), _entries(st, st.v)).view(B, c["kv"], T, per, c["dim"])
    st.out.copy_(out.permute(0, 2, 1, 3, 4).reshape(B, T, c["heads"], c["dim"])[b, t])
    if st.weight is not None:
        st.weight[st.slot.long()] += s.sum(dim=(2, 3))
    return _outputs(st)


def _of_logits(st, x):
    """Into the state's outputs what logits x [rows, vocab] (fp32 or fp64) give."""
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1, dtype=torch.float64)
    lse = m.squeeze(-1).double() + torch.log(total)
    t = st.tokens.long()
    lp = x.gather(1, t.clamp(min=0)[:, None]).squeeze(1).double() - lse
    st.logprob.copy_(torch.where(t < 0, 0.0, lp))
    d.clamp_(min=-1e4).mul_(e)
    st.entropy.copy_(torch.log(total) - d.sum(-1, dtype=torch.float64) / total)
    if st.top_ids is not None:
        v, i = torch.sort(x, dim=-1, descending=True, stable=True)
        st.top_ids.copy_(i[:, :st.top_ids.shape[1]])
        st.top_lp.copy_(v[:, :st.top_ids.shape[1]] - lse[:, None])
    return _scores(st)


def _logprobs(st):
    return _of_logits(st, st.logits[:, :st.case["vocab"]].float())


def _lm(st):
    # the alternatives' order is settled in 64 bits: of the 150,000 logits some lie next to each other
    kind = torch.float64 if st.top_ids is not None else torch.float32
    nibble = torch.arange(0, 32, 4, device=st.w.device, dtype=torch.int32)
    q = (st.w[:, :, None] >> nibble & 15).view(st.w.shape[0], -1, GROUP).to(kind)
    w = torch.addcmul(st.b.to(kind)[..., None], q, st.s.to(kind)[..., None]).flatten(1)
    return _of_logits(st, torch.matmul(st.x.to(kind), w.t()))


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("logprobs", "lm"):
        R, V, out = case["rows"], case["vocab"], case["rows"] * (12 + 8 * case["top"])
        if kind == "logprobs":
            return {"bytes": R * V * (4 if case["dtype"] == "fp32" else 2) + out, "flops": 6 * R * V}
        H = case["hidden"]
        return {"bytes": V * H // 2 + V * H // GROUP * 4 + 2 * R * H + out, "flops": 2 * R * V * H}
    B, heads, kv, dim = case["seqs"], case["heads"], case["kv"], case["dim"]
    lens, toks = _lens(case), _tokens(case)
    R, entry = sum(toks), 2 * kv * (dim // 2 + dim // 16)
    window, sinks = case["window"], case["sinks"]
    # appended: the projection's rows in, the rotated queries and the entries out
    new = R * (2 * (heads + 2 * kv) * dim + entry) if case["append"] else 0
    if kind == "decode":
        seen = sum(_seen(n, window, sinks) for n in lens)
        return {"bytes": seen * entry + 4 * B * heads * dim + (8 * kv * seen if case["weight"] else 0) + new,
                "flops": 4 * heads * dim * seen}
    read = pairs = 0
    for n, t in zip(lens, toks):
        first = n - t
        low = max(0, first + 1 - window) if window else 0
        read += n - low + min(sinks, low)
        pairs += sum(_seen(i + 1, window, sinks) for i in range(first, n))
    return {"bytes": read * entry + 4 * R * heads * dim + new, "flops": 4 * heads * dim * pairs}


# ---- the same in 64 bits -----------------------------------------------------

def _unpacked64(raw, params, low, high):
    """fp64 values of bytes raw [n, dim / 2] (low nibbles first) with params bf16 [n, groups, 2], dims of a group of 64."""
    q = torch.empty((raw.shape[0], 2 * raw.shape[1]), dtype=torch.float64, device=raw.device)
    q[:, low], q[:, high] = (raw % 16).double(), (raw // 16).double()
    s, b = (params[..., i].double().repeat_interleave(64, -1) for i in (0, 1))
    return q * s + b


def _read64(st, b, head, values):
    """Sequence b's keys or values of one kv head, fp64 [entries, dim]."""
    c, n = st.case, int(st.len[b])
    page, half = c["page"], c["dim"] // 2
    ids = st.table[b, :-(-n // page)].long()
    block = (st.v if values else st.k).pool[ids, head]
    raw, words = block[:, :page * half], block[:, page * half:].contiguous().view(torch.bfloat16)
    raw = raw.view(-1, half, page).permute(0, 2, 1) if values else raw.view(-1, page, half)
    words = words.view(len(ids), c["dim"] // 64, page, 2).permute(0, 2, 1, 3)
    d = torch.arange(half, device=raw.device)
    return _unpacked64(raw.reshape(-1, half), words.reshape(-1, c["dim"] // 64, 2), d, d + half)[:n]


def _stored64(x):
    """What 4 bits hold of x [..., dim] in fp64, and (scale, bias) bf16 [..., groups, 2]."""
    y = x.reshape(*x.shape[:-1], -1, 64)
    least = y.min(-1, keepdim=True).values
    scale = ((y.max(-1, keepdim=True).values - least) / 15).to(torch.bfloat16)
    bias = least.to(torch.bfloat16)
    q = torch.clamp(torch.round((y - bias.double()) / scale.double().clamp(min=1e-300)), 0, 15)
    return (q * scale.double() + bias.double()).reshape(x.shape), torch.cat([scale, bias], -1)


def _scores64(logits, tokens, top):
    p = torch.log_softmax(logits, 1)
    found = {"logprob": torch.stack([p[i, t] if t >= 0 else p.new_zeros(()) for i, t in enumerate(tokens.tolist())]),
             "entropy": -torch.xlogy(p.exp(), p.exp()).sum(1), "top_ids": None, "top_logprobs": None}
    if top:
        # by value, then by index: pairs of the largest ones, with all that tie with the last of them
        ids = []
        for row in logits:
            edge = torch.topk(row, top).values[-1]
            among = torch.nonzero(row >= edge).flatten().tolist()
            ids.append(sorted(among, key=lambda i: (-float(row[i]), i))[:top])
        found["top_ids"] = torch.tensor(ids, dtype=torch.int32)
        found["top_logprobs"] = p.gather(1, found["top_ids"].long().to(p.device))
    return found


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "logprobs":
        return _scores64(st.logits[:, :case["vocab"]].double(), st.tokens, case["top"])
    if kind == "lm":
        cols = torch.arange(case["hidden"], device="cuda")
        logits = torch.empty((case["rows"], case["vocab"]), dtype=torch.float64, device="cuda")
        for v in range(0, case["vocab"], 16384):
            word = st.w[v:v + 16384].long() & 0xffffffff
            q = (word[:, cols // 8] >> (cols % 8 * 4)) % 16
            w = q.double() * st.s[v:v + 16384].double()[:, cols // 64] + st.b[v:v + 16384].double()[:, cols // 64]
            logits[:, v:v + 16384] = st.x.double() @ w.T
        return _scores64(logits, st.tokens, case["top"])
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    lens, toks = _lens(case), _tokens(case)
    per = heads // kv
    out = torch.zeros((sum(toks), heads, dim), dtype=torch.float64, device="cuda")
    q_all = st.q.double()
    gathered = None if st.weight is None else st.weight.double()
    k_par, v_par = st.k.params.double(), st.v.params.double()
    turns = torch.arange(dim // 2, device="cuda", dtype=torch.float64) * (-2.0 / dim)
    at = 0
    for b, (n, t) in enumerate(zip(lens, toks)):
        kn = vn = None
        if case["append"]:
            x = st.qkv[at:at + t].double().view(t, heads + 2 * kv, dim)
            where = torch.arange(n - t, n, device="cuda")
            angle = where.double().unsqueeze(1) * torch.exp(turns * math.log(THETA))
            turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)

            def rotated(y, w):
                y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
                z = torch.complex(y[..., :dim // 2], y[..., dim // 2:]) * turn
                return torch.cat([z.real, z.imag], -1)

            q_all[at:at + t] = rotated(x[:, :heads], st.q_norm)
            kn, kp = _stored64(rotated(x[:, heads:heads + kv], st.k_norm))
            vn, vp = _stored64(x[:, heads + kv:])
            pages = st.table[b].long()[where // page]
            k_par[pages, :, where % page], v_par[pages, :, where % page] = kp.double(), vp.double()
            if gathered is not None:
                gathered[int(st.slot[b]), :, n - t:n] = 0.0
        here = torch.arange(n - t, n, device="cuda").unsqueeze(1)
        other = torch.arange(n, device="cuda").unsqueeze(0)
        hidden = other > here
        if case["window"]:
            hidden = hidden | ((here - other >= case["window"]) & (other >= case["sinks"]))
        for h in range(kv):
            keys, values = _read64(st, b, h, False), _read64(st, b, h, True)
            if kn is not None:
                keys[n - t:], values[n - t:] = kn[:, h], vn[:, h]
            for j in range(h * per, (h + 1) * per):
                # (the query in the type that the call hands on)
                q = q_all[at:at + t, j].bfloat16().double()
                p = torch.softmax((q @ keys.T / dim ** 0.5).masked_fill(hidden, float("-inf")), 1)
                out[at:at + t, j] = p @ values
                if gathered is not None:
                    gathered[int(st.slot[b]), h, :n] += p.sum(0)
        at += t
    found = {"out": out, "weight": gathered}
    if case["append"]:
        found.update(q=q_all, k_params=k_par, v_params=v_par)
    return found
