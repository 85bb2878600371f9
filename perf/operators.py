"""The operators of the paged K/V cache, as cases that can be timed and checked.

Kinds of case:

  * ``write``: the K/V rows of new tokens into an f16 cache (``mlg_kv_write``); the pool comes back.
  * ``store``: the same rows written and read back (``mlg_kv_write`` + ``mlg_kv_read``), as a
    program does that checks or moves what its cache holds; q8_0 caches quantise on the way.
  * ``read``: whole sequences out of the cache as f32 rows (``mlg_kv_read``).
  * ``attend``: attention of each sequence's new tokens over its cached keys (``mlg_attn_paged``).

The cache (values of the pool, all offsets in elements of a head's tile):

  page   [heads][K, V][page / 32 tiles of 32 tokens]
  K tile f16:  (token, dim) at ((dim/32 * 2 + token/4%2) * 64 + dim/8%4 * 16 + token/8 * 4 + token%4) * 8 + dim%8
  K tile q8_0: (token, dim) at ((dim/32 * 64 + dim/8%4 * 16 + token/8 * 4 + token%4) * 2 + token/4%2) * 8 + dim%8
  V tile f16:  (token, dim) at (dim/16 * 64 + token/8 * 16 + dim%16) * 8 + token%8
  V tile q8_0: (token, dim) at ((dim/32 * 64 + token/8 * 16 + dim%16) * 2 + dim/16%2) * 8 + token%8
  q8_0 tiles: 32 * head size bytes, then the f16 scale of (token, dims 32 b .. 32 b + 31) at b * 32 + token

Sequence i has ctx[i] tokens, the last row_off[i + 1] - row_off[i] of them new.
"""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"f16": 1, "q8_0": 8}  # ggml type ids


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one decode step of 32 sentences: each layer appends one token's K/V per sentence
        dict(name="write_step32", kind="write", type="f16", heads=16, hd=64, page=64, seqs=32, new_lo=1, new_hi=1,
             single=0.0, past_lo=5, past_hi=199, mix=1),
        # forced target prefixes of a batch of ragged requests go into an 8-bit cache of the large model
        dict(name="store_prefixes_q8", kind="store", type="q8_0", heads=16, hd=128, page=64, seqs=24, new_lo=3,
             new_hi=611, single=0.2, past_lo=0, past_hi=300, mix=2),
        # one long document's keys and values, few wide K/V heads
        dict(name="store_document_q8", kind="store", type="q8_0", heads=8, hd=128, page=128, seqs=1, new_lo=32001,
             new_hi=32001, single=0.0, past_lo=77, past_hi=77, mix=3),
        # sequences taken out of the cache (moved to another device or to host memory)
        dict(name="read_sequences_f16", kind="read", type="f16", heads=16, hd=64, page=32, seqs=8, new_lo=211,
             new_hi=1501, single=0.0, past_lo=0, past_hi=0, mix=4),
        # the smallest call: one sentence, one token, a few dozen keys
        dict(name="attend_one", kind="attend", type="f16", heads=16, group=1, hd=64, page=64, seqs=1, new_lo=1,
             new_hi=1, single=0.0, past_lo=44, past_hi=44, causal=True, mix=5),
        # a decode step of 32 sentences up to the model's longest output
        dict(name="attend_step32", kind="attend", type="f16", heads=16, group=1, hd=64, page=64, seqs=32, new_lo=1,
             new_hi=1, single=0.0, past_lo=5, past_hi=199, causal=True, mix=6),
        # a decode step of a serving batch of the large model over 8-bit caches of whole documents
        dict(name="attend_step64_q8", kind="attend", type="q8_0", heads=16, group=1, hd=128, page=64, seqs=64,
             new_lo=1, new_hi=1, single=0.0, past_lo=90, past_hi=2300, causal=True, mix=7),
        # few sequences with very long contexts, four query heads to a K/V head
        dict(name="attend_long", kind="attend", type="f16", heads=8, group=4, hd=128, page=256, seqs=3, new_lo=1,
             new_hi=1, single=0.0, past_lo=60001, past_hi=100002, causal=True, mix=8),
        # cross attention of a beam step: the four beams of a sentence read one copy of its source
        dict(name="attend_beams", kind="attend", type="f16", heads=16, group=1, hd=64, page=32, seqs=8, new_lo=4,
             new_hi=4, single=0.0, past_lo=9, past_hi=420, causal=False, mix=9),
        # dynamic batching: most requests decode one token while others bring in a chunk of their prompt
        dict(name="attend_mixed_q8", kind="attend", type="q8_0", heads=8, group=2, hd=64, page=64, seqs=40, new_lo=33,
             new_hi=517, single=0.7, past_lo=0, past_hi=1700, causal=True, mix=10),
        # scoring short continuations, wide heads shared seven to one
        dict(name="attend_wide_heads_q8", kind="attend", type="q8_0", heads=2, group=7, hd=256, page=32, seqs=5,
             new_lo=17, new_hi=131, single=0.0, past_lo=200, past_hi=900, causal=True, mix=11),
        # the largest: a long prompt's chunk over what is there of it already
        dict(name="attend_prompt", kind="attend", type="f16", heads=16, group=1, hd=64, page=128, seqs=1, new_lo=4001,
             new_hi=4001, single=0.0, past_lo=3999, past_hi=3999, causal=True, mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "store", "read", "attend", "attend", "attend", "attend", "attend"])
    hd = rng.choice([32, 64, 64, 128, 128, 256])
    c = dict(kind=kind, type="f16" if kind == "write" else rng.choice(["f16", "q8_0"]), heads=rng.choice([1, 2, 4, 8, 16, 16]),
             hd=hd, page=rng.choice([32, 64, 128, 256]), mix=rng.randrange(1 << 20))
    if kind != "attend":
        most = max(1, (1 << 24) // (c["heads"] * hd))  # values of K and of V at most
        hi = _log(rng, 1, min(16001, most))
        n = max(1, min(_log(rng, 1, 64), most // hi))
        past = 0 if kind == "read" else _log(rng, 1, 700)
        c.update(seqs=n, new_lo=max(1, hi // rng.choice([1, 2, 9])), new_hi=hi, single=rng.choice([0.0, 0.3]),
                 past_lo=past // 3, past_hi=past)
        return c
    c.update(group=rng.choice([1, 1, 1, 2, 4, 7, 8]), causal=rng.random() < 0.8)
    if rng.random() < 0.5:  # single tokens, or a beam's worth
        rows = 1 if c["causal"] else rng.choice([1, 2, 4, 5])
        hi = _log(rng, 2, 60001)
        n = max(1, min(_log(rng, 1, 64), (1 << 28) // (hi * c["heads"] * hd)))
        c.update(seqs=n, new_lo=rows, new_hi=rows, single=0.0, past_lo=max(1, hi // rng.choice([1, 2, 9])), past_hi=hi)
    else:  # chunks, a few single tokens among them
        hi = _log(rng, 2, 2001)
        past = _log(rng, 1, 4001)
        heads = c["heads"] * c["group"]
        while hi > 1 and hi * (past + hi) * heads * hd > 24_000_000_000:
            hi, past = hi // 2, past // 2 + 1
        n = max(1, min(_log(rng, 1, 32), (1 << 27) // (hi * (past + hi) * heads * max(1, hd // 128)),
                       (1 << 24) // ((past + hi) * c["heads"] * hd)))
        c.update(seqs=n, new_lo=max(1, hi // rng.choice([1, 3, 9])), new_hi=hi, single=rng.choice([0.0, 0.0, 0.5]),
                 past_lo=past // rng.choice([1, 4]), past_hi=past)
    return c


def _spans(case):
    """(new tokens, tokens in the cache after them) of every sequence: the case's own, whatever the seed."""
    r = random.Random(case["mix"])
    new = [1 if i and r.random() < case["single"] else r.randint(case["new_lo"], case["new_hi"])
           for i in range(case["seqs"])]
    new[0] = case["new_hi"]
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in new]
    past[-1] = case["past_hi"]
    return [(n, n + p) for n, p in zip(new, past)]


def _tile_bytes(case):
    return (64 if case["type"] == "f16" else 34) * case["hd"]


def work(case):
    spans, hd, kvh = _spans(case), case["hd"], case["heads"]
    token = 2 * kvh * _tile_bytes(case) // 32  # cache bytes of a token's K and V
    rows = sum(n for n, _ in spans)
    if case["kind"] != "attend":
        moved = {"write": 1, "read": 1, "store": 2}[case["kind"]]  # times that the f32 rows pass
        return {"bytes": rows * (token + moved * 2 * kvh * hd * 4), "flops": 0}
    h = kvh * case["group"]
    seen = sum(n * c - n * (n - 1) // 2 if case["causal"] else n * c for n, c in spans)
    return {"bytes": sum(c for _, c in spans) * token + 2 * rows * h * hd * 4, "flops": 4 * seen * h * hd}


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    spans, hd, kvh, page = _spans(case), case["hd"], case["heads"], case["page"]
    need = [-(-c // page) for _, c in spans]
    pages, width = sum(need) + 2, max(need)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    # every sequence's pages lie anywhere in the pool; entries past its last page are not read
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    slot = first[:, None] + torch.arange(width, device="cuda")
    have = torch.arange(width, device="cuda") < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(have, order[slot.clamp(max=pages - 1)], 0).to(torch.int32).contiguous()
    tb = _tile_bytes(case)
    if case["type"] == "f16":
        pool = torch.empty(pages * kvh * 2 * (page // 32) * tb // 2, dtype=torch.float16, device="cuda")
        pool.normal_(generator=g)
        pool = pool.view(torch.uint8)
    else:  # blocks as quantised normal values have them
        pool = torch.empty(pages * kvh * 2 * (page // 32), tb, dtype=torch.uint8, device="cuda")
        q = torch.empty(pool.shape[0], 32 * hd, dtype=torch.float16, device="cuda").normal_(0, 50, generator=g)
        pool[:, :32 * hd] = q.round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
        d = torch.empty(pool.shape[0], hd, dtype=torch.float16, device="cuda").uniform_(0.016, 0.024, generator=g)
        pool[:, 32 * hd:] = d.view(torch.uint8)
        pool = pool.view(-1)
    rows = sum(n for n, _ in spans)
    off = [0]
    for n, _ in spans:
        off.append(off[-1] + n)
    s = dict(case=case, pool=pool, table=table, pages=pages, rows=rows, max_new=max(n for n, _ in spans),
             max_ctx=max(c for _, c in spans), row_off=torch.tensor(off, dtype=torch.int32, device="cuda"),
             ctx=torch.tensor([c for _, c in spans], dtype=torch.int32, device="cuda"))

    def normal(*shape, std=1.0):
        return torch.empty(*shape, device="cuda").normal_(0, std, generator=g)

    if case["kind"] == "attend":
        s["q"] = normal(rows, kvh * case["group"], hd, std=1.5)
        s["out"] = torch.zeros_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(hd)
    else:
        if case["kind"] != "read":
            s["k"], s["v"] = normal(rows, kvh, hd), normal(rows, kvh, hd)
        if case["kind"] != "write":
            s["k_out"], s["v_out"] = torch.zeros(rows, kvh, hd, device="cuda"), torch.zeros(rows, kvh, hd, device="cuda")
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "attend":
        return _attend(state)
    if kind != "read":
        _write(state)
    return state["pool"].view(torch.float16) if kind == "write" else _read(state)


def _run_own(s):
    import ctypes

    from malaga_amd import _lib

    c = s["case"]
    lib = _lib.load()
    if "cache" not in s:  # what a program keeps: the cache's description and the attention's workspace
        s["cache"] = _lib.KvCache(TYPES[c["type"]], c["heads"], c["hd"], c["page"], s["pages"], s["pool"].data_ptr(),
                                  s["table"].data_ptr(), c["seqs"], s["table"].shape[1])
        if c["kind"] == "attend":
            n = lib.mlg_attn_paged_scratch(ctypes.byref(s["cache"]), c["heads"] * c["group"], s["rows"], s["max_new"],
                                           s["max_ctx"])
            s["scratch"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
            s["scratch_bytes"] = n
    cache = ctypes.byref(s["cache"])
    stream = torch.cuda.current_stream().cuda_stream
    at = s["row_off"].data_ptr(), s["ctx"].data_ptr(), s["rows"], s["max_new"]
    if c["kind"] == "attend":
        h, hd = c["heads"] * c["group"], c["hd"]
        _lib.check(lib.mlg_attn_paged(cache, s["q"].data_ptr(), h * hd, h, s["scale"], int(c["causal"]), *at, s["max_ctx"],
                                      s["out"].data_ptr(), h * hd, s["scratch"].data_ptr(), s["scratch_bytes"], None,
                                      stream))
        return s["out"]
    ld = c["heads"] * c["hd"]
    if c["kind"] != "read":
        _lib.check(lib.mlg_kv_write(cache, s["k"].data_ptr(), ld, s["v"].data_ptr(), ld, *at, None, stream))
        if c["kind"] == "write":
            return s["pool"].view(torch.float16)
    _lib.check(lib.mlg_kv_read(cache, s["k_out"].data_ptr(), ld, s["v_out"].data_ptr(), ld, *at, None, stream))
    return s["k_out"], s["v_out"]


# ------------------------------------------------------------------ the plain forms

def _rows_at(s):
    """Sequence and position of every new row."""
    off, ctx = s["row_off"].long(), s["ctx"].long()
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(off[1:], row, right=True)
    return seq, ctx[seq] - (off[seq + 1] - row)


def _places(s):
    """Elements of the pool's tiles that hold the new rows: their tile's first byte [rows, heads, K/V] and, in the tile,
    K's and V's element [rows, hd] and the scale's [rows, hd / 32]."""
    c = s["case"]
    seq, pos = _rows_at(s)
    page, tb = c["page"], _tile_bytes(c)
    p = s["table"].long()[seq, pos // page]
    head = torch.arange(c["heads"], device="cuda")[:, None]
    kv = torch.arange(2, device="cuda")
    tiles = page // 32
    tile = (((p[:, None, None] * c["heads"] + head) * 2 + kv) * tiles + (pos % page // 32)[:, None, None]) * tb
    t, d = (pos % 32)[:, None], torch.arange(c["hd"], device="cuda")
    if c["type"] == "f16":
        ke = ((d // 32 * 2 + t // 4 % 2) * 64 + d // 8 % 4 * 16 + t // 8 * 4 + t % 4) * 8 + d % 8
        ve = (d // 16 * 64 + t // 8 * 16 + d % 16) * 8 + t % 8
    else:
        ke = ((d // 32 * 64 + d // 8 % 4 * 16 + t // 8 * 4 + t % 4) * 2 + t // 4 % 2) * 8 + d % 8
        ve = ((d // 32 * 64 + t // 8 * 16 + d % 16) * 2 + d // 16 % 2) * 8 + t % 8
    return tile, ke, ve, torch.arange(c["hd"] // 32, device="cuda") * 32 + t


def _quantise(x):
    """q8_0 blocks of 32 values: d = max |x| / 127, whole numbers round(x (1 / d)), ties away from zero."""
    x = x.view(*x.shape[:-1], -1, 32)
    d = (x.abs().amax(-1).double() / 127).float()  # in 64 bits: a division by a number may multiply by its inverse
    y = x * torch.where(d > 0, 1 / d.double(), 0).float()[..., None]
    whole = y.trunc()
    return (whole + torch.where((y - whole).abs() >= 0.5, y.sign(), 0)).flatten(-2), d


def _write(s):
    c = s["case"]
    tile, ke, ve, se = _places(s)
    if c["type"] == "f16":
        pool = s["pool"].view(torch.float16)
        pool[tile[:, :, :1] // 2 + ke[:, None]] = s["k"].half()
        pool[tile[:, :, 1:] // 2 + ve[:, None]] = s["v"].half()
        return
    (qk, dk), (qv, dv) = _quantise(s["k"]), _quantise(s["v"])
    pool, scales = s["pool"].view(torch.int8), s["pool"].view(torch.float16)
    pool[tile[:, :, :1] + ke[:, None]] = qk.to(torch.int8)
    pool[tile[:, :, 1:] + ve[:, None]] = qv.to(torch.int8)
    first = tile // 2 + 16 * c["hd"]
    scales[first[:, :, :1] + se[:, None]] = dk.half()
    scales[first[:, :, 1:] + se[:, None]] = dv.half()


def _read(s):
    c = s["case"]
    tile, ke, ve, se = _places(s)
    if c["type"] == "f16":
        pool = s["pool"].view(torch.float16)
        return pool[tile[:, :, :1] // 2 + ke[:, None]].float(), pool[tile[:, :, 1:] // 2 + ve[:, None]].float()
    pool, scales = s["pool"].view(torch.int8), s["pool"].view(torch.float16)
    first = tile // 2 + 16 * c["hd"]
    dk = scales[first[:, :, :1] + se[:, None]].float().repeat_interleave(32, -1)
    dv = scales[first[:, :, 1:] + se[:, None]].float().repeat_interleave(32, -1)
    return pool[tile[:, :, :1] + ke[:, None]].float() * dk, pool[tile[:, :, 1:] + ve[:, None]].float() * dv


def _dense(s):
    """K and V of every sequence's pages as f32 [seqs, heads, tokens, hd]."""
    c = s["case"]
    n, width = s["table"].shape
    hd, kvh, tiles = c["hd"], c["heads"], c["page"] // 32
    got = s["pool"].view(s["pages"], -1)[s["table"].long()].view(n, width, kvh, 2, tiles, _tile_bytes(c))
    got = got.permute(3, 0, 2, 1, 4, 5)  # [K/V, seqs, heads, pages, tiles, bytes]
    k, v = got[0].contiguous(), got[1].contiguous()
    lead = (n, kvh, width, tiles)
    if c["type"] == "f16":
        # K [dim block, token/4%2, dim/8%4, token/8, token%4, dim%8], V [dim/16, token/8, dim%16, token%8]
        k = k.view(torch.float16).view(*lead, hd // 32, 2, 4, 4, 4, 8).permute(0, 1, 2, 3, 7, 5, 8, 4, 6, 9)
        v = v.view(torch.float16).view(*lead, hd // 16, 4, 16, 8).permute(0, 1, 2, 3, 5, 7, 4, 6)
        return k.float().reshape(n, kvh, -1, hd), v.float().reshape(n, kvh, -1, hd)
    dk, dv = (x[..., 32 * hd:].contiguous().view(torch.float16).view(*lead, hd // 32, 32).transpose(-1, -2).float()
              for x in (k, v))
    k, v = (x[..., :32 * hd].contiguous().view(torch.int8) for x in (k, v))
    # K [dim block, dim/8%4, token/8, token%4, token/4%2, dim%8], V [dim block, token/8, dim%16, dim/16%2, token%8]
    k = k.view(*lead, hd // 32, 4, 4, 4, 2, 8).permute(0, 1, 2, 3, 6, 8, 7, 4, 5, 9)
    v = v.view(*lead, hd // 32, 4, 16, 2, 8).permute(0, 1, 2, 3, 5, 8, 4, 7, 6)
    k = k.reshape(*lead, 32, hd // 32, 32).float() * dk[..., None]
    v = v.reshape(*lead, 32, hd // 32, 32).float() * dv[..., None]
    return k.reshape(n, kvh, -1, hd), v.reshape(n, kvh, -1, hd)


def _attend(s):
    c = s["case"]
    k, v = _dense(s)
    k, v = k[:, :, :s["max_ctx"]].contiguous(), v[:, :, :s["max_ctx"]]
    n, kvh, hd, g, m = c["seqs"], c["heads"], c["hd"], c["group"], s["max_new"]
    off, ctx = s["row_off"].long(), s["ctx"].long()
    t = torch.arange(m, device="cuda")
    new = off[1:] - off[:-1]
    row = (off[:-1, None] + t).clamp(max=s["rows"] - 1)  # [seqs, m], rows past a sequence's last masked below
    seen = ctx[:, None] - new[:, None] + t + 1 if c["causal"] else ctx[:, None].expand(n, m)
    seen = torch.where(t < new[:, None], seen, 0)
    q = s["q"][row].view(n, m, kvh, g, hd).permute(0, 2, 1, 3, 4).reshape(n, kvh, m * g, hd)
    score = (q @ k.transpose(-1, -2).contiguous()).mul_(s["scale"])
    hidden = torch.arange(k.shape[2], device="cuda") >= seen[:, :, None]  # [seqs, m, keys]
    score = score.view(n, kvh, m, g, -1).masked_fill_(hidden[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(n, kvh, m * g, -1) @ v.contiguous()).view(n, kvh, m, g, hd) / torch.where(total > 0, total, 1)
    o = o.permute(0, 2, 1, 3, 4).reshape(n * m, kvh * g, hd)
    seq, pos = _rows_at(s)
    return o[seq * m + pos - (ctx - new)[seq]].contiguous()


# ------------------------------------------------------------------ 64 bits

def _cached(s, i, head, which, count):
    """Tokens 0 .. count - 1 of sequence i in 64 bits, [count, hd], value by value from where the layout puts them."""
    c = s["case"]
    hd, page, eight = c["hd"], c["page"], c["type"] == "q8_0"
    size = _tile_bytes(c)
    tok = torch.arange(count, device="cuda")
    at = s["table"].long()[i][tok.div(page, rounding_mode="floor")] * c["heads"] + head
    base = ((at * 2 + which) * (page // 32) + tok.remainder(page).div(32, rounding_mode="floor")) * size
    t, e = tok.remainder(32).unsqueeze(1), torch.arange(hd, device="cuda").unsqueeze(0)
    if which == 0:
        lane = (e >> 3 & 3) * 16 + (t >> 3) * 4 + (t & 3)
        piece = (((e >> 5) * 64 + lane) * 2 + (t >> 2 & 1)) if eight else (((e >> 5) * 2 + (t >> 2 & 1)) * 64 + lane)
        place = piece * 8 + (e & 7)
    else:
        lane = (t >> 3) * 16 + (e & 15)
        piece = (((e >> 5) * 64 + lane) * 2 + (e >> 4 & 1)) if eight else ((e >> 4) * 64 + lane)
        place = piece * 8 + (t & 7)
    if not eight:
        return s["pool"].view(torch.float16)[(base >> 1).unsqueeze(1) + place].double()
    d = s["pool"].view(torch.float16)[(base + 32 * hd >> 1).unsqueeze(1) + (e >> 5) * 32 + t]
    return s["pool"].view(torch.int8)[base.unsqueeze(1) + place].double() * d.double()


def _stored(x, kind):
    """What a cache of this type holds for rows x, in 64 bits."""
    if kind == "f16":
        return x.half().double()
    b = x.double().reshape(-1, 32)
    d = (b.abs().max(1).values / 127.0).float().double()  # the definition rounds d, 1 / d and x / d to f32
    inv = torch.where(d > 0, (1.0 / d.clamp(min=1e-300)).float().double(), torch.zeros_like(d))
    y = (b * inv[:, None]).float().double()
    q = torch.floor(y.abs() + 0.5) * torch.sign(y)
    return (q * d.half().double()[:, None]).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    spans, kind = _spans(case), case["kind"]
    if kind == "store":
        return _stored(s["k"], case["type"]), _stored(s["v"], case["type"])
    if kind == "write":
        pool, at, hd = s["pool"].view(torch.float16).double(), 0, case["hd"]
        for i, (n, c) in enumerate(spans):
            pos = torch.arange(c - n, c, device="cuda")
            where = s["table"].long()[i][pos // case["page"]] * case["heads"]
            t, e = (pos & 31).unsqueeze(1), torch.arange(hd, device="cuda").unsqueeze(0)
            for h in range(case["heads"]):
                for which, x in enumerate((s["k"], s["v"])):
                    base = (((where + h) * 2 + which) * (case["page"] // 32) + (pos % case["page"] >> 5)) * 32 * hd
                    place = (((e >> 5) * 2 + (t >> 2 & 1)) * 64 + (e >> 3 & 3) * 16 + (t >> 3) * 4 + (t & 3)) * 8 + (e & 7) \
                        if which == 0 else ((e >> 4) * 64 + (t >> 3) * 16 + (e & 15)) * 8 + (t & 7)
                    pool[base.unsqueeze(1) + place] = _stored(x[at:at + n, h], "f16")
            at += n
        return pool
    if kind == "read":
        got = [torch.cat([torch.stack([_cached(s, i, h, w, c)[c - n:] for h in range(case["heads"])], 1)
                          for i, (n, c) in enumerate(spans)]) for w in (0, 1)]
        return got[0], got[1]
    out, at, g = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0, case["group"]
    for i, (n, c) in enumerate(spans):
        last = (torch.arange(c - n, c, device="cuda") if case["causal"] else torch.full((n,), c - 1, device="cuda"))
        hidden = torch.arange(c, device="cuda").unsqueeze(0) > last.unsqueeze(1)
        for h in range(case["heads"]):
            k, v = _cached(s, i, h, 0, c), _cached(s, i, h, 1, c)
            for j in range(h * g, (h + 1) * g):
                a = torch.mm(s["q"][at:at + n, j].double(), k.t().contiguous()) * s["scale"]
                a[hidden] = -math.inf
                out[at:at + n, j] = torch.mm(torch.softmax(a, 1), v)
        at += n
    return out
