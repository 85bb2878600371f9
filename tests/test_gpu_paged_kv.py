"""The paged K/V cache on the GPU: writing, reading and attending it against plain 64-bit numpy, and the
three together as a decoding program runs them."""
import ctypes as C

import numpy as np
import pytest
import torch

import malaga_amd as M
from malaga_amd import _lib

pytestmark = pytest.mark.gpu
F16, Q8_0 = _lib.F16, _lib.Q8_0
lib = _lib.load()
KINDS = [F16, Q8_0]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def u32(a):
    return dev(np.asarray(a, dtype=np.uint32).view(np.int32))


class Cache:
    """A pool whose every byte is NaN until written (f16 NaN values; q8_0 NaN scales), and its table."""

    def __init__(self, kind, heads, hd, page, seqs, table_len, pages=None, seed=0):
        self.kind, self.heads, self.hd, self.page, self.seqs, self.table_len = kind, heads, hd, page, seqs, table_len
        self.pages = pages or seqs * table_len + 3
        self.bytes = lib.mlg_kv_page_bytes(kind, heads, hd, page)
        self.pool = torch.full((self.pages * self.bytes // 2,), 0x7e7e, dtype=torch.int16, device="cuda")
        ids = np.random.default_rng(seed).permutation(self.pages)[: seqs * table_len].astype(np.uint32)
        self.ids = ids.reshape(seqs, table_len)
        self.table = u32(self.ids)

    @property
    def c(self):
        return _lib.KvCache(self.kind, self.heads, self.hd, self.page, self.pages, self.pool.data_ptr(),
                            self.table.data_ptr(), self.seqs, self.table_len)

    def stored(self, x):
        """What the cache holds for f32 rows x (numpy, rounded as the codec rounds)."""
        if self.kind == F16:
            with np.errstate(over="ignore"):
                return x.astype(np.float16).astype(np.float32)
        return M.dequantize(Q8_0, M.quantize(Q8_0, x), x.size).reshape(x.shape)


def rows_of(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)


def stream():
    return torch.cuda.current_stream().cuda_stream


def put(cache, k, v, new, ctx, off=True, max_new=None, bad=None, rows=None, call=None):
    """Writes rows k, v [rows, heads, hd] (or strided views of them)."""
    o, x = u32(rows_of(new)) if off else None, u32(ctx)
    _lib.check((call or lib.mlg_kv_write)(
        C.byref(cache.c), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), o.data_ptr() if off else None,
        x.data_ptr(), len(k) if rows is None else rows, max_new or max(max(new), 1), bad.data_ptr() if bad is not None else None,
        stream()))
    torch.cuda.synchronize()


def get(cache, k, v, new, ctx, **kw):
    put(cache, k, v, new, ctx, call=lib.mlg_kv_read, **kw)


def attend(cache, q, new, ctx, scale, causal=True, off=True, max_new=None, max_ctx=0, out=None, bad=None, rows=None,
           sync=True):
    heads = q.shape[1]
    out = torch.full(q.shape, 7.0, device="cuda") if out is None else out
    o, x = u32(rows_of(new)) if off else None, u32(ctx)
    m, rows = max_new or max(max(new), 1), len(q) if rows is None else rows
    n = lib.mlg_attn_paged_scratch(C.byref(cache.c), heads, rows, m, max_ctx)
    scratch = torch.full((max(n // 4, 1),), float("nan"), device="cuda")
    _lib.check(lib.mlg_attn_paged(C.byref(cache.c), q.data_ptr(), q.stride(0), heads, scale, int(causal),
                                  o.data_ptr() if off else None, x.data_ptr(), rows, m, max_ctx, out.data_ptr(),
                                  out.stride(0), scratch.data_ptr(), n, bad.data_ptr() if bad is not None else None,
                                  stream()))
    if sync:
        torch.cuda.synchronize()
    return out


def reference(q, k, v, n, ctx, scale, causal, tol=True):
    """Attention of q [n, H, hd] over k, v [ctx, Hkv, hd] in 64 bits, and how far f32 arithmetic may be from it.

    A score's f32 error: hd products and sums in any order, the two-term q (2^-22), and the scale:
    (hd + 16) 2^-24 sum |q k| scale; p is off by that much relatively, plus 2^-22 (exp2 and the subtraction
    of the maximum, in log2 units: |s| 1.45 2^-24 each), and out, a mean weighted by p, by twice p's error
    times max |v|, plus the f32 sums over the tokens: 32 at once, so ctx / 32 + 64 roundings."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    g = q.shape[1] // k.shape[1]
    out, err = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(q.shape[1]):
        for t in range(n):
            seen = min(max(ctx - n + t + 1, 0), ctx) if causal else ctx
            if not seen:
                continue
            kk, vv = k[:seen, h // g], v[:seen, h // g]
            s = kk @ q[t, h] * scale
            p = np.exp(s - s.max())
            out[t, h] = p @ vv / p.sum()
            a = (np.abs(kk) @ np.abs(q[t, h])).max() * abs(scale)
            err[t, h] = (2 * ((q.shape[2] + 16) * 2.0 ** -24 * a + 2.0 ** -22 + 4 * np.abs(s).max() * 2.0 ** -24) +
                         (ctx / 32 + 64) * 2.0 ** -24) * np.abs(vv).max()
    return out, err


def filled(kind, heads, hd, page, spans, seed, table_len=None, std=1.0):
    """A cache with ctx tokens of every sequence, and what it holds of them per sequence."""
    rng = np.random.default_rng(seed)
    ctx = [c for _, c in spans]
    cache = Cache(kind, heads, hd, page, len(spans), table_len or max(1, -(-max(ctx) // page)), seed=seed)
    k = rng.normal(0, std, (sum(ctx), heads, hd)).astype(np.float32)
    v = rng.normal(0, 1, (sum(ctx), heads, hd)).astype(np.float32)
    if sum(ctx):
        put(cache, dev(k), dev(v), ctx, ctx)
    at = np.cumsum([0] + ctx)
    kd, vd = cache.stored(k), cache.stored(v)
    return cache, [(kd[a:b], vd[a:b]) for a, b in zip(at, at[1:])], rng


SPANS = [(1, 1), (1, 33), (0, 40), (3, 2), (5, 64), (0, 0), (33, 33), (2, 0), (31, 97), (1, 64), (17, 130)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,heads,page", [(32, 3, 32), (64, 2, 64), (128, 1, 128), (256, 2, 32), (64, 1, 256)])
def test_written_rows_read_back_as_the_codec_rounds_them(kind, hd, heads, page):
    """Ragged writes at positions anywhere in a tile, in two calls (the second next to what the first left),
    from strided rows; values beside the written ones keep what they were."""
    rng = np.random.default_rng(hd + heads)
    new, past = [1, 33, 0, 7, 64, 2], [0, 5, 9, 30, 31, 63]
    ctx = [a + b for a, b in zip(new, past)]
    cache = Cache(kind, heads, hd, page, len(new), -(-max(ctx) // page), seed=hd)
    both = []
    for n, c in ((past, past), (new, ctx)):
        rows = rng.normal(0, 1, (sum(n), 3, heads, hd)).astype(np.float32)
        rows *= 10.0 ** rng.integers(-3, 4, (sum(n), 3, heads, 1)).astype(np.float32)
        rows[rng.random(rows.shape) < 0.02] = 0.0
        fused = dev(rows)
        put(cache, fused[:, 1], fused[:, 2], n, c)
        both.append((rows[:, 1], rows[:, 2]))
    for which in range(2):
        want, at = [], [0, 0]
        for i, (n, p) in enumerate(zip(new, past)):
            want += [both[0][which][at[0]:at[0] + p], both[1][which][at[1]:at[1] + n]]
            at = [at[0] + p, at[1] + n]
        want = cache.stored(np.concatenate(want))
        out = [torch.full((sum(ctx) + 1, heads, hd + 4), 5.0, device="cuda") for _ in range(2)]
        views = [o.view(len(o), -1)[:, : heads * hd].unflatten(1, (heads, hd)) for o in out]
        get(cache, *views, ctx, ctx)
        got = views[which].cpu().numpy()
        assert np.array_equal(got[:-1], want)
        assert (got[-1] == 5).all() and (out[which].view(len(out[which]), -1)[:, heads * hd:] == 5).all()
    # bytes of the pool that hold no token are as they were
    pool = cache.pool.view(torch.uint8).cpu().numpy()
    held = np.zeros(pool.size, bool)
    sb = C.c_int64()
    for i, c in enumerate(ctx):
        for pos in range(c):
            for h in range(heads):
                for which in range(2):
                    for d in range(hd):
                        at = lib.mlg_debug_kv_place(C.byref(cache.c), int(cache.ids[i, pos // page]), h, which, pos, d,
                                                    C.byref(sb))
                        held[at: at + (2 if kind == F16 else 1)] = True
                        if sb.value >= 0:
                            held[sb.value: sb.value + 2] = True
        if c > 40:
            break  # the first sequences are enough
    first = sum(1 for _ in range(i + 1))
    ids = cache.ids[:first].reshape(-1)
    for pid in ids:
        part = slice(int(pid) * cache.bytes, (int(pid) + 1) * cache.bytes)
        assert (pool[part][~held[part]] == 0x7e).all()


def test_values_that_are_not_finite_and_the_edges_of_the_formats():
    x = np.zeros((4, 1, 64), np.float32)
    x[0, 0, :4] = [np.inf, -np.inf, np.nan, 1.0]
    x[1, 0, :3] = [65504.0, 65519.9, 65536.0]
    x[2, 0, :3] = [2.0 ** -24, 2.0 ** -25, 3.0 * 2.0 ** -25]
    x[3, 0, 0], x[3, 0, 32] = 1e-39, 3e38
    c = Cache(F16, 1, 64, 32, 1, 1)
    put(c, dev(x), dev(x), [4], [4])
    k, v = torch.zeros(4, 1, 64, device="cuda"), torch.zeros(4, 1, 64, device="cuda")
    get(c, k, v, [4], [4])
    want = c.stored(x)
    assert np.array_equal(k.cpu().numpy(), want, equal_nan=True) and np.array_equal(v.cpu().numpy(), want, equal_nan=True)
    c = Cache(Q8_0, 1, 64, 32, 1, 1)
    put(c, dev(x), dev(x), [4], [4])
    get(c, k, v, [4], [4])
    got = k.cpu().numpy()
    assert np.array_equal(got, v.cpu().numpy(), equal_nan=True)
    assert np.isnan(got[0, 0, :32]).all() and (got[0, 0, 32:] == 0).all()  # the whole block, and no other
    assert np.array_equal(got[1:3], c.stored(x[1:3]))
    assert (got[3, 0, :32] == 0).all() and not np.isfinite(got[3, 0, 32])  # a scale beyond f16


def test_quotients_next_to_a_half_round_as_the_codec_rounds_them():
    """q8_0 values whose quotient by the scale is a half of a whole number or a few units in the last place
    beside it, for many scales: a product and a sum taken in one rounding would move some of them."""
    rng = np.random.default_rng(17)
    n, heads, hd = 512, 8, 64
    amax = rng.uniform(0.5, 4.0, (n, heads, 2, 1)).astype(np.float32)
    d = (amax / np.float32(127)).astype(np.float32)
    half = rng.integers(0, 126, (n, heads, 2, 32)).astype(np.float32) + np.float32(0.5)
    x = (half * d).astype(np.float32)
    x = (x.view(np.int32) + rng.integers(-2, 3, x.shape)).astype(np.int32).view(np.float32)
    x *= rng.choice([-1.0, 1.0], x.shape).astype(np.float32)
    x[..., 5:6] = amax
    x = x.reshape(n, heads, hd)
    c = Cache(Q8_0, heads, hd, 64, 1, n // 64)
    put(c, dev(x), dev(x[::-1].copy()), [n], [n])
    k, v = torch.zeros(n, heads, hd, device="cuda"), torch.zeros(n, heads, hd, device="cuda")
    get(c, k, v, [n], [n])
    assert np.array_equal(k.cpu().numpy(), c.stored(x)) and np.array_equal(v.cpu().numpy(), c.stored(x[::-1].copy()))


ATTEND = [  # kind, hd, K/V heads, group, page
    (F16, 64, 2, 1, 64), (Q8_0, 64, 2, 1, 64), (F16, 32, 1, 3, 32), (Q8_0, 32, 2, 2, 256), (F16, 128, 1, 5, 128),
    (Q8_0, 128, 2, 1, 32), (F16, 256, 1, 2, 64), (Q8_0, 256, 1, 7, 32), (F16, 64, 1, 16, 32), (Q8_0, 64, 1, 24, 64),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kind,hd,heads,group,page", ATTEND)
def test_attention_of_ragged_chunks(kind, hd, heads, group, page, causal):
    """Single tokens beside chunks, sequences without rows or without tokens, rows that see nothing, tokens
    that end inside a tile; whatever no sequence owns in the pool is NaN."""
    cache, held, rng = filled(kind, heads, hd, page, SPANS, 3 * hd + group)
    new, ctx = [n for n, _ in SPANS], [c for _, c in SPANS]
    q = rng.normal(0, 1, (sum(new), heads * group, hd)).astype(np.float32)
    q *= 2.0 ** rng.integers(-4, 2, (sum(new), heads * group, 1)).astype(np.float32)
    scale = 1 / np.sqrt(hd)
    got = attend(cache, dev(q), new, ctx, scale, causal).cpu().numpy()
    for i, (n, c) in enumerate(SPANS):
        a = rows_of(new)[i]
        want, err = reference(q[a:a + n], *held[i], n, c, scale, causal)
        assert (np.abs(got[a:a + n] - want) <= err).all(), (i, n, c)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 4])
def test_attention_of_long_contexts_in_splits(kind, n):
    """One sequence long enough that its tokens are split over workgroups, beside short ones; the bound on
    the tokens changes the plan, not the result beyond rounding; repeats are equal bit for bit."""
    spans = [(n, 7001), (n, 5), (n, 2048), (n, 33)]
    cache, held, rng = filled(kind, 2, 64, 128, spans, 77)
    q = rng.normal(0, 1, (4 * n, 2, 64)).astype(np.float32)
    new, ctx = [a for a, _ in spans], [c for _, c in spans]
    assert lib.mlg_attn_paged_scratch(C.byref(cache.c), 2, 4 * n, n, 0) > 0
    got = [attend(cache, dev(q), new, ctx, 0.125, max_ctx=m).cpu().numpy() for m in (0, 0, 1, 600, 7001)]
    assert np.array_equal(got[0], got[1])
    for i, (_, c) in enumerate(spans):
        want, err = reference(q[i * n:(i + 1) * n], *held[i], n, c, 0.125, True)
        for g in got:
            assert (np.abs(g[i * n:(i + 1) * n] - want) <= err).all(), i


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,group,n,past", [(64, 1, 300, 211), (128, 2, 129, 0), (64, 3, 90, 1000), (32, 8, 70, 64),
                                             (256, 1, 140, 37)])
def test_attention_of_long_chunks(kind, hd, group, n, past):
    spans = [(n, n + past), (1, 50), (n // 2, n // 2 + 3)]
    cache, held, rng = filled(kind, 1, hd, 64, spans, n)
    new, ctx = [a for a, _ in spans], [c for _, c in spans]
    q = rng.normal(0, 1, (sum(new), group, hd)).astype(np.float32)
    got = attend(cache, dev(q), new, ctx, 1 / np.sqrt(hd)).cpu().numpy()
    for i, (m, c) in enumerate(spans):
        a = rows_of(new)[i]
        want, err = reference(q[a:a + m], *held[i], m, c, 1 / np.sqrt(hd), True)
        assert (np.abs(got[a:a + m] - want) <= err).all(), i


@pytest.mark.parametrize("n", [6, 150])
@pytest.mark.parametrize("kind", KINDS)
def test_tokens_that_a_row_does_not_see_have_no_influence(kind, n):
    """Inf and NaN in the K and V of a chunk's later token: rows before it are as if it were not there, rows
    from it on get what the formula gives them (NaN)."""
    ctx, at = n + 40, n - 3  # row `at` of the chunk is the token with the bad values
    rng = np.random.default_rng(5)
    k, v = (rng.normal(0, 1, (ctx, 1, 64)).astype(np.float32) for _ in range(2))
    q = rng.normal(0, 1, (n, 1, 64)).astype(np.float32)
    out = []
    for bad in (False, True):
        cache = Cache(kind, 1, 64, 32, 1, -(-ctx // 32), seed=1)
        kk, vv = k.copy(), v.copy()
        if bad:
            kk[40 + at, 0, 3], vv[40 + at, 0, 5], vv[40 + at, 0, 40] = np.nan, np.inf, np.nan
        put(cache, dev(kk), dev(vv), [ctx], [ctx])
        out.append(attend(cache, dev(q), [n], [ctx], 0.125).cpu().numpy())
    assert np.array_equal(out[0][:at], out[1][:at])
    assert np.isnan(out[1][at:]).all() and np.isfinite(out[0]).all()


def test_an_infinite_value_reaches_its_own_dimension_alone():
    """V of a seen token holds inf in one dim (f16): that dim is not finite, the others are; in a chunk, only
    for the rows that see it."""
    rng = np.random.default_rng(6)
    ctx, n = 70, 9
    k, v = (rng.normal(0, 1, (ctx, 1, 64)).astype(np.float32) for _ in range(2))
    v[64, 0, 17] = np.inf
    q = rng.normal(0, 1, (n, 1, 64)).astype(np.float32)
    cache = Cache(F16, 1, 64, 64, 1, 2)
    put(cache, dev(k), dev(v), [ctx], [ctx])
    got = attend(cache, dev(q), [n], [ctx], 0.125).cpu().numpy()[:, 0]
    sees = np.arange(n) + ctx - n >= 64
    assert np.isfinite(got[~sees]).all() and not np.isfinite(got[sees][:, 17]).any()
    assert np.isfinite(np.delete(got[sees], 17, 1)).all()


@pytest.mark.parametrize("kind", KINDS)
def test_sizes_of_the_operands(kind):
    """Queries from 1e-30 to 1e30 (the scale bringing the scores back), scales of V from tiny to large: the
    result is as exact as for ordinary sizes."""
    spans = [(2, 90)]
    for vs, qs in ((1e-3, 1e-30), (100.0, 1e30), (1.0, 1.0)):
        rng = np.random.default_rng(9)
        cache = Cache(kind, 1, 64, 32, 1, 3)
        k = rng.normal(0, 1, (90, 1, 64)).astype(np.float32)
        v = (rng.normal(0, 1, (90, 1, 64)) * vs).astype(np.float32)
        v[:45] *= np.float32(1 / 64)  # larger scales come later
        put(cache, dev(k), dev(v), [90], [90])
        q = (rng.normal(0, 1, (2, 1, 64)) * qs).astype(np.float32)
        got = attend(cache, dev(q), [2], [90], 0.125 / qs).cpu().numpy()
        want, err = reference(q, cache.stored(k), cache.stored(v), 2, 90, float(np.float32(0.125 / qs)), True)
        assert (np.abs(got - want) <= err).all(), (vs, qs)


@pytest.mark.parametrize("scale", [0.0, -0.125, 0.125])
@pytest.mark.parametrize("n", [2, 40])
def test_scales_of_any_sign(n, scale):
    """Scale 0 weighs all that a row sees alike; a negative one prefers what a positive one avoids."""
    for kind in KINDS:
        cache, held, rng = filled(kind, 1, 64, 32, [(n, 75)], 6)
        q = rng.normal(0, 1, (n, 2, 64)).astype(np.float32)
        got = attend(cache, dev(q), [n], [75], scale).cpu().numpy()
        want, err = reference(q, *held[0], n, 75, scale, True)
        assert (np.abs(got - want) <= err).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_values_of_zero_before_others(hd, n):
    """q8_0: long runs of V that is zero, in all blocks or in one, before the first scale that is not."""
    rng = np.random.default_rng(12)
    ctx = 700
    k, v = (rng.normal(0, 1, (ctx, 1, hd)).astype(np.float32) for _ in range(2))
    v[:400] = 0
    v[400:600, :, :32] = 0
    cache = Cache(Q8_0, 1, hd, 64, 1, 11)
    put(cache, dev(k), dev(v), [ctx], [ctx])
    q = rng.normal(0, 1, (n, 1, hd)).astype(np.float32)
    got = attend(cache, dev(q), [n], [ctx], 0.125).cpu().numpy()
    want, err = reference(q, cache.stored(k), cache.stored(v), n, ctx, 0.125, True)
    assert (np.abs(got - want) <= err).all()


@pytest.mark.parametrize("hd,heads,seqs,longest", [(32, 2, 150, 2100), (64, 1, 90, 4100), (256, 1, 70, 1500)])
@pytest.mark.parametrize("kind", KINDS)
def test_many_sequences_in_splits(kind, hd, heads, seqs, longest):
    """More sequences than a wave has lanes, ragged and some without rows, a bad one among them, their tokens
    split: the join finds every row's sequence, and no other row."""
    rng = np.random.default_rng(seqs)
    ctx = rng.integers(1, 60, seqs).tolist()
    ctx[3], ctx[-1] = longest, longest - 77
    new = [min(c, int(x)) for c, x in zip(ctx, rng.integers(0, 3, seqs))]
    new[3], new[-1] = 2, 1
    cache, held, rng = filled(kind, heads, hd, 64, list(zip(new, ctx)), seqs)
    q = rng.normal(0, 1, (sum(new) + 3, heads, hd)).astype(np.float32)
    assert lib.mlg_attn_paged_scratch(C.byref(cache.c), heads, len(q), 2, 0) > 0
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    told = list(ctx)
    told[5] = 64 * cache.table_len + 1  # more than its table row holds
    got = attend(cache, dev(q), new, told, 1 / np.sqrt(hd), bad=bad).cpu().numpy()
    assert bad.item() == 1 and (got[sum(new):] == 7).all()
    off = rows_of(new)
    assert (got[off[5]:off[6]] == 0).all()
    for i in (0, 2, 3, 4, 6, 63, 64, 65, seqs - 2, seqs - 1):
        want, err = reference(q[off[i]:off[i + 1]], *held[i], new[i], ctx[i], 1 / np.sqrt(hd), True)
        assert (np.abs(got[off[i]:off[i + 1]] - want) <= err).all(), i


@pytest.mark.parametrize("n", [1, 50])
def test_out_in_the_place_of_q(n):
    cache, held, rng = filled(F16, 2, 64, 32, [(n, 90), (n, 64)], 15)
    q = dev(rng.normal(0, 1, (2 * n, 4, 64)).astype(np.float32))
    want = attend(cache, q, [n, n], [90, 64], 0.125)
    attend(cache, q, [n, n], [90, 64], 0.125, out=q)
    assert torch.equal(q, want)


def test_calls_on_two_streams_at_once():
    """Two caches written and attended on two streams without a wait between them: each as if alone."""
    made = [filled(kind, 2, 64, 64, [(1, 3000), (1, 40)], 20 + kind) for kind in KINDS]
    qs = [dev(rng.normal(0, 1, (2, 2, 64)).astype(np.float32)) for _, _, rng in made]
    want = [attend(c, q, [1, 1], [3000, 40], 0.125) for (c, _, _), q in zip(made, qs)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in made], []
    for _ in range(20):
        for st, (c, _, _), q in zip(streams, made, qs):
            with torch.cuda.stream(st):
                got.append(attend(c, q, [1, 1], [3000, 40], 0.125, sync=False))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])


def test_a_query_that_is_not_finite_spoils_its_own_row_alone():
    cache, held, rng = filled(F16, 1, 64, 32, [(4, 50)], 3)
    q = rng.normal(0, 1, (4, 1, 64)).astype(np.float32)
    clean = attend(cache, dev(q), [4], [50], 0.125).cpu().numpy()
    q[1, 0, 3], q[2, 0, 9] = np.nan, np.inf
    got = attend(cache, dev(q), [4], [50], 0.125).cpu().numpy()
    assert np.isnan(got[1:3]).all() and np.array_equal(got[[0, 3]], clean[[0, 3]])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [2, 60])
def test_pages_and_sequences_that_cannot_be_used(kind, n):
    """A page id past the pool, and sequences whose rows or tokens do not fit: flagged, never followed, the
    others as ever."""
    spans = [(n, 130), (n, 130), (n, 130)]
    cache, held, rng = filled(kind, 2, 64, 32, spans, 11, table_len=5)
    q = dev(rng.normal(0, 1, (3 * n, 2, 64)).astype(np.float32))
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    new, ctx = [n] * 3, [130] * 3
    good = attend(cache, q, new, ctx, 0.125, bad=bad)
    assert bad.item() == 0
    # sequence 1's second page does not exist: its tokens 32 .. 63 are no keys
    ids = cache.ids.copy()
    ids[1, 1] = cache.pages
    cache.table = u32(ids)
    got = attend(cache, q, new, ctx, 0.125, bad=bad)
    assert bad.item() == 1
    assert torch.equal(got[:n], good[:n]) and torch.equal(got[2 * n:], good[2 * n:])
    keep = np.r_[0:32, 64:130]
    want, err = reference(q[n:2 * n].cpu().numpy(), held[1][0][keep], held[1][1][keep], n, 98, 0.125, True)
    if 130 - n >= 64:  # every row sees all that is left of the page and what lies before it
        assert (np.abs(got[n:2 * n].cpu().numpy() - want) <= err).all()
    bad.zero_()
    k, v = torch.full((390, 2, 64), 5.0, device="cuda"), torch.full((390, 2, 64), 5.0, device="cuda")
    get(cache, k, v, [130] * 3, ctx, bad=bad)
    assert bad.item() == 1 and (k[130 + 32:130 + 64] == 0).all() and (v[130 + 32:130 + 64] == 0).all()
    assert np.array_equal(k[390 - 130:].cpu().numpy(), held[2][0])
    before = cache.pool.clone()
    ids[0, 4] = 0xffffffff
    cache.table = u32(ids)
    bad.zero_()
    put(cache, torch.ones(2, 2, 64, device="cuda"), torch.ones(2, 2, 64, device="cuda"), [2, 0, 0], [130, 130, 130],
        bad=bad)
    assert bad.item() == 1 and torch.equal(before, cache.pool)
    cache.table = u32(cache.ids)
    # more tokens than the table holds; rows past max_new; rows past the arrays
    for new2, ctx2, rows, m in ((new, [130, 161, 130], 3 * n, n), (new, [130, 0xffffffff, 130], 3 * n, n),
                                ([n, n + 1, n - 1], ctx, 3 * n, n)):
        bad.zero_()
        got = attend(cache, q, new2, ctx2, 0.125, bad=bad, max_new=m, rows=rows)
        assert bad.item() == 1
        assert torch.equal(got[:n], good[:n])
        assert (got[n:2 * n] == 0).all()
    before = cache.pool.clone()
    bad.zero_()
    put(cache, k[:3 * n], v[:3 * n], new, [130, 161, n - 1], bad=bad)  # sequence 2: more rows than tokens
    assert bad.item() == 1
    changed = (before != cache.pool).view(cache.pages, -1).any(1).nonzero().view(-1).tolist()
    assert set(changed) <= set(int(i) for i in cache.ids[0])


def test_rows_behind_the_last_sequence_are_left_alone():
    cache, held, rng = filled(F16, 1, 64, 32, [(3, 40), (1, 40)], 4)
    q = dev(rng.normal(0, 1, (9, 1, 64)).astype(np.float32))
    out = attend(cache, q, [3, 1], [40, 40], 0.125)
    assert (out[4:] == 7).all() and (out[:4] != 7).any()


def test_uniform_rows_without_offsets_and_strided_arrays():
    """row_off NULL: max_new rows each; q a slice of a fused projection's rows, out wider than it needs."""
    for n in (1, 5):
        spans = [(n, 77), (n, 40), (n, 33)]
        cache, held, rng = filled(Q8_0, 2, 64, 32, spans, 8)
        fused = dev(rng.normal(0, 1, (3 * n, 8, 64)).astype(np.float32))
        q, wide = fused[:, 2:6], torch.full((3 * n, 6, 64), 7.0, device="cuda")
        a = attend(cache, q, [n] * 3, [77, 40, 33], 0.125, off=False, out=wide[:, :4])
        b = attend(cache, q.contiguous(), [n] * 3, [77, 40, 33], 0.125)
        assert torch.equal(a, b) and (wide[:, 4:] == 7).all()


def test_a_cache_of_more_than_4_gib():
    """Pages on both sides of 2^32 bytes: an offset cut to 32 bits would land in the first ones."""
    heads, hd, page = 16, 128, 256
    pb = lib.mlg_kv_page_bytes(F16, heads, hd, page)
    pages = (1 << 32) // pb + 6
    cache = Cache(F16, heads, hd, page, 1, 2, pages=4)
    cache.pool = torch.zeros(pages * pb // 2, dtype=torch.float16, device="cuda")
    cache.pages, cache.table = pages, u32([[pages - 1, (1 << 32) // pb]])
    rng = np.random.default_rng(2)
    k, v = (rng.normal(0, 1, (300, heads, hd)).astype(np.float32) for _ in range(2))
    put(cache, dev(k), dev(v), [300], [300])
    assert not cache.pool[: 4 * pb // 2].any()
    rk, rv = torch.zeros(300, heads, hd, device="cuda"), torch.zeros(300, heads, hd, device="cuda")
    get(cache, rk, rv, [300], [300])
    assert np.array_equal(rk.cpu().numpy(), cache.stored(k)) and np.array_equal(rv.cpu().numpy(), cache.stored(v))
    q = rng.normal(0, 1, (2, heads, hd)).astype(np.float32)
    got = attend(cache, dev(q), [2], [300], 0.09).cpu().numpy()
    want, err = reference(q, cache.stored(k), cache.stored(v), 2, 300, float(np.float32(0.09)), True)
    assert (np.abs(got - want) <= err).all()


@pytest.mark.parametrize("kind", KINDS)
def test_decoding_with_the_three_together(kind):
    """As a program decodes: prompts of different lengths written and attended as one ragged chunk, then
    token after token for the sequences that still run, pages handed out as they fill; every output against
    dense attention over what the cache should hold."""
    heads, group, hd, page = 2, 2, 64, 32
    rng = np.random.default_rng(21)
    prompts, steps = [37, 1, 64, 30], 36
    cache = Cache(kind, heads, hd, page, 4, 4, seed=5)
    k = [np.zeros((0, heads, hd), np.float32) for _ in prompts]
    v = [np.zeros((0, heads, hd), np.float32) for _ in prompts]
    for step in range(steps + 1):
        new = prompts if step == 0 else [1 if step <= 9 * (i + 1) else 0 for i in range(4)]
        rows = rng.normal(0, 1, (sum(new), heads * (group + 2), hd)).astype(np.float32)
        fused, at = dev(rows), 0
        for i, n in enumerate(new):
            k[i] = np.concatenate([k[i], cache.stored(rows[at:at + n, heads * group:heads * (group + 1)])]) if n else k[i]
            v[i] = np.concatenate([v[i], cache.stored(rows[at:at + n, heads * (group + 1):])]) if n else v[i]
            at += n
        ctx = [len(x) for x in k]
        put(cache, fused[:, heads * group:heads * (group + 1)], fused[:, heads * (group + 1):], new, ctx)
        got = attend(cache, fused[:, :heads * group], new, ctx, 0.125).cpu().numpy()
        if step not in (0, 1, 8, 20, steps):
            continue
        at = 0
        for i, n in enumerate(new):
            want, err = reference(rows[at:at + n, :heads * group], k[i], v[i], n, ctx[i], 0.125, True)
            assert (np.abs(got[at:at + n] - want) <= err).all(), (step, i)
            at += n


def test_captured_step_replayed_as_the_cache_grows():
    """One token's write and attention captured once and replayed with the tokens counted on the device, the
    eager calls of the same step on a second cache between the replays: equal bit for bit.  A second graph
    with its own scratch replays on another stream meanwhile."""
    heads, hd, page, seqs = 2, 64, 32, 3
    rng = np.random.default_rng(31)
    caches = [Cache(Q8_0, heads, hd, page, seqs, 40, seed=2) for _ in range(3)]
    start = [700, 31, 1]
    k0 = rng.normal(0, 1, (2, sum(start), heads, hd)).astype(np.float32)
    for c in caches:
        put(c, dev(k0[0]), dev(k0[1]), start, start)
    x = torch.zeros(seqs, 3 * heads, hd, device="cuda")
    ctx = u32(start)
    n = lib.mlg_attn_paged_scratch(C.byref(caches[0].c), heads, seqs, 1, 1280)
    assert n > 0
    outs = [torch.zeros(seqs, heads, hd, device="cuda") for _ in range(3)]
    scratch = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(3)]

    def step(i):
        c, ld = caches[i].c, 3 * heads * hd
        kp, vp = x[:, heads:].data_ptr(), x[:, 2 * heads:].data_ptr()
        _lib.check(lib.mlg_kv_write(C.byref(c), kp, ld, vp, ld, None, ctx.data_ptr(), seqs, 1, None, stream()))
        _lib.check(lib.mlg_attn_paged(C.byref(c), x.data_ptr(), ld, heads, 0.125, 1, None, ctx.data_ptr(), seqs, 1, 1280,
                                      outs[i].data_ptr(), heads * hd, scratch[i].data_ptr(), n, None, stream()))

    graphs, side = [], torch.cuda.Stream()
    for i in (1, 2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(i)
        graphs.append(g)
    for t in range(1, 6):
        x.copy_(dev(rng.normal(0, 1, (seqs, 3 * heads, hd)).astype(np.float32)))
        ctx.copy_(u32([s + t for s in start]))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        step(0)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]), t
        assert outs[0].abs().sum() > 0
    assert torch.equal(caches[0].pool, caches[1].pool) and torch.equal(caches[0].pool, caches[2].pool)


def test_sequences_that_share_pages():
    """Two sequences whose first pages are one prefix's, attended together: each as over a copy of its own."""
    cache, held, rng = filled(F16, 2, 64, 32, [(1, 64), (1, 90), (1, 90)], 13, table_len=3)
    ids = cache.ids.copy()
    ids[2, :2] = ids[1, :2]  # sequence 2: sequence 1's first 64 tokens, then its own
    cache.table = u32(ids)
    q = rng.normal(0, 1, (3, 2, 64)).astype(np.float32)
    got = attend(cache, dev(q), [1, 1, 1], [64, 90, 90], 0.125).cpu().numpy()
    kv = [np.concatenate([held[1][w][:64], held[2][w][64:]]) for w in (0, 1)]
    for i, (k, v) in enumerate((held[0], held[1], kv)):
        want, err = reference(q[i:i + 1], k, v, 1, len(k), 0.125, True)
        assert (np.abs(got[i:i + 1] - want) <= err).all()
