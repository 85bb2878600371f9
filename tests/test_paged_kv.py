"""The paged K/V cache without a GPU: where the layout puts every value, what the kernels take a
sequence's rows and tokens to be, and the refusals of the entry points."""
import ctypes as C

import numpy as np
import pytest

from malaga_amd import _lib

F16, Q8_0 = _lib.F16, _lib.Q8_0
lib = _lib.load()


def cache(**kw):
    a = dict(type=F16, heads=2, head_size=64, page=64, pages=3, pool=4096, table=8192, seqs=2, table_len=4)
    a.update(kw)
    return _lib.KvCache(*[a[n] for n, _ in _lib.KvCache._fields_])


@pytest.mark.parametrize("t", [F16, Q8_0])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("page", [32, 128])
def test_every_value_has_a_place_of_its_own(t, hd, page):
    """Pages, heads, K and V, tokens and dims fill the pool's bytes exactly once, scales included, and
    lie where the header's formulas say."""
    heads, pages = 2, 2
    c = cache(type=t, heads=heads, head_size=hd, page=page, pages=pages)
    pb = lib.mlg_kv_page_bytes(t, heads, hd, page)
    tile = (64 if t == F16 else 34) * hd
    assert pb == heads * 2 * page // 32 * tile
    seen = np.zeros(pages * pb, np.int32)
    sb = C.c_int64()
    for pid in range(pages):
        for head in range(heads):
            for which in range(2):
                for pos in range(page):
                    x = pos % 32
                    for d in range(hd):
                        at = lib.mlg_debug_kv_place(C.byref(c), pid, head, which, 5 * page + pos, d, C.byref(sb))
                        if which == 0 and t == F16:
                            e = ((d // 32 * 2 + x // 4 % 2) * 64 + d // 8 % 4 * 16 + x // 8 * 4 + x % 4) * 8 + d % 8
                        elif which == 0:
                            e = ((d // 32 * 64 + d // 8 % 4 * 16 + x // 8 * 4 + x % 4) * 2 + x // 4 % 2) * 8 + d % 8
                        elif t == F16:
                            e = (d // 16 * 64 + x // 8 * 16 + d % 16) * 8 + x % 8
                        else:
                            e = ((d // 32 * 64 + x // 8 * 16 + d % 16) * 2 + d // 16 % 2) * 8 + x % 8
                        base = (((pid * heads + head) * 2 + which) * (page // 32) + pos // 32) * tile
                        assert at == base + (2 * e if t == F16 else e)
                        seen[at: at + (2 if t == F16 else 1)] += 1
                        if t == Q8_0:
                            assert sb.value == base + 32 * hd + (d // 32 * 32 + x) * 2
                            if d % 32 == 0:
                                seen[sb.value: sb.value + 2] += 1
                        else:
                            assert sb.value == -1
    assert (seen == 1).all()


def test_places_past_32_bits_and_out_of_range():
    c = cache(type=Q8_0, heads=16, head_size=128, page=256, pages=1 << 20, table_len=1 << 15)
    pb = lib.mlg_kv_page_bytes(Q8_0, 16, 128, 256)
    assert lib.mlg_debug_kv_place(C.byref(c), (1 << 20) - 1, 15, 1, 255, 127, None) > ((1 << 20) - 1) * pb
    assert lib.mlg_debug_kv_place(C.byref(c), (1 << 20) - 1, 15, 1, 255, 127, None) < (1 << 20) * pb
    for bad in [(1 << 20, 0, 0, 0, 0), (0, 16, 0, 0, 0), (0, 0, 2, 0, 0), (0, 0, 0, -1, 0), (0, 0, 0, 0, 128)]:
        assert lib.mlg_debug_kv_place(C.byref(c), *bad, None) == -1


def seq(c, off, ctx, rows, max_new, i):
    o = None if off is None else np.array(off, np.uint32)
    x = np.array(ctx, np.uint32)
    v = [C.c_int() for _ in range(4)]
    _lib.check(lib.mlg_debug_kv_seq(C.byref(c), None if o is None else o.ctypes.data, x.ctypes.data, rows, max_new, i,
                                    *[C.byref(e) for e in v]))
    return tuple(e.value for e in v)


def test_rows_and_tokens_of_a_sequence():
    c = cache(seqs=3, table_len=4, page=64)  # 256 tokens at most
    assert seq(c, [0, 5, 5, 9], [256, 0, 4], 9, 5, 0) == (0, 5, 256, 1)
    assert seq(c, [0, 5, 5, 9], [256, 0, 4], 9, 5, 1) == (5, 0, 0, 1)  # no rows, no tokens
    assert seq(c, [0, 5, 5, 9], [256, 0, 4], 9, 5, 2) == (5, 4, 4, 1)
    assert seq(c, None, [1, 2, 3], 9, 3, 2) == (6, 3, 3, 1)


@pytest.mark.parametrize("off,ctx,rows,max_new,want", [
    ([0, 4], [257], 4, 4, (0, 4, 0, 0)),            # more tokens than the table row holds
    ([0, 4], [0xffffffff], 4, 4, (0, 4, 0, 0)),
    ([0, 4], [9], 4, 3, (0, 3, 0, 0)),              # more rows than max_new
    ([0, 4], [9], 3, 4, (0, 3, 0, 0)),              # past the arrays' rows
    ([4, 2], [9], 8, 4, (4, 0, 0, 0)),              # falling
    ([0xfffffff0, 0xffffffff], [9], 8, 20, (8, 0, 0, 0)),
    ([2, 0xffffffff], [9], 8, 4, (2, 4, 0, 0)),
])
def test_sequences_that_cannot_be_followed(off, ctx, rows, max_new, want):
    first, n, tokens, usable = seq(cache(seqs=1), off, ctx, rows, max_new, 0)
    assert (first, n, tokens, usable) == want
    assert 0 <= first <= rows and first + n <= rows and n <= max_new


def write(c, ld=128, rows=4, max_new=4, k=16, v=32, ctx=64, off=48, ldv=None):
    return lib.mlg_kv_write(c, k, ld, v, ld if ldv is None else ldv, off, ctx, rows, max_new, None, None)


def read(c, ld=128, rows=4, max_new=4, k=16, v=32, ctx=64, off=48, ldv=None):
    return lib.mlg_kv_read(c, k, ld, v, ld if ldv is None else ldv, off, ctx, rows, max_new, None, None)


def attend(c, ld=256, rows=4, max_new=4, k=16, v=32, ctx=64, off=48, ldv=None, heads=4, scale=0.125, max_ctx=0,
           scratch=None, size=0):
    return lib.mlg_attn_paged(c, k, ld, heads, scale, 1, off, ctx, rows, max_new, max_ctx, v,
                              ld if ldv is None else ldv, scratch, size, None, None)


@pytest.mark.parametrize("call", [write, read, attend])
def test_refusals_before_any_launch(call):
    """Host checks: none of these pointers is memory."""
    INV, UNS = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED
    assert call(None) == INV
    for kw in (dict(pool=None), dict(table=None), dict(heads=0), dict(pages=0), dict(seqs=-1), dict(table_len=0),
               dict(pool=4104), dict(page=256, table_len=1 << 23)):
        assert call(C.byref(cache(**kw))) == INV, kw
    for kw in (dict(type=_lib.F32), dict(type=_lib.Q4_K), dict(type=_lib.BF16), dict(head_size=16), dict(head_size=96),
               dict(page=16), dict(page=48), dict(page=512), dict(page=0)):
        assert call(C.byref(cache(**kw))) == UNS, kw
    c = C.byref(cache())
    for kw in (dict(k=None), dict(v=None), dict(ctx=None), dict(rows=-1), dict(max_new=0), dict(k=8), dict(v=24),
               dict(ld=124), dict(ld=258), dict(ldv=64), dict(ldv=259), dict(off=None, rows=7)):
        assert call(c, **kw) == INV, kw
        assert _lib.load().mlg_last_error()


def test_refusals_of_the_attention():
    INV = _lib.ERR_INVALID
    c = cache()
    for kw in (dict(heads=0), dict(heads=3), dict(heads=-2), dict(scale=float("inf")), dict(scale=float("nan")),
               dict(max_ctx=-1)):
        assert attend(C.byref(c), **kw) == INV, kw
    # one sequence over a long table: the call splits its tokens and needs scratch
    c = cache(seqs=1, table_len=2048, page=256)
    need = lib.mlg_attn_paged_scratch(C.byref(c), 4, 1, 1, 0)
    assert need > 0
    for kw in (dict(), dict(scratch=64, size=need - 1), dict(scratch=72, size=need)):
        assert attend(C.byref(c), rows=1, max_new=1, **kw) == INV, kw
        assert b"scratch" in lib.mlg_last_error()
    # a bound on the tokens bounds the plan; nothing to plan where the arguments are not usable
    assert lib.mlg_attn_paged_scratch(C.byref(c), 4, 1, 1, 40) == 0
    assert lib.mlg_attn_paged_scratch(None, 4, 1, 1, 0) == 0
    assert lib.mlg_attn_paged_scratch(C.byref(c), 3, 1, 1, 0) == 0
    assert lib.mlg_attn_paged_scratch(C.byref(cache(page=48)), 4, 1, 1, 0) == 0


@pytest.mark.parametrize("call", [write, read, attend])
def test_sizes_beyond_the_kernels_indexes(call):
    """Pages of 2^32 bytes, and launches of more workgroups or rows than a grid or an int has."""
    big = cache(heads=1 << 18, head_size=128, page=256)
    assert call(C.byref(big), ld=1 << 27, ldv=1 << 27, **(dict(heads=1 << 18) if call is attend else {})) == _lib.ERR_INVALID
    wide = cache(seqs=1 << 30, heads=8)
    assert call(C.byref(wide), ld=1024, **(dict(heads=8, scratch=16, size=1 << 62) if call is attend else {})) == \
        _lib.ERR_INVALID
    if call is attend:
        assert attend(C.byref(cache(seqs=1, heads=1)), ld=1 << 20, ldv=1 << 20, heads=1 << 14, max_new=1 << 20,
                      scratch=16, size=1 << 62) == _lib.ERR_INVALID


@pytest.mark.parametrize("call", [write, read, attend])
def test_nothing_to_do_is_ok(call):
    """No sequences, or no rows: no launch, so no device either."""
    assert call(C.byref(cache(seqs=0))) == _lib.OK
    assert call(C.byref(cache()), rows=0) == _lib.OK


def test_page_bytes():
    assert lib.mlg_kv_page_bytes(F16, 16, 64, 64) == 16 * 64 * 64 * 2 * 2
    assert lib.mlg_kv_page_bytes(Q8_0, 16, 64, 64) == 16 * 64 * 64 * 2 * 34 // 32
    for a in [(F16, 0, 64, 64), (F16, 16, 48, 64), (F16, 16, 64, 16), (_lib.F32, 16, 64, 64), (_lib.Q6_K, 16, 256, 64)]:
        assert lib.mlg_kv_page_bytes(*a) == -1
