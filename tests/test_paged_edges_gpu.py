"""Paged-cache operators at the edges of what their arguments allow.

Attention is held to the 64-bit formula and tolerance of ``test_paged_gpu``; everything else is compared exactly.
"""

import math

import pytest
import torch

from test_paged_gpu import DEV, UNIT, Book, attention_64, check_attention, ints
from tiktoktechjam2026_b200 import PagedKVCache, _lib, ops

gpu = pytest.mark.gpu

# Calls for each kernel of the attention: (new tokens, tokens before them, KV heads, query heads).  "item": short rows
# over short tables; "rows": short rows, tables past 640 KB of cache, more than 32 (sequence, KV head) pairs; "chunk":
# more than 16 rows; "few": short rows over a long cache, at most 16 pairs.
LONG = {16: 11000, 32: 6000, 64: 3000, 128: 1500, 256: 800}


def call_of(route, hd):
    if route == "item":
        return [1, 2, 3, 1], [0, 15, 297, 63], 2, 4
    if route == "rows":
        return [1, 2, 1, 4, 1, 1, 3, 1, 1], [LONG[hd], 5, 64, 700, 0, 129, LONG[hd] // 2, 1, 300], 4, 8
    if route == "few":
        return [1, 3], [LONG[hd], 70], 2, 4
    return [1, 130, 40, 300], [300, 64, 500, 0], 2, 4


def word_is_clear():
    word = _lib.c_uint()
    return _lib.lib().tt_device_error(_lib.ctypes.byref(word), 0) == 0


# ------------------------------------------------------------------------------------- order of kernels
@gpu
@pytest.mark.parametrize("news,past,hd,room", [
    ([60, 33], [4, 0], 64, 0),            # chunk kernel, one key tile for each item: nothing is cut
    ([300, 200], [5000, 0], 64, 0),       # chunk kernel, items are cut
    ([1] * 40, [3] * 40, 128, 2000),      # rows kernel, one tile for each item, in a wide table
    ([1] * 40, [1500] * 40, 128, 0),      # rows kernel, items are cut
])
def test_graph_node_after_attention_sees_its_rows(tt_lib, news, past, hd, room):
    """A captured consumer of the output depends on the last kernel of the call alone: that one ends after the first."""
    totals = [n + p for n, p in zip(news, past)]
    book = Book(31, totals + ([room] if room else []), 2, hd, 64, torch.float16)
    slots = book.slots[: len(news)].contiguous()
    cu = [0]
    for t in news:
        cu.append(cu[-1] + t)
    q = torch.randn(cu[-1], 4, hd, device=DEV).half()
    out = torch.zeros(cu[-1], 4 * hd, dtype=torch.float16, device=DEV)
    seen = torch.zeros_like(out)
    call = lambda: ops.paged_attention(q, book.pages_k, book.pages_v, book.tables, book.lens, cu_q, slots=slots, out=out)  # noqa: E731
    cu_q = ints(cu)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
        seen.copy_(out)
    for _ in range(20):
        q.normal_()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = seen.clone()
        call()
        assert torch.equal(replayed, out)
    assert word_is_clear()


@gpu
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 3)])
def test_attention_where_a_half_sees_few_tiles(tt_lib, hd, window, sinks):
    """Of an item's two query tiles one is empty, or sees only some of the key tiles that pass through the ring."""
    news, past = [20, 129, 200, 1], [9000, 3000, 64, 5000]
    book = Book(hd, [n + p for n, p in zip(news, past)], 1, hd, 64, torch.bfloat16)
    for heads in (1, 5):
        check_attention(book, news, heads, torch.bfloat16, window=window, sinks=sinks)


@gpu
def test_compact_skips_entries_that_name_a_free_page(tt_lib):
    """A table entry whose page has no count stays as it is; the live pages move as ever."""
    k = torch.randn(2, 8, 1, 16, 16, device=DEV).half()
    v = torch.randn(2, 8, 1, 16, 16, device=DEV).half()
    k0, v0 = k.clone(), v.clone()
    tables, lens, refs = ints([[2, 7, -1], [6, 5, 9]]), ints([32, 0]), ints([0, 0, 1, 0, 0, 0, 0, 1])
    for _ in range(3):  # (the call's scratch is memory that earlier work has written)
        junk = torch.full((64,), 1 << 28, dtype=torch.int32, device=DEV)
        del junk
        live = ops.cache_compact(k, v, tables, lens, refs)
        assert live.item() == 2
        assert tables.tolist() == [[0, 1, -1], [6, 5, 9]] and refs.tolist() == [1, 1, 0, 0, 0, 0, 0, 0]
    for a, b in ((2, 0), (7, 1)):
        k0[:, b], v0[:, b] = k0[:, a], v0[:, a]
    assert torch.equal(k, k0) and torch.equal(v, v0)


# ---------------------------------------------------------------------------------------------- scale
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("route", ["item", "rows", "few", "chunk"])
@pytest.mark.parametrize("scale", [-0.25, 0.0, -0.0, 0.5, 1e-30])
def test_attention_scales(tt_lib, dtype, hd, route, scale):
    """Any finite scale, on every kernel: hidden keys stay hidden whatever its sign."""
    news, past, kv_heads, heads = call_of(route, hd)
    book = Book(hd + 1, [n + p for n, p in zip(news, past)], kv_heads, hd, 64, dtype)
    check_attention(book, news, heads, dtype, scale=scale)
    check_attention(book, news, heads, dtype, scale=scale, window=40, sinks=3)


@gpu
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39, 3e38])
def test_attention_refuses_a_scale_that_is_not_finite(tt_lib, scale):
    book = Book(1, [20, 40], 2, 32, 16, torch.float16)
    q = torch.randn(2, 4, 32, device=DEV).half()
    with pytest.raises(_lib.TTError, match="scale"):
        ops.paged_attention(q, book.pages_k, book.pages_v, book.tables, book.lens, ints([0, 1, 2]), scale=scale)


# --------------------------------------------------------------------------------- reservations and their appends
def _cache_with_one_sequence():
    cache = PagedKVCache(1, 4, 1, 16, slots=4, max_len=96, page=16, device=DEV)
    cache.k.zero_(), cache.v.zero_()
    cu, slot = ints([0, 40]), ints([0])
    status = cache.reserve(cu, slot)
    cache.append(0, torch.ones(40, 1, 16, device=DEV).half(), torch.ones(40, 1, 16, device=DEV).half(), cu, slot,
                 status=status)
    cache.check()
    return cache


@gpu
@pytest.mark.parametrize("between", ["reserve", "fork", "nothing"])
def test_append_of_a_refused_reservation_writes_nothing(tt_lib, between):
    """Whatever is reserved or forked after it: an append goes by the answer to its own reservation."""
    cache = _cache_with_one_sequence()
    k, v = cache.k.clone(), cache.v.clone()
    cu, slots = ints([0, 24, 40]), ints([0, 1])
    refused = cache.reserve(cu, slots)  # two pages, one is free
    if between == "reserve":
        cache.reserve(ints([0, 5]), ints([2]))
        cache.check()
    elif between == "fork":
        cache.fork(ints([0]), ints([3]))
        cache.check()
        k, v = cache.k.clone(), cache.v.clone()  # (the child's copy of the partial page)
    new = torch.full((40, 1, 16), 7.0, device=DEV).half()
    cache.append(0, new, new, cu, slots, status=refused)
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v)
    with pytest.raises(RuntimeError, match="short"):
        cache.check(refused)


@gpu
def test_append_of_an_accepted_reservation_survives_a_refused_call(tt_lib):
    cache = _cache_with_one_sequence()
    cu, slot = ints([0, 8]), ints([0])
    granted = cache.reserve(cu, slot)
    cache.fork(ints([0]), ints([0]))  # not empty
    with pytest.raises(RuntimeError, match="empty"):
        cache.check()
    new = torch.full((8, 1, 16), 7.0, device=DEV).half()
    cache.append(0, new, new, cu, slot, status=granted)
    page = int(cache.tables[0, 2])
    assert torch.all(cache.k[0, page, 0, 8:] == 7) and torch.all(cache.k[0, page, 0, :8] == 1)


@gpu
def test_append_names_its_reservation(tt_lib):
    cache = _cache_with_one_sequence()
    new = torch.zeros(8, 1, 16, device=DEV).half()
    with pytest.raises(TypeError, match="status"):
        cache.append(0, new, new, ints([0, 8]), ints([0]))


# -------------------------------------------------------------------------------------- windows past 32 bits
@gpu
@pytest.mark.parametrize("route", ["item", "chunk"])
def test_attention_window_of_any_size(tt_lib, route):
    """A window or first tokens past every position are as good as all keys, also past 32 bits."""
    news, past, kv_heads, heads = call_of(route, 64)
    book = Book(3, [n + p for n, p in zip(news, past)], kv_heads, 64, 16, torch.float16)
    q = torch.randn(sum(news), heads, 64, device=DEV).half()
    cu = [0]
    for t in news:
        cu.append(cu[-1] + t)
    call = lambda **kw: ops.paged_attention(q, book.pages_k, book.pages_v, book.tables, book.lens, ints(cu),  # noqa: E731
                                            slots=book.slots, **kw)
    want = call()
    for window in (1 << 30, 2**31 - 1, 2**31, 2**32, 2**32 + 5, 2**40):
        assert torch.equal(call(window=window), want)
    for sinks in (2**31 - 1, 2**31, 2**32, 2**32 + 1):
        torch.testing.assert_close(call(window=20, sinks=sinks), want, rtol=2e-3, atol=2e-3)


@gpu
def test_trim_behind_a_window_of_any_size(tt_lib):
    tables, lens, refs = ints([[1, 0, 2, -1]]), ints([48]), ints([1, 1, 1])
    for window, sinks in ((2**31, 0), (2**32, 0), (2**32 + 1, 0), (1, 2**32), (1, 2**31)):
        ops.cache_release(tables, lens, refs, 16, window=window, sinks=sinks)
        assert tables.tolist() == [[1, 0, 2, -1]] and lens.tolist() == [48] and refs.tolist() == [1, 1, 1]
    with pytest.raises(_lib.TTError, match="negative"):
        ops.cache_release(tables, lens, refs, 16, window=-(2**32))
    assert lens.tolist() == [48]


# ------------------------------------------------------------------------------------------- hidden keys
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [1, 4])
def test_hidden_values_weigh_nothing(tt_lib, dtype, hd, heads):
    """The largest finite values at positions that a row does not see leave the row as it is, bit for bit."""
    big = torch.finfo(dtype).max
    book = Book(hd, [228], 1, hd, 32, dtype)
    q = torch.randn(200, heads, hd, device=DEV).to(dtype)
    row = book.tables[book.slot_of[0]].tolist()

    def call(value, lo, hi, window):
        v = book.pages_v.clone()
        for u in range(lo, hi):
            v[row[u // 32], :, u % 32] = value
        return ops.paged_attention(q, book.pages_k, v, book.tables, book.lens, ints([0, 200]), slots=book.slots,
                                   window=window)

    late, none = call(big, 100, 228, 0), call(0.0, 100, 228, 0)
    assert torch.equal(late[:72], none[:72])  # positions 28 .. 99
    late, none = call(big, 0, 60, 30), call(0.0, 0, 60, 30)
    assert torch.equal(late[62:], none[62:])  # positions 90 .. 227 see 61 and later


# ------------------------------------------------------------------------------------- strides of single entries
def odd(t, **strides):
    """t with other strides in dimensions of size one (named d0, d1, ...): the same elements."""
    st = list(t.stride())
    for name, s in strides.items():
        assert t.shape[int(name[1:])] == 1
        st[int(name[1:])] = s
    return t.as_strided(t.shape, st)


@gpu
@pytest.mark.parametrize("total,window", [(40, 0), (9000, 0), (9000, 33)])
def test_strides_of_single_entries_do_not_matter(tt_lib, total, window):
    """One token, one head, one page, one slot, one layer: the stride of that dimension addresses nothing."""
    book = Book(4, [total], 1, 64, 32, torch.float16, spare=0)
    k, v, lens, cu = book.pages_k, book.pages_v, book.lens, ints([0, 1])
    q = torch.randn(1, 4, 64, device=DEV).half()
    want = ops.paged_attention(q, k, v, book.tables, lens, cu, window=window)
    for args in ((odd(q, d0=7), k, v, book.tables), (q, odd(k, d1=5), odd(v, d1=3), book.tables),
                 (q, k, v, odd(book.tables, d0=1))):
        assert torch.equal(ops.paged_attention(*args, lens, cu, window=window), want)
    wide, short = ints([[int(book.tables[0, 0]), 5, 7]]), ints([9])  # (a page whose rows all hold values)
    args = (q, k, v, wide[:, ::2][:, :1], short, cu), (q, k, v, wide[:, :1], short, cu)
    assert torch.equal(ops.paged_attention(*args[0]), ops.paged_attention(*args[1]))
    one = torch.randn(33, 1, 64, device=DEV).half()
    want = ops.paged_attention(one, k, v, book.tables, lens, ints([0, 33]))
    assert torch.equal(ops.paged_attention(odd(one, d1=9), k, v, book.tables, lens, ints([0, 33])), want)


@gpu
def test_append_and_compact_ignore_strides_of_single_entries(tt_lib):
    tables, lens, cu = ints([[0, -1]]), ints([7]), ints([0, 1])
    new = torch.randn(1, 2, 32, device=DEV).half()
    k = torch.zeros(1, 2, 16, 32, dtype=torch.float16, device=DEV)
    want = k.clone()
    want[0, :, 6] = new[0]
    got = [torch.zeros_like(k) for _ in range(2)]
    ops.cache_append(odd(new, d0=3), odd(new, d0=5), odd(got[0], d0=11), odd(got[1], d0=1), tables, lens, cu)
    assert torch.equal(got[0], want) and torch.equal(got[1], want)
    turned = new.transpose(1, 2).contiguous().transpose(1, 2)  # dense in nothing but the token
    got = [torch.zeros_like(k) for _ in range(2)]
    ops.cache_append(odd(turned, d0=3), odd(turned, d0=64), *got, tables, lens, cu)
    assert torch.equal(got[0], want) and torch.equal(got[1], want)
    k1 = torch.randn(1, 3, 1, 16, 32, device=DEV).half()
    k2, refs, table = k1.clone(), ints([0, 0, 1]), ints([[2]])
    ops.cache_compact(odd(k1, d0=13, d2=1), odd(k2, d0=3, d2=7), table, ints([16]), refs)
    assert table.tolist() == [[0]] and torch.equal(k1[:, 0], k1[:, 2]) and torch.equal(k1, k2)


# ------------------------------------------------------------------------------- groupings and routes less travelled
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [16, 64, 128, 256])
@pytest.mark.parametrize("group", [9, 15, 16, 17, 31, 64, 100, 127, 128])
def test_attention_large_groups(tt_lib, dtype, hd, group):
    """9 to 128 query heads to a KV head; from 17 on single tokens take the chunk kernel too."""
    news, past = [1, 1, 5, 40, 0, 2], [0, 700, 64, 100, 9, 2000]
    book = Book(hd + group, [n + p for n, p in zip(news, past)], 2, hd, 32, dtype)
    check_attention(book, news, 2 * group, dtype)
    check_attention(book, news, 2 * group, dtype, window=33, sinks=2, layout="heads")


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (3000, 65)])
def test_attention_short_rows_over_wide_tables(tt_lib, dtype, hd, window, sinks):
    """The rows kernel and its join at every head_dim: ragged tokens, some over caches that are cut."""
    news, past, kv_heads, heads = call_of("rows", hd)
    book = Book(hd + 7, [n + p for n, p in zip(news, past)], kv_heads, hd, 64, dtype)
    check_attention(book, news, heads, dtype, window=window, sinks=sinks)


@gpu
@pytest.mark.parametrize("route", ["rows", "few", "chunk"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_head_dim_8_on_every_kernel(tt_lib, route, dtype):
    news, past, kv_heads, heads = call_of(route, 16)
    book = Book(12, [n + p for n, p in zip(news, past)], kv_heads, 16, 32, dtype)
    check_attention(book, news, heads, dtype, hd_out=8)


@gpu
@pytest.mark.parametrize("hd,dtype,kv_heads,group", [(16, torch.bfloat16, 4, 1), (32, torch.float16, 3, 2),
                                                     (64, torch.bfloat16, 2, 5), (128, torch.bfloat16, 4, 1),
                                                     (256, torch.float16, 2, 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
def test_attention_chunks_and_tokens_in_two_launches(tt_lib, hd, dtype, kv_heads, group, window, sinks):
    """More than two (sequence, KV head) pairs per SM: longer chunks and short rows go by their own kernels."""
    n = 320 // kv_heads + 60
    news = [40 if i % 16 == 0 else (i % 3) for i in range(n)]
    past = [(37 * i) % 90 for i in range(n)]
    past[3] = LONG[hd]
    book = Book(hd + kv_heads, [a + b for a, b in zip(news, past)], kv_heads, hd, 32, dtype)
    check_attention(book, news, kv_heads * group, dtype, window=window, sinks=sinks)


@gpu
@pytest.mark.parametrize("hd,group,page", [(128, 4, 64), (64, 1, 16), (32, 1, 128), (256, 2, 32), (16, 5, 16)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (129, 67), (1000, 4), (5000, 9)])
def test_attention_window_bf16(tt_lib, hd, group, page, window, sinks):
    news, past = [1, 1, 7, 40, 300, 1, 129], [0, 3000, 100, 1500, 64, 130, 1000]
    book = Book(window + hd, [n + p for n, p in zip(news, past)], 1, hd, page, torch.bfloat16)
    check_attention(book, news, group, torch.bfloat16, window=window, sinks=sinks)


# ------------------------------------------------------------------------------------------ huge scores
def _equal_keys(route, hd, dtype, size, sign, top):
    """Rows whose scores are sign * hd ** 0.5 * size ** 2, or `top` times that for every third key -> (own, o, a)."""
    news, past, kv_heads, heads = call_of(route, hd)
    book = Book(hd + 3, [n + p for n, p in zip(news, past)], kv_heads, hd, 64, dtype)
    book.pages_k[~torch.isnan(book.pages_k)] = size
    q = torch.full((sum(news), heads, hd), sign * size, device=DEV).to(dtype)
    cu = [0]
    for b, slot in enumerate(book.slot_of):
        row = book.tables[slot].tolist()
        book.k[b][:] = float(torch.tensor(size).to(dtype))
        book.k[b][::3] *= top
        for u in range(0, book.k[b].shape[0], 3):
            book.pages_k[row[u // 64], :, u % 64] *= top
        cu.append(cu[-1] + news[b])
    got = ops.paged_attention(q, book.pages_k, book.pages_v, book.tables, book.lens, ints(cu), slots=book.slots,
                              max_q_len=max(news))
    got = got.cpu().double().view(-1, heads, hd)
    for b in range(len(news)):
        o, a = attention_64(q[cu[b]:cu[b + 1]].cpu().double(), book.k[b], book.v[b], hd**-0.5, 0, 0)
        yield got[cu[b]:cu[b + 1]], o, a, book.k[b].shape[0] * 2.0**-25 * float(book.v[b].abs().max()) + 2.0**-24


@gpu
@pytest.mark.parametrize("dtype,size", [(torch.float16, 60000.0), (torch.bfloat16, 60000.0), (torch.bfloat16, 2.0**50)])
@pytest.mark.parametrize("hd", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("route", ["item", "rows"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attention_short_rows_huge_scores(tt_lib, dtype, size, hd, route, sign):
    """Queries and keys near the type's largest: equal scores give the mean, a larger one takes its row."""
    u = UNIT[dtype]
    for top in (1.0, 0.5):
        for got, o, a, small in _equal_keys(route, hd, dtype, size, sign, top):
            assert torch.all((got - o).abs() <= 2 * u * o.abs() + 2 * u * a + 2e-4 * a + small)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("route", ["few", "chunk"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("bits", [10, 20, 26])
def test_attention_large_scores(tt_lib, dtype, hd, route, sign, bits):
    """Scaled scores of 2^9 to 2^26 (log2 e included): a score s counts to s 2^-23, so that two weights of a row differ
    by a factor of at most 2^(s 2^-22) from the formula's."""
    size = float(2.0 ** ((bits - 0.5 * math.log2(hd) - math.log2(math.log2(math.e))) / 2) * 0.99)
    size = float(torch.tensor(size).to(dtype))
    s, u = hd**0.5 * size * size * math.log2(math.e), UNIT[dtype]
    assert 2.0 ** (bits - 1) <= s <= 2.0**bits
    for got, o, a, small in _equal_keys(route, hd, dtype, size, sign, 1.0):
        vmax = 8.0  # a row lies within its values, whatever their weights
        tol = (2.0 ** min(s * 2.0**-22, 8.0) - 1) * a + 2 * u * o.abs() + 2 * u * a + 2e-4 * a + small
        assert torch.all((got - o).abs() <= tol) and torch.all(got.abs() <= vmax)


@gpu
def test_attention_without_heads_is_refused(tt_lib):
    book = Book(1, [20, 40], 2, 32, 16, torch.float16)
    q = torch.randn(2, 4, 32, device=DEV).half()
    with pytest.raises(ValueError, match="heads"):
        ops.paged_attention(q[:, :0], book.pages_k, book.pages_v, book.tables, book.lens, ints([0, 1, 2]))
