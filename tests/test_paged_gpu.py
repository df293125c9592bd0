"""Paged-cache operators against plain 64-bit formulas and a plain Python page book.

Attention tolerance, per element, with u the unit roundoff of the 16-bit type
(2^-11 FP16, 2^-9 BF16) and A = sum_u p_u |v_u|: the output is rounded once
(u |o|), every probability once before it multiplies v (u A), the exponential
is good to 1e-4 (1e-4 A), FP32 scores of magnitude s carry hd 2^-24 s (below
1e-4 A here), and an FP16 probability below 2^-14 is off by up to 2^-25
(n 2^-25 max|v|).  The bound is the sum of these, doubled where two terms meet
in one rounding; nothing in it comes from a run.
"""

import math
import random

import pytest
import torch

from tiktoktechjam2026_b200 import _lib, ops

DEV = "cuda:0"
UNIT = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-9}


class Book:
    """A paged cache on the GPU, its pages dealt out at random, with the exact K and V kept per slot."""

    def __init__(self, seed, totals, kv_heads, hd, page, dtype, spare=3, slots=None, poison=True):
        self.g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        n_slots = slots or len(totals)
        self.slot_of = rng.sample(range(n_slots), len(totals))
        width = max([-(-t // page) for t in totals] + [1]) + 1
        need = sum(-(-t // page) for t in totals)
        pages = list(range(need + spare))
        rng.shuffle(pages)
        k = torch.randn(need + spare, kv_heads, page, hd, generator=self.g).to(dtype)
        v = torch.randn(need + spare, kv_heads, page, hd, generator=self.g).to(dtype)
        tables = torch.full((n_slots, width), -1, dtype=torch.int32)
        lens = torch.zeros(n_slots, dtype=torch.int32)
        used = torch.zeros(need + spare, page, dtype=torch.bool)
        self.k, self.v = [], []
        for slot, t in zip(self.slot_of, totals):
            mine = [pages.pop() for _ in range(-(-t // page))]
            tables[slot, : len(mine)] = torch.tensor(mine, dtype=torch.int32)
            lens[slot] = t
            for i, p in enumerate(mine):
                used[p, : min(page, t - i * page)] = True
            at = torch.tensor(mine, dtype=torch.long)
            self.k.append(k[at].permute(0, 2, 1, 3).reshape(-1, kv_heads, hd)[:t].double())
            self.v.append(v[at].permute(0, 2, 1, 3).reshape(-1, kv_heads, hd)[:t].double())
        if poison:  # what no sequence owns holds NaN
            hole = ~used[:, None, :, None].expand(-1, kv_heads, -1, hd)
            k[hole] = float("nan")
            v[hole] = float("nan")
        self.pages_k, self.pages_v = k.to(DEV), v.to(DEV)
        self.tables, self.lens = tables.to(DEV), lens.to(DEV)
        self.slots = torch.tensor(self.slot_of, dtype=torch.int32, device=DEV)


def attention_64(q, k, v, scale, window, sinks):
    """q [T, H, hd], k and v [L, KH, hd] in 64 bits -> (o, sum p |v|) [T, H, hd]."""
    T, H, hd = q.shape
    L, KH, _ = k.shape
    g = H // KH
    o = torch.zeros(T, H, hd, dtype=torch.float64)
    a = torch.zeros_like(o)
    if L == 0 or T == 0:
        return o, a
    t = torch.arange(T)[:, None] + L - T
    u = torch.arange(L)[None, :]
    see = u <= t
    if window:
        see = see & ((t - u < window) | (u < sinks))
    for h in range(H):
        s = (q[:, h] @ k[:, h // g].T) * scale
        s = s.masked_fill(~see, -math.inf)
        m = s.amax(1, keepdim=True)
        p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
        z = p.sum(1, keepdim=True)
        p = torch.where(z > 0, p / z, 0.0)
        o[:, h] = p @ v[:, h // g]
        a[:, h] = p @ v[:, h // g].abs()
    return o, a


def check_attention(book, news, heads, dtype, *, window=0, sinks=0, scale=None, q_gain=1.0, layout="packed", hd_out=None,
                    tail=0, head=0, max_q_len="exact", use_slots=True):
    KH, page, hd = book.pages_k.shape[1:]
    n = sum(news) + tail + head
    hd_out = hd_out or hd
    raw = torch.randn(n, heads, hd, generator=book.g) * q_gain
    if hd_out < hd:
        raw[..., hd_out:] = 0
    raw = raw.to(dtype)
    if layout == "packed":
        buf = torch.full((n, heads + 2 * KH, hd), float("nan"), dtype=dtype)
        buf[:, :heads] = raw
        q = buf.to(DEV)[:, :heads]
    elif layout == "heads":
        q = raw.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    else:
        q = raw.to(DEV)
    cu = [head]
    for t in news:
        cu.append(cu[-1] + t)
    cu_q = torch.tensor(cu, dtype=torch.int32, device=DEV)
    bound = {"exact": max(news + [0]) or None, "none": None, "wrong": 1}[max_q_len]
    scale_ = hd_out**-0.5 if scale is None else scale
    got = ops.paged_attention(q, book.pages_k, book.pages_v, book.tables, book.lens, cu_q,
                              slots=book.slots if use_slots else None, scale=scale, window=window, sinks=sinks,
                              head_dim=hd_out, max_q_len=bound)
    assert got.shape == (n, heads * hd_out) and got.dtype == dtype
    got = got.cpu().double().view(n, heads, hd_out)
    assert torch.all(got[:head] == 0) and torch.all(got[cu[-1]:] == 0)
    u = UNIT[dtype]
    for b, t in enumerate(news):
        if t == 0:
            continue
        o, a = attention_64(raw[cu[b]:cu[b + 1]].double(), book.k[b], book.v[b], scale_, window, sinks)
        vmax = float(book.v[b].abs().max()) if book.v[b].numel() else 0.0
        tol = 2 * u * o.abs() + 2 * u * a + 2e-4 * a + (book.k[b].shape[0] * 2.0**-25 * vmax + 2.0**-24)
        err = (got[cu[b]:cu[b + 1]] - o[..., :hd_out]).abs()
        bad = ~(err <= tol[..., :hd_out])
        assert not bad.any(), (b, t, book.k[b].shape[0], int(bad.sum()), float(err.max()))
    word = _lib.c_uint()
    assert _lib.lib().tt_device_error(_lib.ctypes.byref(word), 0) == 0


gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_attention_tokens(tt_lib, dtype, hd, page):
    """Single tokens, ragged caches: one key, page ends, tile ends, one past them."""
    totals = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 2049]
    book = Book(hd + page, totals, 2, hd, page, dtype, slots=40)
    check_attention(book, [1] * len(totals), 8, dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_attention_chunks(tt_lib, dtype, hd, group):
    """Chunks of every size class in one call, caches from none to long."""
    news = [1, 0, 2, 5, 16, 17, 33, 130, 257, 64, 1, 300]
    past = [0, 70, 64, 3, 0, 500, 128, 0, 77, 1, 900, 129]
    book = Book(hd * group, [n + p for n, p in zip(news, past)], 2, hd, 32, dtype, slots=20)
    check_attention(book, news, 2 * group, dtype, layout="heads")


@gpu
@pytest.mark.parametrize("hd,group,page", [(128, 4, 64), (64, 1, 16), (32, 1, 128), (256, 2, 32), (16, 5, 16)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (128, 64), (129, 67), (1000, 4), (5000, 9)])
def test_attention_window(tt_lib, hd, group, page, window, sinks):
    news = [1, 1, 7, 40, 300, 1, 129]
    past = [0, 3000, 100, 1500, 64, 130, 1000]
    book = Book(window + hd, [n + p for n, p in zip(news, past)], 1, hd, page, torch.float16)
    check_attention(book, news, group, torch.float16, window=window, sinks=sinks)


@gpu
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_attention_window_trimmed_pages(tt_lib, hd):
    """Pages that the window left behind are released and filled with NaN: the result is the same."""
    page, window, sinks = 16, 100, 20
    news, past = [1, 1, 60], [900, 333, 700]
    book = Book(5, [n + p for n, p in zip(news, past)], 2, hd, page, torch.bfloat16)
    refs = torch.zeros(book.pages_k.shape[0], dtype=torch.int32, device=DEV)
    refs[book.tables[book.tables >= 0].long()] = 1
    before = book.lens.clone()
    book.lens -= torch.tensor(news, dtype=torch.int32, device=DEV)[torch.argsort(book.slots)]  # as before the new tokens
    ops.cache_release(book.tables, book.lens, refs, page, window=window, sinks=sinks)
    book.lens.copy_(before)
    assert int((refs == 0).sum()) > 3 + 40
    book.pages_k[refs == 0] = float("nan")
    book.pages_v[refs == 0] = float("nan")
    check_attention(book, news, 4, torch.bfloat16, window=window, sinks=sinks)


@gpu
@pytest.mark.parametrize("max_q_len", ["exact", "none", "wrong"])
@pytest.mark.parametrize("layout", ["packed", "heads", "dense"])
def test_attention_layouts_and_bounds(tt_lib, max_q_len, layout):
    """Strides, rows of no sequence, and a bound that is missing or too small: results never depend on it."""
    news, past = [3, 0, 200, 1], [100, 5, 20, 77]
    book = Book(9, [n + p for n, p in zip(news, past)], 3, 64, 32, torch.float16, slots=9)
    check_attention(book, news, 6, torch.float16, layout=layout, max_q_len=max_q_len, head=5, tail=37)


@gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_rows_before_the_cache(tt_lib, hd):
    """More new tokens than the length: rows at negative positions see nothing and are zero."""
    totals, news = [0, 5, 1, 40], [4, 9, 300, 41]
    book = Book(3, totals, 2, hd, 16, torch.float16)
    check_attention(book, news, 4, torch.float16)
    check_attention(book, news, 4, torch.float16, window=3, sinks=1)


@gpu
@pytest.mark.parametrize("hd", [32, 128])
@pytest.mark.parametrize("gain", [0.0, 30.0])
def test_attention_flat_and_peaked(tt_lib, hd, gain):
    """All scores equal, and scores in the hundreds (one key takes the row)."""
    news, past = [1, 150], [2000, 700]
    book = Book(11, [n + p for n, p in zip(news, past)], 2, hd, 64, torch.bfloat16)
    check_attention(book, news, 4, torch.bfloat16, q_gain=gain)


@gpu
@pytest.mark.parametrize("news", [[1, 1], [40, 150]])
def test_attention_head_dim_8(tt_lib, news):
    """head_dim 8 is stored 16 wide; its spare value features may hold anything."""
    book = Book(2, [300, 200], 4, 16, 16, torch.float16)
    check_attention(book, news, 4, torch.float16, hd_out=8)


@gpu
def test_attention_one_long_sequence(tt_lib):
    """One sequence over the whole GPU, for one token and for a chunk."""
    book = Book(21, [30011], 1, 128, 64, torch.bfloat16)
    check_attention(book, [1], 4, torch.bfloat16)
    check_attention(book, [70], 4, torch.bfloat16)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [16, 64, 128, 256])
@pytest.mark.parametrize("seqs", [1, 2, 3])
@pytest.mark.parametrize("window,sinks", [(0, 0), (4000, 5)])
def test_attention_few_long_sequences(tt_lib, dtype, hd, seqs, window, sinks):
    """Short rows over long caches, few and more (sequence, KV head) pairs than a piece per SM is worth."""
    past = [11003, 4097, 0][:seqs]
    news = [1, 2, 3][:seqs]
    book = Book(hd + seqs, [n + p for n, p in zip(news, past)], 8, hd, 32, dtype)
    check_attention(book, news, 16, dtype, window=window, sinks=sinks)


@gpu
@pytest.mark.parametrize("news_of", ["tokens", "mixed"])
def test_attention_many_sequences(tt_lib, news_of):
    """More sequences than a block has threads, in tables wide enough that items may be cut; some are empty."""
    rng = random.Random(5)
    n = 1300
    news = [rng.choice([1, 1, 1, 0, 3]) if news_of == "tokens" or i % 9 else rng.randint(17, 40) for i in range(n)]
    totals = [t + rng.choice([0, 1, 30, 64, rng.randint(0, 200)]) for t in news]
    totals[7] = news[7] + 1900
    book = Book(77, totals, 1, 128, 64, torch.float16, slots=1400)
    check_attention(book, news, 2, torch.float16)


@gpu
def test_attention_no_sequence(tt_lib):
    """No sequence at all, and sequences without tokens: every row is zero."""
    book = Book(1, [20, 40], 2, 64, 16, torch.float16)
    q = torch.randn(300, 4, 64, device=DEV).half()
    for cu in ([0], [0, 0, 0], [300, 300, 300]):
        for bound in (1, None):
            got = ops.paged_attention(q, book.pages_k, book.pages_v, book.tables, book.lens, ints(cu), max_q_len=bound)
            assert torch.all(got == 0)
    assert ops.paged_attention(q[:0], book.pages_k, book.pages_v, book.tables, book.lens, ints([0, 0, 0])).shape == (0, 256)


@gpu
def test_attention_pool_past_2_31_bytes(tt_lib):
    """Pages past 2^31 values from the start of the pool, K and V interleaved in one buffer."""
    P, KH, page, hd = 36000, 2, 256, 64
    pool = torch.zeros(P, 2, KH, page, hd, dtype=torch.float16, device=DEV)
    k, v = pool[:, 0], pool[:, 1]
    book = Book(4, [500], KH, hd, page, torch.float16, poison=False)
    far = torch.tensor([P - 1, P - 3], device=DEV)
    at = book.tables[0, :2].long()
    k[far], v[far] = book.pages_k[at], book.pages_v[at]
    assert (P - 3) * k.stride(0) > 2**31
    book.tables[0, :2] = far.int()
    book.pages_k, book.pages_v = k, v
    check_attention(book, [1], 4, torch.float16)
    check_attention(book, [90], 4, torch.float16)


@gpu
def test_attention_repeats_bit_for_bit_and_on_a_stream(tt_lib):
    news, past = [1, 80, 1, 400], [5000, 900, 44, 0]
    book = Book(8, [n + p for n, p in zip(news, past)], 2, 128, 32, torch.float16)
    q = torch.randn(sum(news), 8, 128, device=DEV).half()
    cu = torch.tensor([0, 1, 81, 82, 482], dtype=torch.int32, device=DEV)
    args = (q, book.pages_k, book.pages_v, book.tables, book.lens, cu)
    first = ops.paged_attention(*args, slots=book.slots)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [ops.paged_attention(*args, slots=book.slots) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for o in others:
        assert torch.equal(first, o)


@gpu
def test_attention_in_a_graph(tt_lib):
    """Captured once, replayed with other inputs and lengths."""
    book = Book(6, [700, 90], 2, 64, 16, torch.float16)
    q = torch.randn(2, 8, 64, device=DEV).half()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    out = torch.empty(2, 512, dtype=torch.float16, device=DEV)
    call = lambda: ops.paged_attention(q, book.pages_k, book.pages_v, book.tables, book.lens, cu, slots=book.slots, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    q.normal_()
    book.lens -= 1
    graph.replay()
    torch.cuda.synchronize()
    replayed = out.clone()
    call()
    assert torch.equal(replayed, out)


# ------------------------------------------------------------------------------------ pages
class PageBook:
    """The page rules in plain Python."""

    def __init__(self, n_slots, width, n_pages, page):
        self.page, self.width = page, width
        self.tables = [[-1] * width for _ in range(n_slots)]
        self.lens = [0] * n_slots
        self.refs = [0] * n_pages

    def free(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def pages(self, n):
        return -(-n // self.page)

    def reserve(self, slots, news):
        if any(s < 0 or s >= len(self.lens) for s in slots):
            return -2
        if any(self.pages(self.lens[s] + t) > self.width for s, t in zip(slots, news)):
            return -1
        need = sum(self.pages(self.lens[s] + t) - self.pages(self.lens[s]) for s, t in zip(slots, news))
        free = self.free()
        if need > len(free):
            return need - len(free)
        for s, t in zip(slots, news):
            for i in range(self.pages(self.lens[s]), self.pages(self.lens[s] + t)):
                self.tables[s][i] = free.pop(0)
                self.refs[self.tables[s][i]] = 1
            self.lens[s] += t
        return 0

    def fork(self, parents, children):
        if any(not 0 <= s < len(self.lens) for s in parents + children):
            return -2, []
        if len(set(children)) < len(children) or any(self.lens[c] for c in children):
            return -3, []
        need = sum(self.lens[p] % self.page != 0 for p in parents)
        free = self.free()
        if need > len(free):
            return need - len(free), []
        copies, before = [], list(self.lens)  # parents as they were when the call began
        for p, c in zip(parents, children):
            full = before[p] // self.page
            for i in range(full):
                self.tables[c][i] = self.tables[p][i]
                if self.tables[p][i] >= 0:
                    self.refs[self.tables[p][i]] += 1
            if before[p] % self.page:
                new = free.pop(0)
                self.refs[new] = 1
                copies.append((self.tables[p][full], new, before[p] % self.page))
                self.tables[c][full] = new
            self.lens[c] = before[p]
        return 0, copies

    def release(self, slots, window=0, sinks=0):
        for s in slots:
            for i in range(self.width):
                gone = not window or (i * self.page >= sinks and (i + 1) * self.page <= self.lens[s] - window + 1)
                if gone and self.tables[s][i] >= 0:
                    self.refs[self.tables[s][i]] -= 1
                    self.tables[s][i] = -1
            if not window:
                self.lens[s] = 0

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        src = [p for p, r in enumerate(self.refs) if r > 0 and p >= n]
        dst = [p for p, r in enumerate(self.refs) if r == 0 and p < n]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.tables = [[to.get(p, p) for p in row] for row in self.tables]
        return n, list(to.items())


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@gpu
@pytest.mark.parametrize("seed", range(6))
def test_pages_random_programs(tt_lib, seed):
    """Random sequences of calls: tables, lengths, counts, statuses and page contents all match."""
    rng = random.Random(seed)
    page = rng.choice([16, 32, 64])
    n_slots, width, P = rng.choice([3, 24, 80]), 9, rng.choice([20, 150, 9000])
    layers, KH, hd = rng.choice([1, 3]), 2, rng.choice([16, 64])
    plain = PageBook(n_slots, width, P, page)
    tables = torch.full((n_slots, width + 3), -1, dtype=torch.int32, device=DEV)[:, :width]  # padded rows
    lens, refs = ints([0] * n_slots), ints([0] * P)
    k = torch.randn(layers, P, KH, page, hd, device=DEV).half()
    v = torch.randn(layers, P, KH, page, hd, device=DEV).half()
    k0, v0 = k.clone(), v.clone()

    def same():
        assert tables.tolist() == plain.tables
        assert lens.tolist() == plain.lens
        assert refs.tolist() == plain.refs

    for _ in range(40):
        what = rng.choice(["reserve"] * 4 + ["fork", "fork", "release", "trim", "compact"])
        some = rng.sample(range(n_slots), rng.randint(1, n_slots))
        if what == "reserve":
            news = [rng.choice([0, 1, 1, page, rng.randint(1, 3 * page)]) for _ in some]
            cu = [0]
            for t in news:
                cu.append(cu[-1] + t)
            st = ops.cache_reserve(tables, lens, refs, ints(cu), page, slots=ints(some))
            assert st.item() == plain.reserve(some, news)
        elif what == "fork":
            children = [s for s in some if plain.lens[s] == 0 or rng.random() < 0.1]
            parents = [rng.randrange(n_slots) for _ in children]
            if any(p in children and plain.lens[p] for p in parents):
                continue
            st = ops.cache_fork(k, v, tables, lens, refs, ints(parents), ints(children))
            want, copies = plain.fork(parents, children)
            assert st.item() == want
            for a, b, rows in copies:
                k0[:, b, :, :rows], v0[:, b, :, :rows] = k0[:, a, :, :rows], v0[:, a, :, :rows]
        elif what == "release":
            few = some[: max(1, len(some) // 3)]
            ops.cache_release(tables, lens, refs, page, slots=ints(few + few[:1]))
            plain.release(few)
        elif what == "trim":
            window, sinks = rng.randint(1, 4 * page), rng.choice([0, 3, page, page + 1])
            ops.cache_release(tables, lens, refs, page, slots=ints(some), window=window, sinks=sinks)
            plain.release(some, window, sinks)
            for s in some:  # a trimmed sequence's partial page stays: it can still be forked and grow
                assert plain.lens[s] % page == 0 or plain.tables[s][plain.lens[s] // page] >= 0
        else:
            live = ops.cache_compact(k, v, tables, lens, refs)
            n, moves = plain.compact()
            assert live.item() == n
            for a, b in moves:
                k0[:, b], v0[:, b] = k0[:, a], v0[:, a]
        same()
        assert torch.equal(k, k0) and torch.equal(v, v0)


@gpu
def test_reserve_statuses_change_nothing(tt_lib):
    page = 16
    tables = torch.full((4, 5), -1, dtype=torch.int32, device=DEV)
    lens, refs = ints([0, 16, 40, 0]), ints([1] * 4 + [0, 1, 0] + [0] * 2)
    state = [t.clone() for t in (tables, lens, refs)]

    def status(cu, slots=None):
        st = ops.cache_reserve(tables, lens, refs, ints(cu), page, slots=None if slots is None else ints(slots)).item()
        assert all(torch.equal(a, b) for a, b in zip(state, (tables, lens, refs)))
        return st

    assert status([0, 64, 65, 65, 75]) == 2      # 4 + 1 + 0 + 1 pages, 4 free
    assert status([0, 81]) == -1                 # 6 pages in a row of 5
    assert status([0, 1, 2], [1, 4]) == -2
    assert status([0, 1, 2], [-1, 2]) == -2
    assert status([0, 5, 3]) == -2
    assert status([0]) == 0                      # no sequence
    assert status([0, 0, 0, 0, 0]) == 0          # no tokens


@gpu
def test_fork_statuses_change_nothing(tt_lib):
    page = 16
    tables = torch.full((5, 4), -1, dtype=torch.int32, device=DEV)
    tables[0, :2], tables[1, :1] = ints([3, 1]), ints([0])
    lens, refs = ints([20, 16, 0, 0, 0]), ints([1, 1, 0, 1])
    k = torch.randn(4, 1, page, 16, device=DEV).half()
    v = torch.randn(4, 1, page, 16, device=DEV).half()
    state = [t.clone() for t in (tables, lens, refs, k, v)]

    def status(parents, children):
        st = ops.cache_fork(k, v, tables, lens, refs, ints(parents), ints(children)).item()
        assert all(torch.equal(a, b) for a, b in zip(state, (tables, lens, refs, k, v)))
        return st

    assert status([0, 0], [2, 3]) == 1
    assert status([0], [1]) == -3
    assert status([1, 1], [2, 2]) == -3
    assert status([0], [5]) == -2
    assert status([-1], [2]) == -2
    assert status([], []) == 0
    assert status([2], [3]) == 0                 # an empty parent


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["projection", "packed", "dense"])
@pytest.mark.parametrize("hd,KH,page", [(16, 3, 16), (32, 8, 64), (64, 1, 128), (128, 2, 16), (256, 2, 256)])
def test_append(tt_lib, dtype, layout, hd, KH, page):
    """Every value lands in its place and nothing else is touched."""
    news, past = [1, 0, 3, 130, 1, 64, 17], [0, 9, 15, 31, 700, 16, 256]
    totals = [n + p for n, p in zip(news, past)]
    book = Book(hd, totals, KH, hd, page, dtype, slots=11, poison=False)
    n = sum(news) + 6  # rows of no sequence before and after
    k, v = torch.randn(n, KH, hd).to(dtype), torch.randn(n, KH, hd).to(dtype)
    if layout == "projection":
        dk = k.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
        vt = torch.zeros(KH, hd, (n + 7) // 8 * 8, dtype=dtype)
        vt[..., :n] = v.permute(1, 2, 0)
        dv = vt.to(DEV)[..., :n].permute(2, 0, 1)
    elif layout == "packed":
        row = torch.stack([k, v], 1).to(DEV)
        dk, dv = row[:, 0], row[:, 1]
    else:
        dk, dv = k.to(DEV), v.to(DEV)
    cu = [2]
    for t in news:
        cu.append(cu[-1] + t)
    want_k, want_v = book.pages_k.clone(), book.pages_v.clone()
    for b, t in enumerate(news):
        for j in range(t):
            pos = past[b] + j
            p = int(book.tables[book.slot_of[b], pos // page])
            want_k[p, :, pos % page], want_v[p, :, pos % page] = k[cu[b] + j].to(DEV), v[cu[b] + j].to(DEV)
    ops.cache_append(dk, dv, book.pages_k, book.pages_v, book.tables, book.lens, ints(cu), slots=book.slots)
    assert torch.equal(book.pages_k, want_k) and torch.equal(book.pages_v, want_v)


@gpu
def test_append_skips_missing_pages(tt_lib):
    """A token whose page does not exist, or whose slot is outside the table, is dropped."""
    tables = ints([[1, -1], [7, 0]])
    lens = ints([33, 16])
    k = torch.zeros(3, 1, 32, 16, dtype=torch.float16, device=DEV)
    v = torch.zeros_like(k)
    new = torch.ones(4, 1, 16, dtype=torch.float16, device=DEV)
    ops.cache_append(new, new, k, v, tables, lens, ints([0, 2, 3, 4]), slots=ints([0, 1, 9]))
    assert k.sum() == 16 and torch.all(k[1, 0, 31] == 1) and torch.equal(k, v)


@gpu
def test_copy_pages(tt_lib):
    tables, lens = ints([[0, 1]]), ints([0])
    k = torch.randn(2, 9, 3, 16, 32, device=DEV).half()
    v = torch.randn(2, 9, 3, 16, 32, device=DEV).half()
    k0, v0 = k.clone(), v.clone()
    ops.cache_copy_pages(k, v, tables, lens, ints([0, 5, 20, -1]), ints([3, 8, 1, 2]))
    for a, b in ((0, 3), (5, 8)):
        k0[:, b], v0[:, b] = k0[:, a], v0[:, a]
    assert torch.equal(k, k0) and torch.equal(v, v0)


# ----------------------------------------------------------------------------------- refusals
@gpu
def test_refusals(tt_lib):
    book = Book(1, [20, 40], 2, 32, 16, torch.float16)
    q = torch.randn(2, 4, 32, device=DEV).half()
    cu = ints([0, 1, 2])
    k, v, t, n = book.pages_k, book.pages_v, book.tables, book.lens
    refs = ints([0] * k.shape[0])

    def bad(f, *a, exc=ValueError, **kw):
        with pytest.raises(exc):
            f(*a, **kw)

    A = ops.paged_attention
    bad(A, q.float(), k, v, t, n, cu)
    bad(A, q.bfloat16(), k, v, t, n, cu)
    bad(A, q.cpu(), k, v, t, n, cu)
    bad(A, q[..., :16], k, v, t, n, cu)
    bad(A, q[:, :3], k, v, t, n, cu)                                 # 3 heads over 2 KV heads
    bad(A, q, k, v, t.long(), n, cu)
    bad(A, q, k, v, t, n[:1], cu)
    bad(A, q, k, v, t, n, cu, slots=ints([0]))
    bad(A, q, k, v, t, n, ints([0, 1, 2, 2]))                        # more sequences than rows of the table
    bad(A, q, k, v, t, n, cu, window=-1)
    bad(A, q, k, v, t, n, cu, sinks=-1)
    bad(A, q, k, v[:1], t, n, cu)
    bad(A, q, k.transpose(1, 2), v.transpose(1, 2), t, n, cu)        # pages are not contiguous
    bad(A, q, k, v, t, n, cu, out=torch.empty(2, 64, device=DEV).half())
    bad(A, q, k, v, t, n, cu, head_dim=8, exc=_lib.TTError)          # 8 is stored 16 wide, not 32
    odd = torch.randn(2 * 4 * 32 + 8, device=DEV).half()[1:257].view(2, 4, 32)
    bad(A, odd, k, v, t, n, cu, exc=_lib.TTError)                    # misaligned
    wide = torch.randn(2, 4, 36, device=DEV).half()[..., :32]
    bad(A, wide, k, v, t, n, cu, exc=_lib.TTError)                   # rows are not whole 16 bytes apart
    k12 = torch.zeros(4, 2, 24, 32, device=DEV).half()
    bad(A, q, k12, k12, t, n, cu, exc=_lib.TTError)                  # page of 24
    k48 = torch.zeros(4, 2, 16, 48, device=DEV).half()
    bad(A, torch.zeros(2, 4, 48, device=DEV).half(), k48, k48, t, n, cu, exc=_lib.TTError)
    many = torch.zeros(2, 258, 32, device=DEV).half()
    bad(A, many, k, v, t, n, cu, exc=_lib.TTError)                   # 129 query heads to a KV head
    new = torch.zeros(2, 2, 32, device=DEV).half()
    bad(ops.cache_append, new[:, :1], new, k, v, t, n, cu)
    bad(ops.cache_append, new.float(), new, k, v, t, n, cu)
    bad(ops.cache_append, new, new, k[None], v[None], t, n, cu)
    bad(ops.cache_append, torch.zeros(2, 2, 64, device=DEV).half()[..., ::2], new, k, v, t, n, cu, exc=_lib.TTError)
    bad(ops.cache_reserve, t, n, refs, cu, 24, exc=_lib.TTError)
    bad(ops.cache_release, t, n, refs, 16, window=-1, exc=_lib.TTError)
    bad(ops.cache_fork, k, v, t, n, refs, ints([0]), ints([0, 1]))
    bad(ops.cache_compact, k, v, t, n, refs[:-1])
    bad(ops.cache_copy_pages, k, v, t, n, ints([0]), ints([0, 1]))
    word = _lib.c_uint()
    assert _lib.lib().tt_device_error(_lib.ctypes.byref(word), 0) == 0


@gpu
def test_workspace_too_small_is_refused(tt_lib):
    """Calls that may cut an item need their workspace; one that cannot takes none."""
    for total, rc_want in ((6000, _lib.TT_ERR_WORKSPACE), (20, _lib.TT_OK)):
        book = Book(1, [total], 2, 32, 16, torch.float16)
        q = torch.randn(1, 2, 32, device=DEV).half()
        out = torch.zeros(1, 64, dtype=torch.float16, device=DEV)
        c = ops._cache(book.pages_k, book.pages_v, book.tables, book.lens, None)
        ws = torch.empty(64, dtype=torch.uint8, device=DEV)
        for ptr, size in ((ws.data_ptr(), 64), (None, 1 << 40)):
            rc = tt_lib.tt_paged_attention(c, q.data_ptr(), 64, 32, ints([0, 1]).data_ptr(), None, 1, out.data_ptr(), 1, 2,
                                           32, 0, 1.0, 0, 0, 1, ptr, size, torch.cuda.current_stream().cuda_stream)
            assert rc == rc_want and bool(torch.all(out == 0)) == (rc_want != _lib.TT_OK)


def test_cpu_tensors_are_refused():
    t = torch.zeros(2, 3, dtype=torch.int32)
    n = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.cache_reserve(t, n, n, n, 16)
