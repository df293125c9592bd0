"""The paged-cache operators as measured cases: their plain forms and the framework's calls.

Four kinds of case, each one pass over one operator:

* ``attend``  -- attention of a chunk of new tokens over a paged K/V cache, grouped KV heads,
                 optionally with a sliding window and a few first tokens that stay visible;
* ``append``  -- allocate the pages that new tokens need and write one layer's K and V into them;
* ``fork``    -- children that share their parent's full pages and get a copy of its partial one;
* ``compact`` -- trim what a window left behind, free finished sequences, then move the live
                 pages to the front of the pool.

A cache holds K and V pages [pages, kv_heads, page, head_dim] per layer, a page table [slots, width]
(-1 where there is no page), lengths [slots] and reference counts [pages].  Sequence b of a call has
the rows cu_q[b] .. cu_q[b + 1] of its new tokens, whose positions end at lens[slot] - 1.
"""

import math

import torch

own = False

if torch.cuda.is_available():
    DEVICE = torch.device("cuda", torch.cuda.current_device())
else:
    DEVICE = torch.device("cpu")

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------- cases
def _attend(name, dtype, batch, heads, kv_heads, head_dim, page, q, past, window=0, sinks=0, layout="packed"):
    return {"name": name, "op": "attend", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "q_lo": q[0], "q_hi": q[1], "past_lo": past[0], "past_hi": past[1],
            "window": window, "sinks": sinks, "layout": layout}


def _append(name, dtype, batch, kv_heads, head_dim, page, q, past, spare, layout):
    return {"name": name, "op": "append", "dtype": dtype, "batch": batch, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "q_lo": q[0], "q_hi": q[1], "past_lo": past[0], "past_hi": past[1],
            "spare": spare, "layout": layout}


def _fork(name, dtype, layers, parents, copies, kv_heads, head_dim, page, past):
    return {"name": name, "op": "fork", "dtype": dtype, "layers": layers, "parents": parents, "copies": copies,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "past_lo": past[0], "past_hi": past[1]}


def _compact(name, dtype, layers, batch, kv_heads, head_dim, page, past, window, sinks):
    return {"name": name, "op": "compact", "dtype": dtype, "layers": layers, "batch": batch, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "past_lo": past[0], "past_hi": past[1], "window": window,
            "sinks": sinks}


def listed():
    return [
        # One user, one token after a prompt of the benchmark's 1024 tokens, its 8 heads of 32: pure latency.
        _attend("token-one", "fp16", 1, 8, 8, 32, 16, (1, 1), (1000, 1000), layout="projection"),
        # A served batch of the 512-wide model (8 heads of 64), everybody at another place of up to 2048 tokens.
        _attend("token-batch", "fp16", 64, 8, 8, 64, 32, (1, 1), (1, 2047), layout="projection"),
        # Long documents, four query heads to a KV head: the cache is all the traffic.
        _attend("token-long", "bf16", 12, 32, 8, 128, 64, (1, 1), (20011, 65000)),
        # A serving step that mixes prompt chunks with single tokens over caches of up to 8K.
        _attend("chunk-mixed", "fp16", 8, 32, 8, 128, 64, (1, 777), (0, 7400)),
        # One long prompt read in chunks: 2048 new tokens over 30K old ones.
        _attend("chunk-long", "bf16", 1, 16, 4, 128, 128, (2048, 2048), (30001, 30001)),
        # Whole prompts into an empty cache, the benchmark's model (8 heads of 32, 1024 tokens).
        _attend("prompt-batch", "fp16", 32, 8, 8, 32, 64, (900, 1024), (0, 0), layout="projection"),
        # Single tokens far into long streams, held to a window of 1024 and 4 first tokens.
        _attend("window-token", "bf16", 64, 32, 8, 128, 16, (1, 1), (3000, 30000), window=1024, sinks=4),
        # A long prompt under the same window.
        _attend("window-prompt", "fp16", 1, 8, 8, 64, 64, (8111, 8111), (0, 0), window=1024, sinks=4,
                layout="projection"),
        # The cache's side of a decode step, in the form in which the QKV projection leaves K and V.
        _append("append-token", "fp16", 256, 8, 32, 16, (1, 1), (1, 1023), 4096, "projection"),
        # Prompts of any length written at once.
        _append("append-prompt", "bf16", 24, 8, 128, 64, (17, 4096), (0, 300), 1024, "packed"),
        # Several answers to each of a few prompts.
        _fork("fork-answers", "fp16", 4, 16, 7, 8, 64, 64, (33, 2048)),
        # Half the sequences done and a window behind the others: the pool is drawn together.
        _compact("compact-pool", "fp16", 4, 64, 8, 64, 64, (500, 7000), 2048, 4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges as the listed ones, no dearer than the largest of its kind."""
    most = {}
    for c in listed():
        w = work(c)
        a, b = most.get(c["op"], (0, 0))
        most[c["op"]] = (max(a, w["bytes"]), max(b, w["flops"]))
    while True:
        kind = rng.choice(["attend", "attend", "attend", "window", "window", "append", "fork", "compact"])
        dtype = rng.choice(["fp16", "bf16"])
        head_dim = rng.choice([16, 32, 64, 64, 128, 128, 256])
        page = rng.choice([16, 32, 64, 128])
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        layout = rng.choice(["packed", "projection"])
        if kind in ("attend", "window"):
            window, sinks = (0, 0) if kind == "attend" else (_log(rng, 16, 4096), rng.choice([0, 1, 4, 4, 67]))
            q_hi = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 65, 4096)])
            q_lo = rng.choice([1, q_hi, max(1, q_hi // 2)])
            past_hi = _log(rng, 1, 65000)
            past_lo = rng.choice([0, past_hi // 2, past_hi])
            heads = kv_heads * rng.choice([1, 1, 2, 4, 5, 8])
            c = _attend("", dtype, _log(rng, 1, 256), heads, kv_heads, head_dim, page, (q_lo, q_hi),
                        (past_lo, past_hi), window, sinks, layout)
            # The plain form holds a score for every (head, padded query, padded key) in 32 bits.
            if c["batch"] * heads * q_hi * (q_hi + past_hi + page) > 1.2e9:
                continue
            if c["batch"] * kv_heads * head_dim * (q_hi + past_hi + page) > 1.2e9:
                continue
        elif kind == "append":
            q_hi = rng.choice([1, _log(rng, 2, 4096)])
            past_hi = _log(rng, 1, 2048)
            c = _append("", dtype, _log(rng, 1, 512), kv_heads, head_dim, page, (rng.choice([1, q_hi]), q_hi),
                        (0, past_hi), _log(rng, 16, 4096), layout)
        elif kind == "fork":
            past_hi = _log(rng, 2, 4096)
            c = _fork("", dtype, rng.choice([1, 2, 4, 6]), _log(rng, 1, 32), _log(rng, 1, 16), kv_heads, head_dim, page,
                      (rng.choice([1, past_hi]), past_hi))
        else:
            past_hi = _log(rng, 64, 8192)
            c = _compact("", dtype, rng.choice([1, 2, 4, 6]), _log(rng, 2, 128), kv_heads, head_dim, page,
                         (past_hi // 8, past_hi), _log(rng, 64, 4096), rng.choice([0, 4]))
        pages = sum(-(-(t + p) // page) for t, p in _lengths(c)) + c.get("spare", 0)
        if pages * c["kv_heads"] * page * head_dim * c.get("layers", 1) > 0.8e9:
            continue
        w = work(c)
        if w["bytes"] > most[c["op"]][0] or w["flops"] > most[c["op"]][1]:
            continue
        del c["name"]
        return c


def _spread(lo, hi, n, step):
    """n whole numbers over lo .. hi, the ends among them when n > 1, the same for every seed."""
    if n == 1:
        return [hi]
    got = [lo + int((hi - lo + 1) * ((i * step) % 1.0)) for i in range(n)]
    got[0], got[-1] = hi, lo
    return got


def _lengths(c):
    """(new tokens, tokens before them) of each sequence, before the seed shuffles the sequences."""
    n = c["batch"] if "batch" in c else c["parents"]
    return list(zip(_spread(c.get("q_lo", 0), c.get("q_hi", 0), n, 0.6180339887),
                    _spread(c["past_lo"], c["past_hi"], n, 0.7548776662)))


def _sum_min(first, last, cap):
    """sum of min(i, cap) over i = first .. last."""
    mid = min(last, cap)
    ramp = (first + mid) * (mid - first + 1) // 2 if mid >= first else 0
    return ramp + cap * max(0, last - max(first - 1, cap))


def _visible(t, past, window, sinks):
    """(visible (query, key) pairs, keys that some query sees) of t new tokens after `past` old ones."""
    total = past + t
    if window == 0 or window >= total:
        return _sum_min(past + 1, total, total), total
    # Query at position p sees the last min(p + 1, window) keys, and of the first `sinks` those before them.
    near = _sum_min(past + 1, total, window)
    lead = sum(min(sinks, max(0, p + 1 - window)) for p in range(past, total)) if sinks else 0
    first = max(0, past - window + 1)
    return near + lead, total - first + min(first, sinks)


def work(case):
    size = 2
    row = case["kv_heads"] * case["head_dim"] * size
    page = case["page"]
    pairs = _lengths(case)
    if case["op"] == "attend":
        seen = [_visible(t, p, case["window"], case["sinks"]) for t, p in pairs]
        keys = sum(k for _, k in seen)
        q = sum(t for t, _ in pairs) * case["heads"] * case["head_dim"] * size
        return {"bytes": 2 * q + 2 * keys * row + 4 * (keys // page) + 8 * len(pairs),
                "flops": 4 * case["head_dim"] * case["heads"] * sum(n for n, _ in seen)}
    if case["op"] == "append":
        new = sum(t for t, _ in pairs)
        pages = sum(-(-(t + p) // page) - -(-p // page) for t, p in pairs)
        total = sum(-(-(t + p) // page) for t, p in pairs) + case["spare"]
        return {"bytes": 4 * new * row + 12 * pages + 4 * total + 12 * len(pairs), "flops": 0}
    if case["op"] == "fork":
        rows = sum(p % page for _, p in pairs) * case["copies"]
        full = sum(p // page for _, p in pairs) * case["copies"]
        return {"bytes": 4 * rows * row * case["layers"] + 12 * full + 16 * len(pairs) * case["copies"], "flops": 0}
    total = sum(-(-p // page) for _, p in pairs)
    live = sum(_kept(p, page, case["window"], case["sinks"]) for _, p in pairs[::2])
    # The seed deals the pages out: of `live` pages about live * (total - live) / total lie behind the front.
    moved = live * (total - live) // total
    return {"bytes": 4 * moved * row * page * case["layers"] + 16 * total, "flops": 0}


def _kept(length, page, window, sinks):
    """Pages that a sequence of `length` tokens still needs under the window."""
    pages = -(-length // page)
    first, last = -(-sinks // page), max(0, length - window + 1) // page
    return pages - max(0, last - first)


# -------------------------------------------------------------------------------------- inputs
def _rand(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32 if DEVICE.type == "cpu" else dtype).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _state(slots, width, lens, pages, held, order):
    """lens, refs and tables as one int32 buffer: sequence i (slot i) holds `held[i]` pages dealt from `order`."""
    table = torch.full((slots, width), -1, dtype=torch.int32)
    flat = torch.arange(width)[None, :] < torch.tensor(held + [0] * (slots - len(held)))[:, None]
    used = int(sum(held))
    table[flat] = order[:used].to(torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[order[:used]] = 1
    lens = torch.tensor(lens + [0] * (slots - len(lens)), dtype=torch.int32)
    return torch.cat([lens, refs, table.reshape(-1)]).to(DEVICE)


def _parts(state, ints):
    """lens, refs, tables as views of the int32 buffer."""
    s, p, w = state["slots"], state["pages"], state["width"]
    return ints[:s], ints[s:s + p], ints[s + p:].view(s, w)


def prepare(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, page = TYPES[case["dtype"]], case["page"]
    kh, hd, op = case["kv_heads"], case["head_dim"], case["op"]
    pairs = _lengths(case)
    pairs = [pairs[i] for i in torch.randperm(len(pairs), generator=cpu).tolist()]
    if op in ("fork", "compact"):  # released sequences are every second one: keep the order
        pairs = _lengths(case)
    past = [p for _, p in pairs]
    total = [t + p for t, p in pairs]
    st = {"case": case}
    held = [-(-n // page) for n in (total if op == "attend" else past)]
    if op == "attend":
        pages, slots, width = sum(held) + 3, len(pairs), max(held) + 1
        lens = total
    elif op == "append":
        pages, slots = sum(-(-n // page) for n in total) + case["spare"], len(pairs)
        width, lens = max(-(-n // page) for n in total) + 1, past
    elif op == "fork":
        slots = case["parents"] * (1 + case["copies"])
        pages, width, lens = sum(held) + slots, max(held) + 1, past
    else:
        pages, slots, width, lens = sum(held), len(pairs), max(held), past
    order = torch.randperm(pages, generator=cpu)
    st.update(slots=slots, pages=pages, width=width, ints=_state(slots, width, lens, pages, held, order))
    layers = case.get("layers", 1)
    shape = (layers, pages, kh, page, hd) if op in ("fork", "compact") else (pages, kh, page, hd)
    st["k"], st["v"] = _rand(g, dtype, *shape), _rand(g, dtype, *shape)
    if op in ("attend", "append"):
        starts = [0]
        starts += torch.tensor([t for t, _ in pairs]).cumsum(0).tolist()
        n = starts[-1]
        st["cu_q"], st["max_q"], st["tokens"] = _ints(starts), max(t for t, _ in pairs), n
    if op == "attend":
        h = case["heads"]
        if case["layout"] == "projection":  # the QKV projection leaves q head-major
            st["q"] = _rand(g, dtype, h, n, hd).transpose(0, 1)
        else:  # q is the first part of a packed q, k, v row
            st["q"] = _rand(g, dtype, n, h + 2 * kh, hd)[:, :h]
    elif op == "append":
        if case["layout"] == "projection":  # k head-major, v transposed with its rows padded to 8 tokens
            st["new_k"] = _rand(g, dtype, kh, n, hd).transpose(0, 1)
            st["new_v"] = _rand(g, dtype, kh, hd, (n + 7) // 8 * 8)[..., :n].permute(2, 0, 1)
        else:
            row = _rand(g, dtype, n, 3, kh, hd)
            st["new_k"], st["new_v"] = row[:, 1], row[:, 2]
    elif op == "fork":
        f = case["parents"] * case["copies"]
        st["parents"] = _ints([i % case["parents"] for i in range(f)])
        st["children"] = _ints([case["parents"] + i for i in range(f)])
    else:
        st["kept"] = _ints(list(range(0, slots, 2)))
        st["done"] = _ints(list(range(1, slots, 2)))
    return st


# ------------------------------------------------------------------------------------- one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    from tiktoktechjam2026_b200 import ops

    case = st["case"]
    if case["op"] == "attend":
        lens, _, tables = _parts(st, st["ints"])
        return ops.paged_attention(st["q"], st["k"], st["v"], tables, lens, st["cu_q"], window=case["window"],
                                   sinks=case["sinks"], max_q_len=st["max_q"])
    lens, refs, tables = _parts(st, st["ints"].clone())  # the pass starts from the same cache every time
    if case["op"] == "append":
        status = ops.cache_reserve(tables, lens, refs, st["cu_q"], case["page"])
        ops.cache_append(st["new_k"], st["new_v"], st["k"], st["v"], tables, lens, st["cu_q"])
        return [status, lens, refs, tables, st["k"], st["v"]]
    if case["op"] == "fork":
        status = ops.cache_fork(st["k"], st["v"], tables, lens, refs, st["parents"], st["children"])
        return [status, lens, refs, tables, st["k"], st["v"]]
    ops.cache_release(tables, lens, refs, case["page"], slots=st["kept"], window=case["window"], sinks=case["sinks"])
    ops.cache_release(tables, lens, refs, case["page"], slots=st["done"])
    live = ops.cache_compact(st["k"], st["v"], tables, lens, refs)
    return [live, lens, refs, tables, st["k"], st["v"]]


def _run_plain(st):
    case = st["case"]
    if case["op"] == "attend":
        return _plain_attend(st)
    lens, refs, tables = _parts(st, st["ints"].clone())
    page = case["page"]
    if case["op"] == "append":
        return _plain_append(st, lens, refs, tables, page)
    if case["op"] == "fork":
        return _plain_fork(st, lens, refs, tables, page)
    return _plain_compact(st, lens, refs, tables, page)


def _token_place(cu_q, n):
    """Sequence and index within its new tokens of each of n rows."""
    rows = torch.arange(n, device=DEVICE)
    b = (rows[:, None] >= cu_q[None, 1:]).sum(1)
    return b, rows - cu_q.long()[b]


def _plain_attend(st):
    case = st["case"]
    lens, _, tables = _parts(st, st["ints"])
    h, kh, hd, page, window, sinks = (case[x] for x in ("heads", "kv_heads", "head_dim", "page", "window", "sinks"))
    cu, t_max, n = st["cu_q"].long(), st["max_q"], st["tokens"]
    b, w = tables.shape
    at = tables.long().clamp(min=0)
    k = st["k"][at].float().permute(0, 2, 1, 3, 4).reshape(b, kh, w * page, hd)
    v = st["v"][at].float().permute(0, 2, 1, 3, 4).reshape(b, kh, w * page, hd)
    rows = (cu[:-1, None] + torch.arange(t_max, device=DEVICE)).clamp(max=n - 1)
    q = st["q"].float()[rows].permute(0, 2, 1, 3).reshape(b, kh, h // kh * t_max, hd)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(hd ** -0.5).view(b, kh, h // kh, t_max, w * page)
    count = cu[1:] - cu[:-1]
    pos = (lens.long() - count)[:, None] + torch.arange(t_max, device=DEVICE)
    key = torch.arange(w * page, device=DEVICE)
    ok = key <= pos[..., None]
    if window:
        ok = ok & ((key > pos[..., None] - window) | (key < sinks))
    s.masked_fill_(~ok[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    z = s.sum(-1)
    o = torch.matmul(s.view(b, kh, h // kh * t_max, w * page), v).view(b, kh, h // kh, t_max, hd)
    o = torch.where(z[..., None] > 0, o / z[..., None], 0.0)
    seq, j = _token_place(st["cu_q"], n)
    return o.reshape(b, h, t_max, hd)[seq, :, j].reshape(n, h * hd).to(st["q"].dtype)


def _plain_append(st, lens, refs, tables, page):
    cu = st["cu_q"]
    count = cu[1:] - cu[:-1]
    old = (lens + page - 1) // page
    new = (lens + count + page - 1) // page
    upto = torch.cumsum(new - old, 0)
    first, need = upto - (new - old), upto[-1]
    free = torch.argsort((refs != 0).to(torch.int32), stable=True)  # free pages first, lowest first
    rank = torch.cumsum((refs == 0).to(torch.int32), 0) - 1
    short = (need - (refs == 0).sum()).clamp(min=0)
    col = torch.arange(tables.shape[1], device=DEVICE)
    fresh = (col >= old[:, None]) & (col < new[:, None]) & (short == 0)
    pick = (first[:, None] + col - old[:, None]).clamp(0, refs.numel() - 1)
    tables.copy_(torch.where(fresh, free[pick].to(torch.int32), tables))
    refs.copy_(torch.where((refs == 0) & (rank < need) & (short == 0), 1, refs))
    lens.add_(torch.where(short == 0, count, 0))
    b, j = _token_place(cu, st["tokens"])
    pos = (lens - count).long()[b] + j
    at = tables[b, pos // page].long()
    st["k"][at, :, pos % page] = st["new_k"]
    st["v"][at, :, pos % page] = st["new_v"]
    return [short.to(torch.int32).view(1), lens, refs, tables, st["k"], st["v"]]


def _plain_fork(st, lens, refs, tables, page):
    parent, child = st["parents"].long(), st["children"].long()
    size = lens[parent]
    full, part = size // page, size % page
    need = part > 0
    upto = torch.cumsum(need.to(torch.int32), 0)
    short = (upto[-1] - (refs == 0).sum()).clamp(min=0)
    free = torch.argsort((refs != 0).to(torch.int32), stable=True)
    fresh = free[(upto - 1).clamp(0, refs.numel() - 1)].to(torch.int32)
    col = torch.arange(tables.shape[1], device=DEVICE)
    row = torch.where(col < full[:, None], tables[parent], tables[child])
    row = torch.where((col == full[:, None]) & need[:, None], fresh[:, None], row)
    share = (col < full[:, None]) & (tables[parent] >= 0)
    pick = need.nonzero()[:, 0]
    src, dst = tables[parent[pick], full[pick].long()].long(), fresh[pick].long()
    keep = torch.arange(page, device=DEVICE)[:, None] < part[pick][:, None, None, None]
    st["k"][:, dst] = torch.where(keep, st["k"][:, src], st["k"][:, dst])
    st["v"][:, dst] = torch.where(keep, st["v"][:, src], st["v"][:, dst])
    refs.index_add_(0, tables[parent].clamp(min=0).long().reshape(-1), share.reshape(-1).to(torch.int32))
    refs[dst] = 1
    tables[child] = row
    lens[child] = size
    return [short.to(torch.int32).view(1), lens, refs, tables, st["k"], st["v"]]


def _plain_compact(st, lens, refs, tables, page):
    case = st["case"]
    window, sinks = case["window"], case["sinks"]
    col = torch.arange(tables.shape[1], device=DEVICE)
    kept, done = st["kept"].long(), st["done"].long()
    behind = (col * page >= sinks) & ((col + 1) * page <= lens[kept][:, None] - window + 1)
    gone = torch.zeros_like(tables, dtype=torch.bool)
    gone[kept] = behind
    gone[done] = True
    gone &= tables >= 0
    refs.index_add_(0, tables.clamp(min=0).long().reshape(-1), -gone.reshape(-1).to(torch.int32))
    tables.masked_fill_(gone, -1)
    lens[done] = 0
    live, index = refs > 0, torch.arange(refs.numel(), device=DEVICE)
    n = live.sum()
    src = (live & (index >= n)).nonzero()[:, 0]
    dst = (~live & (index < n)).nonzero()[:, 0]
    st["k"][:, dst] = st["k"][:, src]
    st["v"][:, dst] = st["v"][:, src]
    to = index.to(torch.int32)
    to[src] = dst.to(torch.int32)
    refs[dst] = refs[src]
    refs[src] = 0
    tables.copy_(torch.where(tables >= 0, to[tables.clamp(min=0).long()], -1))
    return [n.to(torch.int32).view(1), lens, refs, tables, st["k"], st["v"]]


# ------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["op"] != "attend":
        return None  # page numbers, counts and copied values: nothing is computed
    st = prepare(case, seed)
    h, kh, hd, page, window, sinks = (case[x] for x in ("heads", "kv_heads", "head_dim", "page", "window", "sinks"))
    lens, _, tables = _parts(st, st["ints"])
    out = torch.zeros(st["tokens"], h, hd, dtype=torch.float64, device=DEVICE)
    cu, lens = st["cu_q"].tolist(), lens.tolist()
    for b in range(len(cu) - 1):
        n = lens[b]
        own_pages = tables[b, :-(-n // page)].long()
        for g in range(kh):
            k = st["k"][own_pages, g].reshape(-1, hd)[:n].double()
            v = st["v"][own_pages, g].reshape(-1, hd)[:n].double()
            heads = slice(g * (h // kh), (g + 1) * (h // kh))
            for lo in range(cu[b], cu[b + 1], 512):
                hi = min(lo + 512, cu[b + 1])
                q = st["q"][lo:hi, heads].double()
                s = torch.einsum("thd,ud->thu", q, k) / math.sqrt(hd)
                t = torch.arange(lo, hi, device=DEVICE)[:, None] - cu[b + 1] + n
                u = torch.arange(n, device=DEVICE)[None]
                hidden = u > t
                if window:
                    hidden = hidden | ((t - u >= window) & (u >= sinks))
                p = torch.softmax(s.masked_fill(hidden[:, None], -math.inf), -1)
                out[lo:hi, heads] = torch.einsum("thu,ud->thd", p, v)
    return out.reshape(st["tokens"], h * hd)
