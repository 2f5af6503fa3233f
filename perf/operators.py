"""The paged key/value cache and what fills and reads it, as a serving program runs it, for timing and for comparing results.

Before a step the program turns its requests' lengths into page tables and slots (`M.PageTables`); in each layer it rotates the
new tokens' queries and keys by their positions and puts keys and values into their slots (`M.Rotary`), and the new tokens attend
to their requests' pages (`M.PagedAttention`).  The listed cases go from the smallest decoding step to prompts of thousands of
tokens; `draw` gives further sizes, types, layouts and lengths of the same kinds of work.
"""
import math
import random

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}


def _tables(requests, chunks, new_lo, new_hi, cached_lo, cached_hi, page_size, spare=1.25):
    """spare: pages on the free list over those that the new tokens want (below 1: some requests go without)."""
    return {"op": "tables", "requests": requests, "chunks": chunks, "new_lo": new_lo, "new_hi": new_hi,
            "cached_lo": cached_lo, "cached_hi": cached_hi, "page_size": page_size, "spare": spare}


def _rotary(dtype, tokens, q_heads, kv_heads, head_dim, sections, adjacent=False, page_size=0, far=4096):
    """sections: pairs of each axis, as a text; page_size 0: the gradient's inverse rotation, without a cache."""
    return {"op": "rotary", "dtype": dtype, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "sections": sections, "adjacent": adjacent, "page_size": page_size, "far": far}


def _attention(dtype, requests, chunks, new_lo, new_hi, cached_lo, cached_hi, q_heads, kv_heads, head_dim, page_size, window=0, heads_first=False):
    """chunks: requests with new_lo to new_hi new tokens, the others have one; heads_first: pages hold a block of slots per head."""
    return {"op": "attention", "dtype": dtype, "requests": requests, "chunks": chunks, "new_lo": new_lo, "new_hi": new_hi,
            "cached_lo": cached_lo, "cached_hi": cached_hi, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page_size": page_size, "window": window, "heads_first": heads_first}


def listed():
    return [
        # A decoding step of a small batch: all latency.
        dict(_tables(16, 0, 1, 1, 100, 2048, 16), name="tables_decode"),
        # A step that takes in prompts of very different lengths beside running requests.
        dict(_tables(67, 40, 5, 1501, 1, 4096, 64), name="tables_prompts"),
        # A decoding step's queries and keys, keys and values into the cache.
        dict(_rotary("bf16", 32, 32, 8, 128, "64", page_size=16, far=32768), name="rotary_decode"),
        # A long prompt with images: time, height and width turn their own pairs.
        dict(_rotary("bf16", 4101, 32, 8, 128, "16,24,24", page_size=64), name="rotary_image_prompt"),
        # The gradient through a rotation of half of a head's dims, neighbours paired.
        dict(_rotary("f32", 2048, 16, 16, 80, "20", adjacent=True), name="rotary_f32_gradient"),
        # Decoding with a short context: a few requests, latency counts.
        dict(_attention("bf16", 4, 0, 1, 1, 100, 563, 16, 16, 128, 16), name="attn_decode_short"),
        # Decoding a batch of very different contexts.
        dict(_attention("bf16", 48, 0, 1, 1, 300, 16384, 32, 8, 128, 64), name="attn_decode_batch"),
        # Decoding one request with a very long context, its pages head by head.
        dict(_attention("bf16", 1, 0, 1, 1, 130001, 130001, 32, 8, 128, 32, heads_first=True), name="attn_decode_long"),
        # A prompt's next chunk over what is cached of it.
        dict(_attention("bf16", 1, 1, 2048, 2048, 6001, 6001, 32, 8, 128, 64), name="attn_chunk"),
        # Prompts' chunks and running requests in one batch, head dim 64.
        dict(_attention("bf16", 24, 6, 100, 777, 17, 5000, 16, 2, 64, 16), name="attn_mixed"),
        # The same with layers that see only the last tokens.
        dict(_attention("bf16", 9, 5, 200, 1500, 64, 8192, 16, 4, 96, 128, window=1024), name="attn_window"),
        # A reference run in f32: short chunks, a head of keys per head of queries.
        dict(_attention("f32", 5, 3, 33, 260, 40, 1501, 12, 12, 80, 16), name="attn_f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "rotary", "attention", "attention"])
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "tables":
        requests = _log(rng, 1, 300)
        chunks = rng.choice([0, rng.randint(0, requests)])
        return _tables(requests, chunks, rng.randint(1, 8), _log(rng, 8, max(8, min(1500, 40000 // max(1, chunks)))), rng.randint(1, 64),
                       _log(rng, 64, 8192), rng.choice([1, 8, page, page]), rng.choice([1.25, 1.25, 1.25, 0.7]))
    if kind == "rotary":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        head_dim = rng.choice([64, 80, 96, 128, 128])
        pairs = rng.choice([head_dim // 2, head_dim // 2, head_dim // 4])
        a, b = rng.randint(1, pairs // 3), rng.randint(1, pairs // 3)
        sections = rng.choice(["%d" % pairs, "%d,%d,%d" % (a, b, pairs - a - b)])
        kv = rng.choice([1, 2, 4, 8])
        return _rotary(dtype, _log(rng, 1, 4096), kv * rng.choice([1, 3, 4, 8]), kv, head_dim, sections, rng.random() < 0.3,
                       rng.choice([0, page, page, page]), rng.choice([4096, 131072, 1000000]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    head_dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
    window = rng.choice([0, 0, 0, _log(rng, 16, 2048)])
    if rng.random() < 0.5:  # decoding
        requests = _log(rng, 1, 128)
        cached_hi = _log(rng, 64, max(65, min(60000, int(8e8 / (requests * kv * head_dim * 2 * _SIZE[dtype])))))
        return _attention(dtype, requests, 0, 1, 1, rng.randint(1, 64), cached_hi, kv * group, kv, head_dim, page, window, rng.random() < 0.5)
    requests = _log(rng, 1, 24)
    chunks = rng.randint(1, requests)
    new_hi = _log(rng, 8, 2000 // chunks + 8)
    return _attention(dtype, requests, chunks, rng.randint(1, 8), new_hi, rng.randint(1, 64), _log(rng, 64, 6000), kv * group, kv, head_dim,
                      page, window, rng.random() < 0.5)


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly over their logarithm."""
    return [int(round(hi * (lo / hi) ** (i / max(1, n - 1)))) for i in range(n)]


def _lengths(case):
    """(tokens in the cache, new tokens) of each request; a case's own, whatever the seed."""
    n = case["requests"]
    new = [1] * (n - case["chunks"]) + _spread(case["new_lo"], case["new_hi"], case["chunks"])
    cached = _spread(case["cached_lo"], case["cached_hi"], n)
    random.Random(n).shuffle(cached)
    return list(zip(cached, new))


def _pages(case):
    """What the requests' pages come to: of each before and after the step, and columns of the table."""
    page = case["page_size"]
    have = [-(-c // page) for c, _ in _lengths(case)]
    need = [-(-(c + n) // page) for c, n in _lengths(case)]
    return have, need, max(need) + 1


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def prepare(case, seed):
    order = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, std=1.0):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(_TORCH[dtype])

    def shuffled(n):
        return torch.randperm(n, generator=gen, device="cuda").to(torch.int32)

    if case["op"] == "rotary":
        return _prepare_rotary(case, order, normal, shuffled)
    lengths = _lengths(case)
    order.shuffle(lengths)
    cached, new = [c for c, _ in lengths], [n for _, n in lengths]
    have, need, width = _pages(case)
    page, requests, tokens = case["page_size"], case["requests"], sum(new)
    state = {"case": case, "tokens": tokens, "width": width, "call": None}
    if case["op"] == "tables":
        wanted = sum(need) - sum(have)
        count = int(wanted * case["spare"]) + (2 if case["spare"] > 1 else 0)
        pages = sum(have) + count + 7
        ids = shuffled(pages)
        table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
        taken = 0
        for r, c in enumerate(cached):
            h = -(-c // page)
            table[r, :h] = ids[taken:taken + h]
            taken += h
        state.update(pages=pages, cached=_ints(cached), added=_ints(new), free=ids[taken:taken + count].clone(), free_count=_ints([count]), table=table)
        for name, n in (("starts", requests + 1), ("lengths", requests), ("slots", tokens), ("positions", tokens), ("free_left", 2)):
            state[name] = torch.zeros(n, dtype=torch.int32, device="cuda")
        return state
    dtype, dim, kv = case["dtype"], case["head_dim"], case["kv_heads"]
    pages = sum(need) + 3
    ids = shuffled(pages)
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    taken = 0
    for r, (c, n) in enumerate(lengths):
        h = -(-(c + n) // page)
        table[r, :h] = ids[taken:taken + h]
        taken += h
    shape = (pages, kv, page, dim) if case["heads_first"] else (pages, page, kv, dim)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state.update(
        pages=pages, q=normal((tokens, case["q_heads"], dim), dtype, 2.0),  # scores of a standard deviation of 2
        keys=normal(shape, dtype), values=normal(shape, dtype), table=table, starts=_ints(starts), lengths=_ints([c + n for c, n in lengths]),
        out=torch.zeros((tokens, case["q_heads"], dim), dtype=_TORCH[dtype], device="cuda"), most_new=max(new), longest=max(c + n for c, n in lengths))
    return state


def _prepare_rotary(case, order, normal, shuffled):
    dtype, tokens, dim, kv, page = case["dtype"], case["tokens"], case["head_dim"], case["kv_heads"], case["page_size"]
    pairs = sum(_sections(case))
    axes = len(_sections(case))
    # every axis counts on from a start of its own, as tokens of requests and patches of images do
    at = [order.randrange(case["far"]) for _ in range(axes)]
    steps = torch.arange(tokens, device="cuda", dtype=torch.int64)
    positions = torch.stack([(at[a] + steps // (1 + 17 * a)) % case["far"] for a in range(axes)]).to(torch.int32)
    frequencies = (10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)).to(torch.float32)
    state = {"case": case, "tokens": tokens, "call": None, "positions": positions.contiguous(), "frequencies": frequencies,
             "q": normal((tokens, case["q_heads"], dim), dtype), "k": normal((tokens, kv, dim), dtype),
             "q_out": torch.zeros((tokens, case["q_heads"], dim), dtype=_TORCH[dtype], device="cuda")}
    if page:
        pages = -(-tokens // page) + 2
        shape = (pages, page, kv, dim)
        index = torch.arange(tokens, device="cuda") // page
        slots = shuffled(pages)[index] * page + (torch.arange(tokens, device="cuda") % page).to(torch.int32)
        state.update(pages=pages, v=normal((tokens, kv, dim), dtype), slots=slots.to(torch.int32).contiguous(),
                     keys=torch.zeros(shape, dtype=_TORCH[dtype], device="cuda"), values=torch.zeros(shape, dtype=_TORCH[dtype], device="cuda"))
    else:
        state["k_out"] = torch.zeros((tokens, kv, dim), dtype=_TORCH[dtype], device="cuda")
    return state


def run(state):
    if own:
        return _run_own(state)
    return {"tables": _plain_tables, "rotary": _plain_rotary, "attention": _plain_attention}[state["case"]["op"]](state)


def _run_own(s):
    """What a program keeps per layer: the descriptor and the pointers of its buffers."""
    import morello_amd as M

    case = s["case"]
    if s["call"] is None:
        M.init(0)
        dtype = {"bf16": M.bf16, "f32": M.f32}.get(case.get("dtype"))
        if case["op"] == "tables":
            op = M.PageTables(requests=case["requests"], table_width=s["width"], page_size=case["page_size"], pages=s["pages"],
                              tokens=s["tokens"], free_pages=s["free"].numel())
            tensors = [s[n] for n in ("cached", "added", "free", "free_count", "table", "starts", "lengths", "slots", "positions", "free_left")]
        elif case["op"] == "rotary":
            paged = case["page_size"] > 0
            op = M.Rotary(dtype, tokens=s["tokens"], q_heads=case["q_heads"], kv_heads=case["kv_heads"], head_dim=case["head_dim"],
                          sections=_sections(case), adjacent=case["adjacent"], inverse=not paged, page_size=case["page_size"], pages=s.get("pages", 0))
            names = ("q", "k", "v", "positions", "frequencies", "slots", "q_out", "keys", "values") if paged else \
                ("q", "k", None, "positions", "frequencies", None, "q_out", "k_out", None)
            tensors = [s[n] if n else None for n in names]
        else:
            first = case["heads_first"]
            dim, page, kv = case["head_dim"], case["page_size"], case["kv_heads"]
            strides = (kv * page * dim, dim, page * dim) if first else (page * kv * dim, kv * dim, dim)  # of a page, a slot, a head
            op = M.PagedAttention(dtype, tokens=s["tokens"], requests=case["requests"], q_heads=case["q_heads"], kv_heads=kv, head_dim=dim,
                                  page_size=page, pages=s["pages"], table_width=s["width"], max_new=s["most_new"], window=case["window"],
                                  key_strides=strides, value_strides=strides)
            s["workspace"] = torch.zeros(max(1, op.workspace_bytes()), dtype=torch.uint8, device="cuda")
            tensors = [s[n] for n in ("q", "keys", "values", "table", "starts", "lengths", "out", "workspace")]
        s["call"] = (op, [t.data_ptr() if t is not None else 0 for t in tensors])
    op, pointers = s["call"]
    op.run_async(pointers, torch.cuda.current_stream().cuda_stream)
    if case["op"] == "tables":
        return [s[n] for n in ("table", "starts", "lengths", "slots", "positions", "free_left")]
    if case["op"] == "rotary":
        return [s[n] for n in (("q_out", "keys", "values") if case["page_size"] else ("q_out", "k_out"))]
    return s["out"]


def _plain_tables(s):
    page, width, tokens, pages = s["case"]["page_size"], s["width"], s["tokens"], s["pages"]
    cached, added, free, table = s["cached"].long().clamp(min=0), s["added"].long().clamp(min=0), s["free"].long(), s["table"]
    count = s["free_count"].long().clamp(0, free.numel())
    starts = torch.cat([torch.zeros_like(added[:1]), torch.cumsum(added, 0)]).clamp(max=tokens)
    lengths = cached + starts.diff()
    have = ((cached + page - 1) // page).clamp(max=width)
    drawn = torch.maximum(((lengths + page - 1) // page).clamp(max=width), have) - have
    first = torch.cumsum(drawn, 0) - drawn
    t = torch.arange(tokens, device="cuda")
    there = t < starts[-1]
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=cached.numel() - 1)
    position = cached[r] + t - starts[r]
    column = position // page
    k = first[r] + column - have[r]
    inside = there & (column < width)
    from_list = torch.where(k < count, free[(count - 1 - k).clamp(0, max(0, free.numel() - 1))] if free.numel() else torch.full_like(k, -1), torch.full_like(k, -1))
    number = torch.where(column >= have[r], from_list, table[r, column.clamp(max=width - 1)].long())
    number = torch.where(inside, number, torch.full_like(number, -1))
    opens = inside & (position % page == 0)
    flat = torch.where(opens, r * width + column, torch.full_like(r, table.numel()))
    grown = torch.cat([table.reshape(-1), table.new_zeros(1)]).scatter(0, flat, number.to(torch.int32))  # the rest lands behind the end
    table.copy_(grown[:-1].view_as(table))
    slots = torch.where((number >= 0) & (number < pages), number * page + position % page, torch.full_like(number, -1))
    positions = torch.where(there, position, torch.zeros_like(position))
    total = drawn.sum()
    left = torch.stack([(count[0] - total).clamp(min=0), (total - count[0]).clamp(min=0)])
    return [table] + [x.to(torch.int32) for x in (starts, lengths, slots, positions, left)]


def _turned(x, cos, sin, adjacent):
    """The pairs of the first dims of each head turned, in 32 bits; the dims behind them as they are."""
    pairs = cos.shape[-1]
    f = x.float()
    head, rest = f[..., :2 * pairs], f[..., 2 * pairs:]
    a, b = (head[..., 0::2], head[..., 1::2]) if adjacent else (head[..., :pairs], head[..., pairs:])
    c, s = cos[:, None, :], sin[:, None, :]
    u, w = a * c - b * s, b * c + a * s
    both = torch.stack([u, w], -1).flatten(-2) if adjacent else torch.cat([u, w], -1)
    return torch.cat([both, rest], -1).to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    axis = torch.repeat_interleave(torch.arange(len(_sections(case)), device="cuda"), torch.tensor(_sections(case), device="cuda"))
    angles = s["positions"].double()[axis].T * s["frequencies"].double()
    cos, sin = torch.cos(angles).float(), torch.sin(angles).float()
    if not case["page_size"]:
        s["q_out"].copy_(_turned(s["q"], cos, -sin, case["adjacent"]))
        s["k_out"].copy_(_turned(s["k"], cos, -sin, case["adjacent"]))
        return [s["q_out"], s["k_out"]]
    s["q_out"].copy_(_turned(s["q"], cos, sin, case["adjacent"]))
    at = s["slots"].long()
    s["keys"].view(-1, case["kv_heads"], case["head_dim"])[at] = _turned(s["k"], cos, sin, case["adjacent"])
    s["values"].view(-1, case["kv_heads"], case["head_dim"])[at] = s["v"]
    return [s["q_out"], s["keys"], s["values"]]


def _plain_attention(s):
    """Every request's keys, values and queries side by side as long as the longest ones', in 32 bits."""
    case = s["case"]
    page, kv, dim, longest, most = case["page_size"], case["kv_heads"], case["head_dim"], s["longest"], s["most_new"]
    group, requests = case["q_heads"] // kv, case["requests"]
    at = torch.arange(longest, device="cuda")
    numbers = s["table"][:, at // page].long().clamp(min=0)
    lengths, starts = s["lengths"].long(), s["starts"].long()
    there = at[None, :] < lengths[:, None]

    def rows(cache):
        if case["heads_first"]:
            cache = cache.transpose(1, 2)
        got = cache[numbers, (at % page).expand_as(numbers)].float()
        return (got * there[:, :, None, None]).permute(0, 2, 1, 3).contiguous()  # requests, heads, keys, dims

    i = torch.arange(most, device="cuda")
    new = starts.diff()
    row = (starts[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][row].float().view(requests, most, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(requests, kv, most * group, dim)
    scores = torch.matmul(q * dim ** -0.5, rows(s["keys"]).transpose(2, 3).contiguous()).view(requests, kv, most, group, longest)
    position = (lengths - new)[:, None] + i
    seen = at[None, None, :] <= position[:, :, None]
    if case["window"]:
        seen = seen & (at[None, None, :] > position[:, :, None] - case["window"])
    scores = scores.masked_fill(~seen[:, None, :, None, :], float("-inf"))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = (weights / weights.sum(-1, keepdim=True)).view(requests, kv, most * group, longest)
    got = torch.matmul(weights, rows(s["values"])).view(requests, kv, most, group, dim)
    got = got.permute(0, 2, 1, 3, 4).reshape(requests, most, case["q_heads"], dim).to(_TORCH[case["dtype"]])
    mine = i[None, :] < new[:, None]
    s["out"][row[mine]] = got[mine]
    return s["out"]


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    if 8.0 * case["q_heads"] * sum(n * (c + n) for c, n in _lengths(case)) > 4e10:
        return None
    page, kv, dim = case["page_size"], case["kv_heads"], case["head_dim"]
    group = case["q_heads"] // kv
    out = torch.zeros((s["tokens"], case["q_heads"], dim), dtype=torch.float64, device="cuda")
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for r, length in enumerate(lengths):
        first, end = starts[r], starts[r + 1]
        numbers = s["table"][r, :-(-length // page)].long()
        keys, values = s["keys"][numbers], s["values"][numbers]
        if case["heads_first"]:
            keys, values = keys.transpose(1, 2), values.transpose(1, 2)
        keys, values = (x.reshape(-1, kv, dim)[:length].double() for x in (keys, values))
        where = torch.arange(length - (end - first), length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None, :]
        hidden = key > where
        if case["window"]:
            hidden = hidden | (key <= where - case["window"])
        for h in range(case["q_heads"]):
            score = s["q"][first:end, h].double() @ keys[:, h // group].T.contiguous() / math.sqrt(dim)
            out[first:end, h] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ values[:, h // group].contiguous()
    return out


def _exact_rotary(case, s):
    sections, dim, tokens = _sections(case), case["head_dim"], s["tokens"]
    pairs = sum(sections)
    way = 1.0 if case["page_size"] else -1.0
    first, second = (range(0, 2 * pairs, 2), range(1, 2 * pairs, 2)) if case["adjacent"] else (range(pairs), range(pairs, 2 * pairs))
    results = []
    for x in (s["q"], s["k"]):
        y = x.double().clone()
        pair = 0
        for axis, n in enumerate(sections):
            for _ in range(n):
                turn = torch.polar(torch.ones(tokens, dtype=torch.float64, device="cuda"), way * s["positions"][axis].double() * s["frequencies"][pair].double())
                z = torch.complex(x[..., first[pair]].double(), x[..., second[pair]].double()) * turn[:, None]
                y[..., first[pair]], y[..., second[pair]] = z.real, z.imag
                pair += 1
        results.append(y)
    if not case["page_size"]:
        return results
    caches = []
    for x in (results[1], s["v"].double()):
        cache = torch.zeros((s["pages"] * case["page_size"], case["kv_heads"], dim), dtype=torch.float64, device="cuda")
        cache[s["slots"].long()] = x
        caches.append(cache.view(s["pages"], case["page_size"], case["kv_heads"], dim))
    return [results[0]] + caches


def work(case):
    if case["op"] == "tables":
        have, need, _ = _pages(case)
        tokens = sum(n for _, n in _lengths(case))
        # lengths and the pages drawn are read; starts, lengths, pages, slots and positions written
        return {"bytes": 4 * (4 * case["requests"] + 2 * (sum(need) - sum(have)) + 2 * tokens), "flops": 0}
    size, dim = _SIZE[case["dtype"]], case["head_dim"]
    if case["op"] == "rotary":
        heads = case["q_heads"] + (2 if case["page_size"] else 1) * case["kv_heads"]
        pairs = sum(_sections(case))
        return {"bytes": 2 * size * case["tokens"] * heads * dim + 4 * case["tokens"] * len(_sections(case)) + 4 * pairs,
                "flops": 6 * pairs * case["tokens"] * (case["q_heads"] + case["kv_heads"])}
    keys, pairs, tokens = 0, 0, 0
    window = case["window"] or 1 << 40
    for c, n in _lengths(case):
        keys += min(c + n, window + n - 1)
        pairs += sum(min(p + 1, window) for p in range(c, c + n))
        tokens += n
    return {"bytes": size * dim * (2 * tokens * case["q_heads"] + 2 * keys * case["kv_heads"]), "flops": 4 * pairs * case["q_heads"] * dim}
