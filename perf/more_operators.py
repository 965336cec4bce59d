"""What a decode step needs around the key-value cache, as timed cases: page tables and slot maps built on the GPU (`kv_pages_v1`), rotary positions
forward and backward (`rotary_v1`), rotated rows written into the cache (`kv_cache_rotary_append_v1`), and a cache held in 4 bits, written, read back
and attended to (`kv_cache_append_v1`, `kv_cache_read_v1`, `paged_attention_v1` with the format e2m1).

`own` False: their plain form, elementary torch operations in 32 bits (angles in 64).  `own` True: the library's launches, prepared once and launched
per pass as a serving program does.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
FREE = -1   # of a page table and of a slot map, as signed bits


def listed():
    return [
        # -- page tables and slot maps.  One new token for each of a small batch's sequences: latency
        {"name": "pages_step_48", "op": "pages", "batch": 48, "tokens": 48, "width": 256, "page": 16, "before": 2000, "each": True, "released": 0},
        #    prompts of many requests come in at once, finished ones leave their pages
        {"name": "pages_131072", "op": "pages", "batch": 512, "tokens": 131072, "width": 640, "page": 16, "before": 6000, "each": False, "released": 61},
        # -- rotary positions.  Queries and keys of a long prompt
        {"name": "rotary_16384", "op": "rotary", "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "type": "bf16",
         "backward": False, "far": 16384},
        #    their gradient, in f32: neighbours as pairs, part of the head, positions far out, an odd number of tokens
        {"name": "rotary_back_1003", "op": "rotary", "tokens": 1003, "heads": 12, "kv_heads": 12, "dim": 96, "rotary": 32, "layout": "interleaved",
         "type": "f32", "backward": True, "far": 1000000},
        # -- rotated and written: pieces of five prompts, a quarter of the head rotated
        {"name": "write_8191", "op": "write", "batch": 5, "tokens": 8191, "heads": 16, "kv_heads": 16, "dim": 80, "rotary": 20, "layout": "half", "page": 16,
         "before": 300, "type": "bf16", "far": 100000},
        #    a whole step of one attention block: pages, rotation and cache, attention
        {"name": "step_64x2048", "op": "step", "batch": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "page": 16,
         "max_len": 2048, "ragged": True, "type": "bf16", "far": 0},
        # -- rows of a 4-bit cache: prompts of eight requests written, and what the cache then holds of them (for the prompts' own attention)
        {"name": "append4_16384", "op": "append4", "batch": 8, "tokens": 16384, "kv_heads": 8, "dim": 128, "before": 0, "page": 64, "input": "bf16"},
        #    all of a cache read back
        {"name": "read4_131072", "op": "read4", "batch": 16, "tokens": 131072, "kv_heads": 8, "dim": 128, "before": 0, "page": 64, "output": "bf16"},
        # -- one new token a sequence over a 4-bit cache.  A single user's short context
        {"name": "attend4_1x512", "op": "attend4", "batch": 1, "heads": 16, "kv_heads": 16, "dim": 64, "max_len": 512, "ragged": False, "page": 16,
         "window": 0, "q": "bf16", "out": "f32"},
        #    an ordinary batch of all lengths, one request not begun yet; eight query heads to a key head
        {"name": "attend4_96_ragged", "op": "attend4", "batch": 96, "heads": 32, "kv_heads": 4, "dim": 128, "max_len": 6000, "ragged": True, "page": 64,
         "window": 0, "q": "bf16", "out": "bf16"},
        #    two long documents
        {"name": "attend4_2x131071", "op": "attend4", "batch": 2, "heads": 32, "kv_heads": 8, "dim": 128, "max_len": 131071, "ragged": False, "page": 64,
         "window": 0, "q": "bf16", "out": "bf16"},
        #    f32 queries, a head size between the powers of two, pages of 24, the last 1777 keys only
        {"name": "attend4_window_40", "op": "attend4", "batch": 40, "heads": 24, "kv_heads": 12, "dim": 96, "max_len": 2900, "ragged": True, "page": 24,
         "window": 1777, "q": "f32", "out": "f32"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend4", "attend4", "attend4", "append4", "read4", "rotary", "rotary", "write", "step", "pages"])
    page = rng.choice([16, 16, 32, 64, 64, 128, 24, 8])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 12, 16])
    group = rng.choice([1, 2, 3, 4, 4, 8, 16] if kv_heads < 8 else [1, 1, 2, 4, 4, 5])
    if op == "pages":
        batch = _log(rng, 1, 1000)
        tokens = batch if rng.random() < 0.4 else batch + _log(rng, 1, 131072 - batch)
        before, page = _log(rng, 1, 8000), rng.choice([16, 16, 32, 64, 1, 7, 24])
        width = -(-(before + min(tokens, 4 * (tokens // batch) + 64)) // page)
        while batch * width > 1 << 20:
            width, before = width // 2 + 1, before // 2
        return {"op": op, "batch": batch, "tokens": tokens, "width": width, "page": page, "before": max(1, min(before, width * page // 4)),
                "each": tokens == batch, "released": 0 if tokens == batch or batch < 4 else rng.randrange(batch // 4)}
    if op in ("attend4", "append4", "read4"):
        dim = rng.choice([64, 128, 128, 128, 32, 96, 160, 256])
        rows = (1 << 27) // (kv_heads * dim)
        batch = _log(rng, 1, 256)
        if op == "attend4":
            max_len = _log(rng, 1, max(1, min(131072, rows // batch)))
            return {"op": op, "batch": batch, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "max_len": max_len, "ragged": rng.random() < 0.7,
                    "page": page, "window": rng.choice([0, 0, 0, _log(rng, 1, max(2, max_len))]), "q": rng.choice(["bf16", "bf16", "f32"]),
                    "out": rng.choice(["bf16", "f32"])}
        tokens = batch + _log(rng, 1, max(2, min(1 << 17, (1 << (24 if op == "append4" else 26)) // (kv_heads * dim) - batch)))
        case = {"op": op, "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "before": rng.choice([0, 0, _log(rng, 1, 500)]), "page": page}
        case["input" if op == "append4" else "output"] = rng.choice(["bf16", "f32"])
        return case
    dim = rng.choice([64, 64, 128, 128, 128, 32, 80, 96, 256])
    rotary = rng.choice([dim, dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)])
    case = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "layout": rng.choice(["half", "half", "interleaved"]),
            "type": rng.choice(["bf16", "bf16", "f32"]), "far": _log(rng, 1, 2000000)}
    room = (1 << 26) // (dim * kv_heads * (group + 1))
    if op == "rotary":
        return {**case, "tokens": _log(rng, 1, room), "backward": rng.random() < 0.4}
    batch = _log(rng, 1, min(256, max(1, room // 2)))
    if op == "write":
        return {**case, "batch": batch, "tokens": batch + _log(rng, 1, max(2, min(1 << 15, room // 2 - batch))), "before": rng.choice([0, 0, _log(rng, 1, 500)]),
                "page": page}
    return {**case, "batch": batch, "max_len": _log(rng, 1, max(1, min(65536, (1 << 26) // (kv_heads * dim * batch)))), "ragged": rng.random() < 0.7,
            "page": page, "far": 0}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------

def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _below(g, top, shape):
    return torch.randint(0, top, shape, generator=g, device="cuda", dtype=torch.int64)


def _divided(x, by):
    """Quotients by a plain number (which torch would make a product with its reciprocal)."""
    return x / torch.full((), by, dtype=x.dtype, device=x.device)


def _codes4(y):
    """The nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 by number, ties to the even one; 8 more for a minus."""
    a, code = y.abs(), torch.zeros(y.shape, dtype=torch.uint8, device=y.device)
    for at, with_it in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= at) if with_it else (a > at)
    return code + 8 * torch.signbit(y).to(torch.uint8)


def _quantised4(x):
    """Packed codes (the even column in the low half), block scales' bytes and row scales of f32 rows."""
    m = x.abs().amax(-1, keepdim=True)
    some = m >= 2.0 ** -100
    one = torch.where(some, m, torch.ones((), device=x.device))
    scale = torch.where(some, _divided(m, 2688.0), torch.zeros((), device=x.device))
    blocks = x.unflatten(-1, (-1, 16))
    b = (blocks.abs().amax(-1) * (torch.full((), 448.0, device=x.device) / one)).to(torch.float8_e4m3fn)
    b = torch.where(some, b.view(torch.uint8), torch.zeros((), dtype=torch.uint8, device=x.device))
    step = (b.view(torch.float8_e4m3fn).float() * scale).unsqueeze(-1)
    r = torch.where(step > 0, torch.ones((), device=x.device) / torch.where(step > 0, step, torch.ones((), device=x.device)), torch.zeros((), device=x.device))
    code = _codes4(blocks * r).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, b, scale.squeeze(-1)


def _widened4(code, b):
    """f32 values of codes with their block scales (exact)."""
    value = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    x = torch.stack([value[(code & 15).int()], value[(code >> 4).int()]], -1).flatten(-2)
    return (x.unflatten(-1, (-1, 16)) * b.view(torch.float8_e4m3fn).float().unsqueeze(-1)).flatten(-2)


def _parts4(cache, case, pages):
    """A 4-bit cache's two parts: codes [pages][kv_heads][page][dim / 2] and, behind them, block scales [pages][kv_heads][page][dim / 16]."""
    rows = pages * case["kv_heads"] * case["page"]
    codes = rows * case["dim"] // 2
    shape = (pages, case["kv_heads"], case["page"], -1)
    return cache[:codes].view(shape), cache[codes:].view(shape)


def _lengths(g, case):
    """Cached tokens of each sequence, the new one included."""
    batch, top = case["batch"], case["max_len"]
    if not case["ragged"]:
        return torch.full((batch,), top, dtype=torch.int32, device="cuda")
    n = torch.randint(1, top + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = top
    if batch > 2 and case["op"] == "attend4":
        n[1] = 0   # a slot of the batch without a request
    return n


def _counts(g, batch, tokens):
    """How new tokens fall on the sequences."""
    if tokens == batch:
        return torch.ones(batch, dtype=torch.int64, device="cuda")
    cuts = torch.sort(_below(g, tokens + 1, (batch - 1,))).values
    return torch.diff(torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), tokens)]))


def _offsets(n):
    return torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), n.cumsum(0)]).to(torch.int32)


def _table(g, lengths, width, page, pages):
    """Pages in no order, a sequence's table of them; the pages that are left over."""
    used = (lengths.long() + page - 1) // page
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), width), FREE, dtype=torch.int32, device="cuda")
    taken = int(used.sum())
    table[torch.arange(width, device="cuda") < used.unsqueeze(1)] = order[:taken]
    return table, order[taken:]


def _cache(g, case, pages, bits):
    """What an earlier life of the cache left in every slot; some channels of the keys are several times as large as the others."""
    page, kv_heads, dim = case["page"], case["kv_heads"], case["dim"]
    spread, s = torch.exp(0.5 * _normal(g, dim)), {}
    for name, by in (("k", spread), ("v", 1.0)):
        shape = (pages, kv_heads, page, dim)
        if bits == 16:
            s[name + "_cache"] = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        else:
            s[name + "_cache"] = torch.empty(pages * kv_heads * page * dim * 9 // 16, dtype=torch.uint8, device="cuda")
            s[name + "_scales"] = torch.empty(shape[:3], device="cuda")
            codes, blocks = _parts4(s[name + "_cache"], case, pages)
        step = max(1, (1 << 25) // (kv_heads * page * dim))
        for at in range(0, pages, step):
            x = _normal(g, (min(step, pages - at),) + shape[1:]) * by
            if bits == 16:
                s[name + "_cache"][at:at + step] = x.to(torch.bfloat16)
            else:
                codes[at:at + step], blocks[at:at + step], s[name + "_scales"][at:at + step] = _quantised4(x)
    return s


def _frequencies(case):
    r = case["rotary"]
    f = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    return (f / 4 if case["far"] > 32768 else f).float()   # (scaled for long contexts)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, page = case["op"], case.get("page")
    s = {"case": case}
    if op == "pages":
        batch, width, tokens = case["batch"], case["width"], case["tokens"]
        released = torch.zeros(batch, dtype=torch.int32, device="cuda")
        released[torch.randperm(batch, generator=g, device="cuda")[:case["released"]]] = 1
        n = _counts(g, batch, tokens) if not case["each"] else torch.ones(batch, dtype=torch.int64, device="cuda")
        n = torch.where(released > 0, torch.zeros_like(n), n)   # (their slots stand empty for now)
        if not case["each"]:
            n = torch.minimum(n, torch.full_like(n, width * page - case["before"]))
        before = 1 + _below(g, case["before"], (batch,))
        s["lengths"] = before.to(torch.int32)
        pages = (tokens + batch * case["before"]) // page + batch   # enough for all at their longest
        s["table"], left = _table(g, s["lengths"], width, page, pages)
        s["free"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
        s["free"][:len(left)] = left
        s["free_count"] = torch.tensor([len(left)], dtype=torch.int32, device="cuda")
        s["counts"] = None if case["each"] else n.to(torch.int32)
        s["released"] = released if case["released"] else None
    elif op == "rotary":
        dt = DTYPES[case["type"]]
        s["positions"] = _below(g, case["far"], (1,)).add(torch.arange(case["tokens"], device="cuda")).to(torch.int32)
        s["q"], s["k"] = (_normal(g, (case["tokens"], case[h], case["dim"]), dt) for h in ("heads", "kv_heads"))
    elif op in ("write", "step"):
        dt = DTYPES[case["type"]]
        if op == "write":
            n = _counts(g, case["batch"], case["tokens"])
            s["lengths"] = (n + _below(g, case["before"] + 1, (case["batch"],))).to(torch.int32)
            width, tokens = -(-(case["tokens"] + case["before"]) // page), case["tokens"]
            pages = (case["tokens"] + case["batch"] * case["before"]) // page + case["batch"]
            s["table"], _ = _table(g, s["lengths"], width, page, pages)
            offsets = _offsets(n).long()
            t = torch.arange(tokens, device="cuda")
            seq = torch.searchsorted(offsets, t, right=True) - 1
            at = s["lengths"].long()[seq] - offsets[seq + 1] + t
            s["slots"] = (s["table"].long()[seq, at // page] * page + at % page).to(torch.int32)
            s["positions"] = (at + _below(g, case["far"], (1,))).to(torch.int32)   # (far: rows behind a prefix that is kept elsewhere)
        else:
            after = _lengths(g, case)
            s["lengths"] = after - 1
            width, tokens = -(-case["max_len"] // page), case["batch"]
            pages = case["batch"] * width
            s["table"], left = _table(g, s["lengths"], width, page, pages)
            s["free"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
            s["free"][:len(left)] = left
            s["free_count"] = torch.tensor([len(left)], dtype=torch.int32, device="cuda")
            s["counts"], s["released"] = torch.ones(tokens, dtype=torch.int32, device="cuda"), None
            s["o"] = torch.zeros(case["batch"], case["heads"], case["dim"], dtype=dt, device="cuda")
        s["q"], s["k"], s["v"] = (_normal(g, (tokens, case[h], case["dim"]), dt) for h in ("heads", "kv_heads", "kv_heads"))
        s["width"], s["pages"] = width, pages
        s.update(_cache(g, case, pages, 16))
    elif op == "attend4":
        s["lengths"] = _lengths(g, case)
        s["width"] = -(-case["max_len"] // page)
        s["pages"] = case["batch"] * s["width"]
        s["table"], _ = _table(g, s["lengths"], s["width"], page, s["pages"])
        s.update(_cache(g, case, s["pages"], 4))
        s["q"] = _normal(g, (case["batch"], case["heads"], case["dim"]), DTYPES[case["q"]])
        s["o"] = torch.zeros(case["batch"], case["heads"], case["dim"], dtype=DTYPES[case["out"]], device="cuda")
        s["lse"] = torch.zeros(case["batch"], case["heads"], device="cuda") if case["out"] == "f32" else None
    else:
        n = _counts(g, case["batch"], case["tokens"])
        s["lengths"], s["offsets"] = (n + _below(g, case["before"] + 1, (case["batch"],))).to(torch.int32), _offsets(n)
        s["width"] = -(-(case["tokens"] + case["before"]) // page)
        s["pages"] = (case["tokens"] + case["batch"] * case["before"]) // page + case["batch"]
        s["table"], _ = _table(g, s["lengths"], s["width"], page, s["pages"])
        s.update(_cache(g, case, s["pages"], 4))
        shape = (case["tokens"], case["kv_heads"], case["dim"])
        if op == "append4":
            s["k"], s["v"] = (_normal(g, shape, DTYPES[case["input"]]) for _ in range(2))
        s["k_out"], s["v_out"] = (torch.zeros(shape, dtype=DTYPES[case.get("output", "f32")], device="cuda") for _ in range(2))
    if "rotary" in case:
        s["frequencies"] = _frequencies(case)
        s["q_out"] = torch.zeros_like(s["q"])
        if op == "rotary":
            s["k_out"] = torch.zeros_like(s["k"])
    if op in ("pages", "step"):
        count = case["tokens"] if "tokens" in case else case["batch"]
        s["next_lengths"], s["next_free_count"] = torch.zeros_like(s["lengths"]), torch.zeros_like(s["free_count"])
        s["offsets"] = torch.zeros(case["batch"] + 1, dtype=torch.int32, device="cuda")
        s["positions"], s["slots"] = (torch.zeros(count, dtype=torch.int32, device="cuda") for _ in range(2))
    if own:
        s["launches"], s["stream"] = _prepared(s)
    return s


# ---- the library's launches ----------------------------------------------------------------------------------------------------------

_ctx = None


def _prepared(s):
    """The launches of one pass, in order."""
    import fe2o3_b200 as fe
    global _ctx
    if _ctx is None:
        ctx = fe.GpuContext(torch.cuda.current_device())
        _ctx = (ctx, ctx.default_stream())
    ctx, stream = _ctx
    case, op, launches = s["case"], s["case"]["op"], []
    code = {torch.float32: fe.DTYPE_F32, torch.bfloat16: fe.DTYPE_BF16}
    dim, kv_heads, heads = case.get("dim"), case.get("kv_heads"), case.get("heads")

    def packed(*names):   # strides of contiguous rows
        return {k: v for n in names for k, v in ((n + "_token_stride", (heads if n[0] == "q" else kv_heads) * dim), (n + "_head_stride", dim))}

    layout = {"half": fe.ROTARY_HALF, "interleaved": fe.ROTARY_INTERLEAVED}.get(case.get("layout"))
    if op in ("pages", "step"):
        launches.append(fe.prepare(ctx, "kv_pages_v1", counts=s["counts"], release=s["released"], lengths=s["lengths"], free_count=s["free_count"],
                                   page_table=s["table"], free_pages=s["free"], next_lengths=s["next_lengths"], next_free_count=s["next_free_count"],
                                   token_offsets=s["offsets"], positions=s["positions"], slots=s["slots"], batch=case["batch"],
                                   table_width=s["table"].shape[1], page_size=case["page"], tokens=len(s["slots"])))
    if op == "rotary":
        launches.append(fe.prepare(ctx, "rotary_v1", q=s["q"], k=s["k"], positions=s["positions"], frequencies=s["frequencies"], q_output=s["q_out"],
                                   k_output=s["k_out"], tokens=case["tokens"], heads=heads, kv_heads=kv_heads, dim=dim, rotary_dim=case["rotary"],
                                   layout=layout, dtype=code[s["q"].dtype], backward=int(case["backward"]), scale=1.0,
                                   **packed("q", "k", "q_output", "k_output")))
    if "k_cache" in s:
        cache = {n: s[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales") if n in s}
        cache.update(kv_heads=kv_heads, dim=dim, page_size=case["page"], format=fe.KV_E2M1 if "k_scales" in s else fe.KV_BF16)
        book = dict(page_table=s["table"], lengths=s.get("next_lengths", s["lengths"]), batch=case["batch"], table_width=s["width"])
    if op in ("write", "step"):
        launches.append(fe.prepare(ctx, "kv_cache_rotary_append_v1", q=s["q"], k=s["k"], v=s["v"], positions=s["positions"], slots=s["slots"],
                                   frequencies=s["frequencies"], q_output=s["q_out"], tokens=len(s["slots"]), heads=heads, rotary_dim=case["rotary"],
                                   layout=layout, input_dtype=code[s["q"].dtype], scale=1.0, **packed("q", "k", "v", "q_output"), **cache))
    if op == "append4":
        launches.append(fe.prepare(ctx, "kv_cache_append_v1", k=s["k"], v=s["v"], token_offsets=s["offsets"], tokens=case["tokens"],
                                   input_dtype=code[s["k"].dtype], **packed("k", "v"), **cache, **book))
    if op in ("append4", "read4"):
        launches.append(fe.prepare(ctx, "kv_cache_read_v1", k=s["k_out"], v=s["v_out"], token_offsets=s["offsets"], tokens=case["tokens"],
                                   output_dtype=code[s["k_out"].dtype], **packed("k", "v"), **cache, **book))
    if "o" in s:
        launches.append(fe.prepare(ctx, "paged_attention_v1", q=s["q_out"] if op == "step" else s["q"], output=s["o"], lse=s.get("lse"), heads=heads,
                                   q_stride=heads * dim, q_head_stride=dim, scale=1 / math.sqrt(dim), window=case.get("window", 0),
                                   q_dtype=code[s["q"].dtype], output_dtype=code[s["o"].dtype], **cache, **book))
    return launches, stream


# ---- the plain forms -----------------------------------------------------------------------------------------------------------------

def _plain_pages(s):
    case = s["case"]
    page, (batch, width), tokens = case["page"], s["table"].shape, len(s["slots"])
    lengths, table, top = s["lengths"].long(), s["table"].long(), s["free_count"].long()
    gone = s["released"] > 0 if s["released"] is not None else torch.zeros(batch, dtype=torch.bool, device="cuda")
    column, stack = torch.arange(width, device="cuda"), torch.cat([s["free"].long(), torch.zeros(1, dtype=torch.int64, device="cuda")])
    back = torch.where(gone, (lengths + page - 1) // page, 0)
    behind = top + back.cumsum(0) - back
    at = torch.where(column < back.unsqueeze(1), behind.unsqueeze(1) + back.unsqueeze(1) - 1 - column, len(stack) - 1)   # (the rest goes where nothing reads)
    stack[at] = table
    top = top + back.sum()
    lengths = torch.where(gone, 0, lengths)
    n = s["counts"].long() if s["counts"] is not None else (lengths > 0).long()
    held, need = (lengths + page - 1) // page, (lengths + n + page - 1) // page
    first = (need - held).cumsum(0) - need   # + column: which of the new pages
    mine = (column >= held.unsqueeze(1)) & (column < need.unsqueeze(1))
    table = torch.where(mine, stack[(top - 1 - first.unsqueeze(1) - column).clamp(min=0, max=len(stack) - 1)], table)
    ends = n.cumsum(0)
    t = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(ends, t, right=True).clamp(max=batch - 1)
    position = lengths[seq] + t - (ends - n)[seq]
    slot = table[seq, (position // page).clamp(max=width - 1)] * page + position % page
    inside = t < ends[-1]
    s["table"].copy_(table)
    s["free"].copy_(stack[:-1])
    s["next_lengths"].copy_(lengths + n)
    s["next_free_count"].copy_(top - (need - held).sum())
    s["offsets"].copy_(torch.cat([ends.new_zeros(1), ends]))
    s["positions"].copy_(torch.where(inside, position, 0))
    s["slots"].copy_(torch.where(inside, slot, FREE))


def _rotated(x, positions, frequencies, layout, sign, dtype):
    """Rows [tokens][heads][dim] with the pairs of their first columns turned, in `dtype`."""
    r = 2 * len(frequencies)
    angle = positions.double().view(-1, 1) * frequencies.double()
    c, s = torch.cos(angle).to(dtype).unsqueeze(1), sign * torch.sin(angle).to(dtype).unsqueeze(1)
    x = x.to(dtype)
    turned, rest = x[..., :r], x[..., r:]
    if layout == "half":
        a, b = turned[..., :r // 2], turned[..., r // 2:]
        return torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), rest], -1)


def _plain_write(s):
    case, page = s["case"], s["case"]["page"]
    s["q_out"], k = (_rotated(s[n], s["positions"], s["frequencies"], case["layout"], 1.0, torch.float32).to(s[n].dtype if n == "q" else torch.bfloat16)
                     for n in ("q", "k"))
    at = s["slots"].long()
    s["k_cache"][at // page, :, at % page] = k
    s["v_cache"][at // page, :, at % page] = s["v"].to(torch.bfloat16)


def _held(s, name, where, dtype):
    """What rows (page, head or all, slot) of one side of the cache stand for."""
    if "k_scales" not in s:
        return s[name + "_cache"][where].to(dtype)
    codes, blocks = _parts4(s[name + "_cache"], s["case"], s["pages"])
    return _widened4(codes[where], blocks[where]).to(dtype) * s[name + "_scales"][where].to(dtype).unsqueeze(-1)


def _plain_attend(s, q, lengths):
    case = s["case"]
    batch, kv_heads, page, dim = case["batch"], case["kv_heads"], case["page"], case["dim"]
    table = s["table"].long().clamp(min=0)

    def gathered(name):   # [batch][kv_heads][positions][dim]
        return _held(s, name, table, torch.float32).transpose(1, 2).reshape(batch, kv_heads, s["width"] * page, dim)

    q = q.float().view(batch, kv_heads, case["heads"] // kv_heads, dim)
    scores = q @ gathered("k").transpose(2, 3) * (1 / math.sqrt(dim))
    at, n = torch.arange(s["width"] * page, device="cuda"), lengths.long().view(batch, 1, 1, 1)
    keep = at < n
    if case.get("window"):
        keep = keep & (at >= n - case["window"])
    scores = torch.where(keep, scores, torch.full((), -math.inf, device="cuda"))
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = (p @ gathered("v")) / torch.where(total > 0, total, torch.ones((), device="cuda"))
    lse = torch.where(total > 0, top + torch.log(total), torch.full((), -math.inf, device="cuda"))
    return o.view(batch, case["heads"], dim).to(s["o"].dtype), lse.view(batch, case["heads"])


def _slots(s):
    """(page, slot) of every new token's row."""
    page, offsets = s["case"]["page"], s["offsets"].long()
    t = torch.arange(s["case"]["tokens"], device="cuda")
    seq = torch.searchsorted(offsets, t, right=True) - 1
    position = s["lengths"].long()[seq] - offsets[seq + 1] + t
    return s["table"].long()[seq, position // page], position % page


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op in ("pages", "step"):
        _plain_pages(s)
    if op == "rotary":
        for n in "qk":
            s[n + "_out"] = _rotated(s[n], s["positions"], s["frequencies"], case["layout"], -1.0 if case["backward"] else 1.0, torch.float32).to(s[n].dtype)
    if op in ("write", "step"):
        _plain_write(s)
    if op == "append4":
        page, slot = _slots(s)
        for n in "kv":
            codes, blocks = _parts4(s[n + "_cache"], case, s["pages"])
            codes[page, :, slot], blocks[page, :, slot], s[n + "_scales"][page, :, slot] = _quantised4(s[n].float())
    if op in ("append4", "read4"):
        page, slot = _slots(s)
        for n in "kv":
            s[n + "_out"] = _held(s, n, (page, slice(None), slot), torch.float32).to(s[n + "_out"].dtype)
    if op in ("attend4", "step"):
        s["o"], lse = _plain_attend(s, s["q_out"] if op == "step" else s["q"], s["next_lengths"] if op == "step" else s["lengths"])
        if s.get("lse") is not None:
            s["lse"] = lse


_OUTPUTS = {"pages": ("table", "free", "next_lengths", "next_free_count", "offsets", "positions", "slots"), "rotary": ("q_out", "k_out"),
            "write": ("q_out", "k_cache", "v_cache"), "step": ("o", "q_out", "table", "next_lengths", "next_free_count", "positions", "slots", "k_cache", "v_cache"),
            "append4": ("k_out", "v_out"), "read4": ("k_out", "v_out"), "attend4": ("o", "lse")}


def run(state):
    if own:
        for launch in state["launches"]:
            launch.launch(state["stream"])
    else:
        _plain(state)
    return {n: state[n] for n in _OUTPUTS[state["case"]["op"]] if state.get(n) is not None}


def work(case):
    op, page = case["op"], case.get("page")
    if op == "pages":
        new = case["tokens"] // page
        return {"bytes": 8 * case["tokens"] + 8 * new + case["batch"] * (12 if case["each"] else 20), "flops": 0}
    kv_heads, dim = case["kv_heads"], case["dim"]
    size = lambda name: 4 if case[name] == "f32" else 2  # noqa: E731
    row = dim * 9 / 16 + 4   # of one side of a 4-bit cache
    if op in ("append4", "read4"):
        rows = 2 * case["tokens"] * kv_heads
        moved = rows * (row + dim * size("input" if op == "append4" else "output"))
        if op == "append4":   # and what was written, read back as f32
            moved += rows * (row + dim * 4)
        return {"bytes": int(moved + case["tokens"] * 4 // page + 8 * case["batch"]), "flops": 0}
    if op in ("rotary", "write", "step"):
        tokens = case["tokens"] if "tokens" in case else case["batch"]
        rows = case["heads"] + kv_heads
        moved = tokens * (rows * dim * 2 * size("type") + 4)
        if op != "rotary":   # k goes into a cache of 16 bits, and v from its rows
            moved += tokens * (kv_heads * dim * 4 + 4)
        flops = 3 * tokens * rows * case["rotary"]
        if op != "step":
            return {"bytes": moved, "flops": flops}
    top = case["max_len"]
    # lengths spread evenly over [1, max_len], the first at max_len, and one of an attending batch at zero
    n = [top] * case["batch"]
    if case["ragged"]:
        n = [top] + [(2 * i + 1) * top // (2 * max(1, case["batch"] - 1)) + 1 for i in range(case["batch"] - 1)]
    if op == "step":
        seen = sum(n)
        return {"bytes": int(moved + seen * (4 * kv_heads * dim + 4 / page) + case["batch"] * (case["heads"] * dim * size("type") + 16)),
                "flops": flops + 4 * seen * case["heads"] * dim}
    seen = sum(min(x, case["window"] or x) for x in n)
    return {"bytes": int(seen * (2 * kv_heads * row + 4 / page) + case["batch"] * (case["heads"] * dim * (size("q") + size("out")) + 4)),
            "flops": 4 * seen * case["heads"] * dim}


# ---- the definitions -----------------------------------------------------------------------------------------------------------------

def _exact_pages(s):
    """The stack of free pages and the sequences one after another, on the host."""
    page, table, stack = s["case"]["page"], s["table"].tolist(), s["free"].tolist()
    top, lengths, room = int(s["free_count"]), s["lengths"].tolist(), len(s["slots"])
    for b, gone in enumerate(s["released"].tolist() if s["released"] is not None else []):
        if gone:
            for i in reversed(range(-(-lengths[b] // page))):
                stack[top] = table[b][i]
                top += 1
            lengths[b] = 0
    counts = s["counts"].tolist() if s["counts"] is not None else [int(n > 0) for n in lengths]
    offsets, positions, slots = [0], [], []
    for b, n in enumerate(counts):
        for i in range(-(-lengths[b] // page), -(-(lengths[b] + n) // page)):
            top -= 1
            table[b][i] = stack[top]
        for p in range(lengths[b], lengths[b] + n):
            positions.append(p)
            slots.append(table[b][p // page] * page + p % page)
        lengths[b] += n
        offsets.append(offsets[-1] + n)
    over = room - len(slots)
    out = {"table": table, "free": stack, "next_lengths": lengths, "next_free_count": [top], "offsets": offsets, "positions": positions + [0] * over,
           "slots": slots + [FREE] * over}
    return {k: torch.tensor(v, dtype=torch.int32, device="cuda") for k, v in out.items()}


def _value4(codes, blocks, scales):
    """What bits stand for: a sign, two exponent bits and one more (0 is subnormal); block scales of four exponent bits and three more."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    sign, e, m = 1 - 2 * (c // 8), c // 2 % 4, c % 2
    value = sign * torch.where(e > 0, (1 + m / 2) * 2 ** (e - 1), m / 2)
    e, m = (blocks >> 3).double(), (blocks & 7).double()
    scale = torch.where(e > 0, (1 + m / 8) * 2 ** (e - 7), m * 2.0 ** -9) * scales.double().unsqueeze(-1)
    return (value.unflatten(-1, (-1, 16)) * scale.unsqueeze(-1)).flatten(-2)


def _stored4(x):
    """What a 4-bit cache holds of rows x: steps and quotients are rounded to 32 bits by definition."""
    f = lambda t: t.float().double()  # noqa: E731
    x = x.double()
    m = x.abs().amax(-1, keepdim=True)
    scale = f(m / 2688)
    blocks = x.unflatten(-1, (-1, 16))
    b = f(blocks.abs().amax(-1) * f(448 / m.clamp(min=2.0 ** -100))).to(torch.float8_e4m3fn).double()
    step = f(b * scale).unsqueeze(-1)
    y = f(blocks * f(1 / step.clamp(min=2.0 ** -126)))
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    hi = torch.searchsorted(grid, y.abs().contiguous()).clamp(1, 7)
    down, up = y.abs() - grid[hi - 1], grid[hi] - y.abs()
    nearest = torch.where((down < up) | ((down == up) & (hi % 2 == 1)), hi - 1, hi)
    value = torch.copysign(grid[nearest], y) * b.unsqueeze(-1) * scale.unsqueeze(-1)
    return torch.where((m >= 2.0 ** -100).unsqueeze(-1), value, torch.zeros((), dtype=torch.float64, device=x.device)).flatten(-2)


def _turned(x, positions, frequencies, layout, sign):
    """As complex numbers: a pair times the unit number of its angle."""
    r = 2 * len(frequencies)
    unit = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), sign * positions.double().view(-1, 1, 1) * frequencies.double())
    x = x.double().clone()
    first, second = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    z = torch.complex(x[..., first], x[..., second]) * unit
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact(case, seed):
    """The definition in 64 bits, from the same inputs."""
    s = prepare(case, seed)
    op, page = case["op"], case.get("page")
    if op == "pages":
        return _exact_pages(s)
    dim, kv_heads, out = case["dim"], case["kv_heads"], {}
    if op == "rotary":
        return {n + "_out": _turned(s[n], s["positions"], s["frequencies"], case["layout"], -1 if case["backward"] else 1) for n in "qk"}
    lengths = s["lengths"]
    if op == "step":
        out = {n: x for n, x in _exact_pages(s).items() if n in _OUTPUTS["step"]}
        s["table"], s["positions"], s["slots"], lengths = out["table"], out["positions"], out["slots"], out["next_lengths"]
    if op in ("write", "step"):
        q, k = (_turned(s[n], s["positions"], s["frequencies"], case["layout"], 1) for n in "qk")
        at = s["slots"].long()
        for n, x in (("k", k), ("v", s["v"])):
            held = s[n + "_cache"].double()
            held[at // page, :, at % page] = x.double()
            out[n + "_cache"] = s[n + "_cache"] = held
        out["q_out"] = s["q"] = q
        if op == "write":
            return out
    table, rows = s["table"].long(), lengths.tolist()

    def held(name, b, first, end):   # [kv_heads][end - first][dim]: what the cache holds
        at = torch.arange(first, end, device="cuda")
        where = (table[b, at // page], slice(None), at % page)
        if "k_scales" not in s:
            return s[name + "_cache"][where].double().transpose(0, 1)
        codes, blocks = _parts4(s[name + "_cache"], case, s["pages"])
        return _value4(codes[where], blocks[where], s[name + "_scales"][where]).transpose(0, 1)

    if op in ("append4", "read4"):
        begin = s["offsets"].tolist()
        for n in "kv":
            out[n + "_out"] = _stored4(s[n]) if op == "append4" else torch.cat(
                [held(n, b, m - (begin[b + 1] - begin[b]), m).transpose(0, 1) for b, m in enumerate(rows)])
        return out
    q = s["q"].double().view(case["batch"], kv_heads, -1, dim)
    o, lse = torch.zeros_like(q), torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(rows):
        first = max(0, n - case["window"]) if case.get("window") else 0
        if n:
            k, v = (held(name, b, first, n) for name in "kv")
            score = (q[b] @ k.transpose(1, 2)) / math.sqrt(dim)
            lse[b] = torch.logsumexp(score, -1)
            o[b] = torch.softmax(score, -1) @ v
    out["o"] = o.view(case["batch"], case["heads"], dim)
    if s.get("lse") is not None:
        out["lse"] = lse.view(case["batch"], case["heads"])
    return out
