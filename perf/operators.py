"""The serving operators over a paged key-value cache, as timed cases: new tokens written into the pages (`kv_cache_append_v1`),
rows read back (`kv_cache_read_v1`), and one new token a sequence that attends to them (`paged_attention_v1`).

`own` False: their plain form, elementary torch operations in 32 bits.  `own` True: the library's launches, prepared once and
launched per pass as a serving program does.
"""
import math

import torch

own = False

FORMATS = {"bf16": 0, "e4m3": 1, "i8": 2}
TOP = {"e4m3": 448.0, "i8": 127.0}   # the largest code of a row
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # -- one new token a sequence.  A single user's short context: the latency of a launch counts
        {"name": "attend_1x512", "op": "attend", "batch": 1, "heads": 16, "kv_heads": 16, "dim": 64, "max_len": 512, "ragged": False,
         "page": 16, "window": 0, "format": "bf16", "q": "bf16", "out": "f32"},
        #    an ordinary batch of requests of all lengths, one of them not begun yet; four query heads to a key head
        {"name": "attend_64_ragged", "op": "attend", "batch": 64, "heads": 32, "kv_heads": 8, "dim": 128, "max_len": 4096,
         "ragged": True, "page": 16, "window": 0, "format": "bf16", "q": "bf16", "out": "bf16"},
        #    two long documents: eight (sequence, key head) pairs each, far fewer than there are SMs
        {"name": "attend_2x131071", "op": "attend", "batch": 2, "heads": 32, "kv_heads": 8, "dim": 128, "max_len": 131071,
         "ragged": False, "page": 64, "window": 0, "format": "bf16", "q": "bf16", "out": "bf16"},
        #    8-bit caches, for larger batches in the same memory: floating, eight query heads to a key head
        {"name": "attend_e4m3_96_ragged", "op": "attend", "batch": 96, "heads": 32, "kv_heads": 4, "dim": 128, "max_len": 6000,
         "ragged": True, "page": 64, "window": 0, "format": "e4m3", "q": "bf16", "out": "bf16"},
        #    and integer, all query heads on one key head
        {"name": "attend_i8_one_kv_head", "op": "attend", "batch": 40, "heads": 16, "kv_heads": 1, "dim": 128, "max_len": 20000,
         "ragged": True, "page": 32, "window": 0, "format": "i8", "q": "bf16", "out": "f32"},
        #    f32 queries, a head size between the powers of two, pages of 24, the last 777 keys only
        {"name": "attend_window_24x1900", "op": "attend", "batch": 24, "heads": 12, "kv_heads": 12, "dim": 96, "max_len": 1900,
         "ragged": True, "page": 24, "window": 777, "format": "bf16", "q": "f32", "out": "f32"},
        # -- a whole decode step of one attention block: the new token is written, then attends to all before it and itself
        {"name": "step_32x2048", "op": "step", "batch": 32, "heads": 16, "kv_heads": 16, "dim": 64, "max_len": 2048, "ragged": True,
         "page": 16, "window": 0, "format": "bf16", "q": "bf16", "out": "f32"},
        # -- writing alone: the new tokens of a large batch
        {"name": "append_256", "op": "append", "batch": 256, "tokens": 256, "kv_heads": 8, "dim": 128, "before": 400, "page": 16,
         "format": "bf16", "input": "bf16"},
        #    prompts of eight requests into an 8-bit cache, and what it then holds of them
        {"name": "append_e4m3_16384", "op": "append", "batch": 8, "tokens": 16384, "kv_heads": 8, "dim": 128, "before": 0, "page": 64,
         "format": "e4m3", "input": "bf16"},
        #    later pieces of three prompts, f32 rows, ends inside pages
        {"name": "append_i8_5001", "op": "append", "batch": 3, "tokens": 5001, "kv_heads": 12, "dim": 64, "before": 333, "page": 16,
         "format": "i8", "input": "f32"},
        # -- reading back: all of a cache into contiguous rows (a prefix handed to another engine), and a short piece
        {"name": "read_131072", "op": "read", "batch": 16, "tokens": 131072, "kv_heads": 8, "dim": 128, "before": 0, "page": 64,
         "format": "bf16", "output": "bf16"},
        {"name": "read_i8_37", "op": "read", "batch": 2, "tokens": 37, "kv_heads": 16, "dim": 64, "before": 50, "page": 16,
         "format": "i8", "output": "f32"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "step", "append", "read"])
    dim = rng.choice([64, 64, 128, 128, 128, 32, 80, 96, 256])
    page = rng.choice([16, 16, 32, 64, 64, 128, 24, 8, 1])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 12, 16])
    form = rng.choice(["bf16", "e4m3", "i8"])
    if op in ("attend", "step"):
        group = rng.choice([1, 2, 3, 4, 4, 8, 16] if kv_heads < 8 else [1, 1, 2, 4, 4, 5])
        rows = (1 << 27) // (kv_heads * dim)
        batch = _log(rng, 1, 256)
        max_len = _log(rng, 1, max(1, min(131072, rows // batch)))
        window = rng.choice([0, 0, 0, _log(rng, 1, max(2, max_len))])
        return {"op": op, "batch": batch, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "max_len": max_len,
                "ragged": rng.random() < 0.7, "page": page, "window": window, "format": "bf16" if op == "step" else form,
                "q": rng.choice(["bf16", "bf16", "f32"]), "out": rng.choice(["bf16", "f32"])}
    batch = _log(rng, 1, 256)
    tokens = batch + _log(rng, 1, max(2, min(1 << 17, (1 << (25 if op == "append" else 26)) // (kv_heads * dim) - batch)))
    case = {"op": op, "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "before": rng.choice([0, 0, _log(rng, 1, 500)]),
            "page": page, "format": form}
    case["input" if op == "append" else "output"] = rng.choice(["bf16", "f32"])
    return case


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _quantised(x, form):
    """Codes and scales of f32 rows: scale = largest magnitude / largest code, code = the rounded quotient."""
    scale = x.abs().amax(-1) / torch.full((), TOP[form], device=x.device)   # (by a plain number it would be a product)
    y = torch.where(scale.unsqueeze(-1) > 0, x / scale.unsqueeze(-1), torch.zeros((), device=x.device))
    code = y.to(torch.float8_e4m3fn).view(torch.uint8) if form == "e4m3" else torch.round(y).to(torch.int8)
    return code, scale


def _widened(code, form):
    return code.view(torch.float8_e4m3fn).float() if form == "e4m3" else code.float()


def _lengths(g, case):
    """Cached tokens of each sequence, the new one included."""
    batch, top = case["batch"], case["max_len"]
    if not case["ragged"]:
        return torch.full((batch,), top, dtype=torch.int32, device="cuda")
    n = torch.randint(1, top + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = top
    if batch > 2 and case["op"] == "attend":
        n[1] = 0   # a slot of the batch without a request
    return n


def _pieces(g, case):
    """How the new tokens fall on the sequences: offsets of their rows, and each sequence's length with them."""
    batch, tokens = case["batch"], case["tokens"]
    if tokens == batch:
        n = torch.ones(batch, dtype=torch.int64, device="cuda")
    else:
        cuts = torch.sort(torch.randint(0, tokens + 1, (batch - 1,), generator=g, device="cuda")).values
        ends = torch.cat([cuts, torch.tensor([tokens], device="cuda")])
        n = torch.diff(ends, prepend=torch.zeros(1, dtype=ends.dtype, device="cuda"))
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), n.cumsum(0)]).to(torch.int32)
    before = torch.randint(0, case["before"] + 1, (batch,), generator=g, device="cuda")
    return offsets, (n + before).to(torch.int32)


def _cache(g, case, lengths):
    """Pages in no order, a sequence's table of them, and what an earlier life of the cache left in every slot."""
    page, kv_heads, dim, form = case["page"], case["kv_heads"], case["dim"], case["format"]
    if "max_len" in case:   # room for every sequence at its longest
        width = -(-case["max_len"] // page)
        pages = case["batch"] * width
    else:
        width = -(-(case["tokens"] + case["before"]) // page)
        pages = (case["tokens"] + case["batch"] * case["before"]) // page + case["batch"]
    used = (lengths.long() + page - 1) // page
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda") < used.unsqueeze(1)] = order[:int(used.sum())]
    state = {"table": table, "width": width, "pages": pages}
    # some channels of the keys are several times as large as the others
    spread = torch.exp(0.5 * torch.randn(dim, generator=g, device="cuda"))
    for name, by in (("k", spread), ("v", 1.0)):
        shape = (pages, kv_heads, page, dim)
        if form == "bf16":
            state[name + "_cache"] = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        else:
            state[name + "_cache"] = torch.empty(shape, dtype=torch.uint8 if form == "e4m3" else torch.int8, device="cuda")
            state[name + "_scales"] = torch.empty(shape[:3], device="cuda")
        step = max(1, (1 << 26) // (kv_heads * page * dim))
        for at in range(0, pages, step):
            x = _normal(g, (min(step, pages - at),) + shape[1:], torch.float32) * by
            if form == "bf16":
                state[name + "_cache"][at:at + step] = x.to(torch.bfloat16)
            else:
                state[name + "_cache"][at:at + step], state[name + "_scales"][at:at + step] = _quantised(x, form)
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, kv_heads, dim = case["op"], case["kv_heads"], case["dim"]
    if op in ("attend", "step"):
        lengths = _lengths(g, case)
        s = _cache(g, case, lengths)
        s["lengths"], s["offsets"] = lengths, None
        s["q"] = _normal(g, (case["batch"], case["heads"], dim), DTYPES[case["q"]])
        s["o"] = torch.zeros(case["batch"], case["heads"], dim, dtype=DTYPES[case["out"]], device="cuda")
        s["lse"] = torch.zeros(case["batch"], case["heads"], device="cuda") if case["out"] == "f32" else None
        if op == "step":
            s["k"], s["v"] = (_normal(g, (case["batch"], kv_heads, dim), torch.bfloat16) for _ in range(2))
    else:
        offsets, lengths = _pieces(g, case)
        s = _cache(g, case, lengths)
        s["lengths"], s["offsets"] = lengths, None if op == "append" and case["tokens"] == case["batch"] else offsets
        shape = (case["tokens"], kv_heads, dim)
        if op == "append":
            s["k"], s["v"] = (_normal(g, shape, DTYPES[case["input"]]) for _ in range(2))
        if op == "read" or case["format"] != "bf16":   # rows read back: f32 ones show every bit of an 8-bit cache
            s["k_out"], s["v_out"] = (torch.zeros(shape, dtype=DTYPES[case.get("output", "f32")], device="cuda") for _ in range(2))
    s["case"] = case
    if own:
        s["launches"], s["stream"] = _prepared(s)
    return s


_ctx = None


def _prepared(s):
    """The library's launches of one pass, in order."""
    import fe2o3_b200 as fe
    global _ctx
    if _ctx is None:
        ctx = fe.GpuContext(torch.cuda.current_device())
        _ctx = (ctx, ctx.default_stream())
    ctx, stream = _ctx
    case = s["case"]
    kv_heads, dim = case["kv_heads"], case["dim"]
    cache = {n: s[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales") if n in s}
    cache.update(page_table=s["table"], lengths=s["lengths"], batch=case["batch"], kv_heads=kv_heads, dim=dim,
                 page_size=case["page"], table_width=s["width"], format=FORMATS[case["format"]])
    rows = dict(k_token_stride=kv_heads * dim, k_head_stride=dim, v_token_stride=kv_heads * dim, v_head_stride=dim)
    code = {torch.float32: fe.DTYPE_F32, torch.bfloat16: fe.DTYPE_BF16}
    launches = []
    if "k" in s:
        launches.append(fe.prepare(ctx, "kv_cache_append_v1", k=s["k"], v=s["v"], token_offsets=s["offsets"],
                                   tokens=case.get("tokens", case["batch"]), input_dtype=code[s["k"].dtype], **rows, **cache))
    if "k_out" in s:
        launches.append(fe.prepare(ctx, "kv_cache_read_v1", k=s["k_out"], v=s["v_out"], token_offsets=s["offsets"],
                                   tokens=case["tokens"], output_dtype=code[s["k_out"].dtype], **rows, **cache))
    if "q" in s:
        launches.append(fe.prepare(ctx, "paged_attention_v1", q=s["q"], output=s["o"], lse=s["lse"], heads=case["heads"],
                                   q_stride=case["heads"] * dim, q_head_stride=dim, scale=1 / math.sqrt(dim), window=case["window"],
                                   q_dtype=code[s["q"].dtype], output_dtype=code[s["o"].dtype], **cache))
    return launches, stream


def _slots(s):
    """(page, slot) of every new token's row."""
    case, lengths = s["case"], s["lengths"].long()
    if s["offsets"] is None:
        seq = torch.arange(case["batch"], device="cuda")
        position = lengths - 1
    else:
        offsets = s["offsets"].long()
        t = torch.arange(case["tokens"], device="cuda")
        seq = torch.searchsorted(offsets, t, right=True) - 1
        position = lengths[seq] - offsets[seq + 1] + t
    return s["table"].long()[seq, position // case["page"]], position % case["page"]


def _plain_append(s):
    form = s["case"]["format"]
    page, slot = _slots(s)
    for name in ("k", "v"):
        if form == "bf16":
            s[name + "_cache"][page, :, slot] = s[name].to(torch.bfloat16)
        else:
            s[name + "_cache"][page, :, slot], s[name + "_scales"][page, :, slot] = _quantised(s[name].float(), form)


def _plain_rows(s, name, page, slot):
    """f32 rows of one side of the cache."""
    form = s["case"]["format"]
    x = s[name + "_cache"][page, :, slot]
    return x.float() if form == "bf16" else _widened(x, form) * s[name + "_scales"][page, :, slot].unsqueeze(-1)


def _plain_attend(s):
    case = s["case"]
    batch, kv_heads, page, dim, form = case["batch"], case["kv_heads"], case["page"], case["dim"], case["format"]
    table = s["table"].long().clamp(min=0)

    def gathered(name):   # [batch][kv_heads][positions][dim]
        x = s[name + "_cache"][table].transpose(1, 2)
        x = x.float() if form == "bf16" else _widened(x, form) * s[name + "_scales"][table].transpose(1, 2).unsqueeze(-1)
        return x.reshape(batch, kv_heads, s["width"] * page, dim)

    q = s["q"].float().view(batch, kv_heads, case["heads"] // kv_heads, dim)
    scores = q @ gathered("k").transpose(2, 3) * (1 / math.sqrt(dim))
    at, n = torch.arange(s["width"] * page, device="cuda"), s["lengths"].long().view(batch, 1, 1, 1)
    keep = at < n
    if case["window"]:
        keep = keep & (at >= n - case["window"])
    scores = torch.where(keep, scores, torch.full((), -math.inf, device="cuda"))
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = (p @ gathered("v")) / torch.where(total > 0, total, torch.ones((), device="cuda"))
    lse = torch.where(total > 0, top + torch.log(total), torch.full((), -math.inf, device="cuda"))
    return o.view(batch, case["heads"], dim).to(s["o"].dtype), lse.view(batch, case["heads"])


def run(state):
    s, out = state, {}
    if own:
        for launch in s["launches"]:
            launch.launch(s["stream"])
        if "q" in s:
            out["o"] = s["o"]
            if s["lse"] is not None:
                out["lse"] = s["lse"]
        if "k_out" in s:
            out["k"], out["v"] = s["k_out"], s["v_out"]
    else:
        if "k" in s:
            _plain_append(s)
        if "q" in s:
            out["o"], lse = _plain_attend(s)
            if s["lse"] is not None:
                out["lse"] = lse
        if "k_out" in s:
            page, slot = _slots(s)
            out["k"], out["v"] = (_plain_rows(s, name, page, slot).to(s[name + "_out"].dtype) for name in ("k", "v"))
    if "k" in s and s["case"]["format"] == "bf16":   # the whole cache, as it is after the write
        out["k_cache"], out["v_cache"] = s["k_cache"], s["v_cache"]
    return out


def work(case):
    kv_heads, dim, page, form = case["kv_heads"], case["dim"], case["page"], case["format"]
    row = dim * (2 if form == "bf16" else 1) + (0 if form == "bf16" else 4)   # of one side, with its scale
    size = lambda name: 4 if case[name] == "f32" else 2  # noqa: E731
    if case["op"] in ("append", "read"):
        rows = 2 * case["tokens"] * kv_heads
        moved = rows * (row + dim * size("input" if case["op"] == "append" else "output"))
        if case["op"] == "append" and form != "bf16":   # and what was written, read back as f32
            moved += rows * (row + dim * 4)
        return {"bytes": moved + case["tokens"] * 4 // page + 8 * case["batch"], "flops": 0}
    top = case["max_len"]
    # lengths spread evenly over [1, max_len], the first at max_len, and one of an attending batch at zero
    n = [top] * case["batch"]
    if case["ragged"]:
        n = [top] + [(2 * i + 1) * top // (2 * max(1, case["batch"] - 1)) + 1 for i in range(case["batch"] - 1)]
    seen = sum(min(x, case["window"] or x) for x in n)
    moved = seen * (2 * kv_heads * row + 4 / page) + case["batch"] * (case["heads"] * dim * (size("q") + size("out")) + 4)
    if case["op"] == "step":
        moved += case["batch"] * kv_heads * 4 * row
    return {"bytes": moved, "flops": 4 * seen * case["heads"] * dim}


def exact(case, seed):
    """The definition, sequence by sequence in 64 bits, from the same inputs."""
    s = prepare(case, seed)
    form, page, dim = case["format"], case["page"], case["dim"]
    lengths, table = s["lengths"].tolist(), s["table"].long()

    def held(name, b, first, end):   # [kv_heads][end - first][dim]: what the codes stand for
        at = torch.arange(first, end, device="cuda")
        where = (table[b, at // page], slice(None), at % page)
        x = s[name + "_cache"][where]
        x = x.view(torch.float8_e4m3fn).double() if form == "e4m3" else x.double()
        if form != "bf16":
            x = x * s[name + "_scales"][where].double().unsqueeze(-1)
        return x.transpose(0, 1)

    def stored(x):   # what a cache of this format holds of rows x; quotients are rounded to 32 bits by definition
        x = x.double()
        if form == "bf16":
            return x.bfloat16().double()
        scale = (x.abs().amax(-1, keepdim=True) / TOP[form]).float().double()
        y = (x / scale).float()
        y = y.to(torch.float8_e4m3fn).double() if form == "e4m3" else y.double().round()
        return torch.where(scale > 0, y * scale, torch.zeros((), dtype=torch.float64, device="cuda"))

    out = {}
    if "k" in s and form == "bf16":
        for name in ("k", "v"):
            x = s[name + "_cache"].clone()
            begin = s["offsets"].tolist() if s["offsets"] is not None else list(range(case["batch"] + 1))
            for b, n in enumerate(lengths):
                at = torch.arange(n - (begin[b + 1] - begin[b]), n, device="cuda")
                x[table[b, at // page], :, at % page] = s[name][begin[b]:begin[b + 1]].bfloat16()
            s[name + "_cache"] = x
            out[name + "_cache"] = x.double()
    if "k_out" in s:
        for name in ("k", "v"):
            if case["op"] == "append":
                out[name] = stored(s[name])
                continue
            begin = s["offsets"].tolist()
            out[name] = torch.cat([held(name, b, n - (begin[b + 1] - begin[b]), n).transpose(0, 1) for b, n in enumerate(lengths)])
    if "q" in s:
        q = s["q"].double().view(case["batch"], case["kv_heads"], -1, dim)
        o, lse = torch.zeros_like(q), torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lengths):
            first = max(0, n - case["window"]) if case["window"] else 0
            if n:
                k, v = (held(name, b, first, n) for name in ("k", "v"))
                score = (q[b] @ k.transpose(1, 2)) / math.sqrt(dim)
                lse[b] = torch.logsumexp(score, -1)
                o[b] = torch.softmax(score, -1) @ v
        out["o"] = o.view(case["batch"], case["heads"], dim)
        if s["lse"] is not None:
            out["lse"] = lse.view(case["batch"], case["heads"])
    return out
