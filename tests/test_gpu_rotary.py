"""Rotary positions on the GPU against 64 bits, forward and backward, and rotated rows written into the key-value cache, bit for bit."""
import math

import numpy as np
import pytest

from test_gpu_kv_cache import CODE, Cache, from_bf16, gpu, rows_in, to_bf16  # noqa: F401  (gpu is a fixture)
from test_gpu_kv_e2m1 import Four

pytestmark = pytest.mark.gpu
f32 = np.float32
LAYOUTS = {"half": 0, "interleaved": 1}


def frequencies(r, base=10000.0):
    return (base ** (-np.arange(0, r, 2) / max(r, 1))).astype(f32)


def turned64(x, positions, freq, layout, scale=1.0, backward=False):
    """Rows [tokens][heads][dim] in 64 bits; the angles' whole turns are taken off in integers (positions below 2^31, frequencies f32)."""
    r = 2 * len(freq)
    angle = np.zeros((len(positions), len(freq)))
    for i, p in enumerate(positions):
        for j, f in enumerate(freq):
            n, d = float(f).as_integer_ratio()
            turns = (int(p) * n * INVERSE_2PI // d) % (1 << 200)
            angle[i, j] = turns / (1 << 200) * 2 * math.pi
    c, s = scale * np.cos(angle)[:, None], scale * np.sin(angle)[:, None] * (-1 if backward else 1)
    x = x.astype(np.float64).copy()
    first, second = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    a, b = x[..., first].copy(), x[..., second].copy()
    x[..., first], x[..., second] = a * c - b * s, a * s + b * c
    return x


def _inverse_2pi():
    """2^200 / (2 pi), by Machin's formula in integers."""
    one = 1 << 460

    def atan_inverse(n):
        term = total = one // n
        k = 1
        while term:
            term //= -n * n
            k += 2
            total += term // k
        return total
    pi = 4 * (4 * atan_inverse(5) - atan_inverse(239))
    return (one << 200) // (2 * pi)


INVERSE_2PI = _inverse_2pi()


def check(got, want, x, freq, layout, dtype, scale=1.0):
    """|o - e| <= 2^-21 |s| (|a| + |b|) of the pair: sine and cosine are off by 2^-23 at most (sincospif's 2 units of the last place at
    values up to 1, and their share of the angle's rounding, 2^-24), scaled by 2^-24, and two products and a sum of f32 add 2^-23; a bf16 output is off by
    half a step more, 2^-8 of it."""
    r = 2 * len(freq)
    first, second = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    pair = np.abs(x[..., first]) + np.abs(x[..., second])
    bound = np.zeros(want.shape)
    bound[..., first] = bound[..., second] = 2.0 ** -21 * abs(scale) * pair
    if dtype == "bf16":
        bound[..., :r] += 2.0 ** -8 * np.abs(want[..., :r])
    err = np.abs(got - want)
    assert (err <= bound).all(), (float(err.max()), float((err / np.maximum(bound, 1e-30)).max()))


def packed(heads, kv_heads, dim, *names):
    return {k: v for n in names for k, v in ((n + "_token_stride", (heads if n[0] == "q" else kv_heads) * dim), (n + "_head_stride", dim))}


def launch(gpu, op, **kw):  # noqa: F811
    fe, torch, ctx, stream = gpu
    p = fe.prepare(ctx, op, **kw)
    try:
        p.launch_and_wait(stream, 20000)
    finally:
        p.destroy()


def rotate(gpu, q, k, positions, freq, layout, backward=False, scale=1.0, out=None):  # noqa: F811
    torch = gpu[1]
    (T, H, D), KH = q.shape, 0 if k is None else k.shape[1]
    qo, ko = out if out else (torch.full_like(q, 7.0), None if k is None else torch.full_like(k, 7.0))
    launch(gpu, "rotary_v1", q=q, k=k, positions=positions, frequencies=torch.from_numpy(freq).cuda(), q_output=qo, k_output=ko, tokens=T, heads=H,
           kv_heads=KH, dim=D, rotary_dim=2 * len(freq), layout=LAYOUTS[layout], dtype=int(q.dtype == torch.bfloat16), backward=int(backward), scale=scale,
           **packed(H, KH, D, "q", "k", "q_output", "k_output"))
    return qo, ko


def up32(torch, a):
    return torch.from_numpy(np.asarray(a, np.uint32).view(np.int32)).cuda()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,rotary", [(16, 16), (16, 2), (32, 32), (48, 20), (64, 64), (64, 32), (80, 20), (80, 80), (96, 24), (112, 48), (128, 128), (128, 64),
                                        (128, 126), (256, 256), (256, 64), (208, 0), (240, 16)])
def test_rows_against_64_bits(gpu, layout, dtype, dim, rotary):  # noqa: F811
    torch = gpu[1]
    T, H, KH = 37, 5, 2
    rng = np.random.default_rng(dim + rotary)
    (q, qv), (k, kv) = (rows_in(torch, rng.normal(size=(T, h, dim)), dtype) for h in (H, KH))
    at = rng.integers(0, 5000, T)
    at[:3] = 0, 1, 131071
    freq = frequencies(rotary)
    for backward, scale in ((False, 1.0), (True, 1.0), (False, 1.25)):
        got = rotate(gpu, q, k, up32(torch, at), freq, layout, backward, scale)
        for o, x in zip(got, (qv, kv)):
            check(o.float().cpu().numpy(), turned64(x, at, freq, layout, scale, backward), x, freq, layout, dtype, scale)
            rest = o[..., rotary:]
            assert torch.equal(rest, (q if x is qv else k)[..., rotary:])


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 0), (1, 128, 8), (3, 0, 2), (148, 16, 16), (149, 7, 1), (1000, 3, 3), (20011, 2, 1), (15000, 1, 0), (2, 1000, 3)])
def test_numbers_of_rows(gpu, tokens, heads, kv_heads):  # noqa: F811
    """One token to many, by one launch; without positions a row's number is its position."""
    torch = gpu[1]
    rng = np.random.default_rng(tokens)
    q, k = (torch.randn(tokens, h, 64, device="cuda").bfloat16() if h else None for h in (heads, kv_heads))
    freq = frequencies(64)
    if q is None:
        q = torch.zeros(tokens, 0, 64, device="cuda", dtype=torch.bfloat16)
    for layout in LAYOUTS:
        got = rotate(gpu, q, k, None, freq, layout)
        some = np.unique(np.concatenate([rng.integers(0, tokens, 20), [0, tokens - 1]]))
        for o, x in zip(got, (q, k)):
            if x is None or x.shape[1] == 0:
                continue
            xv = x[some].float().cpu().numpy()
            check(o[some].float().cpu().numpy(), turned64(xv, some, freq, layout), xv, freq, layout, "bf16")
            assert float((o.float().norm() / x.float().norm() - 1).abs()) < 1e-3   # (every row: lengths stay)
            assert float((o.float().norm(dim=-1) - x.float().norm(dim=-1)).abs().max() / 8) < 2.0 ** -8


def test_far_positions(gpu):  # noqa: F811
    """Up to the last one of 31 bits, and beyond: the angle has 32-bit accuracy all the same."""
    torch = gpu[1]
    at = np.array([2 ** 20 + 1, 2 ** 24 + 1, 2 ** 27 - 3, 2 ** 31 - 1, 2 ** 32 - 1], np.uint32)
    rng = np.random.default_rng(1)
    x, xv = rows_in(torch, rng.normal(size=(5, 2, 64)), "f32")
    for freq in (frequencies(64), frequencies(64, 500000.0), np.linspace(0.9, 1.1, 32).astype(f32), np.full(32, np.pi, f32)):
        got, _ = rotate(gpu, x, None, up32(torch, at), freq, "half")
        check(got.cpu().numpy(), turned64(xv, at, freq, "half"), xv, freq, "half", "f32")


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dim,rotary", [(64, 64), (80, 20), (96, 72)])
def test_the_gradient_is_the_transpose(gpu, layout, dim, rotary):  # noqa: F811
    """<g, R x> = <R^T g, x>, and R^T against differences: the operator is linear, so a difference of any size is the derivative."""
    torch = gpu[1]
    T, H = 9, 3
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x, w, e = (torch.randn(T, H, dim, generator=g, device="cuda") for _ in range(3))
    at, freq = up32(torch, np.arange(T) * 1000 + 7), frequencies(rotary)
    y, back = rotate(gpu, x, None, at, freq, layout, scale=1.5)[0], rotate(gpu, w, None, at, freq, layout, backward=True, scale=1.5)[0]
    size = float(x.norm() * w.norm()) * 1.5
    assert abs(float((y.double() * w.double()).sum() - (back.double() * x.double()).sum())) <= 2.0 ** -20 * size
    moved = rotate(gpu, x + e, None, at, freq, layout, scale=1.5)[0]
    assert abs(float(((moved.double() - y.double()) * w.double()).sum() - (back.double() * e.double()).sum())) <= 2.0 ** -18 * size
    there = rotate(gpu, rotate(gpu, x, None, at, freq, layout)[0], None, at, freq, layout, backward=True)[0]
    assert float((there - x).abs().max()) <= 2.0 ** -20 * float(x.abs().max())


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rotary", [64, 20, 24])
def test_in_place_and_inside_fused_rows(gpu, layout, dtype, rotary):  # noqa: F811
    """q and k turned where they lie, inside rows [q | k | v]; the rest of the rows stays; heads before tokens; starts on odd elements."""
    torch = gpu[1]
    T, H, KH, D = 300, 4, 2, 64
    freq, at = frequencies(rotary), np.arange(T) * 3
    x, xv = rows_in(torch, np.random.default_rng(2).normal(size=(T, (H + 2 * KH) * D)), dtype)
    want = [turned64(v, at, freq, layout) for v in (xv[:, :H * D].reshape(T, H, D), xv[:, H * D:(H + KH) * D].reshape(T, KH, D))]
    ts, eb = (H + 2 * KH) * D, x.element_size()
    q, k = (x.data_ptr(), (T - 1) * ts + H * D), (x.data_ptr() + H * D * eb, (T - 1) * ts + KH * D)
    kw = dict(positions=up32(torch, at), frequencies=torch.from_numpy(freq).cuda(), tokens=T, heads=H, kv_heads=KH, dim=D, rotary_dim=rotary,
              layout=LAYOUTS[layout], dtype=int(dtype == "bf16"), backward=0, scale=1.0)
    strides = {n + s: v for n in ("q", "k", "q_output", "k_output") for s, v in (("_token_stride", ts), ("_head_stride", D))}
    launch(gpu, "rotary_v1", q=q, k=k, q_output=q, k_output=k, **kw, **strides)
    got = x.float().cpu().numpy()
    check(got[:, :H * D].reshape(T, H, D), want[0], xv[:, :H * D].reshape(T, H, D), freq, layout, dtype)
    check(got[:, H * D:(H + KH) * D].reshape(T, KH, D), want[1], xv[:, H * D:(H + KH) * D].reshape(T, KH, D), freq, layout, dtype)
    assert (got[:, (H + KH) * D:] == xv[:, (H + KH) * D:]).all()
    # [heads][tokens][dim], and rows three elements apart that start on an odd one
    for hs, ts, off in ((T * D, D, 0), (D + 3, H * (D + 3), 1)):
        extent = (T - 1) * ts + (H - 1) * hs + D
        at_ = off + np.arange(T)[:, None, None] * ts + np.arange(H)[None, :, None] * hs + np.arange(D)
        x, xv = rows_in(torch, np.random.default_rng(3).normal(size=off + extent + 9), dtype)
        rows = (x.data_ptr() + off * x.element_size(), extent)
        launch(gpu, "rotary_v1", q=rows, q_output=rows, **{**kw, "kv_heads": 0}, q_token_stride=ts, q_head_stride=hs, q_output_token_stride=ts,
               q_output_head_stride=hs)
        got = x.float().cpu().numpy()
        check(got[at_], turned64(xv[at_], at, freq, layout), xv[at_], freq, layout, dtype)
        outside = np.ones(len(got), bool)
        outside[at_] = False
        assert (got[outside] == xv[outside]).all()


def test_infinities_and_nan_stay_in_their_pairs(gpu):  # noqa: F811
    torch = gpu[1]
    x = torch.randn(4, 2, 64, device="cuda")
    x[1, 0, 5], x[2, 1, 40], x[3, 0, 63] = math.inf, math.nan, math.nan
    got = rotate(gpu, x, None, up32(torch, [3, 4, 5, 6]), frequencies(48), "half")[0].cpu().numpy()
    bad = np.zeros(got.shape, bool)
    bad[1, 0, [5, 29]] = bad[2, 1, [16, 40]] = bad[3, 0, 63] = True
    assert (np.isfinite(got) == ~bad).all()
    bits = torch.tensor([0x7f81 + i for i in range(64)], dtype=torch.int16, device="cuda").view(torch.bfloat16).reshape(1, 1, 64)
    got = rotate(gpu, bits, None, up32(torch, [3]), frequencies(32), "half")[0]
    assert torch.equal(got.view(torch.int16)[..., 32:], bits.view(torch.int16)[..., 32:])   # what is not turned stays bit for bit


# ---- into the cache -------------------------------------------------------------------------------------------------

FORMATS = ["bf16", "e4m3", "i8", "e2m1"]


def cache_of(gpu, form, lengths, kv_heads, dim, page, **kw):  # noqa: F811
    return Four(gpu, lengths, kv_heads, dim, page, **kw) if form == "e2m1" else Cache(gpu, form, lengths, kv_heads, dim, page, **kw)


def cache_args(c):
    return {k: v for k, v in c.args().items() if k not in ("page_table", "lengths", "batch", "table_width")}


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,page", [(4, 4, 64, 64, 16), (8, 2, 128, 128, 64), (3, 1, 96, 24, 24), (12, 3, 96, 48, 8), (0, 2, 32, 32, 16),
                                                            (2, 2, 256, 128, 8), (5, 5, 128, 0, 16), (6, 2, 160, 96, 8)])
def test_rotated_rows_in_the_cache(gpu, form, dtype, layout, heads, kv_heads, dim, rotary, page):  # noqa: F811
    """k in f32 as rotary_v1 gives it, then as the cache's rules have it: bit for bit; tokens without a slot are left out."""
    torch = gpu[1]
    new, T = [5, 0, 1, 70, 2], 81
    lengths = [9, 3, 1, 80, 5]
    c = cache_of(gpu, form, lengths, kv_heads, dim, page, seed=dim).to_gpu()
    rng = np.random.default_rng(dim + rotary)
    seq = np.concatenate([np.full(n, b) for b, n in enumerate(new)] + [np.full(T - sum(new), -1)]).astype(int)
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lengths, new)] + [np.zeros(T - sum(new), int)])
    slots = np.full(T, 0xffffffff, np.uint32)
    for t in range(T):
        if seq[t] >= 0:
            slots[t] = c.table[seq[t], pos[t] // page] * page + pos[t] % page
    slots[40] = 0xffffffff                                   # one in the middle too
    seq[40] = -1
    (q, _), (k, _), (v, vv) = (rows_in(torch, rng.normal(size=(T, h, dim)) * np.exp(rng.normal(size=(T, h, 1))), dtype) for h in (heads, kv_heads, kv_heads))
    freq = frequencies(rotary)
    qo = torch.full_like(q, 7.0)
    launch(gpu, "kv_cache_rotary_append_v1", q=q if heads else None, k=k, v=v, positions=up32(torch, pos) if rotary else None, slots=up32(torch, slots),
           frequencies=torch.from_numpy(freq).cuda(), q_output=qo if heads else None, tokens=T, heads=heads, rotary_dim=rotary, layout=LAYOUTS[layout],
           input_dtype=int(dtype == "bf16"), scale=1.25, **packed(heads, kv_heads, dim, "q", "k", "v", "q_output"), **cache_args(c))
    if rotary:
        want_q = rotate(gpu, q, None, up32(torch, pos), freq, layout, scale=1.25)[0]
        want_k = rotate(gpu, k.float(), None, up32(torch, pos), freq, layout, scale=1.25)[0].cpu().numpy()
    else:
        want_q, want_k = q, k.float().cpu().numpy()
    kept = seq >= 0
    assert torch.equal(qo[torch.from_numpy(kept).cuda()], want_q[torch.from_numpy(kept).cuda()])
    assert (qo[torch.from_numpy(~kept).cuda()] == 7).all()
    for t in np.nonzero(kept)[0]:
        c.put(0, seq[t], [pos[t]], want_k[t:t + 1])
        c.put(1, seq[t], [pos[t]], vv[t:t + 1])
    c.assert_same()


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,rotary", [(32, 32), (64, 20), (128, 64), (256, 256)])
def test_queries_and_keys_in_one_warp(gpu, form, dtype, dim, rotary):  # noqa: F811
    """Any number of queries beside any number of keys: rows that are only turned and rows that are quantised meet in a warp, and some tokens are left out."""
    torch = gpu[1]
    rng = np.random.default_rng(dim)
    for heads, kv_heads, T in ((1, 1, 3), (2, 1, 77), (3, 2, 40), (5, 1, 601), (7, 3, 50), (9, 5, 33), (1, 9, 64), (0, 1, 5)):
        c = cache_of(gpu, form, [T], kv_heads, dim, 8, seed=heads).to_gpu()
        pos = np.arange(T)
        slots = (c.table[0, pos // 8].astype(np.int64) * 8 + pos % 8).astype(np.uint32)
        drop = rng.random(T) < 0.2
        slots[drop] = 0xffffffff
        (q, _), (k, _), (v, vv) = (rows_in(torch, rng.normal(size=(T, h, dim)), dtype) for h in (heads, kv_heads, kv_heads))
        qo, freq = torch.full_like(q, 7.0), frequencies(rotary)
        launch(gpu, "kv_cache_rotary_append_v1", q=q if heads else None, k=k, v=v, positions=up32(torch, pos), slots=up32(torch, slots),
               frequencies=torch.from_numpy(freq).cuda(), q_output=qo if heads else None, tokens=T, heads=heads, rotary_dim=rotary, layout=0,
               input_dtype=int(dtype == "bf16"), scale=1.0, **packed(heads, kv_heads, dim, "q", "k", "v", "q_output"), **cache_args(c))
        keep, there = np.nonzero(~drop)[0], torch.from_numpy(~drop).cuda()
        if heads:
            assert torch.equal(qo[there], rotate(gpu, q, None, up32(torch, pos), freq, "half")[0][there]) and (qo[~there] == 7).all()
        if len(keep):
            c.put(0, 0, pos[keep], rotate(gpu, k.float(), None, up32(torch, pos), freq, "half")[0].cpu().numpy()[keep])
            c.put(1, 0, pos[keep], vv[keep])
        c.assert_same()


@pytest.mark.parametrize("form", FORMATS)
def test_many_tokens_and_strided_rows(gpu, form):  # noqa: F811
    """Fused rows [q | k | v] of a long prompt, read as they lie; starts on odd elements."""
    torch = gpu[1]
    T, H, KH, D, page = 5003, 3, 2, 64, 16
    c = cache_of(gpu, form, [T], KH, D, page).to_gpu()
    at = np.arange(T)
    slots = (c.table[0, at // page].astype(np.int64) * page + at % page).astype(np.uint32)
    freq = torch.from_numpy(frequencies(D)).cuda()
    for dtype, off in (("bf16", 0), ("f32", 0), ("bf16", 1), ("f32", 3)):
        ts = (H + 2 * KH) * D + (off and 5)
        x, xv = rows_in(torch, np.random.default_rng(off).normal(size=off + T * ts), dtype)
        eb = x.element_size()
        part = lambda head, n: (x.data_ptr() + (off + head * D) * eb, (T - 1) * ts + n * D)  # noqa: E731
        qo = torch.zeros(T, H, D, device="cuda", dtype=x.dtype)
        strides = {n + s: v for n in "qkv" for s, v in (("_token_stride", ts), ("_head_stride", D))}
        launch(gpu, "kv_cache_rotary_append_v1", q=part(0, H), k=part(H, KH), v=part(H + KH, KH), positions=up32(torch, at), slots=up32(torch, slots),
               frequencies=freq, q_output=qo, tokens=T, heads=H, rotary_dim=D, layout=0, input_dtype=int(dtype == "bf16"), scale=1.0, **strides,
               q_output_token_stride=H * D, q_output_head_stride=D, **cache_args(c))
        rows = torch.from_numpy(xv[off:off + T * ts].reshape(T, ts)[:, :(H + 2 * KH) * D].reshape(T, H + 2 * KH, D).copy()).cuda()
        both = rotate(gpu, rows[:, :H + KH].contiguous(), None, up32(torch, at), frequencies(D), "half")[0]
        assert torch.equal(qo, both[:, :H].to(x.dtype))
        c.put(0, 0, at, both[:, H:].cpu().numpy())
        c.put(1, 0, at, rows[:, H + KH:].cpu().numpy())
        c.assert_same()


def test_slots_outside_the_cache_are_reported_and_left_out(gpu):  # noqa: F811
    fe, torch, ctx, stream = gpu
    for form in FORMATS:
        c = cache_of(gpu, form, [8], 2, 32, 8).to_gpu()
        x = torch.ones(4, 2, 32, device="cuda")
        last = c.pages * 8
        slots = np.array([last, 0xfffffffe, 0xffffffff, c.table[0, 0] * 8 + 3], np.uint32)
        qo = torch.full((4, 2, 32), 7.0, device="cuda")
        with pytest.raises(fe.Fe2o3Error):
            launch(gpu, "kv_cache_rotary_append_v1", q=x, k=x, v=x, positions=up32(torch, [0] * 4), slots=up32(torch, slots),
                   frequencies=torch.from_numpy(frequencies(32)).cuda(), q_output=qo, tokens=4, heads=2, rotary_dim=32, layout=0, input_dtype=0, scale=1.0,
                   **packed(2, 2, 32, "q", "k", "v", "q_output"), **cache_args(c))
        for side in range(2):
            c.put(side, 0, [3], np.ones((1, 2, 32), f32))
        c.assert_same()
        assert (qo[:3] == 7).all() and (qo[3] == 1).all()


def test_infinities_in_rows_of_the_cache(gpu):  # noqa: F811
    """A pair with an infinity makes its row what the cache's format says of one; V's bits stay as they are in bf16."""
    torch = gpu[1]
    for form in FORMATS:
        c = cache_of(gpu, form, [3], 1, 32, 8).to_gpu()
        k = torch.ones(3, 1, 32, device="cuda", dtype=torch.bfloat16)
        k[1, 0, 4] = math.inf
        v = torch.ones(3, 1, 32, device="cuda", dtype=torch.bfloat16)
        if form == "bf16":
            v.view(torch.int16)[2, 0] = 0x7f81
        slots = c.table[0, 0] * 8 + np.arange(3, dtype=np.uint32)
        launch(gpu, "kv_cache_rotary_append_v1", k=k, v=v, positions=up32(torch, [0, 0, 0]), slots=up32(torch, slots),
               frequencies=torch.from_numpy(frequencies(16)).cuda(), tokens=3, heads=0, rotary_dim=16, layout=0, input_dtype=1, scale=1.0,
               **packed(0, 1, 32, "q", "k", "v", "q_output"), **cache_args(c))
        if form == "bf16":
            got = c.d["v_cache"].view(torch.int16)[int(c.table[0, 0]), 0, :3]
            assert (got[2] == 0x7f81).all() and (got[:2] == 0x3f80).all()
            assert not torch.isfinite(c.d["k_cache"].view(torch.bfloat16)[int(c.table[0, 0]), 0, 1, 4])
        else:
            assert torch.isnan(c.d["k_scales"][int(c.table[0, 0]), 0, 1]) and torch.isfinite(c.d["k_scales"][int(c.table[0, 0]), 0, [0, 2]]).all()
