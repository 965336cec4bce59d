"""Whole decode steps on the GPU: pages planned there, rotary positions, caches of every format, attention, as a serving program keeps them."""
import os
import sys

import numpy as np
import pytest

from test_gpu_kv_cache import attention64, check_attention, gpu, rows_in  # noqa: F401  (gpu is a fixture)
from test_gpu_rotary import check, turned64

pytestmark = pytest.mark.gpu
f32 = np.float32
FORMATS = ["bf16", "e4m3", "i8", "e2m1"]


def code(fe, form):
    return {"bf16": fe.KV_BF16, "e4m3": fe.KV_E4M3, "i8": fe.KV_I8, "e2m1": fe.KV_E2M1}[form]


class Held:
    """Rows of a cache, as attention64 asks for them: [sequence][side] -> [positions][kv_heads][dim]."""

    def __init__(self, torch, cache):
        n = read_lengths(cache)
        k, v = (torch.zeros(max(1, int(n.sum())), cache.kv_heads, cache.dim, device="cuda") for _ in range(2))
        cache.read(k, v, n)
        ends = np.concatenate([[0], np.cumsum(n)])
        self.rows = [[x.cpu().numpy()[a:b].astype(np.float64) for x in (k, v)] for a, b in zip(ends, ends[1:])]
        self.lengths, self.kv_heads, self.dim = n, cache.kv_heads, cache.dim

    def get(self, side, b, positions):
        return self.rows[b][side][positions]


def read_lengths(cache):
    return cache.device_lengths.to_host_vec(cache.stream).astype(np.int64)


def near(form, got, want):
    """Rows as a cache of this format holds them: off by half a step of the code at the row's (4 bits: the block's) largest magnitude, twice that for
    its scale's own rounding, and 2^-20 of it for the rotation's f32."""
    step = {"bf16": 2.0 ** -8, "e4m3": 2.0 ** -4, "i8": 1 / 127, "e2m1": 1.07 / 6}[form]
    if form == "bf16":
        top = np.abs(want)
    else:
        top = np.abs(want).max(-1, keepdims=True) * np.ones_like(want)
    assert (np.abs(got - want) <= step * top + 2.0 ** -20 * np.abs(want).max(-1, keepdims=True)).all()


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scaling", [None, "yarn"])
def test_prompts_and_captured_steps(gpu, form, dtype, scaling):  # noqa: F811
    """Prompts of unlike lengths, one sequence not begun; then steps replayed from one graph, over page ends; one ends and another takes its slot."""
    fe, torch, ctx, stream = gpu
    from fe2o3_b200.kv_cache import DecodeStep, PagedKvCache
    from fe2o3_b200.rotary import Rotary
    B, H, KH, D, page = 4, 8, 2, 64, 16
    rotary = Rotary(ctx, stream, 48, fe.ROTARY_INTERLEAVED if dtype == "f32" else fe.ROTARY_HALF, scaling=scaling, factor=4.0 if scaling else 1.0, trained=100)
    layout, freq = "interleaved" if dtype == "f32" else "half", rotary.frequencies.to_host_vec(stream)
    cache = PagedKvCache(ctx, stream, B, 120, KH, D, page, format=code(fe, form), tokens=200)
    rng = np.random.default_rng(5)

    def prompts(counts, release=None):
        T, before = int(np.sum(counts)), read_lengths(cache)
        (q, qv), (k, kv), (v, vv) = (rows_in(torch, rng.normal(size=(T, h, D)), dtype) for h in (H, KH, KH))
        turned = torch.zeros_like(q)
        cache.extend(counts, release)
        cache.append(k, v, q=q, q_out=turned, heads=H, rotary=rotary)
        stream.synchronize()
        first = np.where(release, 0, before) if release is not None else before
        at = np.concatenate([np.arange(n, n + m) for n, m in zip(first, counts)])
        check(turned.float().cpu().numpy(), turned64(qv, at, freq, layout, rotary.scale), qv, freq, layout, dtype, rotary.scale)
        held, ends = Held(torch, cache), np.concatenate([[0], np.cumsum(counts)])
        assert (held.lengths == first + counts).all()
        for b in range(B):
            if counts[b]:
                near(form, held.rows[b][0][-counts[b]:], turned64(kv[ends[b]:ends[b + 1]], at[ends[b]:ends[b + 1]], freq, layout, rotary.scale))
                near(form, held.rows[b][1][-counts[b]:], vv[ends[b]:ends[b + 1]].astype(np.float64))

    prompts(np.array([17, 0, 1, 60]))
    q, k, v = (torch.zeros(B, h, D, dtype=torch.bfloat16 if dtype == "bf16" else torch.float32, device="cuda") for h in (H, KH, KH))
    out, lse = torch.zeros(B, H, D, device="cuda"), torch.zeros(B, H, device="cuda")
    step = DecodeStep(cache, q, k, v, out, H, lse=lse, rotary=rotary)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step.run(ctx.wrap_stream(side.cuda_stream))
    for i in range(24):
        if i == 20:
            prompts(np.array([0, 5, 0, 33]), np.array([False, False, False, True]))
        new = [rows_in(torch, rng.normal(size=(B, h, D)), dtype) for h in (H, KH, KH)]
        for t, (x, _) in zip((q, k, v), new):
            t.copy_(x)
        before = read_lengths(cache)
        torch.cuda.synchronize()
        graph.replay() if i % 5 else step.run()
        torch.cuda.synchronize()
        if i % 4 and i < 19:
            continue
        held = Held(torch, cache)
        assert (held.lengths == before + (before > 0)).all()
        turned = torch.as_tensor(step.turned, device="cuda").view(torch.bfloat16 if dtype == "bf16" else torch.float32).view(B, H, D).float().cpu().numpy()
        at_work = before > 0
        check(turned[at_work], turned64(new[0][1][at_work], before[at_work], freq, layout, rotary.scale), new[0][1][at_work], freq, layout, dtype, rotary.scale)
        for b in np.nonzero(at_work)[0]:
            near(form, held.rows[b][0][-1:], turned64(new[1][1][b:b + 1], before[b:b + 1], freq, layout, rotary.scale))
        check_attention(held, turned, out.cpu().numpy(), lse.cpu().numpy(), attention64(held, turned, f32(D ** -0.5)), "f32")
    assert ctx.take_kernel_status(stream) == 0
    step.destroy()
    cache.free()
    rotary.free()


@pytest.mark.parametrize("form", FORMATS)
def test_both_books_give_the_same(gpu, form):  # noqa: F811
    """The host's book and the device's: the same pages, the same caches, bit for bit, and the same outputs."""
    fe, torch, ctx, stream = gpu
    from fe2o3_b200.kv_cache import DecodeStep, PagedKvCache
    B, H, KH, D = 5, 6, 3, 96
    caches = [PagedKvCache(ctx, stream, B, 90, KH, D, 8, pages=40, format=code(fe, form), tokens=t) for t in (None, 150)]
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    q, k1, v1 = (torch.randn(B, h, D, generator=g, device="cuda").bfloat16() for h in (H, KH, KH))
    outs = [torch.zeros(B, H, D, device="cuda") for _ in caches]
    steps = [DecodeStep(c, q, k1, v1, o, H) for c, o in zip(caches, outs)]
    for counts, gone in (([9, 0, 30, 1, 16], None), ([0, 20, 0, 7, 0], None), ([0, 0, 0, 3, 11], [0, 0, 1, 0, 1]), ([2, 2, 2, 2, 2], None)):
        k, v = (torch.randn(sum(counts), KH, D, generator=g, device="cuda").bfloat16() for _ in range(2))
        for c in caches:
            c.extend(counts, gone)
            c.append(k, v)
        for _ in range(3):
            q.copy_(torch.randn(B, H, D, generator=g, device="cuda"))
            torch.cuda.synchronize()
            for s in steps:
                s.run()
        stream.synchronize()
        assert torch.equal(outs[0], outs[1])
        for name in ("k_cache", "v_cache", "k_scales", "v_scales", "device_lengths"):
            a, b = (getattr(c, name) for c in caches)
            assert a is b is None or (a.to_host_vec(stream).view(np.uint8) == b.to_host_vec(stream).view(np.uint8)).all(), name
    for c in caches:
        c.release(0)
    assert (read_lengths(caches[0]) == read_lengths(caches[1])).all() and read_lengths(caches[1])[0] == 0
    assert ctx.take_kernel_status(stream) == 0
    for x in steps + [c for c in caches]:
        x.destroy() if hasattr(x, "destroy") else x.free()


def test_what_does_not_fit_is_reported_and_changes_nothing(gpu):  # noqa: F811
    fe, torch, ctx, stream = gpu
    from fe2o3_b200.kv_cache import DecodeStep, PagedKvCache
    from fe2o3_b200.rotary import Rotary
    ctx.take_kernel_status(stream)
    cache = PagedKvCache(ctx, stream, 2, 64, 1, 32, 8, pages=3, format=fe.KV_E2M1, tokens=40)
    x = torch.ones(40, 1, 32, device="cuda")
    for bad in ([41, 0], [1], [-1, 1]):
        with pytest.raises(ValueError):
            cache.extend(bad)
    cache.extend([8, 16])
    cache.append(x[:24], x[:24])
    assert ctx.take_kernel_status(stream) == 0 and read_lengths(cache).tolist() == [8, 16]
    before = cache.k_cache.to_host_vec(stream)
    y = torch.full((2, 1, 32), 2.0, device="cuda")
    step = DecodeStep(cache, y, y, y, torch.zeros(2, 1, 32, device="cuda"), 1)
    step.run()                                              # no page is left for either
    assert ctx.take_kernel_status(stream) == 7 and read_lengths(cache).tolist() == [8, 16]
    assert (cache.k_cache.to_host_vec(stream) == before).all()
    cache.release(1)
    step.run()
    assert ctx.take_kernel_status(stream) == 0 and read_lengths(cache).tolist() == [9, 0]
    rotary = Rotary(ctx, stream, 32)
    host = PagedKvCache(ctx, stream, 2, 64, 1, 32, 8, format=fe.KV_E2M1)
    with pytest.raises(ValueError):
        DecodeStep(host, y, y, y, y, 1, rotary=rotary)
    host.extend([1, 1])
    with pytest.raises(ValueError):
        host.append(y, y, q=y, q_out=torch.zeros_like(y), heads=1, rotary=rotary)
    with pytest.raises(ValueError):
        cache.append(y, y, q=y, q_out=torch.zeros_like(y), heads=1)
    for one in (dict(q=y), dict(q_out=torch.zeros_like(y))):
        with pytest.raises(ValueError):
            cache.append(y, y, heads=1, rotary=rotary, **one)
    small = PagedKvCache(ctx, stream, 2, 64, 1, 32, 8, pages=3, format=fe.KV_E2M1)
    small.extend([8, 9])
    with pytest.raises(MemoryError):                        # the host's book: what is released comes back with the error
        small.extend([9, 17], [0, 1])
    assert small.table.lengths.tolist() == [8, 9] and read_lengths(small).tolist() == [8, 9] and len(small.table.free) == 0
    small.extend([0, 16], [1, 1])
    assert read_lengths(small).tolist() == [0, 16]
    small.free()
    with pytest.raises(TypeError):
        cache.append(y, y, q=y.bfloat16(), q_out=torch.zeros_like(y), heads=1, rotary=rotary)
    plain = DecodeStep(host, y, y, y, torch.zeros(2, 1, 32, device="cuda"), 1)
    with pytest.raises(ValueError):
        plain.run(ctx.create_stream())
    for c in (step, plain):
        c.destroy()
    cache.free(), host.free(), rotary.free()


def test_rotary_object(gpu):  # noqa: F811
    """In place and not, with and without keys; the way back gives the rows again."""
    fe, torch, ctx, stream = gpu
    from fe2o3_b200.rotary import Rotary
    rotary = Rotary(ctx, stream, 64, base=500000.0, scaling="ntk", factor=2.0)
    freq = rotary.frequencies.to_host_vec(stream)
    (q, qv), (k, kv) = (rows_in(torch, np.random.default_rng(h).normal(size=(30, h, 128)), "f32") for h in (4, 2))
    at = torch.arange(100, 130, dtype=torch.int32, device="cuda")
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    rotary.apply(q, k, at, 4, 2, 128, q_out=qo, k_out=ko)
    for o, x in ((qo, qv), (ko, kv)):
        check(o.cpu().numpy(), turned64(x, np.arange(100, 130), freq, "half"), x, freq, "half", "f32")
    rotary.apply(q, None, at, 4, 0, 128)
    assert torch.equal(q, qo)
    rotary.apply(q, None, at, 4, 0, 128, backward=True)
    assert float((q - torch.from_numpy(qv).cuda()).abs().max()) <= 2.0 ** -19 * np.abs(qv).max()
    with pytest.raises(TypeError):
        rotary.apply(q, k.bfloat16(), at, 4, 2, 128)
    with pytest.raises(ValueError):
        rotary.apply(q[:, ::2], None, at, 2, 0, 128)
    rotary.free()


@pytest.mark.parametrize("more", [["--format", "e2m1"], ["--rotary", "64"], ["--format", "e2m1", "--rotary", "32"], ["--format", "i8", "--rotary", "20"]])
def test_example_runs(gpu, more):  # noqa: F811
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import paged_decode
    off = paged_decode.main(["--sequences", "16", "--prompt", "37", "--steps", "20", "--heads", "4", "--dim", "64"] + more)
    assert off <= 2.0 ** -8   # (bf16 outputs)


@pytest.mark.parametrize("form", ["bf16", "e2m1"])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("captured", [False, True])
def test_a_step_that_does_not_fit_gives_nothing(gpu, form, turned, captured):  # noqa: F811
    """Not the step before it once more, for no sequence, and the next step that fits is right again."""
    fe, torch, ctx, stream = gpu
    from fe2o3_b200.kv_cache import DecodeStep, PagedKvCache
    from fe2o3_b200.rotary import Rotary
    ctx.take_kernel_status(stream)
    B, H, KH, D = 3, 4, 2, 64
    cache = PagedKvCache(ctx, stream, B, 64, KH, D, 8, pages=6, format=code(fe, form), tokens=40)
    rotary = Rotary(ctx, stream, D) if turned else None
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    new = lambda n, h: torch.randn(n, h, D, generator=g, device="cuda")  # noqa: E731
    cache.extend([14, 9, 0])
    cache.append(new(23, KH), new(23, KH))
    q, k, v = new(B, H), new(B, KH), new(B, KH)
    out, lse = (torch.full(s, 7.0, device="cuda") for s in ((B, H, D), (B, H)))
    step = DecodeStep(cache, q, k, v, out, H, lse=lse, rotary=rotary)
    run = step.run
    if captured:
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            step.run(ctx.wrap_stream(side.cuda_stream))
        run = graph.replay

    def stepped():
        for t, h in ((q, H), (k, KH), (v, KH)):
            t.copy_(new(B, h))
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        return out.cpu().numpy(), lse.cpu().numpy()

    def right(o, l):
        held = Held(torch, cache)
        at = torch.as_tensor(step.turned, device="cuda").view(torch.float32).view(B, H, D) if turned else q
        check_attention(held, at.cpu().numpy(), o, l, attention64(held, at.cpu().numpy(), f32(D ** -0.5)), "f32")

    for _ in range(2):                                      # to 16 positions and 11
        right(*stepped())
    assert ctx.take_kernel_status(stream) == 0 and read_lengths(cache).tolist() == [16, 11, 0]
    cache.extend([0, 0, 16])                                # the last two pages
    cache.append(new(16, KH), new(16, KH))
    before = cache.k_cache.to_host_vec(stream)
    for _ in range(2):                                      # the first and the third want a page, the second does not
        o, l = stepped()
        assert (o == 0).all() and (l == -np.inf).all()
        assert ctx.take_kernel_status(stream) == 7 and read_lengths(cache).tolist() == [16, 11, 16]
        assert (cache.k_cache.to_host_vec(stream) == before).all()
    cache.release(2)
    right(*stepped())
    assert ctx.take_kernel_status(stream) == 0 and read_lengths(cache).tolist() == [17, 12, 0]
    step.destroy()
    cache.free()
    if rotary:
        rotary.free()


def near_by_blocks(got, want):
    """4-bit rows block by block.  m: the row's largest magnitude, s = m / 2688; t = 448 m_g / m of a block, b its e4m3 scale.  Codes lie at most 2 apart, so an
    element is off by b s at most where 6 b s reaches the block's largest, which b >= t gives, and by 6 s (t - b) more where it does not.  From t = 2^-6 on b
    is within 2^-4 of t: (1 + 2^-4) / 6 m_g either way.  Below, b is off by 2^-10 at most: m_g / 6 + 2^-10 s, or 6 * 2^-10 s for what is cut off (all of a block
    whose scale becomes 0).  2^-20 for the f32 quotients and products of the definition, and of the row's largest for the rotation's."""
    blocks = lambda x: np.abs(x).reshape(*x.shape[:-1], -1, 16)  # noqa: E731
    m, of_block = np.abs(want).max(-1)[..., None, None], blocks(want).max(-1, keepdims=True)
    t = 448 * of_block / np.maximum(m, 1e-300)
    bound = np.where(t >= 2.0 ** -6, 1.0625 / 6 * of_block, np.maximum(of_block / 6 + 2.0 ** -10 * m / 2688, 2.0 ** -10 * m / 448))
    assert (blocks(got - want) <= bound * (1 + 2.0 ** -20) + 2.0 ** -20 * m).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim,rotary_dim", [(64, 64), (128, 20), (96, 0)])
def test_four_bit_rows_block_by_block(gpu, dtype, dim, rotary_dim):  # noqa: F811
    """Blocks far below the row's largest, down to such as are lost, through a prompt and a step; a block of another size than its own is noticed."""
    fe, torch, ctx, stream = gpu
    from fe2o3_b200.kv_cache import DecodeStep, PagedKvCache
    from fe2o3_b200.rotary import Rotary
    B, H, KH, T = 2, 2, 2, 70
    rng = np.random.default_rng(dim)
    cache, rotary = PagedKvCache(ctx, stream, B, T + 1, KH, dim, 16, format=fe.KV_E2M1, tokens=B * T), Rotary(ctx, stream, rotary_dim)
    freq = rotary.frequencies.to_host_vec(stream) if rotary_dim else np.zeros(0, f32)

    def rows(n):
        of_block = 2.0 ** -rng.integers(0, 20, (n, KH, dim // 16))
        of_block[..., 0] = 1
        return rows_in(torch, rng.normal(size=(n, KH, dim)) * of_block.repeat(16, -1), dtype)
    (k, kv), (v, vv), (k1, k1v), (v1, v1v) = rows(B * T), rows(B * T), rows(B), rows(B)
    cache.extend([T, T])
    cache.append(k, v, rotary=rotary)
    step = DecodeStep(cache, torch.zeros(B, H, dim, dtype=k.dtype, device="cuda"), k1, v1, torch.zeros(B, H, dim, device="cuda"), H, rotary=rotary)
    step.run()
    held, at = Held(torch, cache), np.arange(T + 1)
    for b in range(B):
        part = slice(b * T, (b + 1) * T)
        want_k = turned64(np.concatenate([kv[part], k1v[b:b + 1]]), at, freq, "half")
        want_v = np.concatenate([vv[part], v1v[b:b + 1]]).astype(np.float64)
        near_by_blocks(held.rows[b][0], want_k)
        near_by_blocks(held.rows[b][1], want_v)
        # the smallest block of a row that is not lost, twice as large
        wrong, size = held.rows[b][1].copy(), np.abs(want_v).reshape(T + 1, KH, -1, 16).max(-1)
        worst = np.unravel_index(np.argmin(np.where(size * 448 >= 2.0 ** -6 * size.max(-1, keepdims=True), size / size.max(-1, keepdims=True), np.inf)), size.shape)
        wrong.reshape(T + 1, KH, -1, 16)[worst] *= 2
        with pytest.raises(AssertionError):
            near_by_blocks(wrong, want_v)
    assert ctx.take_kernel_status(stream) == 0
    step.destroy()
    cache.free()
    rotary.free()
