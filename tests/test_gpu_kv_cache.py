"""The paged key-value cache on the GPU: what is written into the pages, what is read back, and the attention of one new
token over them, against plain implementations in 64 bits (quantisation: the same f32 quotients, bit for bit).

Every slot of a cache that no test row was written to holds NaN, so a kernel that lets one of them into a result shows it.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

FORMATS = ["bf16", "e4m3", "i8"]
CODE = {"bf16": 0, "e4m3": 1, "i8": 2}
TOP = {"e4m3": 448.0, "i8": 127.0}


@pytest.fixture(scope="module")
def gpu():
    import torch
    import fe2o3_b200 as fe
    ctx = fe.GpuContext(0)
    return fe, torch, ctx, ctx.default_stream()


# ---- the format's rules, in numpy -------------------------------------------------------------------------------

def e4m3_values():
    """The value of every code: sign, four exponent bits (bias 7), three mantissa bits; 0x7f is NaN."""
    v = np.zeros(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v[c] = np.nan if c & 127 == 127 else (-1) ** (c >> 7) * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return v


E4M3 = e4m3_values()


def nearest_e4m3(y):
    """Codes of the nearest values, ties to the even code."""
    grid, a = E4M3[:127], np.abs(y.astype(np.float64))
    hi = np.clip(np.searchsorted(grid, a), 1, 126)
    lo = hi - 1
    down, up = a - grid[lo], grid[hi] - a
    c = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    return c | (np.signbit(y).astype(np.uint8) << 7)


def to_bf16(x):
    b = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7fff + (b >> 16 & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (np.asarray(b).astype(np.uint32) << 16).view(np.float32)


def quantised(x, form):
    """Codes (bytes) and scales of f32 rows."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1)
    with np.errstate(all="ignore"):
        scale = np.abs(x).max(-1) / np.float32(TOP[form])
        y = np.where(scale[..., None] > 0, x / scale[..., None], np.float32(0)).astype(np.float32)
        y[bad] = 0
        code = nearest_e4m3(y) if form == "e4m3" else np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
    return code, np.where(bad, np.float32(np.nan), scale).astype(np.float32)


def values_of(code, scale, form):
    """f64 values that stored rows stand for (scale None: bf16)."""
    if form == "bf16":
        return from_bf16(code).astype(np.float64)
    v = E4M3[code] if form == "e4m3" else code.view(np.int8).astype(np.float64)
    return v * scale[..., None].astype(np.float64)


class Cache:
    """Pages in no order with NaN in every slot; numpy holds what the GPU should hold."""

    def __init__(self, gpu, form, lengths, kv_heads, dim, page, seed=0, spare=3, width=None):
        self.fe, self.torch, self.ctx, self.stream = gpu
        self.form, self.kv_heads, self.dim, self.page = form, kv_heads, dim, page
        self.lengths = np.asarray(lengths, np.int64)
        rng = np.random.default_rng(seed)
        used = -(-self.lengths // page)
        self.width = max(1, int(used.max(initial=1)) + 1) if width is None else width
        self.pages = int(used.sum()) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(lengths), self.width), 0xffffffff, np.uint32)
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (self.pages, kv_heads, page, dim)
        fill, dt = (0x7fff, np.uint16) if form == "bf16" else (0x7f, np.uint8)
        self.code = [np.full(shape, fill, dt) for _ in range(2)]
        self.scale = [np.full(shape[:3], np.nan, np.float32) for _ in range(2)]

    def up(self, a):
        a = np.ascontiguousarray(a)
        signed = {np.dtype(np.uint32): np.int32, np.dtype(np.uint16): np.int16}.get(a.dtype)
        return self.torch.from_numpy(a.view(signed) if signed else a).cuda()

    def to_gpu(self):
        self.d = {"k_cache": self.up(self.code[0]), "v_cache": self.up(self.code[1]), "page_table": self.up(self.table),
                  "lengths": self.up(self.lengths.astype(np.uint32))}
        if self.form != "bf16":
            self.d.update(k_scales=self.up(self.scale[0]), v_scales=self.up(self.scale[1]))
        return self

    def args(self):
        return dict(self.d, batch=len(self.lengths), kv_heads=self.kv_heads, dim=self.dim, page_size=self.page,
                    table_width=self.width, format=CODE[self.form])

    def where(self, b, positions):
        positions = np.asarray(positions, np.int64)
        return self.table[b, positions // self.page].astype(np.int64), positions % self.page

    def put(self, side, b, positions, rows):
        """rows [n][kv_heads][dim] f32 into numpy's cache."""
        p, s = self.where(b, positions)
        if self.form == "bf16":
            self.code[side][p, :, s] = to_bf16(rows)
        else:
            self.code[side][p, :, s], self.scale[side][p, :, s] = quantised(rows, self.form)

    def get(self, side, b, positions):
        p, s = self.where(b, positions)
        return values_of(self.code[side][p, :, s], self.scale[side][p, :, s], self.form)

    def assert_same(self):
        """The GPU's cache is numpy's, every slot of it."""
        for i, n in enumerate("kv"):
            got = self.d[n + "_cache"].cpu().numpy().view(self.code[i].dtype)
            assert (got == self.code[i]).all(), (n, int((got != self.code[i]).sum()))
            if self.form != "bf16":
                got = self.d[n + "_scales"].cpu().numpy()
                assert ((got == self.scale[i]) | (np.isnan(got) & np.isnan(self.scale[i]))).all(), n

    def launch(self, op, **kw):
        p = self.fe.prepare(self.ctx, op, **{**self.args(), **kw})
        try:
            p.launch_and_wait(self.stream, 20000)
        finally:
            p.destroy()


def rows_in(torch, x, dtype):
    """A contiguous GPU tensor of rows, and the f32 values that the kernel sees."""
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda()
    if dtype == "bf16":
        t = t.to(torch.bfloat16)
    return t, t.float().cpu().numpy()


def contiguous(kv_heads, dim):
    return dict(k_token_stride=kv_heads * dim, k_head_stride=dim, v_token_stride=kv_heads * dim, v_head_stride=dim)


# ---- append and read ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kv_heads,dim,page", [(1, 16, 1), (3, 64, 16), (8, 128, 64), (2, 96, 24), (5, 256, 7), (12, 80, 16), (33, 32, 8)])
def test_append_and_read_back_bit_exact(gpu, form, dtype, kv_heads, dim, page):
    fe, torch, ctx, stream = gpu
    rng = np.random.default_rng(dim + page)
    new = [5, 0, 1, 70, 0, 2]                      # sequences without new tokens too
    lengths = [n + o for n, o in zip(new, [0, 9, 3, 13, 0, page])]
    c = Cache(gpu, form, lengths, kv_heads, dim, page).to_gpu()
    T = sum(new)
    offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
    rows = [rows_in(torch, rng.normal(size=(T, kv_heads, dim)) * np.exp(rng.normal(size=(T, kv_heads, 1)) * 3), dtype) for _ in range(2)]
    d = {torch.float32: 0, torch.bfloat16: 1}[rows[0][0].dtype]
    kw = dict(token_offsets=c.up(offsets), tokens=T, **contiguous(kv_heads, dim))
    c.launch("kv_cache_append_v1", k=rows[0][0], v=rows[1][0], input_dtype=d, **kw)
    for b, n in enumerate(new):
        if n:
            for side in range(2):
                c.put(side, b, np.arange(lengths[b] - n, lengths[b]), rows[side][1][offsets[b]:offsets[b + 1]])
    c.assert_same()
    for out, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        k, v = (torch.full((T, kv_heads, dim), math.nan, dtype=out, device="cuda") for _ in range(2))
        c.launch("kv_cache_read_v1", k=k, v=v, output_dtype=code, **kw)
        for side, got in enumerate((k, v)):
            want = np.concatenate([c.get(side, b, np.arange(lengths[b] - n, lengths[b])) for b, n in enumerate(new) if n])
            want = want.astype(np.float32)          # one rounding of the exact product
            if code:
                want = from_bf16(to_bf16(want))
            assert (got.float().cpu().numpy() == want).all()
    c.assert_same()


@pytest.mark.parametrize("form", FORMATS)
def test_append_special_rows(gpu, form):
    """Rows of zeros, of the smallest and the largest numbers, ties of the rounding, infinities and NaN."""
    fe, torch, ctx, stream = gpu
    rng = np.random.default_rng(5)
    kv_heads, dim, page = 2, 32, 4
    x = rng.normal(size=(14, kv_heads, dim)).astype(np.float32)
    x[0] = 0
    x[1] = -0.0
    x[2] *= 1e-41
    x[3] *= 1e-44
    x[4] = np.where(rng.random((kv_heads, dim)) < .5, 3.4028235e38, -3.4028235e38)
    x[5] *= 1e38 / np.abs(x[5]).max()
    x[6, 0, 3] = np.inf
    x[7, 1, 31] = -np.inf
    x[8, 0, 0] = np.nan
    x[9] = np.linspace(-127, 127, dim) if form == "i8" else np.linspace(-448, 448, dim)
    x[10] = np.arange(dim) + 0.5                    # halves, with the largest 127: ties of i8
    x[10, :, -1] = 127
    x[11] = np.float32(448) * np.arange(dim) / 256  # the midpoints of e4m3's coarsest steps among them
    x[11, :, -1] = 448
    x[12] = from_bf16(np.uint16(0x3f80) + np.arange(dim, dtype=np.uint16))
    x[13] = 1 + np.arange(dim) * 2.0 ** -9          # bf16 ties
    n = len(x)
    c = Cache(gpu, form, [n], kv_heads, dim, page).to_gpu()
    if form == "bf16":                              # bf16 holds infinities; NaN by itself: any payload
        x[8, 0, 0] = 1
    t = torch.from_numpy(x).cuda()
    kw = dict(token_offsets=c.up(np.array([0, n], np.uint32)), tokens=n, **contiguous(kv_heads, dim))
    c.launch("kv_cache_append_v1", k=t, v=t, input_dtype=0, **kw)
    for side in range(2):
        c.put(side, 0, np.arange(n), x)
    c.assert_same()
    k, v = torch.zeros_like(t), torch.zeros_like(t)
    c.launch("kv_cache_read_v1", k=k, v=v, output_dtype=0, **kw)
    with np.errstate(all="ignore"):
        want = c.get(0, 0, np.arange(n)).astype(np.float32)
    got = k.cpu().numpy()
    assert ((got == want) | (np.isnan(got) & np.isnan(want))).all()
    assert torch.equal(k.nan_to_num(7.0), v.nan_to_num(7.0))
    if form != "bf16":
        assert np.isnan(got[6, 0]).all() and np.isnan(got[7, 1]).all() and np.isnan(got[8, 0]).all() and np.isfinite(got[6, 1]).all()


@pytest.mark.parametrize("form", ["e4m3", "i8"])
def test_append_rows_of_subnormal_scales(gpu, form):
    """A scale of few bits may be a third below max / C: its quotients go up to the largest code, with their sign."""
    top = np.arange(1, 1200)                       # times the smallest number
    x = np.zeros((len(top), 1, 16), np.float32)
    x[:, 0, 0], x[:, 0, 1], x[:, 0, 2] = top * 2.0 ** -149, -top * 2.0 ** -149, top // 2 * 2.0 ** -149
    c = Cache(gpu, form, [len(top)], 1, 16, 16).to_gpu()
    rows = c.up(x)
    c.launch("kv_cache_append_v1", k=rows, v=rows, input_dtype=0, token_offsets=c.up(np.array([0, len(top)], np.uint32)), tokens=len(top), **contiguous(1, 16))
    for side in range(2):
        c.put(side, 0, np.arange(len(top)), x)
    c.assert_same()


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_keeps_the_sign_of_zero(gpu, form, dtype):
    """-0 among ordinary numbers is e4m3's code 0x80, 0 its code 0; so are numbers that round to 0, at every size of the scale."""
    rng = np.random.default_rng(15)
    size = np.array([2.0 ** -120, 2.0 ** -70, 2.0 ** -61, 2.0 ** -59, 1e-6, 1.0, 300.0, 2.0 ** 50, 2.0 ** 70, 2.0 ** 110])
    x = (rng.normal(size=(len(size), 2, 48)) * size[:, None, None]).astype(np.float32)
    x[:, :, 0:48:5], x[:, :, 1:48:5] = -0.0, 0.0
    x[:, :, 2:48:5] *= np.float32(2.0 ** -20)
    c = Cache(gpu, form, [len(size)], 2, 48, 4).to_gpu()
    t, xv = rows_in(c.torch, x, dtype)
    kw = dict(token_offsets=c.up(np.array([0, len(size)], np.uint32)), tokens=len(size), **contiguous(2, 48))
    c.launch("kv_cache_append_v1", k=t, v=t, input_dtype=int(dtype == "bf16"), **kw)
    for side in range(2):
        c.put(side, 0, np.arange(len(size)), xv)
    c.assert_same()
    out = [c.torch.zeros(len(size), 2, 48, device="cuda") for _ in range(2)]
    c.launch("kv_cache_read_v1", k=out[0], v=out[1], output_dtype=0, **kw)
    if form != "i8":
        assert (np.signbit(out[0].cpu().numpy()) == np.signbit(xv)).all()


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("layout", ["token_major", "head_major", "fused", "odd"])
def test_strided_rows(gpu, form, layout):
    """One new token a sequence without offsets; rows inside wider storage, heads before tokens, starts on odd elements."""
    fe, torch, ctx, stream = gpu
    kv_heads, dim, page, B = 4, 64, 16, 19
    rng = np.random.default_rng(3)
    lengths = rng.integers(1, 60, B)
    c = Cache(gpu, form, lengths, kv_heads, dim, page).to_gpu()
    ts, hs, off = {"token_major": (kv_heads * dim, dim, 0), "head_major": (dim, B * dim, 0), "fused": (3 * kv_heads * dim, dim, kv_heads * dim),
                   "odd": (kv_heads * (dim + 3) + 5, dim + 3, 1)}[layout]
    extent = (B - 1) * ts + (kv_heads - 1) * hs + dim
    at = off + np.arange(B)[:, None, None] * ts + np.arange(kv_heads)[None, :, None] * hs + np.arange(dim)
    store = [torch.from_numpy(rng.normal(size=off + extent + 9).astype(np.float32)).cuda().to(torch.bfloat16) for _ in range(2)]
    sl = lambda t: (t.data_ptr() + off * t.element_size(), extent)  # noqa: E731
    strides = dict(k_token_stride=ts, k_head_stride=hs, v_token_stride=ts, v_head_stride=hs)
    c.launch("kv_cache_append_v1", k=sl(store[0]), v=sl(store[1]), tokens=B, input_dtype=1, **strides)
    for side in range(2):
        rows = store[side].float().cpu().numpy()[at]
        for b in range(B):
            c.put(side, b, [lengths[b] - 1], rows[b:b + 1])
    c.assert_same()
    for code, dt in ((0, torch.float32), (1, torch.bfloat16)):
        out = [torch.full((off + extent + 9,), 7.0, device="cuda", dtype=dt) for _ in range(2)]
        c.launch("kv_cache_read_v1", k=sl(out[0]), v=sl(out[1]), tokens=B, output_dtype=code, **strides)
        for side in range(2):
            want = np.full(off + extent + 9, 7.0, np.float32)
            want[at] = np.stack([c.get(side, b, [lengths[b] - 1])[0] for b in range(B)]).astype(np.float32)
            if code:
                want = from_bf16(to_bf16(want))
            assert (out[side].float().cpu().numpy() == want).all()


def test_rows_that_do_not_fit_are_reported_and_left_out(gpu):
    fe, torch, ctx, stream = gpu
    kv_heads, dim, page = 2, 16, 4
    for form in FORMATS:
        # sequence 0: more new tokens than positions; 1: fine; 2: longer than its table; 3: a page outside the cache
        c = Cache(gpu, form, [8, 6, 8, 7], kv_heads, dim, page, width=2)
        c.table[3, 1] = c.pages
        c.to_gpu()
        x = torch.ones(8, kv_heads, dim, device="cuda")
        offsets = c.up(np.array([0, 3, 4, 5, 8], np.uint32))
        lengths = c.up(np.array([2, 6, 9, 7], np.uint32))
        kw = dict(token_offsets=offsets, tokens=8, lengths=lengths, **contiguous(kv_heads, dim))
        with pytest.raises(fe.Fe2o3Error) as e:
            c.launch("kv_cache_append_v1", k=x, v=x, input_dtype=0, **kw)
        assert e.value.name == "KernelStatus"
        for side in range(2):
            c.put(side, 1, [5], np.ones((1, kv_heads, dim), np.float32))
        c.assert_same()
        k, v = (torch.full((8, kv_heads, dim), 5.0, device="cuda") for _ in range(2))
        with pytest.raises(fe.Fe2o3Error):
            c.launch("kv_cache_read_v1", k=k, v=v, output_dtype=0, **kw)
        got = k.cpu().numpy()
        assert (got[[0, 1, 2, 4]] == 5).all()       # left as they were
        assert np.abs(got[3] - 1).max() <= 2 ** -20
        assert (got[5:] == 0).all()                 # positions 4 to 6 of sequence 3 lie in the page outside
        # offsets that do not cover every row: rows before the first and after the last belong to no sequence
        kw["token_offsets"] = c.up(np.array([3, 3, 4, 4, 4], np.uint32))
        k.fill_(5.0)
        with pytest.raises(fe.Fe2o3Error):
            c.launch("kv_cache_read_v1", k=k, v=v, output_dtype=0, **kw)
        got = k.cpu().numpy()
        assert np.abs(got[3] - 1).max() <= 2 ** -20 and (got[[0, 1, 2, 4, 5, 6, 7]] == 5).all()


# ---- attention ------------------------------------------------------------------------------------------------------

def filled(gpu, form, lengths, kv_heads, dim, page, seed=1, **kw):
    """A cache whose sequences hold normal rows, keys with channels of unlike size."""
    c = Cache(gpu, form, lengths, kv_heads, dim, page, seed=seed, **kw)
    rng = np.random.default_rng(seed)
    spread = np.exp(0.5 * rng.normal(size=dim))
    for b, n in enumerate(c.lengths):
        for side, by in ((0, spread), (1, 1.0)):
            if n:
                c.put(side, b, np.arange(n), rng.normal(size=(n, kv_heads, dim)) * by)
    return c.to_gpu()


def attention64(c, q, scale, window=0, lengths=None):
    """o, lse, sum p|v| and the largest sum of |q k| a row, in 64 bits."""
    B, H, D = q.shape
    G = H // c.kv_heads
    o, lse, mag, big = np.zeros((B, H, D)), np.full((B, H), -np.inf), np.zeros((B, H, D)), np.zeros((B, H))
    for b, n in enumerate(c.lengths if lengths is None else lengths):
        if n == 0:
            continue
        at = np.arange(max(0, n - window) if window else 0, n)
        k, v = c.get(0, b, at), c.get(1, b, at)
        for h in range(H):
            kk, vv = k[:, h // G], v[:, h // G]
            s = kk @ q[b, h].astype(np.float64) * scale
            top = s.max()
            with np.errstate(invalid="ignore"):
                p = np.exp(s - top)
                lse[b, h] = top + np.log(p.sum())
                p /= p.sum()
                o[b, h], mag[b, h] = p @ vv, p @ np.abs(vv)
                big[b, h] = (np.abs(kk) @ np.abs(q[b, h].astype(np.float64))).max() * abs(scale)
    return o, lse, mag, big


def check_attention(c, q, got, lse, want, out):
    """|o - e| <= (2 d + 2^-19 + n 2^-24) sum p|v|: d bounds the error of a score (dim products of f32 size added by a unit
    that truncates, 2^-23 each, and the roundings of its scale, maximum and logarithm's base, 2^-22 of it), the rest the
    exponential's and the sums'.  A bf16 output: 16-bit probabilities (2^-15) and its own rounding (2^-9 of it, doubled
    for a tie that falls the other way)."""
    o, l64, mag, big = want
    d = ((c.dim + 8) * 2.0 ** -23 + 2.0 ** -22) * big
    n = np.asarray(c.lengths, np.float64)[:, None]
    bound = (2 * d + 2.0 ** -19 + n * 2.0 ** -24)[..., None] * mag + 1e-37
    if out == "bf16":
        bound = bound + 2.0 ** -15 * mag + 2.0 ** -8 * np.abs(o)
    err = np.abs(got - o)
    assert np.isfinite(got).all() and (err <= bound).all(), (float((err / bound).max()), float(err.max()))
    if lse is not None:
        empty = np.isinf(l64)
        assert (lse[empty] == -np.inf).all()
        lb = (d + 2.0 ** -20 + n * 2.0 ** -24 + 2.0 ** -22 * np.abs(np.where(empty, 0, l64)))[~empty]
        assert (np.abs(lse[~empty] - l64[~empty]) <= lb).all()


def attend(c, q, scale, window=0, out="f32", want_lse=True, stream=None, **kw):
    torch, fe = c.torch, c.fe
    B, H, D = q.shape
    o = torch.full((B, H, D), 7.0, dtype=torch.float32 if out == "f32" else torch.bfloat16, device="cuda")
    lse = torch.full((B, H), 7.0, device="cuda") if want_lse else None
    args = {**c.args(), "q": q, "output": o, "lse": lse, "heads": H, "q_stride": H * D, "q_head_stride": D, "scale": scale,
            "window": window, "q_dtype": 0 if q.dtype == torch.float32 else 1, "output_dtype": 0 if out == "f32" else 1, **kw}
    p = fe.prepare(c.ctx, "paged_attention_v1", **args)
    try:
        p.launch_and_wait(stream or c.stream, 20000)
    finally:
        p.destroy()
    return o.float().cpu().numpy(), None if lse is None else lse.cpu().numpy()


def queries(torch, B, H, D, dtype, seed=9, by=1.0):
    q = np.random.default_rng(seed).normal(size=(B, H, D)) * by
    return rows_in(torch, q, dtype)


EDGES = [0, 1, 2, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 200]


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (8, 2), (16, 2), (24, 8), (12, 1), (40, 1), (66, 2), (130, 1)])
def test_attention_heads(gpu, form, heads, kv_heads):
    c = filled(gpu, form, EDGES, kv_heads, 64, 16)
    q, qv = queries(c.torch, len(EDGES), heads, 64, "bf16")
    got, lse = attend(c, q, 0.125)
    check_attention(c, qv, got, lse, attention64(c, qv, 0.125), "f32")


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128, 160, 192, 208, 256])
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16")])
def test_attention_head_sizes_and_types(gpu, form, dim, dtype, out):
    lengths = [0, 1, 16, 33, 100, 300]
    c = filled(gpu, form, lengths, 2, dim, 24)
    q, qv = queries(c.torch, len(lengths), 6, dim, dtype)
    scale = 1 / math.sqrt(dim)
    got, lse = attend(c, q, scale, out=out)
    check_attention(c, qv, got, lse, attention64(c, qv, np.float32(scale)), out)


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dim", [48, 112, 128, 144, 256])
@pytest.mark.parametrize("group", [9, 16, 20])
def test_attention_groups_above_eight(gpu, form, dim, group):
    """Sixteen query heads at once, and more than one chunk of them, at every build's width of a row."""
    lengths = [0, 1, 17, 90, 260]
    c = filled(gpu, form, lengths, 2, dim, 16)
    for dtype, out in (("bf16", "f32"), ("f32", "f32"), ("f32", "bf16")):
        q, qv = queries(c.torch, len(lengths), 2 * group, dim, dtype)
        got, lse = attend(c, q, dim ** -0.5, out=out)
        check_attention(c, qv, got, lse, attention64(c, qv, np.float32(dim ** -0.5)), out)


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dim", [16, 48, 80, 96, 144, 208, 256])
@pytest.mark.parametrize("page", [1, 3, 20])
def test_attention_row_by_row(gpu, form, dim, page):
    """Pages that take no boxes, with rows narrower than their build's: the columns past a head's are zeros that no copy touches."""
    lengths = [0, 1, 33, 100, 301, 64]
    c = filled(gpu, form, lengths, 2, dim, page)
    for group in (3, 11):
        q, qv = queries(c.torch, len(lengths), 2 * group, dim, "bf16")
        for window in (0, 50):
            got, lse = attend(c, q, dim ** -0.5, window=window)
            check_attention(c, qv, got, lse, attention64(c, qv, np.float32(dim ** -0.5), window), "f32")


@pytest.mark.parametrize("form", ["e4m3", "i8"])
@pytest.mark.parametrize("dim", [64, 96, 256])
def test_attention_scales_that_start_on_any_float(gpu, form, dim):
    """Scales off 16 bytes go row by row too, and the rows of an append and a read find them."""
    lengths = [5, 0, 70, 200]
    c = filled(gpu, form, lengths, 3, dim, 32)
    q, qv = queries(c.torch, len(lengths), 12, dim, "bf16")
    n = c.pages * 3 * 32
    for off in (1, 2, 3):
        held = [c.torch.full((n + 8,), math.nan, device="cuda") for _ in range(2)]
        for t, name in zip(held, ("k_scales", "v_scales")):
            t[off:off + n] = c.d[name].reshape(-1)
        scales = dict(k_scales=(held[0].data_ptr() + 4 * off, n), v_scales=(held[1].data_ptr() + 4 * off, n))
        got, lse = attend(c, q, dim ** -0.5, **scales)
        check_attention(c, qv, got, lse, attention64(c, qv, np.float32(dim ** -0.5)), "f32")
        rows, out = (c.torch.randn(200, 3, dim, device="cuda") for _ in range(2))
        kw = dict(token_offsets=c.up(np.array([0, 0, 0, 0, 200], np.uint32)), tokens=200, **contiguous(3, dim), **scales)
        c.launch("kv_cache_append_v1", k=rows, v=rows, input_dtype=0, **kw)
        c.launch("kv_cache_read_v1", k=out, v=c.torch.empty_like(out), output_dtype=0, **kw)
        code, scale = quantised(rows.cpu().numpy(), form)
        assert (out.cpu().numpy() == values_of(code, scale, form).astype(np.float32)).all()
        assert all(t[:off].isnan().all() and t[off + n:].isnan().all() for t in held)
        c.to_gpu()


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dim,group", [(64, 4), (128, 1), (128, 9), (80, 16)])
def test_attention_bf16_output_is_the_f32_one_rounded(gpu, form, dim, group):
    """The output's type changes its last rounding and nothing before it: bit for bit."""
    c = filled(gpu, form, EDGES + [1000, 3000], 2, dim, 16)
    for dtype in ("bf16", "f32"):
        q, _ = queries(c.torch, len(EDGES) + 2, 2 * group, dim, dtype, by=0.5)
        whole, lse = attend(c, q, dim ** -0.5)
        short, lse2 = attend(c, q, dim ** -0.5, out="bf16")
        assert (short == from_bf16(to_bf16(whole))).all() and (lse == lse2).all()


@pytest.mark.parametrize("page", [1, 3, 8, 16, 40, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 5, 16, 50, 128, 1000])
def test_attention_pages_and_windows(gpu, page, window):
    for form, group in (("bf16", 1), ("i8", 4)):
        c = filled(gpu, form, EDGES, 2, 64, page)
        q, qv = queries(c.torch, len(EDGES), 2 * group, 64, "bf16")
        got, lse = attend(c, q, 0.125, window=window)
        check_attention(c, qv, got, lse, attention64(c, qv, 0.125, window), "f32")


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("lengths,heads,kv_heads", [([30011], 4, 1), ([5000, 3], 8, 8), ([9000, 0, 1, 8999, 20], 10, 2), ([70] * 300, 2, 2),
                                                    ([1] * 700, 3, 1), (list(range(0, 500, 3)), 4, 2), ([2049] * 9, 8, 1),
                                                    ([i % 7 * 9 for i in range(1500)], 2, 1), ([64] * 33 + [20000] + [0] * 40, 3, 3)])
def test_attention_split_and_joined(gpu, form, lengths, heads, kv_heads):
    """Few long sequences, many short ones, and both: the pieces that blocks compute meet in every way."""
    c = filled(gpu, form, lengths, kv_heads, 32, 16)
    q, qv = queries(c.torch, len(lengths), heads, 32, "bf16", by=2.0)
    scale = 32 ** -0.5
    got, lse = attend(c, q, scale)
    check_attention(c, qv, got, lse, attention64(c, qv, np.float32(scale)), "f32")
    again, lse2 = attend(c, q, scale)
    assert (got == again).all() and (lse == lse2).all()        # whichever block comes last


def test_attention_query_strides_and_no_lse(gpu):
    fe, torch, ctx, stream = gpu
    B, H, D = 7, 6, 48
    c = filled(gpu, "bf16", [3, 40, 0, 129, 64, 1, 17], 2, D, 16)
    for dtype in ("f32", "bf16"):
        store, sv = queries(torch, B, H + 3, D + 5, dtype)
        flat = store.reshape(-1)
        hs, bs, off = D + 5, (H + 3) * (D + 5), D + 7
        at = off + np.arange(B)[:, None, None] * bs + np.arange(H)[None, :, None] * hs + np.arange(D)
        qv = sv.reshape(-1)[at]
        view = (flat.data_ptr() + off * flat.element_size(), (B - 1) * bs + (H - 1) * hs + D)
        o = torch.full((B, H, D), 7.0, device="cuda")
        c.launch("paged_attention_v1", q=view, output=o, heads=H, q_stride=bs, q_head_stride=hs, scale=0.2, window=0,
                 q_dtype=0 if dtype == "f32" else 1, output_dtype=0)
        check_attention(c, qv, o.cpu().numpy(), None, attention64(c, qv, np.float32(0.2)), "f32")
    # one query for all heads (stride 0), one for all sequences
    q1, qv1 = queries(torch, 1, 1, D, "bf16")
    o = torch.full((B, H, D), 7.0, device="cuda")
    c.launch("paged_attention_v1", q=q1, output=o, heads=H, q_stride=0, q_head_stride=0, scale=0.2, window=0, q_dtype=1, output_dtype=0)
    qv = np.broadcast_to(qv1, (B, H, D))
    check_attention(c, qv, o.cpu().numpy(), None, attention64(c, qv, np.float32(0.2)), "f32")


@pytest.mark.parametrize("scale", [0.0, -0.3, 25.0])
def test_attention_scales(gpu, scale):
    """Equal weights, reversed order, and scores so far apart that most weights vanish."""
    c = filled(gpu, "bf16", [1, 50, 700], 1, 64, 16)
    q, qv = queries(c.torch, 3, 4, 64, "bf16")
    got, lse = attend(c, q, scale)
    check_attention(c, qv, got, lse, attention64(c, qv, np.float32(scale)), "f32")


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("octaves", [6, 12, 18])
def test_attention_one_weight_far_above_the_others(gpu, form, octaves):
    """A column in which the row of the largest weight is 0 is the small weights' sum, to the same accuracy."""
    c = Cache(gpu, form, [2, 40, 3000], 1, 64, 16)
    rng = np.random.default_rng(11)
    for b, n in enumerate(c.lengths):
        k, v = np.zeros((n, 1, 64)), rng.normal(size=(n, 1, 64))
        k[n // 2, 0, 0] = octaves * math.log(2)
        v[n // 2, 0, 1:] = 0
        c.put(0, b, np.arange(n), k)
        c.put(1, b, np.arange(n), v)
    c.to_gpu()
    q = c.torch.zeros(3, 2, 64, dtype=c.torch.float32, device="cuda")
    q[:, 0, 0], q[:, 1, 0] = 1.0, 0.75
    qv = q.cpu().numpy()
    for out in ("f32", "bf16"):
        got, lse = attend(c, q, 1.0, out=out)
        check_attention(c, qv, got, lse, attention64(c, qv, 1.0), out)


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("octaves", [10, 20, 30, 45, 60])
def test_attention_values_of_unlike_size(gpu, form, octaves):
    """A row of values far larger than the others, which one head of a pair gives next to no weight and the other next to all
    of it: each head has the accuracy that its own products of probability and value allow, wherever the row lies.  (i8 rounds a
    small value of a row to 0, and what lies under a 0 of the heaviest row is held as the next test says: here no value is small.)"""
    lengths = [2, 20, 40, 333, 3000] + [300] * 200
    c = Cache(gpu, form, lengths, 1, 16, 16)
    rng = np.random.default_rng(12)
    for b, n in enumerate(c.lengths):
        big = [0, n - 1, n // 2, n // 3][b % 4]
        k, v = rng.normal(size=(n, 1, 16)) * 0.01, rng.normal(size=(n, 1, 16)) * 2.0 ** -octaves
        k[:, 0, 0], v[big] = 0.0, rng.choice([-1, 1], (1, 16)) * rng.uniform(0.5, 1, (1, 16)) if form == "i8" else rng.normal(size=(1, 16))
        k[big, 0, 0] = (octaves + 6) * math.log(2)
        if b % 3 == 0:
            v[(big + 1) % n] = 0                    # and a row of zeros
        c.put(0, b, np.arange(n), k)
        c.put(1, b, np.arange(n), v)
    c.to_gpu()
    q = rng.normal(size=(len(lengths), 4, 16))
    q[:, :, 0] = [-1.0, 1.0, -1.5, 0.0]
    for dtype, out in (("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")):
        qt, qv = rows_in(c.torch, q, dtype)
        got, lse = attend(c, qt, 1.0, out=out)
        check_attention(c, qv, got, lse, attention64(c, qv, 1.0), out)


@pytest.mark.parametrize("form", ["e4m3", "i8"])
@pytest.mark.parametrize("octaves", [24, 30, 36, 50])
def test_attention_small_weights_of_8_bit_caches(gpu, form, octaves):
    """Weights are held to 2^-25 where the head's largest, probability times scale, lies in [2^14, 2^15): to 2^-39 of it, times the
    largest code for each key.  A column in which the row of the largest weight is 0 shows it."""
    c = Cache(gpu, form, [2, 40, 3000], 1, 64, 16)
    rng = np.random.default_rng(13)
    for b, n in enumerate(c.lengths):
        k, v = np.zeros((n, 1, 64)), rng.normal(size=(n, 1, 64))
        k[n // 2, 0, 0] = octaves * math.log(2)
        v[n // 2, 0, 1:] = 0
        c.put(0, b, np.arange(n), k)
        c.put(1, b, np.arange(n), v)
    c.to_gpu()
    q = c.torch.zeros(3, 1, 64, dtype=c.torch.float32, device="cuda")
    q[:, :, 0] = 1.0
    got, lse = attend(c, q, 1.0)
    o, l64, mag, big = attention64(c, q.cpu().numpy(), 1.0)
    n = np.asarray(c.lengths, np.float64)[:, None, None]
    d = (72 * 2.0 ** -23 + 2.0 ** -22) * big[..., None]
    largest = mag.max(-1, keepdims=True)            # the largest weight times the largest code, at least
    assert (np.abs(got - o) <= (2 * d + 2.0 ** -19 + n * 2.0 ** -24) * mag + n * 2.0 ** -39 * largest).all()
    assert octaves > 30 or (np.abs(got - o)[1:, :, 1:] <= 0.1 * mag[1:, :, 1:]).all()   # (some bits of them are still there)


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("score", [2.0 ** 18, 2.0 ** 22, -2.0 ** 24, 2.0 ** 26, 2.0 ** 30, -2.0 ** 34])
def test_attention_equal_scores_far_from_zero(gpu, form, score):
    """Every key has the same score, however large: the output is the mean of the values, whose rows are of unlike size."""
    lengths = [1, 2, 31, 100, 999]
    c = Cache(gpu, form, lengths, 1, 16, 16)
    rng = np.random.default_rng(17)
    for b, n in enumerate(c.lengths):
        k, v = np.zeros((n, 1, 16)), rng.normal(size=(n, 1, 16)) * 2.0 ** rng.integers(0, 12, (n, 1, 1))
        k[:, 0, 0] = score
        c.put(0, b, np.arange(n), k)
        c.put(1, b, np.arange(n), v)
    c.to_gpu()
    q = c.torch.zeros(len(lengths), 3, 16, device="cuda")
    q[:, 0, 0], q[:, 2, 0] = 1.0, 0.75
    got, _ = attend(c, q, 1.0)
    for b, n in enumerate(lengths):
        v = c.get(1, b, np.arange(n))[:, 0]
        assert (np.abs(got[b] - v.mean(0)) <= (2.0 ** -19 + n * 2.0 ** -24) * np.abs(v).mean(0) + n * 2.0 ** -39 * np.abs(v).max()).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gap", [60.0, 95.0, 200.0, math.inf])
def test_attention_largest_values_without_weight(gpu, dtype, gap):
    """Rows of the largest numbers that bf16 holds, `gap` below the other keys' scores: they count with their weight and, where that
    is 0, not at all.  (A weight below f32's normal numbers may be 0: 2^-126 of the value.)"""
    lengths = [2, 30, 700]
    c = Cache(gpu, "bf16", lengths, 1, 16, 16)
    rng = np.random.default_rng(18)
    for b, n in enumerate(c.lengths):
        k, v = np.zeros((n, 1, 16)), rng.normal(size=(n, 1, 16))
        far = [0, n // 2, n - 1][b]
        k[far, 0, 0], v[far] = -gap, from_bf16(np.full((1, 16), 0x7f7f, np.uint16))
        c.put(0, b, np.arange(n), k)
        c.put(1, b, np.arange(n), v)
    c.to_gpu()
    q, qv = rows_in(c.torch, np.eye(1, 16)[None].repeat(3, 0), dtype)
    got, lse = attend(c, q, 1.0)
    with np.errstate(all="ignore"):
        o, l64, mag, big = attention64(c, qv, 1.0)
    n = np.asarray(lengths, np.float64)[:, None]
    weight = np.exp(-gap)
    bound = (2 * (24 * 2.0 ** -23 + 2.0 ** -22) * min(gap, 100.0) + 2.0 ** -19 + n * 2.0 ** -24)[..., None] * mag
    bound = bound + (weight * 3.4e38 if weight < 2.0 ** -126 else 0.0)
    assert (np.abs(got - o) <= bound).all() and (np.abs(lse - l64) <= 1e-5).all()
    # a query element far below the others, times the largest keys
    c = Cache(gpu, "bf16", [50], 1, 16, 16)
    k, v = np.zeros((50, 1, 16)), rng.normal(size=(50, 1, 16))
    k[:, 0, 1] = np.linspace(-3e38, 3e38, 50)
    c.put(0, 0, np.arange(50), k)
    c.put(1, 0, np.arange(50), v)
    c.to_gpu()
    q = np.zeros((1, 1, 16))
    q[0, 0, 1] = 2.0 ** -124
    qt, qv = rows_in(c.torch, q, dtype)
    got, lse = attend(c, qt, 1.0)
    check_attention(c, qv, got, lse, attention64(c, qv, 1.0), "f32")


def test_attention_rising_scores(gpu):
    """Scores that rise all along (every block moves the maximum) and fall all along."""
    for sign in (1, -1):
        c = Cache(gpu, "bf16", [1500, 333], 1, 16, 16)
        rng = np.random.default_rng(2)
        for b, n in enumerate(c.lengths):
            k = np.zeros((n, 1, 16))
            k[:, 0, 0] = sign * np.linspace(-60, 60, n)
            c.put(0, b, np.arange(n), k)
            c.put(1, b, np.arange(n), rng.normal(size=(n, 1, 16)))
        c.to_gpu()
        q = c.torch.zeros(2, 3, 16, dtype=c.torch.bfloat16, device="cuda")
        q[:, :, 0] = c.torch.tensor([1.0, 8.0, -3.0])
        got, lse = attend(c, q, 1.0)
        qv = q.float().cpu().numpy()
        check_attention(c, qv, got, lse, attention64(c, qv, 1.0), "f32")


@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_attention_infinities_and_nan(gpu, out):
    """What a cached row holds goes into its own (sequence, key head) only, as the formula has it."""
    fe, torch, ctx, stream = gpu
    n, D = 90, 32
    c = Cache(gpu, "bf16", [n] * 6, 2, D, 16)
    rng = np.random.default_rng(4)
    rows = rng.normal(size=(2, 6, n, 2, D)).astype(np.float32)
    q = np.abs(rng.normal(size=(6, 4, D))).astype(np.float32)
    rows[1, 0, 40, 0, 5] = np.inf          # a value: that column of heads 0 and 1
    rows[1, 1, 40, 0, 5] = np.nan
    rows[0, 2, 70, 1, 3] = np.inf          # a key with positive queries: score +inf, no softmax
    rows[0, 3, 70, 1, 3] = -np.inf         # score -inf: weight zero
    rows[0, 4, :, 0, 3] = -np.inf          # every score -inf: no softmax either
    rows[0, 5, 11, 0, 3] = np.nan
    for b in range(6):
        for side in range(2):
            c.put(side, b, np.arange(n), rows[side, b])
    c.code[0][np.isnan(from_bf16(c.code[0]))] = 0x7fc0
    c.to_gpu()
    qt, qv = rows_in(torch, q, "bf16")
    got, lse = attend(c, qt, 0.1, out=out)
    fine = np.ones((6, 4, D), bool)
    assert (got[0, :2, 5] == np.inf).all()
    assert np.isnan(got[1, :2, 5]).all()
    fine[0:2, :2, 5] = False
    assert np.isnan(got[2, 2:]).all() and np.isnan(got[4, :2]).all() and np.isnan(got[5, :2]).all()
    fine[2, 2:] = fine[4, :2] = fine[5, :2] = False
    for b, h, d in ((0, 0, 5), (1, 0, 5)):
        rows[1, b, 40, h, d] = 0
        c.put(1, b, np.arange(n), rows[1, b])
    with np.errstate(all="ignore"):
        o, l64, mag, big = attention64(c, qv, np.float32(0.1))
    big = np.where(np.isfinite(big), big, 12.0)
    bound = (2 * ((D + 8) * 2.0 ** -23 + 2.0 ** -22) * big + 2.0 ** -18)[..., None] * mag
    if out == "bf16":
        bound = bound + 2.0 ** -15 * mag + 2.0 ** -8 * np.abs(o)
    assert np.isfinite(got[fine]).all() and (np.abs(got - o)[fine] <= bound[fine]).all()
    keep = np.isfinite(l64)
    assert (np.abs(lse - l64)[keep] <= 1e-4).all()
    # an 8-bit row with a NaN scale: NaN in its own key head alone
    for form in ("e4m3", "i8"):
        c = filled(gpu, form, [n, n], 2, D, 16)
        p, s = c.where(0, [33])
        for side in range(2):
            c.scale[side][p, 0, s] = np.nan
        c.to_gpu()
        qt, qv = queries(torch, 2, 4, D, "bf16")
        got, lse = attend(c, qt, 0.1, out=out)
        assert np.isnan(got[0, :2]).all() and np.isfinite(got[0, 2:]).all() and np.isfinite(got[1]).all()


def test_attention_reports(gpu):
    """A length that the table cannot hold: reported, that sequence alone unwritten.  A page outside the cache: reported,
    its rows count as zeros."""
    fe, torch, ctx, stream = gpu
    for form in FORMATS:
        c = filled(gpu, form, [30, 64, 20], 2, 64, 16, width=4)
        q, qv = queries(torch, 3, 4, 64, "bf16")
        o = torch.full((3, 4, 64), 7.0, device="cuda")
        kw = dict(q=q, output=o, heads=4, q_stride=256, q_head_stride=64, scale=0.125, window=0, q_dtype=1, output_dtype=0)
        with pytest.raises(fe.Fe2o3Error) as e:
            c.launch("paged_attention_v1", lengths=c.up(np.array([30, 65, 20], np.uint32)), **kw)
        assert e.value.name == "KernelStatus"
        got, want = o.cpu().numpy(), attention64(c, qv, 0.125)
        assert (got[1] == 7).all()
        for b in (0, 2):
            assert np.abs(got[b] - want[0][b]).max() <= 1e-4
        page = c.table[0, 1]
        c.table[0, 1] = 0x80000000
        c.to_gpu()
        with pytest.raises(fe.Fe2o3Error):
            c.launch("paged_attention_v1", **kw)
        c.table[0, 1] = page
        for side in range(2):
            c.code[side][page], c.scale[side][page] = 0, 0
        want = attention64(c, qv, 0.125)
        assert np.abs(o.cpu().numpy() - want[0]).max() <= 1e-4
        got, _ = attend(c.to_gpu(), q, 0.125)                    # and the next launch is as ever
        check_attention(c, qv, got, None, want, "f32")


def test_attention_of_an_empty_batch_and_of_empty_sequences(gpu):
    fe, torch, ctx, stream = gpu
    for B in (0, 1, 200):
        c = Cache(gpu, "bf16", [0] * B, 2, 64, 16, width=1).to_gpu()
        q, _ = queries(torch, B, 4, 64, "bf16")
        got, lse = attend(c, q, 0.125)
        assert (got == 0).all() and (lse == -np.inf).all()
    # a cache without pages
    c = Cache(gpu, "e4m3", [0, 0], 2, 64, 16, spare=0, width=0).to_gpu()
    q, _ = queries(torch, 2, 4, 64, "bf16")
    got, lse = attend(c, q, 0.125)
    assert (got == 0).all() and (lse == -np.inf).all()


def test_attention_on_other_streams(gpu):
    """Two prepared launches on two streams at once, each with its own workspace; many passes of one on one stream."""
    fe, torch, ctx, stream = gpu
    c = filled(gpu, "bf16", [4000, 77, 2500], 2, 64, 16)
    q, qv = queries(torch, 3, 8, 64, "bf16")
    want = attention64(c, qv, 0.125)
    streams = [ctx.create_stream() for _ in range(2)]
    outs = [torch.zeros(3, 8, 64, device="cuda") for _ in range(2)]
    ps = [fe.prepare(ctx, "paged_attention_v1", q=q, output=o, heads=8, q_stride=512, q_head_stride=64, scale=0.125, window=0, q_dtype=1,
                     output_dtype=0, **c.args()) for o in outs]
    torch.cuda.synchronize()
    for _ in range(50):
        for p, s in zip(ps, streams):
            p.launch(s)
    for s in streams:
        s.synchronize()
    for p, o in zip(ps, outs):
        check_attention(c, qv, o.cpu().numpy(), None, want, "f32")
        p.destroy()
    assert ctx.take_kernel_status(stream) == 0


def test_attention_plans_of_one_kernel_stand_side_by_side(gpu):
    """Prepared launches that share a kernel and differ in types, groups and pages: each works whichever was prepared last,
    and a workspace that was given back starts again at zero."""
    fe, torch, ctx, stream = gpu
    plans = []
    for form, dim, group, dtype, page in [("bf16", 128, 8, "f32", 16), ("bf16", 128, 1, "bf16", 24), ("bf16", 128, 7, "bf16", 16),
                                          ("i8", 128, 16, "f32", 64), ("i8", 128, 9, "bf16", 3)]:
        c = filled(gpu, form, [700, 0, 65], 1, dim, page)
        q, qv = queries(torch, 3, group, dim, dtype)
        o = torch.zeros(3, group, dim, device="cuda")
        p = fe.prepare(ctx, "paged_attention_v1", q=q, output=o, heads=group, q_stride=group * dim, q_head_stride=dim, scale=dim ** -0.5,
                       window=0, q_dtype=0 if dtype == "f32" else 1, output_dtype=0, **c.args())
        plans.append((c, q, qv, o, p, attention64(c, qv, np.float32(dim ** -0.5))))
    for order in (plans, plans[::-1]):
        for c, q, qv, o, p, want in order:
            o.fill_(7.0)
            torch.cuda.synchronize()
            p.launch_and_wait(stream, 20000)
            check_attention(c, qv, o.cpu().numpy(), None, want, "f32")
    for x in plans:
        x[4].destroy()
    for c, q, qv, o, _, want in plans:
        got, lse = attend(c, q, c.dim ** -0.5)
        check_attention(c, qv, got, lse, want, "f32")


def test_attention_workspaces_of_many_geometries(gpu):
    """Prepared and destroyed one after another, launches for all sizes of a batch share a few pieces: one of each power of two up to
    the largest need (16 MiB at most), in one or two slabs of 64 MiB."""
    fe, torch, ctx, stream = gpu
    c = Cache(gpu, "bf16", [0], 1, 128, 16, width=16).to_gpu()
    lengths, table = torch.zeros(100, dtype=torch.int32, device="cuda"), torch.zeros(100 * 16, dtype=torch.int32, device="cuda")
    q, o = torch.zeros(100, 8, 128, device="cuda"), torch.zeros(100, 8, 128, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for batch in range(1, 101):
        args = {**c.args(), "batch": batch, "lengths": lengths[:batch], "page_table": table[:batch * 16], "q": q[:batch], "output": o[:batch]}
        fe.prepare(ctx, "paged_attention_v1", heads=8, q_stride=1024, q_head_stride=128, scale=1.0, window=0, q_dtype=0, output_dtype=0, **args).destroy()
    assert before - torch.cuda.mem_get_info()[0] <= 130 << 20


def test_decode_steps_replay_from_one_graph(gpu):
    """Append and attention captured once; lengths grow in device memory between replays, over page ends."""
    fe, torch, ctx, stream = gpu
    B, H, KH, D, page, steps = 3, 8, 2, 64, 16, 20
    start = np.array([1, 14, 40])
    for form in FORMATS:
        c = Cache(gpu, form, start + steps, KH, D, page)
        rng = np.random.default_rng(8)
        for b, n in enumerate(start):
            for side in range(2):
                c.put(side, b, np.arange(n), rng.normal(size=(n, KH, D)))
        c.to_gpu()
        lengths = c.up(start.astype(np.uint32))
        k, v = (torch.zeros(B, KH, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        q, o = torch.zeros(B, H, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(B, H, D, device="cuda")
        args = {**c.args(), "lengths": lengths}
        ap = fe.prepare(ctx, "kv_cache_append_v1", k=k, v=v, tokens=B, input_dtype=1, **contiguous(KH, D), **args)
        at = fe.prepare(ctx, "paged_attention_v1", q=q, output=o, heads=H, q_stride=H * D, q_head_stride=D, scale=0.125, window=0, q_dtype=1,
                        output_dtype=0, **args)
        side_stream = torch.cuda.Stream()
        with torch.cuda.stream(side_stream):
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=side_stream):
                s = ctx.wrap_stream(side_stream.cuda_stream)
                lengths.add_(1)
                ap.launch(s)
                at.launch(s)
        for step in range(steps):
            new = [rows_in(torch, rng.normal(size=(B, KH, D)), "bf16") for _ in range(2)]
            qt, qv = queries(torch, B, H, D, "bf16", seed=step)
            k.copy_(new[0][0]), v.copy_(new[1][0]), q.copy_(qt)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            now = start + step + 1
            for b in range(B):
                for sd in range(2):
                    c.put(sd, b, [now[b] - 1], new[sd][1][b:b + 1])
            check_attention(c, qv, o.cpu().numpy(), None, attention64(c, qv, 0.125, lengths=now), "f32")
        c.assert_same()
        assert ctx.take_kernel_status(stream) == 0
        ap.destroy(), at.destroy()


@pytest.mark.parametrize("form", ["bf16", "i8"])
def test_rows_beyond_32_bits(gpu, form):
    """A cache of more than 2^32 elements a side: its last pages are written, read and attended to."""
    fe, torch, ctx, stream = gpu
    KH, D, page = 8, 128, 64
    pages = (1 << 32) // (KH * D * page) + 40
    dt = torch.int16 if form == "bf16" else torch.int8
    caches = [torch.empty(pages, KH, page, D, dtype=dt, device="cuda") for _ in range(2)]
    scales = [torch.empty(pages, KH, page, device="cuda") if form != "bf16" else None for _ in range(2)]
    n = 150
    table = torch.tensor([[pages - 1, 3, pages - 39]], dtype=torch.int32, device="cuda")
    base = dict(k_cache=caches[0], v_cache=caches[1], k_scales=scales[0], v_scales=scales[1], page_table=table,
                lengths=torch.tensor([n], dtype=torch.int32, device="cuda"), batch=1, kv_heads=KH, dim=D, page_size=page, table_width=3,
                format=CODE[form])
    rng = np.random.default_rng(6)
    rows = [rows_in(torch, rng.normal(size=(n, KH, D)), "bf16") for _ in range(2)]
    kw = dict(token_offsets=torch.tensor([0, n], dtype=torch.int32, device="cuda"), tokens=n, **contiguous(KH, D))
    fe.prepare(ctx, "kv_cache_append_v1", k=rows[0][0], v=rows[1][0], input_dtype=1, **kw, **base).launch_and_wait(stream)
    back = [torch.zeros(n, KH, D, device="cuda") for _ in range(2)]
    fe.prepare(ctx, "kv_cache_read_v1", k=back[0], v=back[1], output_dtype=0, **kw, **base).launch_and_wait(stream)
    held = []
    for side in range(2):
        x = rows[side][1]
        held.append(x.astype(np.float64) if form == "bf16" else values_of(*quantised(x, form), form))
        assert (back[side].cpu().numpy() == held[side].astype(np.float32)).all()
    q, qv = queries(torch, 1, KH, D, "bf16")
    o = torch.zeros(1, KH, D, device="cuda")
    fe.prepare(ctx, "paged_attention_v1", q=q, output=o, heads=KH, q_stride=KH * D, q_head_stride=D, scale=D ** -0.5, window=0, q_dtype=1,
               output_dtype=0, **base).launch_and_wait(stream)
    s = np.einsum("hd,nhd->hn", qv[0].astype(np.float64), held[0]) * D ** -0.5
    p = np.exp(s - s.max(-1, keepdims=True))
    want = np.einsum("hn,nhd->hd", p / p.sum(-1, keepdims=True), held[1])
    assert np.abs(o.cpu().numpy()[0] - want).max() <= 1e-4


# ---- the cache as a serving program keeps it ---------------------------------------------------------------------------

@pytest.mark.parametrize("form", FORMATS)
def test_cache_object_serves_prompts_and_steps(gpu, form):
    """Prompts of unlike lengths, steps over page ends, a request that ends and another that takes its place."""
    fe, torch, ctx, stream = gpu
    from fe2o3_b200.kv_cache import DecodeStep, PagedKvCache
    B, H, KH, D = 4, 6, 2, 48
    cache = PagedKvCache(ctx, stream, sequences=B, positions=64, kv_heads=KH, dim=D, page_size=8, pages=14, format=CODE[form])
    rng = np.random.default_rng(11)
    held = [[np.zeros((0, KH, D)) for _ in range(B)] for _ in range(2)]   # f64 values, by side and sequence

    def keep(side, b, rows):
        code = to_bf16(rows) if form == "bf16" else quantised(rows, form)
        values = values_of(code, None, form) if form == "bf16" else values_of(*code, form)
        held[side][b] = np.concatenate([held[side][b], values])

    def prompt(counts):
        cache.extend(counts)
        rows = [rows_in(torch, rng.normal(size=(sum(counts), KH, D)), "f32") for _ in range(2)]
        torch.cuda.synchronize()
        cache.append(rows[0][0], rows[1][0])
        at = np.concatenate([[0], np.cumsum(counts)])
        for side in range(2):
            for b in range(B):
                keep(side, b, rows[side][1][at[b]:at[b + 1]])

    q, k, v = (torch.zeros(B, n, D, dtype=torch.bfloat16, device="cuda") for n in (H, KH, KH))
    out, lse = torch.zeros(B, H, D, device="cuda"), torch.zeros(B, H, device="cuda")
    step = DecodeStep(cache, q, k, v, out, heads=H, lse=lse)

    def steps(n):
        for _ in range(n):
            new = [rows_in(torch, rng.normal(size=(B, m, D)), "bf16") for m in (H, KH, KH)]
            for t, (x, _) in zip((q, k, v), new):
                t.copy_(x)
            torch.cuda.synchronize()
            step.run()
            stream.synchronize()
            got = out.cpu().numpy()
            for b in range(B):
                if len(held[0][b]) == 0:
                    assert (got[b] == 0).all() and (lse[b].cpu().numpy() == -np.inf).all()
                    continue
                for side in range(2):
                    keep(side, b, new[1 + side][1][b:b + 1])
                for h in range(H):
                    s = held[0][b][:, h // 3] @ new[0][1][b, h].astype(np.float64) * D ** -0.5
                    p = np.exp(s - s.max())
                    want = p @ held[1][b][:, h // 3] / p.sum()
                    assert np.abs(got[b, h] - want).max() <= 1e-4
        assert ctx.take_kernel_status(stream) == 0

    prompt([7, 0, 20, 1])
    steps(3)
    cache.release(2)
    for side in range(2):
        held[side][2] = np.zeros((0, KH, D))
    steps(2)
    prompt([0, 9, 30, 0])
    steps(9)
    counts = [len(x) for x in held[0]]
    assert cache.table.lengths.tolist() == counts
    back = [torch.zeros(sum(counts), KH, D, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    cache.read(back[0], back[1], counts)
    for side in range(2):
        assert (back[side].cpu().numpy() == np.concatenate(held[side]).astype(np.float32)).all()
    with pytest.raises(MemoryError):
        cache.extend([0, 40, 0, 0])
    once = torch.zeros(B, H, D, device="cuda")
    torch.cuda.synchronize()
    cache.attend(q, once, H)
    stream.synchronize()
    assert torch.equal(once, out)
    step.destroy()
    cache.free()


def test_example_runs(gpu):
    import os
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, os.path.join(root, "examples"))
    try:
        import paged_decode
    finally:
        sys.path.pop(0)
    # bf16 projections and residuals of unit size: two roundings of 2^-9 a step on either side of the comparison
    assert paged_decode.main(["--sequences", "16", "--prompt", "40", "--steps", "5", "--heads", "4", "--dim", "64", "--format", "bf16"]) <= 2e-2
