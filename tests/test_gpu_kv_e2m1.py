"""The key-value cache in 4 bits on the GPU: what is written, bit for bit, what is read back, and attention over it against 64 bits.

Every slot of a cache that no test row was written to holds NaN (in its row scale and its block scales).
"""
import math

import numpy as np
import pytest

from test_gpu_kv_cache import (E4M3, EDGES, Cache, attend, attention64, check_attention, contiguous, from_bf16, gpu, nearest_e4m3, queries, rows_in,
                               to_bf16)  # noqa: F401  (gpu is a fixture)

pytestmark = pytest.mark.gpu

E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])
f32 = np.float32


def nearest_e2m1(y):
    """Codes of the nearest values, ties to the even code; beyond 6 it stays 6."""
    a = np.abs(y.astype(np.float64))
    hi = np.clip(np.searchsorted(E2M1[:8], a), 1, 7)
    down, up = a - E2M1[hi - 1], E2M1[hi] - a
    c = np.where((down < up) | ((down == up) & (hi % 2 == 1)), hi - 1, hi).astype(np.uint8)
    return c | (np.signbit(y).astype(np.uint8) << 3)


def quantised4(x):
    """Codes (one a byte), block scales' bytes and row scales of f32 rows."""
    x = np.asarray(x, f32)
    with np.errstate(all="ignore"):
        m = np.abs(x).max(-1)
        bad, none = ~np.isfinite(x).all(-1), m < f32(2.0 ** -100)
        scale = np.where(bad, f32(np.nan), np.where(none, f32(0), m / f32(2688))).astype(f32)
        up = np.where(bad | none, f32(0), f32(448) / m).astype(f32)
        blocks = x.reshape(x.shape[:-1] + (-1, 16))
        y = (np.abs(blocks).max(-1) * up[..., None]).astype(f32)
        b = np.where((bad | none)[..., None], np.uint8(0), nearest_e4m3(y))
        factor = (f32(1) / (E4M3[b].astype(f32) * scale[..., None])).astype(f32)
        code = nearest_e2m1((blocks * factor[..., None]).astype(f32))
    code = np.where(b[..., None] == 0, np.uint8(0), code).reshape(x.shape)
    return code, b, scale


def values4(code, b, scale):
    """f64 values that stored rows stand for."""
    v = E2M1[code].reshape(code.shape[:-1] + (-1, 16)) * E4M3[b][..., None]
    return v.reshape(code.shape) * scale[..., None].astype(np.float64)


class Four(Cache):
    def __init__(self, gpu, lengths, kv_heads, dim, page, **kw):  # noqa: F811
        super().__init__(gpu, "i8", lengths, kv_heads, dim, page, **kw)
        self.code = [np.full((self.pages, kv_heads, page, dim), 5, np.uint8) for _ in range(2)]
        self.block = [np.full((self.pages, kv_heads, page, dim // 16), 0x7f, np.uint8) for _ in range(2)]

    def packed(self, side):
        c = self.code[side]
        return np.concatenate([(c[..., 0::2] | c[..., 1::2] << 4).reshape(-1), self.block[side].reshape(-1)])

    def to_gpu(self):
        self.d = {"k_cache": self.up(self.packed(0)), "v_cache": self.up(self.packed(1)), "page_table": self.up(self.table),
                  "lengths": self.up(self.lengths.astype(np.uint32)), "k_scales": self.up(self.scale[0]), "v_scales": self.up(self.scale[1])}
        return self

    def args(self):
        return {**super().args(), "format": self.fe.KV_E2M1}

    def put(self, side, b, positions, rows):
        p, s = self.where(b, positions)
        self.code[side][p, :, s], self.block[side][p, :, s], self.scale[side][p, :, s] = quantised4(rows)

    def get(self, side, b, positions):
        p, s = self.where(b, positions)
        return values4(self.code[side][p, :, s], self.block[side][p, :, s], self.scale[side][p, :, s])

    def assert_same(self):
        for i, n in enumerate("kv"):
            got, want = self.d[n + "_cache"].cpu().numpy(), self.packed(i)
            assert (got == want).all(), (n, np.nonzero(got != want)[0][:8], len(want))
            got = self.d[n + "_scales"].cpu().numpy()
            assert ((got == self.scale[i]) | (np.isnan(got) & np.isnan(self.scale[i]))).all(), n


def filled(gpu, lengths, kv_heads, dim, page, seed=1, **kw):  # noqa: F811
    c = Four(gpu, lengths, kv_heads, dim, page, seed=seed, **kw)
    rng = np.random.default_rng(seed)
    spread = np.exp(0.5 * rng.normal(size=dim))
    for b, n in enumerate(c.lengths):
        for side, by in ((0, spread), (1, 1.0)):
            if n:
                c.put(side, b, np.arange(n), rng.normal(size=(n, kv_heads, dim)) * by)
    return c.to_gpu()


# ---- append and read ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kv_heads,dim,page", [(1, 32, 8), (3, 64, 16), (8, 128, 64), (2, 96, 24), (5, 256, 8), (4, 160, 40), (33, 32, 16), (2, 224, 8)])
def test_append_and_read_back_bit_exact(gpu, dtype, kv_heads, dim, page):  # noqa: F811
    torch = gpu[1]
    rng = np.random.default_rng(dim + page)
    new = [5, 0, 1, 70, 0, 2]
    lengths = [n + o for n, o in zip(new, [0, 9, 3, 13, 0, page])]
    c = Four(gpu, lengths, kv_heads, dim, page).to_gpu()
    T = sum(new)
    offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
    rows = [rows_in(torch, rng.normal(size=(T, kv_heads, dim)) * np.exp(rng.normal(size=(T, kv_heads, 1)) * 3) *
                    np.exp(rng.normal(size=(T, kv_heads, dim // 16)) * 2).repeat(16, -1), dtype) for _ in range(2)]
    kw = dict(token_offsets=c.up(offsets), tokens=T, **contiguous(kv_heads, dim))
    c.launch("kv_cache_append_v1", k=rows[0][0], v=rows[1][0], input_dtype=int(dtype == "bf16"), **kw)
    for b, n in enumerate(new):
        if n:
            for side in range(2):
                c.put(side, b, np.arange(lengths[b] - n, lengths[b]), rows[side][1][offsets[b]:offsets[b + 1]])
    c.assert_same()
    for out, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        k, v = (torch.full((T, kv_heads, dim), math.nan, dtype=out, device="cuda") for _ in range(2))
        c.launch("kv_cache_read_v1", k=k, v=v, output_dtype=code, **kw)
        for side, got in enumerate((k, v)):
            want = np.concatenate([c.get(side, b, np.arange(lengths[b] - n, lengths[b])) for b, n in enumerate(new) if n]).astype(f32)
            assert (got.float().cpu().numpy() == (from_bf16(to_bf16(want)) if code else want)).all()
    c.assert_same()


def test_append_special_rows(gpu):  # noqa: F811
    """Zeros of both signs, blocks of zeros, numbers below and at the smallest that are kept, the largest, infinities and NaN, ties."""
    rng = np.random.default_rng(5)
    n, kv_heads, dim = 16, 2, 64
    x = rng.normal(size=(n, kv_heads, dim)).astype(f32)
    x[0], x[1] = 0, -0.0
    x[2, :, 16:32] = -0.0                                   # a block of zeros among others
    x[3, :, ::3] = -0.0
    x[4] *= f32(2.0 ** -120)
    x[5] = np.where(rng.random((kv_heads, dim)) < .5, 1, -1) * f32(2.0 ** -100)
    x[6] = np.where(rng.random((kv_heads, dim)) < .5, 1, -1) * np.nextafter(f32(2.0 ** -100), f32(0))
    x[7] = np.where(rng.random((kv_heads, dim)) < .5, 3.4028235e38, -3.4028235e38)
    x[8] *= f32(1e38) / np.abs(x[8]).max()
    x[9, 0, 3], x[10, 1, 63], x[11, 0, 40] = np.inf, -np.inf, np.nan
    x[12] = np.tile(np.array([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 5.5, 6], f32), dim // 16) * np.repeat([1, 2, 4, -448], 16)   # ties
    x[13, :, :16] *= f32(2.0 ** -12)                        # block scales that are subnormal, or round to 0
    x[13, :, 16:32] *= f32(2.0 ** -15)
    x[14, :, 32:] *= f32(1e-30)
    x[15, :, 1:] = 0
    for dtype in ("f32", "bf16"):
        c = Four(gpu, [n], kv_heads, dim, 8).to_gpu()
        t, xv = rows_in(c.torch, x, dtype)
        kw = dict(token_offsets=c.up(np.array([0, n], np.uint32)), tokens=n, **contiguous(kv_heads, dim))
        c.launch("kv_cache_append_v1", k=t, v=t, input_dtype=int(dtype == "bf16"), **kw)
        for side in range(2):
            c.put(side, 0, np.arange(n), xv)
        c.assert_same()
        k, v = (c.torch.zeros(n, kv_heads, dim, device="cuda") for _ in range(2))
        c.launch("kv_cache_read_v1", k=k, v=v, output_dtype=0, **kw)
        got, want = k.cpu().numpy(), c.get(0, 0, np.arange(n)).astype(f32)
        assert ((got == want) | (np.isnan(got) & np.isnan(want))).all()
        assert np.isnan(got[9, 0]).all() and np.isnan(got[10, 1]).all() and np.isnan(got[11, 0]).all() and np.isfinite(got[9, 1]).all()
        assert (got[4] == 0).all() and (got[6] == 0).all() == (dtype == "f32")   # (as bf16 it is 2^-100)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_error_of_a_row(gpu, dtype):  # noqa: F811
    """Half a step of the code, with a block scale off by a sixteenth: |x - read| <= (1 + 2^-4) / 6 of the block's largest magnitude where
    its scale is a normal e4m3 number (codes 4 and 6 are 2 apart and half of that is a sixth of 6), and nothing beyond 6 is asked for but by
    that sixteenth."""
    rng = np.random.default_rng(6)
    n, kv_heads, dim = 300, 4, 128
    c = Four(gpu, [n], kv_heads, dim, 16).to_gpu()
    t, xv = rows_in(c.torch, rng.normal(size=(n, kv_heads, dim)), dtype)
    kw = dict(token_offsets=c.up(np.array([0, n], np.uint32)), tokens=n, **contiguous(kv_heads, dim))
    c.launch("kv_cache_append_v1", k=t, v=t, input_dtype=int(dtype == "bf16"), **kw)
    k, v = (c.torch.zeros(n, kv_heads, dim, device="cuda") for _ in range(2))
    c.launch("kv_cache_read_v1", k=k, v=v, output_dtype=0, **kw)
    off = np.abs(k.cpu().numpy() - xv).reshape(n, kv_heads, -1, 16)
    largest = np.abs(xv).reshape(n, kv_heads, -1, 16).max(-1, keepdims=True)
    assert (off <= largest * (1 + 2.0 ** -4) / 6 * (1 + 1e-5)).all()


@pytest.mark.parametrize("layout", ["token_major", "head_major", "fused", "odd"])
def test_strided_rows(gpu, layout):  # noqa: F811
    torch = gpu[1]
    kv_heads, dim, page, B = 4, 64, 16, 19
    rng = np.random.default_rng(3)
    lengths = rng.integers(1, 60, B)
    c = Four(gpu, lengths, kv_heads, dim, page).to_gpu()
    ts, hs, off = {"token_major": (kv_heads * dim, dim, 0), "head_major": (dim, B * dim, 0), "fused": (3 * kv_heads * dim, dim, kv_heads * dim),
                   "odd": (kv_heads * (dim + 3) + 5, dim + 3, 1)}[layout]
    extent = (B - 1) * ts + (kv_heads - 1) * hs + dim
    at = off + np.arange(B)[:, None, None] * ts + np.arange(kv_heads)[None, :, None] * hs + np.arange(dim)
    strides = dict(k_token_stride=ts, k_head_stride=hs, v_token_stride=ts, v_head_stride=hs)
    for code, dt in ((0, torch.float32), (1, torch.bfloat16)):
        store = [torch.from_numpy(rng.normal(size=off + extent + 9).astype(f32)).cuda().to(dt) for _ in range(2)]
        sl = lambda t: (t.data_ptr() + off * t.element_size(), extent)  # noqa: E731
        c.launch("kv_cache_append_v1", k=sl(store[0]), v=sl(store[1]), tokens=B, input_dtype=code, **strides)
        for side in range(2):
            rows = store[side].float().cpu().numpy()[at]
            for b in range(B):
                c.put(side, b, [lengths[b] - 1], rows[b:b + 1])
        c.assert_same()
        out = [torch.full((off + extent + 9,), 7.0, device="cuda", dtype=dt) for _ in range(2)]
        c.launch("kv_cache_read_v1", k=sl(out[0]), v=sl(out[1]), tokens=B, output_dtype=code, **strides)
        for side in range(2):
            want = np.full(off + extent + 9, 7.0, f32)
            want[at] = np.stack([c.get(side, b, [lengths[b] - 1])[0] for b in range(B)]).astype(f32)
            assert (out[side].float().cpu().numpy() == (from_bf16(to_bf16(want)) if code else want)).all()


def test_rows_that_do_not_fit_are_reported_and_left_out(gpu):  # noqa: F811
    fe, torch = gpu[:2]
    c = Four(gpu, [16, 14, 16, 15], 2, 32, 8, width=2)
    c.table[3, 1] = c.pages
    c.to_gpu()
    x = torch.ones(8, 2, 32, device="cuda")
    kw = dict(token_offsets=c.up(np.array([0, 3, 4, 5, 8], np.uint32)), tokens=8, lengths=c.up(np.array([2, 14, 17, 15], np.uint32)), **contiguous(2, 32))
    with pytest.raises(fe.Fe2o3Error):
        c.launch("kv_cache_append_v1", k=x, v=x, input_dtype=0, **kw)
    for side in range(2):
        c.put(side, 1, [13], np.ones((1, 2, 32), f32))
    c.assert_same()
    k, v = (torch.full((8, 2, 32), 5.0, device="cuda") for _ in range(2))
    with pytest.raises(fe.Fe2o3Error):
        c.launch("kv_cache_read_v1", k=k, v=v, output_dtype=0, **kw)
    got = k.cpu().numpy()
    assert (got[[0, 1, 2, 4]] == 5).all() and (got[5:] == 0).all() and np.abs(got[3] - 1).max() <= 1 / 6


# ---- attention ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (8, 2), (16, 2), (24, 8), (12, 1), (40, 1), (66, 2), (130, 1)])
def test_attention_heads(gpu, heads, kv_heads):  # noqa: F811
    c = filled(gpu, EDGES, kv_heads, 64, 16)
    q, qv = queries(c.torch, len(EDGES), heads, 64, "bf16")
    got, lse = attend(c, q, 0.125)
    check_attention(c, qv, got, lse, attention64(c, qv, 0.125), "f32")


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("group", [3, 8, 9, 16, 20])
def test_attention_head_sizes_and_types(gpu, dim, dtype, out, group):  # noqa: F811
    lengths = [0, 1, 16, 33, 100, 300]
    c = filled(gpu, lengths, 2, dim, 24)
    q, qv = queries(c.torch, len(lengths), 2 * group, dim, dtype)
    scale = 1 / math.sqrt(dim)
    got, lse = attend(c, q, scale, out=out)
    check_attention(c, qv, got, lse, attention64(c, qv, f32(scale)), out)


@pytest.mark.parametrize("dim,group", [(64, 4), (128, 1), (128, 9), (256, 16)])
def test_attention_bf16_output_is_the_f32_one_rounded(gpu, dim, group):  # noqa: F811
    c = filled(gpu, EDGES + [1000, 3000], 2, dim, 16)
    for dtype in ("bf16", "f32"):
        q, _ = queries(c.torch, len(EDGES) + 2, 2 * group, dim, dtype, by=0.5)
        whole, lse = attend(c, q, dim ** -0.5)
        short, lse2 = attend(c, q, dim ** -0.5, out="bf16")
        assert (short == from_bf16(to_bf16(whole))).all() and (lse == lse2).all()


@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 5, 16, 50, 128, 1000])
def test_attention_pages_and_windows(gpu, page, window):  # noqa: F811
    for dim, group in ((64, 1), (128, 4), (256, 2)):
        c = filled(gpu, EDGES, 2, dim, page)
        q, qv = queries(c.torch, len(EDGES), 2 * group, dim, "bf16")
        got, lse = attend(c, q, 0.125, window=window)
        check_attention(c, qv, got, lse, attention64(c, qv, 0.125, window), "f32")


@pytest.mark.parametrize("dim", [32, 128])
@pytest.mark.parametrize("lengths,heads,kv_heads", [([30011], 4, 1), ([5000, 3], 8, 8), ([9000, 0, 1, 8999, 20], 10, 2), ([70] * 300, 2, 2),
                                                    ([1] * 700, 3, 1), (list(range(0, 500, 3)), 4, 2), ([2049] * 9, 8, 1),
                                                    ([i % 7 * 9 for i in range(1500)], 2, 1), ([64] * 33 + [20000] + [0] * 40, 3, 3)])
def test_attention_split_and_joined(gpu, lengths, heads, kv_heads, dim):  # noqa: F811
    c = filled(gpu, lengths, kv_heads, dim, 16)
    q, qv = queries(c.torch, len(lengths), heads, dim, "bf16", by=2.0)
    scale = dim ** -0.5
    got, lse = attend(c, q, scale)
    check_attention(c, qv, got, lse, attention64(c, qv, f32(scale)), "f32")
    again, lse2 = attend(c, q, scale)
    assert (got == again).all() and (lse == lse2).all()


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("group,dtype", [(1, "bf16"), (4, "f32"), (8, "bf16")])
def test_attention_tables_with_room_for_long_rows(gpu, dim, group, dtype):  # noqa: F811
    """Tables of 4096 positions and more, in pages of whole tiles of 64 keys: lengths around those, empty ones, windows, pieces that blocks join."""
    for page, lengths in ((64, EDGES + [1000, 4096, 4500]), (128, [9000, 0, 1, 8999, 20]), (192, [64] * 33 + [5000] + [0] * 9)):
        c = filled(gpu, lengths, 2, dim, page, width=-(-9100 // page))
        q, qv = queries(c.torch, len(lengths), 2 * group, dim, dtype)
        for window in (0, 4100):
            got, lse = attend(c, q, dim ** -0.5, window=window)
            check_attention(c, qv, got, lse, attention64(c, qv, f32(dim ** -0.5), window), "f32")
        again, lse2 = attend(c, q, dim ** -0.5, window=4100)
        assert (got == again).all() and (lse == lse2).all()


@pytest.mark.parametrize("octaves", [10, 20, 30, 45, 60])
def test_attention_values_of_unlike_size(gpu, octaves):  # noqa: F811
    """A row of values far larger than the others, which one head gives next to no weight and another next to all of it.  (No value of it is small
    against its row: 4 bits round those to 0, and what lies under a 0 of the heaviest row is held as the weights are.)"""
    lengths = [2, 20, 40, 333, 3000] + [300] * 50
    for dim in (32, 128):
        c = Four(gpu, lengths, 1, dim, 16)
        rng = np.random.default_rng(12)
        for b, n in enumerate(c.lengths):
            big = [0, n - 1, n // 2, n // 3][b % 4]
            k, v = rng.normal(size=(n, 1, dim)) * 0.01, rng.normal(size=(n, 1, dim)) * 2.0 ** -octaves
            k[:, 0, 0], v[big] = 0.0, rng.choice([-1, 1], (1, dim)) * rng.uniform(0.5, 1, (1, dim))
            k[big, 0, 0] = (octaves + 6) * math.log(2)
            if b % 3 == 0:
                v[(big + 1) % n] = 0
            c.put(0, b, np.arange(n), k)
            c.put(1, b, np.arange(n), v)
        c.to_gpu()
        q = rng.normal(size=(len(lengths), 4, dim))
        q[:, :, 0] = [-1.0, 1.0, -1.5, 0.0]
        for dtype, out in (("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")):
            qt, qv = rows_in(c.torch, q, dtype)
            got, lse = attend(c, qt, 1.0, out=out)
            check_attention(c, qv, got, lse, attention64(c, qv, 1.0), out)


@pytest.mark.parametrize("page,width", [(16, None), (64, 80)])
@pytest.mark.parametrize("rise", [0.5, 3.0, 5.5, 20.0])
def test_attention_rising_scores_over_rows_of_zeros(gpu, page, width, rise):  # noqa: F811
    """Scores that rise tile by tile, by less or more than what moves the maximum kept, while the values are zeros; then tiny, ordinary and the largest
    ones.  Many sequences of the same, for several tiles a warp."""
    n, many = 1200, 500
    for size in (0.0, 2.0 ** -90, 1.0, 1e37):
        c = Four(gpu, [n], 1, 64, page, width=width)
        k, v = np.zeros((n, 1, 64)), np.zeros((n, 1, 64))
        k[:, 0, 0] = np.minimum(np.arange(n) // 64, 12) * rise
        v[-100:] = np.random.default_rng(1).choice([-1, 1], (100, 1, 64)) * size
        c.put(0, 0, np.arange(n), k)
        c.put(1, 0, np.arange(n), v)
        c.to_gpu()
        q = c.torch.zeros(many, 3, 64, device="cuda")
        q[:, :, 0] = c.torch.tensor([1.0, 0.3, -1.0])
        got, lse = attend(c, q, 1.0, batch=many, page_table=c.up(c.table.repeat(many, 0)), lengths=c.up(np.full(many, n, np.uint32)))
        o, l64, mag, big = attention64(c, q[:1].cpu().numpy(), 1.0)
        d = (72 * 2.0 ** -23 + 2.0 ** -22) * big
        # a probability below f32's normal numbers, 2^-126, is 0; a weight is held to 2^-25 in units of at most 2^118, the least largest one's, and
        # counts up to 2688 times: 2^-131 a key (probabilities against the first maximum kept are at most 2^8, and their sum no less than 2^-8 ones)
        least = n * 2.0 ** 16 * (2.0 ** -126 * size + 2.0 ** -131)
        bound = (2 * d + 2.0 ** -19 + n * 2.0 ** -24)[..., None] * mag + n * 2.0 ** -39 * mag.max(-1, keepdims=True) + least
        assert (np.abs(got - o) <= bound).all(), (size, float(np.nanmax(np.abs(got - o) / bound)), np.isnan(got).sum())
        assert (np.abs(lse - l64) <= d + 2.0 ** -20 + n * 2.0 ** -24 + 2.0 ** -22 * np.abs(l64)).all()


@pytest.mark.parametrize("spread", [2, 6, 10])
def test_attention_blocks_of_unlike_size(gpu, spread):  # noqa: F811
    """Blocks of 16 columns whose sizes lie 2^spread apart, in keys and in values, each column to its own accuracy."""
    lengths = [1, 37, 700]
    for dim in (64, 96, 128, 256):
        c = Four(gpu, lengths, 2, dim, 16)
        rng = np.random.default_rng(dim)
        by = 2.0 ** (-spread * rng.random((2, dim // 16))).repeat(16, -1)
        for b, n in enumerate(c.lengths):
            for side in range(2):
                c.put(side, b, np.arange(n), rng.normal(size=(n, 2, dim)) * by[side])
        c.to_gpu()
        q, qv = queries(c.torch, 3, 8, dim, "bf16")
        got, lse = attend(c, q, dim ** -0.5)
        check_attention(c, qv, got, lse, attention64(c, qv, f32(dim ** -0.5)), "f32")


@pytest.mark.parametrize("scale", [0.0, -0.3, 25.0])
def test_attention_scales(gpu, scale):  # noqa: F811
    """At 25 a weight or two is far above the others, and 4 bits hold many a column of its row as 0: what is left there are the small weights.
    A weight, probability times row scale, is held to 2^-25 where the head's largest, W, lies in [2^14, 2^15): to 2^-39 W.  Its key adds that
    times at most 2688, a row's largest code times block scale, to a column; W times 2688 is the heaviest row's largest element times its
    probability (6 times 448 is what the largest element of every row becomes), no more than the largest sum of p|v| of the head's columns:
    n keys add n 2^-39 of that to the bound of the other tests."""
    c = filled(gpu, [1, 50, 700], 1, 64, 16)
    q, qv = queries(c.torch, 3, 4, 64, "bf16")
    got, lse = attend(c, q, scale)
    o, l64, mag, big = attention64(c, qv, f32(scale))
    n = np.asarray(c.lengths, np.float64)[:, None]
    d = ((c.dim + 8) * 2.0 ** -23 + 2.0 ** -22) * big
    bound = (2 * d + 2.0 ** -19 + n * 2.0 ** -24)[..., None] * mag + (n * 2.0 ** -39)[..., None] * mag.max(-1, keepdims=True)
    assert (np.abs(got - o) <= bound).all(), float((np.abs(got - o) / bound).max())
    check_attention(c, qv, o, lse, (o, l64, mag, big), "f32")


def test_attention_infinities_and_nan(gpu):  # noqa: F811
    """A row that held an infinity or a NaN is NaN for its own (sequence, key head) and nothing else."""
    c = filled(gpu, [40, 41, 300, 17], 2, 64, 16)
    rows = np.ones((1, 2, 64), f32)
    rows[0, 1, 5] = np.inf
    c.put(0, 1, [7], rows)
    rows[0, 1, 5] = np.nan
    c.put(1, 2, [299], rows)
    c.to_gpu()
    q, qv = queries(c.torch, 4, 4, 64, "bf16")
    got, lse = attend(c, q, 0.125)
    assert np.isnan(got[1, 2:]).all() and np.isnan(lse[1, 2:]).all() and np.isnan(got[2, 2:]).all()
    keep = np.ones((4, 4), bool)
    keep[1, 2:] = keep[2, 2:] = False
    with np.errstate(all="ignore"):
        o = attention64(c, qv, 0.125)[0]
    assert np.abs(got[keep] - o[keep]).max() <= 1e-4 and np.isfinite(lse[1:3, :2]).all() and np.isfinite(lse[2]).all()


@pytest.mark.parametrize("page,width", [(16, None), (64, 70)])
def test_attention_reports(gpu, page, width):  # noqa: F811
    """A length that the table cannot hold leaves that sequence unwritten; rows of a page outside the cache count as zeros; a cache without pages."""
    fe, torch, ctx, stream = gpu
    lengths = [page * 5 // 2, 30, 2 * page + 1]
    c = filled(gpu, lengths, 2, 64, page, width=width)
    q, qv = queries(torch, 3, 4, 64, "bf16")
    want = attention64(c, qv, 0.125)[0]
    o = torch.full((3, 4, 64), 7.0, device="cuda")
    kw = dict(q=q, output=o, heads=4, q_stride=256, q_head_stride=64, scale=0.125, window=0, q_dtype=1, output_dtype=0)
    with pytest.raises(fe.Fe2o3Error):
        c.launch("paged_attention_v1", **kw, lengths=c.up(np.array([lengths[0], c.width * page + 1, lengths[2]], np.uint32)))
    got = o.cpu().numpy()
    assert (got[1] == 7).all() and np.abs(got[[0, 2]] - want[[0, 2]]).max() <= 1e-4
    table = c.table.copy()
    table[2, 1] = c.pages
    with pytest.raises(fe.Fe2o3Error):
        c.launch("paged_attention_v1", **kw, page_table=c.up(table))
    got = o.cpu().numpy()
    k, v = (c.get(side, 2, np.arange(lengths[2])) for side in range(2))
    k[page:2 * page] = v[page:2 * page] = 0
    for h in range(4):
        p = np.exp(k[:, h // 2] @ qv[2, h] * 0.125)
        assert np.abs(got[2, h] - p @ v[:, h // 2] / p.sum()).max() <= 1e-4
    assert np.abs(got[:2] - want[:2]).max() <= 1e-4
    none = dict(k_cache=None, v_cache=None, k_scales=None, v_scales=None)
    with pytest.raises(fe.Fe2o3Error):
        c.launch("paged_attention_v1", **kw, **none)
    assert (o.cpu().numpy() == 0).all()


def test_attention_of_an_empty_batch_and_of_empty_sequences(gpu):  # noqa: F811
    c = filled(gpu, [0, 0, 0], 2, 128, 16)
    q, _ = queries(c.torch, 3, 4, 128, "bf16")
    got, lse = attend(c, q, 0.1)
    assert (got == 0).all() and (lse == -np.inf).all()


def test_rows_beyond_32_bits(gpu):  # noqa: F811
    """A cache whose codes and block scales lie past 2^32 bytes: its last pages are written, read and attended to."""
    fe, torch, ctx, stream = gpu
    KH, D, page, n = 8, 128, 64, 150
    pages = (1 << 32) // (KH * D // 2 * page) + 40
    rows = pages * KH * page
    caches = [torch.empty(rows * D // 16 * 9, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.empty(rows, device="cuda") for _ in range(2)]
    base = dict(k_cache=caches[0], v_cache=caches[1], k_scales=scales[0], v_scales=scales[1], batch=1, kv_heads=KH, dim=D, page_size=page, table_width=3,
                page_table=torch.tensor([[pages - 1, 3, pages - 39]], dtype=torch.int32, device="cuda"),
                lengths=torch.tensor([n], dtype=torch.int32, device="cuda"), format=fe.KV_E2M1)
    rng = np.random.default_rng(6)
    x = [rows_in(torch, rng.normal(size=(n, KH, D)), "bf16") for _ in range(2)]
    kw = dict(token_offsets=torch.tensor([0, n], dtype=torch.int32, device="cuda"), tokens=n, **contiguous(KH, D))
    fe.prepare(ctx, "kv_cache_append_v1", k=x[0][0], v=x[1][0], input_dtype=1, **kw, **base).launch_and_wait(stream)
    back = [torch.zeros(n, KH, D, device="cuda") for _ in range(2)]
    fe.prepare(ctx, "kv_cache_read_v1", k=back[0], v=back[1], output_dtype=0, **kw, **base).launch_and_wait(stream)
    held = [values4(*quantised4(r[1])) for r in x]
    for side in range(2):
        assert (back[side].cpu().numpy() == held[side].astype(f32)).all()
    q, qv = queries(torch, 1, KH, D, "bf16")
    o = torch.zeros(1, KH, D, device="cuda")
    fe.prepare(ctx, "paged_attention_v1", q=q, output=o, heads=KH, q_stride=KH * D, q_head_stride=D, scale=D ** -0.5, window=0, q_dtype=1,
               output_dtype=0, **base).launch_and_wait(stream)
    s = np.einsum("hd,nhd->hn", qv[0].astype(np.float64), held[0]) * D ** -0.5
    p = np.exp(s - s.max(-1, keepdims=True))
    want = np.einsum("hn,nhd->hd", p / p.sum(-1, keepdims=True), held[1])
    assert np.abs(o.cpu().numpy()[0] - want).max() <= 1e-4
