"""A paged key-value cache and the decode step over it, for serving.

`PageTable` is the host's book of pages (no GPU).  `PagedKvCache` owns the cache's device memory in one of three formats
and launches the library's operators on it: `append` writes new tokens' keys and values, `attend` lets one new token a
sequence attend to all its positions, `read` brings rows back.  `DecodeStep` binds the tensors of a step once, so that a
step is two launches and the copy of the lengths; a step in which a sequence begins a page copies the whole page table too
(4 bytes a page that the table has room for), from ordinary memory.

    cache = PagedKvCache(ctx, stream, sequences=8, positions=4096, kv_heads=8, dim=128, format=KV_E4M3)
    cache.extend([prompt_length] * 8)           # pages for the prompts' tokens
    cache.append(k, v)                          # rows [tokens][kv_heads][dim], sequence after sequence
    step = DecodeStep(cache, q, k1, v1, out, heads=32, lse=None)
    for _ in range(n):                          # fill q, k1, v1 on the stream, then
        step.run()

`append`, `extend`, `release` and the steps are enqueued on the cache's stream and do not wait for its launches (but a copy from
ordinary memory may hold the host until the stream has come to it, once it is larger than the driver keeps aside).  What waits:
preparing an attention (`attention`, `DecodeStep`) for the legacy stream, destroying one for the whole device, `attend`, which
does both, and `read` for the cache's stream.
"""
import numpy as np

from . import DTYPE_BF16, DTYPE_F32, KV_BF16, KV_E4M3, KV_I8, DeviceBuffer, prepare


class PageTable:
    """Pages of every sequence, in order, and how many positions each has."""

    FREE = 0xFFFFFFFF

    def __init__(self, sequences, positions, pages, page_size):
        if min(sequences, positions, pages, page_size) < 1:
            raise ValueError("sequences, positions, pages and page_size are at least 1")
        self.page_size = page_size
        self.entries = np.full((sequences, -(-positions // page_size)), self.FREE, np.uint32)
        self.lengths = np.zeros(sequences, np.uint32)
        self.free = list(range(pages - 1, -1, -1))   # the next page is the last of the list

    def extend(self, counts):
        """Positions for `counts[b]` new tokens of every sequence b; all of them or, with an error, none."""
        counts = np.asarray(counts)
        if counts.shape != self.lengths.shape or (counts < 0).any():
            raise ValueError(f"counts has one number, at least 0, for each of the {len(self.lengths)} sequences")
        after = self.lengths.astype(np.int64) + counts
        held, need = -(-self.lengths.astype(np.int64) // self.page_size), -(-after // self.page_size)
        if (need > self.entries.shape[1]).any():
            raise ValueError(f"sequence {int(np.argmax(need))}: more than {self.entries.shape[1] * self.page_size} positions")
        if int((need - held).sum()) > len(self.free):
            raise MemoryError(f"{int((need - held).sum())} pages wanted, {len(self.free)} are free")
        for b in np.nonzero(need > held)[0]:
            for i in range(held[b], need[b]):
                self.entries[b, i] = self.free.pop()
        self.lengths[:] = after

    def release(self, sequence):
        """Gives a finished sequence's pages back; its slot starts again at no positions."""
        used = -(-int(self.lengths[sequence]) // self.page_size)
        self.free.extend(int(p) for p in self.entries[sequence, :used][::-1])
        self.entries[sequence] = self.FREE
        self.lengths[sequence] = 0


def _float_dtype(x, dtype):
    """DTYPE_* of rows: by the tensor's own type, or as said."""
    if dtype is not None:
        return dtype
    name = str(getattr(x, "dtype", ""))
    if name.endswith("bfloat16") or name == "uint16":
        return DTYPE_BF16
    if name.endswith("float32"):
        return DTYPE_F32
    raise TypeError(f"rows are f32 or bf16 (bits as uint16), got {name or type(x)}: say dtype=")


def _contiguous(*tensors):
    for x in tensors:
        if hasattr(x, "is_contiguous") and not x.is_contiguous():
            raise ValueError("a tensor is contiguous here; rows inside wider storage come as (address, elements) with their strides")


def _pair_dtype(k, v, dtype):
    """DTYPE_* of k and v, which are of one type."""
    one = _float_dtype(k, dtype)
    if hasattr(v, "dtype") and _float_dtype(v, dtype) != one:
        raise TypeError(f"k and v are of one type, got {k.dtype} and {v.dtype}")
    return one


class PagedKvCache:
    def __init__(self, ctx, stream, sequences, positions, kv_heads, dim, page_size=16, pages=None, format=KV_BF16):
        """Room for `sequences` of up to `positions` tokens each in `pages` pages (default: enough for all at their
        longest)."""
        self.ctx, self.stream, self.format = ctx, stream, format
        pages = sequences * -(-positions // page_size) if pages is None else pages
        self.table = PageTable(sequences, positions, pages, page_size)
        self.sequences, self.kv_heads, self.dim, self.page_size = sequences, kv_heads, dim, page_size
        rows = pages * kv_heads * page_size
        element = {KV_BF16: np.uint16, KV_E4M3: np.uint8, KV_I8: np.int8}[format]
        self.k_cache, self.v_cache = (DeviceBuffer.zeroed(stream, rows * dim, element) for _ in range(2))
        self.k_scales, self.v_scales = ((DeviceBuffer.zeroed(stream, rows, np.float32) if format != KV_BF16 else None) for _ in range(2))
        self.device_table = DeviceBuffer.from_host(stream, self.table.entries)
        self.device_lengths = DeviceBuffer.from_host(stream, self.table.lengths)
        self.device_offsets = DeviceBuffer.zeroed(stream, sequences + 1, np.uint32)
        self.new_tokens = 0

    def args(self):
        """The cache's own arguments of the three operators."""
        return dict(k_cache=self.k_cache, v_cache=self.v_cache, k_scales=self.k_scales, v_scales=self.v_scales, page_table=self.device_table,
                    lengths=self.device_lengths, batch=self.sequences, kv_heads=self.kv_heads, dim=self.dim, page_size=self.page_size,
                    table_width=self.table.entries.shape[1], format=self.format)

    def _upload(self, pages_changed=True):
        # (arrays in ordinary memory: the copies have read them when the calls return)
        if pages_changed:
            self.device_table.copy_from_host_async(self.stream, self.table.entries)
        self.device_lengths.copy_from_host_async(self.stream, self.table.lengths)

    def extend(self, counts):
        """Positions for new tokens of every sequence; `append` then writes them."""
        before = len(self.table.free)
        self.table.extend(counts)
        offsets = np.zeros(self.sequences + 1, np.uint32)
        offsets[1:] = np.cumsum(counts)
        self.new_tokens = int(offsets[-1])
        self._upload(len(self.table.free) != before)
        self.device_offsets.copy_from_host_async(self.stream, offsets)

    def release(self, sequence):
        self.table.release(sequence)
        self._upload()

    def _rows(self, k, v, tokens, strides):
        _contiguous(k, v)
        packed = (self.kv_heads * self.dim, self.dim)
        (kt, kh), (vt, vh) = strides or (packed, packed)
        return dict(k=k, v=v, tokens=tokens, k_token_stride=kt, k_head_stride=kh, v_token_stride=vt, v_head_stride=vh)

    def _launch(self, op, **kw):
        p = prepare(self.ctx, op, **kw, **self.args())
        try:
            p.launch(self.stream)
        finally:
            p.destroy()

    def append(self, k, v, dtype=None, strides=None):
        """Rows of the tokens of the last `extend`, sequence after sequence: [tokens][kv_heads][dim], or with `strides`
        ((k token, k head), (v token, v head)) in elements, as slices (address, elements)."""
        self._launch("kv_cache_append_v1", token_offsets=self.device_offsets, input_dtype=_pair_dtype(k, v, dtype),
                     **self._rows(k, v, self.new_tokens, strides))

    def read(self, k, v, counts, dtype=None, strides=None):
        """The last `counts[b]` rows of every sequence b into k and v, which are there when this returns."""
        kw = dict(output_dtype=_pair_dtype(k, v, dtype))
        offsets = np.zeros(self.sequences + 1, np.uint32)
        offsets[1:] = np.cumsum(counts)
        kw.update(self._rows(k, v, int(offsets[-1]), strides))
        at = DeviceBuffer.from_host(self.stream, offsets)
        self._launch("kv_cache_read_v1", token_offsets=at, **kw)
        self.stream.synchronize()   # before the offsets go
        at.free()

    def attention(self, q, out, heads, lse=None, scale=None, window=0, q_dtype=None, out_dtype=None, q_strides=None):
        """A prepared launch of `paged_attention_v1` over this cache; the caller launches and destroys it."""
        _contiguous(q, out, lse)
        qs, qh = q_strides or (heads * self.dim, self.dim)
        return prepare(self.ctx, "paged_attention_v1", q=q, output=out, lse=lse, heads=heads, q_stride=qs, q_head_stride=qh,
                       scale=self.dim ** -0.5 if scale is None else scale, window=window, q_dtype=_float_dtype(q, q_dtype),
                       output_dtype=_float_dtype(out, out_dtype), **self.args())

    def attend(self, q, out, heads, **kw):
        """One new token a sequence, q and out [sequences][heads][dim].  Returns when the device is idle, since the launch's workspace
        goes back: a program that attends again and again keeps an `attention` or a `DecodeStep`."""
        p = self.attention(q, out, heads, **kw)
        try:
            p.launch(self.stream)
        finally:
            p.destroy()

    def free(self):
        for b in (self.k_cache, self.v_cache, self.k_scales, self.v_scales, self.device_table, self.device_lengths, self.device_offsets):
            if b is not None:
                b.free()


class DecodeStep:
    """One new token of every sequence at work (of length above 0): its key and value are written, then it attends to all
    positions so far and its own.  The tensors, a row a sequence, stay where they are from step to step; the caller fills
    q, k and v on the cache's stream.  Rows of released sequences are not read, and their output is zeros."""

    def __init__(self, cache, q, k, v, out, heads, lse=None, scale=None, window=0, dtype=None, out_dtype=None, strides=None, q_strides=None):
        self.cache = cache
        self.attend = cache.attention(q, out, heads, lse, scale, window, dtype, out_dtype, q_strides)
        self.append = prepare(cache.ctx, "kv_cache_append_v1", input_dtype=_pair_dtype(k, v, dtype),
                              **cache._rows(k, v, cache.sequences, strides), **cache.args())

    def run(self):
        cache = self.cache
        before = len(cache.table.free)
        cache.table.extend((cache.table.lengths > 0).astype(np.int64))
        cache._upload(len(cache.table.free) != before)
        self.append.launch(cache.stream)
        self.attend.launch(cache.stream)

    def destroy(self):
        self.append.destroy()
        self.attend.destroy()
