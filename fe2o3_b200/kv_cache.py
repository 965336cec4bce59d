"""A paged key-value cache and the decode step over it, for serving.

`PageTable` is the host's book of pages (no GPU), `DevicePages` one on the device, whose steps need nothing from the host and can be
captured in a CUDA graph.  `PagedKvCache` owns the cache's device memory in one of four formats and launches the library's operators on it: `append` writes new tokens' keys and values, `attend` lets one new token a
sequence attend to all its positions, `read` brings rows back.  `DecodeStep` binds the tensors of a step once, so that a
step is two launches and the copy of the lengths, or three launches with a book on the device; a step in which a sequence begins a page copies the whole page table too
(4 bytes a page that the table has room for), from ordinary memory.

    cache = PagedKvCache(ctx, stream, sequences=8, positions=4096, kv_heads=8, dim=128, format=KV_E4M3)
    cache.extend([prompt_length] * 8)           # pages for the prompts' tokens
    cache.append(k, v)                          # rows [tokens][kv_heads][dim], sequence after sequence
    step = DecodeStep(cache, q, k1, v1, out, heads=32, lse=None)
    for _ in range(n):                          # fill q, k1, v1 on the stream, then
        step.run()

    cache = PagedKvCache(ctx, stream, 8, 4096, 8, 128, format=KV_E2M1, tokens=8 * prompt_length)   # with a book on the device
    cache.extend([prompt_length] * 8)
    cache.append(k, v, q=q, q_out=turned, heads=32, rotary=rotary)   # rotary positions on the way
    step = DecodeStep(cache, q1, k1, v1, out, heads=32, rotary=rotary)

`append`, `extend`, `release` and the steps are enqueued on the cache's stream and do not wait for its launches (but a copy from
ordinary memory may hold the host until the stream has come to it, once it is larger than the driver keeps aside).  What waits:
preparing an attention (`attention`, `DecodeStep`) for the legacy stream, destroying one for the whole device, `attend`, which
does both, and `read` for the cache's stream.
"""
import operator

import numpy as np

from . import DTYPE_BF16, DTYPE_F32, KV_BF16, KV_E2M1, KV_E4M3, KV_I8, DeviceBuffer, prepare


def _new_tokens(counts, sequences):
    """New tokens of every sequence, as 64-bit integers."""
    counts = np.asarray(counts)
    if counts.shape != (sequences,) or not (counts >= 0).all() or (counts > 0x7fffffff).any() or (counts.dtype.kind not in "biu" and (counts % 1 != 0).any()):
        raise ValueError(f"counts has a whole number, from 0 on and below 2^31, for each of the {sequences} sequences")
    return counts.astype(np.int64)


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
        counts = _new_tokens(counts, len(self.lengths))
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


def _mask(release, sequences):
    """Which sequences give their pages back: a truth value each."""
    release = np.zeros(sequences, bool) if release is None else np.asarray(release).astype(bool)
    if release.shape != (sequences,):
        raise ValueError(f"release has a truth value for each of the {sequences} sequences")
    return release


class DevicePages:
    """The same book on the device (`kv_pages_v1`): pages go out and come back in the same order.  What does not fit is found there too: it is reported
    (`ctx.take_kernel_status`), and nothing changes.  `tokens`: the most new tokens of an `extend`."""

    def __init__(self, ctx, stream, sequences, positions, pages, page_size, tokens):
        if min(sequences, positions, pages, page_size, tokens) < 1:
            raise ValueError("sequences, positions, pages, page_size and tokens are at least 1")
        self.stream, self.width, self.tokens = stream, -(-positions // page_size), tokens
        self.table = DeviceBuffer.from_host(stream, np.full((sequences, self.width), PageTable.FREE, np.uint32))
        self.free_pages = DeviceBuffer.from_host(stream, np.arange(pages - 1, -1, -1, dtype=np.uint32))
        self.free_count = DeviceBuffer.from_host(stream, np.array([pages], np.uint32))
        zeros = lambda n: DeviceBuffer.zeroed(stream, n, np.uint32)  # noqa: E731
        self.lengths, self.counts, self.released, self.offsets = zeros(sequences), zeros(sequences), zeros(sequences), zeros(sequences + 1)
        self.attended = zeros(sequences)   # lengths after a step, or zeros where it did not fit
        # of an extend's new tokens; and of a step's, a row for every sequence
        self.positions, self.slots, self.step_positions, self.step_slots = zeros(tokens), zeros(tokens), zeros(sequences), zeros(sequences)
        same = dict(lengths=self.lengths, next_lengths=self.lengths, free_count=self.free_count, next_free_count=self.free_count, page_table=self.table,
                    free_pages=self.free_pages, batch=sequences, table_width=self.width, page_size=page_size)
        self._extend = prepare(ctx, "kv_pages_v1", counts=self.counts, release=self.released, token_offsets=self.offsets, positions=self.positions,
                               slots=self.slots, tokens=tokens, **same)
        self._step = prepare(ctx, "kv_pages_v1", positions=self.step_positions, slots=self.step_slots, tokens=sequences, attended=self.attended, **same)

    def extend(self, counts, release=None):
        """Places for `counts[b]` new tokens of every sequence b, after those of `release` (truth values) have given their pages back."""
        n = len(self.lengths)
        counts, release = _new_tokens(counts, n), _mask(release, n).astype(np.uint32)
        if int(counts.sum()) > self.tokens:
            raise ValueError(f"no more than {self.tokens} new tokens at once, got {int(counts.sum())}")
        # (arrays in ordinary memory: the copies have read them when the calls return)
        self.counts.copy_from_host_async(self.stream, counts.astype(np.uint32))
        self.released.copy_from_host_async(self.stream, release)
        self._extend.launch(self.stream)

    def step(self, stream=None):
        """A place for one new token of every sequence at work (of length above 0)."""
        self._step.launch(stream or self.stream)

    def free(self):
        self._extend.destroy()
        self._step.destroy()
        for b in (self.table, self.free_pages, self.free_count, self.lengths, self.counts, self.released, self.offsets, self.positions, self.slots,
                  self.step_positions, self.step_slots, self.attended):
            b.free()


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


def _numbers(**arrays):
    """Positions and slots are read as 32-bit words, one behind the other (addresses with a length say nothing of that)."""
    _contiguous(*arrays.values())
    for name, x in arrays.items():
        if hasattr(x, "dtype") and not str(x.dtype).endswith("int32"):
            raise TypeError(f"{name} are 32-bit integers, got {x.dtype}")


def _pair_dtype(k, v, dtype):
    """DTYPE_* of k and v, which are of one type."""
    one = _float_dtype(k, dtype)
    if hasattr(v, "dtype") and _float_dtype(v, dtype) != one:
        raise TypeError(f"k and v are of one type, got {k.dtype} and {v.dtype}")
    return one


class PagedKvCache:
    def __init__(self, ctx, stream, sequences, positions, kv_heads, dim, page_size=16, pages=None, format=KV_BF16, tokens=None):
        """Room for `sequences` of up to `positions` tokens each in `pages` pages (default: enough for all at their
        longest).  With `tokens`, the most new tokens of one `extend`, the book of pages lies on the device."""
        if format == KV_E2M1 and (dim % 32 or page_size % 8):
            raise ValueError("a 4-bit cache has dim a multiple of 32 and page_size one of 8")
        self.ctx, self.stream, self.format = ctx, stream, format
        pages = sequences * -(-positions // page_size) if pages is None else pages
        self.sequences, self.kv_heads, self.dim, self.page_size = sequences, kv_heads, dim, page_size
        rows = pages * kv_heads * page_size
        element = {KV_BF16: np.uint16, KV_E4M3: np.uint8, KV_I8: np.int8, KV_E2M1: np.uint8}[format]
        row = dim * 9 // 16 if format == KV_E2M1 else dim   # elements
        self.k_cache, self.v_cache = (DeviceBuffer.zeroed(stream, rows * row, element) for _ in range(2))
        self.k_scales, self.v_scales = ((DeviceBuffer.zeroed(stream, rows, np.float32) if format != KV_BF16 else None) for _ in range(2))
        self.new_tokens = 0
        if tokens is not None:
            self.table, self.pages = None, DevicePages(ctx, stream, sequences, positions, pages, page_size, tokens)
            self.device_table, self.device_lengths, self.device_offsets = self.pages.table, self.pages.lengths, self.pages.offsets
            self.table_width = self.pages.width
            return
        self.table, self.pages = PageTable(sequences, positions, pages, page_size), None
        self.table_width = self.table.entries.shape[1]
        self.device_table = DeviceBuffer.from_host(stream, self.table.entries)
        self.device_lengths = DeviceBuffer.from_host(stream, self.table.lengths)
        self.device_offsets = DeviceBuffer.zeroed(stream, sequences + 1, np.uint32)

    def _storage(self):
        return dict(k_cache=self.k_cache, v_cache=self.v_cache, k_scales=self.k_scales, v_scales=self.v_scales, kv_heads=self.kv_heads, dim=self.dim,
                    page_size=self.page_size, format=self.format)

    def args(self):
        """The cache's own arguments of the three operators."""
        return dict(page_table=self.device_table, lengths=self.device_lengths, batch=self.sequences, table_width=self.table_width, **self._storage())

    def _upload(self, pages_changed=True):
        # (arrays in ordinary memory: the copies have read them when the calls return)
        if pages_changed:
            self.device_table.copy_from_host_async(self.stream, self.table.entries)
        self.device_lengths.copy_from_host_async(self.stream, self.table.lengths)

    def extend(self, counts, release=None):
        """Positions for new tokens of every sequence; `append` then writes them.  `release`: truth values, the sequences that give their pages
        back first."""
        if self.pages:
            self.pages.extend(counts, release)
            self.new_tokens = int(np.sum(counts))
            return
        book, before, gone = self.table, len(self.table.free), np.nonzero(_mask(release, self.sequences))[0]
        held = book.entries[gone], book.lengths[gone]   # (copies)
        for b in gone:
            book.release(int(b))
        try:
            book.extend(counts)
        except Exception:   # all or none, what is released too: its pages lie behind those that were free
            book.entries[gone], book.lengths[gone] = held
            del book.free[before:]
            raise
        offsets = np.zeros(self.sequences + 1, np.uint32)
        offsets[1:] = np.cumsum(counts)
        self.new_tokens = int(offsets[-1])
        self._upload(len(self.table.free) != before or release is not None)
        self.device_offsets.copy_from_host_async(self.stream, offsets)

    def release(self, sequence):
        """Gives a finished sequence's pages back; its slot starts again at no positions."""
        if self.pages:
            gone = np.zeros(self.sequences, bool)
            gone[operator.index(sequence)] = True   # (one, no slice or mask of them)
            self.pages.extend([0] * self.sequences, gone)
            self.new_tokens = 0
            return
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

    def rotary_append(self, q, k, v, q_out, heads, rotary, tokens, positions, slots, dtype=None, strides=None, q_strides=None):
        """A prepared launch of `kv_cache_rotary_append_v1` into this cache (q and q_out None: keys and values alone; rotary None: no
        rotation, and queries stay as they are); the caller launches and destroys it.  positions and slots: 32-bit integers, one a token."""
        _contiguous(q, q_out)
        _numbers(positions=positions, slots=slots)
        if q is None or q_out is None or rotary is None:
            q, q_out, heads = None, None, 0
        one = _pair_dtype(k, v, dtype)
        if (hasattr(q, "dtype") and _float_dtype(q, dtype) != one) or (hasattr(q_out, "dtype") and _float_dtype(q_out, dtype) != one):
            raise TypeError("q and its turned rows are of the type of k and v")
        qt, qh = q_strides or (heads * self.dim, self.dim)
        turn = rotary.args() if rotary else dict(frequencies=None, rotary_dim=0, layout=0, scale=1.0)
        return prepare(self.ctx, "kv_cache_rotary_append_v1", q=q, q_output=q_out, heads=heads, input_dtype=one, positions=positions if rotary and rotary.rotary_dim else None,
                       slots=slots, q_token_stride=qt, q_head_stride=qh, q_output_token_stride=heads * self.dim, q_output_head_stride=self.dim,
                       **turn, **self._rows(k, v, tokens, strides), **self._storage())

    def append(self, k, v, dtype=None, strides=None, q=None, q_out=None, heads=0, rotary=None, q_strides=None):
        """Rows of the tokens of the last `extend`, sequence after sequence: [tokens][kv_heads][dim], or with `strides`
        ((k token, k head), (v token, v head)) in elements, as slices (address, elements).  With a book on the device also with rotary positions on
        the way (`rotary`, a fe2o3_b200.rotary.Rotary): keys are turned, and queries q [tokens][heads][dim] into q_out."""
        if (q is None) != (q_out is None) or (q is not None and not rotary):
            raise ValueError("queries come along to be turned, by rotary=, from q into q_out")
        if rotary:
            if not self.pages:
                raise ValueError("rotary positions on the way into the cache need its book on the device: tokens=")
            n = self.new_tokens
            p = self.rotary_append(q, k, v, q_out, heads, rotary, n, (self.pages.positions.as_device_ptr(), n), (self.pages.slots.as_device_ptr(), n), dtype, strides, q_strides)
            try:
                p.launch(self.stream)
            finally:
                p.destroy()
            return
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

    def attention(self, q, out, heads, lse=None, scale=None, window=0, q_dtype=None, out_dtype=None, q_strides=None, lengths=None):
        """A prepared launch of `paged_attention_v1` over this cache, to the positions so far or to the first `lengths` of them; the caller launches and
        destroys it."""
        _contiguous(q, out, lse)
        _numbers(lengths=lengths)
        qs, qh = q_strides or (heads * self.dim, self.dim)
        return prepare(self.ctx, "paged_attention_v1", q=q, output=out, lse=lse, heads=heads, q_stride=qs, q_head_stride=qh,
                       scale=self.dim ** -0.5 if scale is None else scale, window=window, q_dtype=_float_dtype(q, q_dtype),
                       output_dtype=_float_dtype(out, out_dtype), **{**self.args(), **({} if lengths is None else dict(lengths=lengths))})

    def attend(self, q, out, heads, **kw):
        """One new token a sequence, q and out [sequences][heads][dim].  Returns when the device is idle, since the launch's workspace
        goes back: a program that attends again and again keeps an `attention` or a `DecodeStep`."""
        p = self.attention(q, out, heads, **kw)
        try:
            p.launch(self.stream)
        finally:
            p.destroy()

    def free(self):
        for b in (self.k_cache, self.v_cache, self.k_scales, self.v_scales):
            if b is not None:
                b.free()
        for b in (self.pages,) if self.pages else (self.device_table, self.device_lengths, self.device_offsets):
            b.free()


class DecodeStep:
    """One new token of every sequence at work (of length above 0): its key and value are written, then it attends to all
    positions so far and its own.  The tensors, a row a sequence, stay where they are from step to step; the caller fills
    q, k and v on the cache's stream.  Rows of released sequences count for nothing (with the device's book they may be read), and their output is zeros.

    A step that does not fit changes neither book nor cache.  With the host's book `run` raises.  With the device's it cannot know: the step is reported
    (`ctx.take_kernel_status`, which a program asks from time to time), and its output is zeros for every sequence, its log-sum-exp -inf.

    With the cache's book on the device a step is three launches and nothing else, and `run` may be captured in a CUDA graph (on the stream that
    it is given); with `rotary` q and k are turned by their positions on the way (q packed, or with strides, into rows that the step keeps)."""

    def __init__(self, cache, q, k, v, out, heads, lse=None, scale=None, window=0, dtype=None, out_dtype=None, strides=None, q_strides=None, rotary=None):
        self.cache, self.turned = cache, None
        if cache.pages:
            one = _pair_dtype(k, v, dtype)
            if rotary:
                self.turned = DeviceBuffer.zeroed(cache.stream, cache.sequences * heads * cache.dim, np.uint16 if one == DTYPE_BF16 else np.float32)
            self.append = cache.rotary_append(q, k, v, self.turned, heads, rotary, cache.sequences, cache.pages.step_positions, cache.pages.step_slots, dtype,
                                              strides, q_strides)
            if rotary:
                q, q_strides, dtype = self.turned, None, one
            self.attend = cache.attention(q, out, heads, lse, scale, window, dtype, out_dtype, q_strides, lengths=cache.pages.attended)
            return
        if rotary:
            raise ValueError("rotary positions in a decode step need the cache's book on the device: tokens=")
        self.attend = cache.attention(q, out, heads, lse, scale, window, dtype, out_dtype, q_strides)
        self.append = prepare(cache.ctx, "kv_cache_append_v1", input_dtype=_pair_dtype(k, v, dtype),
                              **cache._rows(k, v, cache.sequences, strides), **cache.args())

    def run(self, stream=None):
        cache = self.cache
        if stream is not None and not cache.pages:
            raise ValueError("a step whose book of pages is on the host runs on the cache's stream")
        stream = stream or cache.stream
        if cache.pages:
            cache.pages.step(stream)
        else:
            before = len(cache.table.free)
            cache.table.extend((cache.table.lengths > 0).astype(np.int64))
            cache._upload(len(cache.table.free) != before)
        self.append.launch(stream)
        self.attend.launch(stream)

    def destroy(self):
        self.append.destroy()
        self.attend.destroy()
        if self.turned is not None:
            self.turned.free()
