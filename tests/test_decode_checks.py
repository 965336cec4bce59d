"""Admission of page plans, rotary positions and 4-bit caches: pure host checks, no GPU."""
import math

import pytest
import torch

import fe2o3_b200 as fe
from test_kv_cache_checks import ALL, err, ok, queries, rows, sl


def pages(batch=3, width=4, count=10, tokens=8):
    return dict(counts=sl(0, batch), release=sl(1, batch), lengths=sl(2, batch), free_count=sl(3, 1), page_table=sl(4, batch * width), free_pages=sl(5, count),
                next_lengths=sl(6, batch), next_free_count=sl(7, 1), token_offsets=sl(8, batch + 1), positions=sl(9, tokens), slots=sl(10, tokens),
                batch=batch, table_width=width, page_size=16, tokens=tokens)


def test_page_plans():
    op, kw = "kv_pages_v1", pages()
    ok(op, **kw)
    for name in ("counts", "release", "token_offsets", "positions", "slots"):
        ok(op, **{**kw, name: None})
    ok(op, **{**kw, "next_lengths": kw["lengths"], "next_free_count": kw["free_count"]})
    ok(op, **pages(batch=0, width=0, count=0, tokens=0))
    each = {**kw, "counts": None, "tokens": 2}   # a row for every sequence, where there are rows
    assert err(op, **{**each, "positions": sl(9, 2), "slots": None}) == "UnsupportedShape"
    ok(op, **{**each, "positions": None, "slots": None})
    ok(op, **{**kw, "tokens": 2, "positions": sl(9, 2), "slots": sl(10, 2)})
    ok(op, **pages(batch=8192))
    for bad in (dict(page_size=0), dict(batch=8193), dict(table_width=1 << 31), dict(page_size=1 << 30)):
        assert err(op, **{**kw, **bad}) == "UnsupportedShape", bad
    for name, n in (("counts", 2), ("release", 4), ("lengths", 2), ("free_count", 2), ("page_table", 11), ("next_lengths", 4), ("next_free_count", 0),
                    ("token_offsets", 3), ("positions", 9), ("slots", 7)):
        assert err(op, **{**kw, name: sl(40, n)}) == "Length", name
    assert err(op, **{**kw, "lengths": (0, 3)}) == "NullAddress"
    assert err(op, **{**kw, "slots": sl(10, 8, 2)}) == "Alignment"
    # outputs lie apart, from each other and from what is read; lengths that are only partly the next ones are neither
    for a, b in (("next_lengths", "counts"), ("positions", "slots"), ("next_lengths", "page_table"), ("free_pages", "page_table"), ("token_offsets", "release")):
        assert err(op, **{**kw, a: (kw[b][0], kw[a][1])}) == "OutputAliasesInput", (a, b)
    assert err(op, **{**kw, "next_lengths": (kw["lengths"][0] + 4, 3)}) == "OutputAliasesInput"


def rotary(tokens=5, heads=4, kv_heads=2, dim=64):
    kw = dict(q=sl(0, tokens * heads * dim), k=sl(1, tokens * kv_heads * dim), positions=sl(2, tokens), frequencies=sl(3, 16),
              q_output=sl(4, tokens * heads * dim), k_output=sl(5, tokens * kv_heads * dim), tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotary_dim=32,
              layout=fe.ROTARY_HALF, dtype=fe.DTYPE_F32, backward=0, scale=1.0)
    for n in ("q", "k", "q_output", "k_output"):
        kw.update({n + "_token_stride": (heads if n[0] == "q" else kv_heads) * dim, n + "_head_stride": dim})
    return kw


def test_rotary_rows():
    op, kw = "rotary_v1", rotary()
    ok(op, **kw)
    ok(op, **{**kw, "positions": None})
    ok(op, **{**kw, "layout": fe.ROTARY_INTERLEAVED, "backward": 1, "scale": -2.0})
    ok(op, **{**kw, "kv_heads": 0, "k": None, "k_output": None})
    ok(op, **{**kw, "heads": 0, "q": None, "q_output": None})
    ok(op, **{**kw, "rotary_dim": 0, "frequencies": None})
    ok(op, **rotary(tokens=0))
    for bad in (dict(dim=0), dict(dim=24), dict(dim=272), dict(rotary_dim=31), dict(rotary_dim=66), dict(layout=2), dict(dtype=2), dict(backward=2),
                dict(scale=math.nan), dict(scale=math.inf), dict(heads=65537)):
        assert err(op, **{**kw, **bad}) == "UnsupportedShape", bad
    for name, n in (("q", 5 * 4 * 64 - 1), ("k", 5 * 2 * 64 + 1), ("positions", 4), ("frequencies", 15), ("q_output", 64), ("k_output", 64)):
        assert err(op, **{**kw, name: sl(20, n)}) == "Length", name
    assert err(op, **{**kw, "q": sl(0, 5 * 4 * 64, 2)}) == "Alignment"
    ok(op, **{**kw, "q": sl(0, 5 * 4 * 64, 2), "dtype": fe.DTYPE_BF16})
    # in place with the same strides, and with no others
    ok(op, **{**kw, "q_output": kw["q"], "k_output": kw["k"]})
    head_major = {"q_output_token_stride": 64, "q_output_head_stride": 320}
    ok(op, **{**kw, **head_major})
    assert err(op, **{**kw, "q_output": kw["q"], **head_major}) == "OutputAliasesInput"
    assert err(op, **{**kw, "q_output": kw["k_output"]}) == "Length"
    assert err(op, **{**kw, "q_output": (kw["k_output"][0], 5 * 4 * 64)}) == "OutputAliasesInput"
    assert err(op, **{**kw, "q_output_token_stride": 128, "q_output": sl(4, 4 * 128 + 256)}) == "UnsupportedShape"   # rows that meet
    ok(op, **{**kw, "q_token_stride": 0, "q": sl(0, 256)})                                                          # one row for all tokens


def test_rotary_rows_inside_fused_ones():
    """[q | k | v] in one array: turned where they lie, or one array of turned rows; rows that meet are refused."""
    op, kw = "rotary_v1", rotary()
    ts, n = 8 * 64, 4 * 8 * 64
    strides = {k: ts for k in kw if k.endswith("token_stride")}
    fused = {**kw, **strides, "q": sl(0, n + 256), "k": sl(0, n + 128, 256 * 4)}
    ok(op, **{**fused, "q_output": fused["q"], "k_output": fused["k"]})
    ok(op, **{**fused, "q_output": sl(4, n + 256), "k_output": sl(4, n + 128, 256 * 4)})
    ok(op, **{**fused, "q_output": sl(4, n + 256, 128 * 4), "k_output": sl(4, n + 128)})             # k first
    assert err(op, **{**fused, "q_output": sl(4, n + 256), "k_output": sl(4, n + 128, 255 * 4)}) == "OutputAliasesInput"
    assert err(op, **{**fused, "q_output": sl(4, n + 256), "k_output": sl(4, n + 128, 385 * 4)}) == "OutputAliasesInput"   # into the next token's
    assert err(op, **{**fused, "q_output": fused["q"], "k_output": sl(5, n + 128)}) == "OutputAliasesInput"   # k is read between rows that are written
    assert err(op, **{**fused, "q_output": sl(4, n + 256), "k_output": sl(4, n + 128, 256 * 4), "positions": sl(4, 5, 400 * 4)}) == "OutputAliasesInput"


def four(pages_=10, kv_heads=2, dim=64, page=16, batch=3, width=4):
    n = pages_ * kv_heads * page
    return dict(k_cache=sl(24, n * dim * 9 // 16), v_cache=sl(32, n * dim * 9 // 16), k_scales=sl(40, n), v_scales=sl(41, n), page_table=sl(42, batch * width),
                lengths=sl(43, batch), batch=batch, kv_heads=kv_heads, dim=dim, page_size=page, table_width=width, format=fe.KV_E2M1)


@pytest.mark.parametrize("op,more", ALL)
def test_four_bit_caches(op, more):
    rest = {k: (v[0] + (64 << 20), v[1]) if isinstance(v, tuple) else v for k, v in more().items()}
    kw = {**four(), **rest}
    ok(op, **kw)
    n = 10 * 2 * 16
    for bad in (dict(dim=48), dict(dim=16), dict(dim=288), dict(page_size=12), dict(page_size=1), dict(format=3), dict(format=5)):
        assert err(op, **{**kw, **bad}) == "UnsupportedShape", bad
    assert err(op, **{**kw, "k_cache": sl(24, n * 64 // 2)}) == "Length"              # codes without their block scales
    assert err(op, **{**kw, "v_cache": sl(32, n * 36 - 36 * 32)}) == "Length"
    assert err(op, **{**kw, "k_scales": sl(40, n - 1)}) == "Length"
    assert err(op, **{**kw, "k_scales": sl(40, n, 4)}) == "Alignment"
    assert err(op, **{**kw, "v_scales": sl(41, n, 8)}) == "Alignment"
    assert err(op, **{**kw, "k_cache": sl(24, n * 36, 8)}) == "Alignment"


@pytest.mark.parametrize("cache", ["bf16", "e2m1"])
def test_rotary_append(cache):
    op = "kv_cache_rotary_append_v1"
    base = {k: v for k, v in four().items() if k not in ("page_table", "lengths", "batch", "table_width")}
    if cache == "bf16":
        base.update(format=fe.KV_BF16, k_cache=sl(24, 10 * 2 * 16 * 64), v_cache=sl(32, 10 * 2 * 16 * 64), k_scales=None, v_scales=None)
    r = rotary()
    kw = {**base, **{k: v for k, v in r.items() if not k.startswith("k_output") and k not in ("dtype", "backward", "kv_heads", "dim")}}
    kw.update(v=sl(12, 5 * 2 * 64), v_token_stride=128, v_head_stride=64, slots=sl(13, 5), input_dtype=fe.DTYPE_F32)
    ok(op, **kw)
    ok(op, **{**kw, "rotary_dim": 0, "frequencies": None, "positions": None})
    ok(op, **{**kw, "heads": 0, "q": None, "q_output": None})
    for bad in (dict(rotary_dim=33), dict(rotary_dim=66), dict(layout=2), dict(input_dtype=2), dict(scale=math.nan), dict(format=3), dict(heads=70000), dict(dim=24)):
        assert err(op, **{**kw, **bad}) == "UnsupportedShape", bad
    for name, n in (("q", 1), ("k", 1), ("v", 1), ("slots", 4), ("positions", 6), ("frequencies", 17), ("q_output", 1), ("k_cache", 100)):
        assert err(op, **{**kw, name: sl(50, n)}) == "Length", name
    assert err(op, **{**kw, "positions": None}) == "Length"
    for name in ("q", "k", "v", "slots"):
        assert err(op, **{**kw, "q_output": (kw[name][0], kw["q_output"][1])}) == "OutputAliasesInput", name
    assert err(op, **{**kw, "v": (kw["k_cache"][0], kw["v"][1])}) == "OutputAliasesInput"
    assert err(op, **{**kw, "v_cache": kw["k_cache"]}) == "OutputAliasesInput"
    assert err(op, **{**kw, "q_output_token_stride": 100, "q_output": sl(4, 4 * 100 + 256)}) == "UnsupportedShape"


# ---- what the host works out ------------------------------------------------------------------------------------------

def test_rotary_frequencies():
    import numpy as np
    from fe2o3_b200.rotary import rotary_frequencies
    f, by = rotary_frequencies(64)
    assert f.dtype == np.float32 and by == 1.0 and np.allclose(f, 10000.0 ** (-np.arange(32) / 32), rtol=1e-7, atol=0) and f[0] == 1
    lin, _ = rotary_frequencies(64, scaling="linear", factor=4.0)
    assert np.allclose(lin * 4, f, rtol=1e-6, atol=0)
    ntk, _ = rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert ntk[0] == 1 and np.isclose(ntk[-1] * 8, f[-1], rtol=1e-5) and (np.diff(ntk) < 0).all()
    yarn, by = rotary_frequencies(128, scaling="yarn", factor=16.0, trained=4096)
    plain, _ = rotary_frequencies(128)
    turns = 4096 * plain.astype(np.float64) / (2 * math.pi)
    assert np.isclose(by, 0.1 * math.log(16) + 1)
    assert (yarn[turns > 36] == plain[turns > 36]).all() and np.allclose(yarn[turns < 0.85] * 16, plain[turns < 0.85], rtol=1e-6)
    assert (yarn <= plain).all() and (yarn * 16 >= plain * (1 - 1e-6)).all() and (np.diff(yarn) < 0).all()
    assert len(rotary_frequencies(0)[0]) == 0 and rotary_frequencies(2, scaling="yarn", factor=2.0, trained=100)[0].shape == (1,)
    for bad in (dict(rotary_dim=3), dict(rotary_dim=64, factor=0.5), dict(rotary_dim=64, base=0), dict(rotary_dim=64, scaling="more"),
                dict(rotary_dim=64, scaling="yarn", factor=2.0), dict(rotary_dim=2, scaling="ntk", factor=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_objects_refuse_before_the_device_is_touched():
    from fe2o3_b200.kv_cache import DevicePages, PagedKvCache
    for kw in (dict(dim=48), dict(page_size=12)):
        with pytest.raises(ValueError):
            PagedKvCache(None, None, **{**dict(sequences=1, positions=8, kv_heads=1, dim=64, page_size=8, format=fe.KV_E2M1), **kw})
    with pytest.raises(ValueError):
        DevicePages(None, None, 1, 8, 1, 8, 0)


def test_rotary_object_wants_the_number_of_strided_rows():
    from fe2o3_b200.rotary import Rotary
    rotary = Rotary(None, None, 0)   # (no columns to turn: nothing on a device)
    for q, kw in (((1 << 20, 512), {}), (torch.zeros(4, 512), dict(strides=((512, 64), (512, 64))))):
        with pytest.raises(ValueError):
            rotary.apply(q, None, None, 2, 0, 64, dtype=fe.DTYPE_F32, **kw)


def test_rotary_object_wants_positions_of_32_bits():
    from fe2o3_b200.rotary import Rotary
    rotary, q = Rotary(None, None, 0), torch.zeros(4, 2, 64)
    for positions in (torch.arange(4), torch.arange(4.0), torch.arange(4, dtype=torch.int16)):
        with pytest.raises(TypeError, match="32-bit"):
            rotary.apply(q, None, positions, 2, 0, 64)
    with pytest.raises(ValueError):
        rotary.apply(q, None, torch.arange(8, dtype=torch.int32)[::2], 2, 0, 64)


@pytest.mark.parametrize("name", ["positions", "slots"])
def test_rotated_rows_want_numbers_of_32_bits(name):
    """64-bit numbers read as 32-bit words would be a slot, 0, a slot, 0: the first page's first row, again and again."""
    from fe2o3_b200.kv_cache import PagedKvCache
    from fe2o3_b200.rotary import Rotary
    cache = PagedKvCache.__new__(PagedKvCache)             # (nothing of it is on a GPU before the arguments are looked at)
    rotary, k = Rotary(None, None, 0), torch.zeros(4, 2, 32)
    cache.kv_heads, cache.dim = 2, 32
    good = dict(positions=torch.arange(4, dtype=torch.int32), slots=torch.arange(4, dtype=torch.int32))
    for bad in (torch.arange(4), torch.arange(4.0), torch.arange(4, dtype=torch.int16)):
        with pytest.raises(TypeError, match=name + " are 32-bit"):
            cache.rotary_append(None, k, k, None, 0, rotary, 4, **{**good, name: bad})
    with pytest.raises(ValueError, match="contiguous"):
        cache.rotary_append(None, k, k, None, 0, rotary, 4, **{**good, name: torch.arange(8, dtype=torch.int32)[::2]})


class Copies:
    """A device array of which only what is copied into it counts."""

    def __init__(self):
        self.held = None

    def copy_from_host_async(self, stream, array):
        self.held = array.copy()


def host_book(sequences=3, positions=64, page_size=8, pages=20):
    """A cache with the host's book of pages, nothing of it on a GPU."""
    from fe2o3_b200.kv_cache import PagedKvCache, PageTable
    cache = PagedKvCache.__new__(PagedKvCache)
    cache.pages, cache.stream, cache.sequences, cache.table = None, None, sequences, PageTable(sequences, positions, pages, page_size)
    cache.device_table, cache.device_lengths, cache.device_offsets = Copies(), Copies(), Copies()
    return cache


def device_book(sequences=3, tokens=50):
    """The same with the device's book, whose launches do nothing."""
    from fe2o3_b200.kv_cache import DevicePages, PagedKvCache
    cache, pages = PagedKvCache.__new__(PagedKvCache), DevicePages.__new__(DevicePages)
    pages.stream, pages.tokens, pages.lengths, pages.counts, pages.released = None, tokens, [0] * sequences, Copies(), Copies()
    pages._extend = type("Launch", (), {"launch": lambda self, stream: None})()
    cache.pages, cache.sequences, cache.stream = pages, sequences, None
    return cache


@pytest.mark.parametrize("book", [host_book, device_book])
def test_released_sequences_are_a_truth_value_each(book):
    """A list of sequence numbers is not taken for one: [2] would be sequence 0."""
    cache = book()
    cache.extend([5, 6, 7])
    for bad in ([2], [1, 0], [1, 0, 0, 0], [[1, 0, 0]], 1, []):
        with pytest.raises(ValueError, match="truth value"):
            cache.extend([0, 0, 0], bad)
    if cache.pages:
        assert cache.pages.counts.held.tolist() == [5, 6, 7] and cache.pages.released.held.tolist() == [0, 0, 0]
        cache.extend([0, 1, 0], [True, False, True])
        assert cache.pages.released.held.tolist() == [1, 0, 1]
    else:
        assert cache.table.lengths.tolist() == [5, 6, 7] and len(cache.table.free) == 17
        cache.extend([0, 1, 0], [True, False, True])
        assert cache.table.lengths.tolist() == [0, 7, 0] and cache.device_lengths.held.tolist() == [0, 7, 0] and len(cache.table.free) == 19


def test_extending_the_hosts_book_costs_its_new_pages_alone():
    """The table, the lengths and the list of free pages are not copied for an undoing that `PageTable.extend` does not need."""
    import numpy as np
    cache = host_book()
    copies = []

    class Watched(np.ndarray):
        def copy(self, *args, **kw):
            copies.append(self.shape)
            return super().copy(*args, **kw)

        def __getitem__(self, at):
            out = super().__getitem__(at)
            if isinstance(out, np.ndarray) and out.size and not np.shares_memory(out, self):
                copies.append(out.shape)
            return out

    class Pages(list):
        def __iter__(self):
            copies.append(len(self))
            return super().__iter__()

    book = cache.table
    book.entries, book.free = book.entries.view(Watched), Pages(book.free)
    cache.device_table.copy_from_host_async = lambda stream, array: None
    cache.extend([5, 6, 7])
    assert copies == [] and book.lengths.tolist() == [5, 6, 7]
    with pytest.raises(ValueError):
        cache.extend([0, 100, 0])
    assert copies == []
    with pytest.raises(ValueError):
        cache.extend([0, 100, 0], [1, 0, 0])
    assert copies == [(1, 8)] and book.lengths.tolist() == [5, 6, 7]   # the row of the released sequence


def test_a_release_that_fails_with_its_extend_is_undone():
    import numpy as np
    rng = np.random.default_rng(1)
    cache = host_book(sequences=6, pages=20)
    book, failed = cache.table, 0
    for _ in range(300):
        before = book.entries.copy(), book.lengths.copy(), list(book.free)
        counts, gone = rng.integers(0, 30, 6), rng.random(6) < 0.4
        try:
            cache.extend(counts, gone)
        except (ValueError, MemoryError):
            failed += 1
            assert (book.entries == before[0]).all() and (book.lengths == before[1]).all() and book.free == before[2]
        else:
            assert (book.lengths == np.where(gone, 0, before[1]) + counts).all()
            used = book.entries[book.entries != book.FREE].tolist()
            assert sorted(used + list(book.free)) == list(range(20))
    assert 20 < failed < 280


@pytest.mark.parametrize("book", [host_book, device_book])
def test_a_released_sequence_is_one_of_the_book(book):
    """A number past the end is an error with either book, one below zero counts from the end."""
    cache = book()
    cache.extend([5, 6, 7])
    lengths = lambda: (cache.pages.released.held == 0).tolist() if cache.pages else (cache.table.lengths > 0).tolist()  # noqa: E731
    for bad in (3, -4, 100):
        with pytest.raises(IndexError):
            cache.release(bad)
    assert lengths() == [True, True, True]
    cache.release(-1)
    assert lengths() == [True, True, False]
    cache.release(0)
    assert lengths()[0] is False


@pytest.mark.parametrize("book", [host_book, device_book])
def test_a_released_sequence_is_a_number(book):
    cache = book()
    cache.extend([5, 6, 7])
    for bad in (None, slice(0, 2), [0, 1], "0"):
        with pytest.raises((TypeError, IndexError)):
            cache.release(bad)
    if cache.pages:
        assert cache.pages.released.held.tolist() == [0, 0, 0]
    else:
        assert cache.table.lengths.tolist() == [5, 6, 7]


@pytest.mark.parametrize("book", [host_book, device_book])
def test_new_tokens_are_whole_numbers(book):
    """Also such whose sum leaves 64 bits, and would be 0 there."""
    cache = book(4)
    for bad in ([1.5, 0.5, 0, 0], [1 << 62] * 4, [1 << 31, 0, 0, 0], [1 << 70, 0, 0, 0], [float("nan"), 0, 0, 0], [float("inf"), 0, 0, 0], [-1, 1, 0, 0], [1, 1, 1]):
        with pytest.raises(ValueError):
            cache.extend(bad)
    held = lambda: cache.pages.counts.held if cache.pages else cache.device_lengths.held  # noqa: E731
    assert held() is None
    cache.extend([3.0, True, 0, 2])
    assert held().tolist() == [3, 1, 0, 2] and cache.new_tokens == 6


def test_lengths_to_attend_to():
    """What a plan leaves for the attention of its step: optional, one a sequence, apart from everything else."""
    op, kw = "kv_pages_v1", pages()
    ok(op, **{**kw, "attended": sl(11, 3)})
    for n in (2, 4):
        assert err(op, **{**kw, "attended": sl(11, n)}) == "Length"
    assert err(op, **{**kw, "attended": sl(11, 3, 2)}) == "Alignment"
    for name in ("lengths", "next_lengths", "slots", "page_table"):
        assert err(op, **{**kw, "attended": (kw[name][0], 3)}) == "OutputAliasesInput", name


def test_lengths_of_an_attention_are_32_bits():
    from fe2o3_b200.kv_cache import PagedKvCache
    cache, q = PagedKvCache.__new__(PagedKvCache), torch.zeros(3, 2, 32)
    cache.dim = 32
    for bad in (torch.arange(3), torch.arange(3.0)):
        with pytest.raises(TypeError, match="lengths are 32-bit"):
            cache.attention(q, q, 2, lengths=bad)
    with pytest.raises(ValueError, match="contiguous"):
        cache.attention(q, q, 2, lengths=torch.arange(6, dtype=torch.int32)[::2])
