"""Admission of the paged key-value cache's operators: pure host checks, no GPU."""
import math

import numpy as np
import pytest

import fe2o3_b200 as fe

BASE = 0x7F0000000000


def sl(megabyte, n, off=0):
    return (BASE + (megabyte << 20) + off, n)


def err(op, **kw):
    with pytest.raises(fe.Fe2o3Error) as e:
        fe.check_args(op, fe.make_args(op, **kw))
    return e.value.name


def cache(form=fe.KV_BF16, pages=10, kv_heads=2, dim=64, page=16, batch=3, width=4):
    rows = pages * kv_heads * page
    scales = (0, 0) if form == fe.KV_BF16 else None
    return dict(k_cache=sl(0, rows * dim), v_cache=sl(8, rows * dim), k_scales=scales or sl(16, rows), v_scales=scales or sl(17, rows),
                page_table=sl(18, batch * width), lengths=sl(19, batch), batch=batch, kv_heads=kv_heads, dim=dim, page_size=page,
                table_width=width, format=form)


def rows(tokens=3, kv_heads=2, dim=64):
    n = tokens * kv_heads * dim
    return dict(k=sl(24, n), v=sl(32, n), tokens=tokens, k_token_stride=kv_heads * dim, k_head_stride=dim, v_token_stride=kv_heads * dim,
                v_head_stride=dim)


def queries(batch=3, heads=4, dim=64):
    n = batch * heads * dim
    return dict(q=sl(40, n), output=sl(48, n), lse=sl(56, batch * heads), heads=heads, q_stride=heads * dim, q_head_stride=dim, scale=0.125,
                window=0, q_dtype=fe.DTYPE_BF16, output_dtype=fe.DTYPE_F32)


def ok(op, **kw):
    fe.check_args(op, fe.make_args(op, **kw))


ALL = [("kv_cache_append_v1", rows), ("kv_cache_read_v1", rows), ("paged_attention_v1", queries)]


@pytest.mark.parametrize("op,more", ALL)
@pytest.mark.parametrize("form", [fe.KV_BF16, fe.KV_E4M3, fe.KV_I8])
def test_the_cache(op, more, form):
    kw = {**cache(form), **more()}
    ok(op, **kw)
    for bad in (dict(dim=0), dict(dim=24), dict(dim=272), dict(kv_heads=0), dict(page_size=0), dict(format=3),
                dict(kv_heads=1 << 20, page_size=1 << 20)):
        assert err(op, **{**kw, **bad}) == "UnsupportedShape", bad
    assert err(op, **{**kw, "k_cache": sl(0, 10 * 2 * 16 * 64, 8)}) == "Alignment"
    assert err(op, **{**kw, "v_cache": sl(8, 10 * 2 * 16 * 64, 2)}) == "Alignment"
    assert err(op, **{**kw, "k_cache": sl(0, 10 * 2 * 16 * 64 - 1)}) == "Length"       # not whole pages
    assert err(op, **{**kw, "v_cache": sl(8, 9 * 2 * 16 * 64)}) == "Length"
    assert err(op, **{**kw, "k_cache": (0, 10 * 2 * 16 * 64)}) == "NullAddress"
    assert err(op, **{**kw, "k_scales": sl(16, 5)}) == "Length"                         # none for bf16, one a row otherwise
    assert err(op, **{**kw, "page_table": sl(18, 11)}) == "Length"
    assert err(op, **{**kw, "lengths": sl(19, 4)}) == "Length"
    assert err(op, **{**kw, "lengths": sl(19, 3, 2)}) == "Alignment"


@pytest.mark.parametrize("op", ["kv_cache_append_v1", "kv_cache_read_v1"])
def test_rows_of_new_tokens(op):
    kw = {**cache(), **rows()}
    dtype = "input_dtype" if op == "kv_cache_append_v1" else "output_dtype"
    assert err(op, **{**kw, dtype: 2}) == "UnsupportedShape"
    assert err(op, **{**kw, **rows(4)}) == "UnsupportedShape"                            # one token a sequence without offsets
    more = {**kw, **rows(4), "token_offsets": sl(20, 4)}
    ok(op, **more)
    assert err(op, **{**more, "token_offsets": sl(20, 3)}) == "Length"
    assert err(op, **{**kw, "k": sl(24, 3 * 2 * 64 - 1)}) == "Length"
    assert err(op, **{**kw, "k": sl(24, 3 * 2 * 64, 1), dtype: 1}) == "Alignment"
    assert err(op, **{**kw, "k": sl(24, 3 * 2 * 64, 2), dtype: 0}) == "Alignment"
    ok(op, **{**kw, "k": sl(24, 3 * 2 * 64, 2), dtype: 1})
    # strided rows: (tokens - 1) * token_stride + (kv_heads - 1) * head_stride + dim elements
    ok(op, **{**kw, "k": sl(24, 2 * 1000 + 100 + 64), "k_token_stride": 1000, "k_head_stride": 100})
    ok(op, **{**kw, "k": sl(24, 2 * 64 + 500 + 64), "k_token_stride": 64, "k_head_stride": 500})
    overlapping = {**kw, "v": sl(32, 2 * 60 + 500 + 64), "v_token_stride": 60, "v_head_stride": 500}
    if op == "kv_cache_append_v1":
        ok(op, **overlapping)
    else:
        assert err(op, **overlapping) == "UnsupportedShape"
    empty = {**cache(batch=0), **rows(0)}
    ok(op, **empty)
    # what is written lies apart from what is read
    inside = {**kw, "k": sl(0, 3 * 2 * 64, 4096)}
    assert err(op, **inside) == "OutputAliasesInput"
    assert err(op, **{**kw, "v_cache": sl(0, 10 * 2 * 16 * 64)}) == "OutputAliasesInput" if op == "kv_cache_append_v1" else True


def test_caches_that_are_one_array():
    """What only reads takes K and V from the same array; what writes does not."""
    same = {**cache(), "v_cache": sl(0, 10 * 2 * 16 * 64)}
    ok("kv_cache_read_v1", **{**same, **rows()})
    ok("paged_attention_v1", **{**same, **queries()})
    assert err("kv_cache_append_v1", **{**same, **rows()}) == "OutputAliasesInput"


def test_attention_arguments():
    kw = {**cache(), **queries()}
    op = "paged_attention_v1"
    for bad in (dict(heads=0), dict(heads=3), dict(q_dtype=2), dict(output_dtype=2), dict(scale=math.nan), dict(scale=math.inf)):
        assert err(op, **{**kw, **bad}) == "UnsupportedShape", bad
    ok(op, **{**kw, "lse": None})
    ok(op, **{**kw, "scale": -3.0, "window": 0xffffffff})
    assert err(op, **{**kw, "lse": sl(56, 11)}) == "Length"
    assert err(op, **{**kw, "q": sl(40, 3 * 4 * 64 + 1)}) == "Length"
    assert err(op, **{**kw, "output": sl(48, 3 * 4 * 64 - 1)}) == "Length"
    ok(op, **{**kw, "q": sl(40, 64), "q_stride": 0, "q_head_stride": 0})
    ok(op, **{**kw, "q": sl(40, 2 * 5000 + 3 * 70 + 64), "q_stride": 5000, "q_head_stride": 70})
    assert err(op, **{**kw, "output": sl(40, 3 * 4 * 64)}) == "OutputAliasesInput"
    assert err(op, **{**kw, "output": sl(48, 3 * 4 * 64), "lse": sl(48, 12)}) == "OutputAliasesInput"
    assert err(op, **{**kw, "output": sl(0, 3 * 4 * 64)}) == "OutputAliasesInput"
    big = cache(batch=1 << 20, width=0)
    many = {**big, "lengths": sl(64, 1 << 20), "page_table": (0, 0), "heads": 4096, "kv_heads": 2, "scale": 1.0}
    assert err(op, **many) == "UnsupportedShape"


@pytest.mark.parametrize("batch,fits", [(1 << 29, True), ((1 << 29) + 1, False), ((1 << 31) - 1, False)])
def test_attention_batches_that_can_be_counted(batch, fits):
    """Two places a sequence beside its tiles (2^31 of those, in all of a page table) fit 32 bits."""
    far = lambda i: BASE + (i << 40)  # noqa: E731
    kw = dict(cache(kv_heads=1, dim=16), batch=batch, table_width=1, page_table=(far(1), batch), lengths=(far(2), batch), heads=1,
              q=(far(3), 16), q_stride=0, q_head_stride=0, output=(far(4), 16 * batch), lse=None, scale=1.0, window=0, q_dtype=1, output_dtype=1,
              k_cache=sl(0, 10 * 16 * 16), v_cache=sl(8, 10 * 16 * 16))
    if fits:
        ok("paged_attention_v1", **kw)
    else:
        assert err("paged_attention_v1", **kw) == "UnsupportedShape"


# ---- the host's book of pages ----------------------------------------------------------------------------------------

def test_pages_are_handed_out_and_come_back():
    from fe2o3_b200.kv_cache import PageTable
    t = PageTable(sequences=3, positions=50, pages=9, page_size=16)
    assert t.entries.shape == (3, 4)
    t.extend([16, 0, 33])
    assert t.lengths.tolist() == [16, 0, 33] and len(t.free) == 9 - 1 - 3
    t.extend([1, 15, 15])                                # 17, 15, 48: one page each for the first two
    assert len(t.free) == 3
    used = [int(p) for row, n in zip(t.entries, (2, 1, 3)) for p in row[:n]]
    assert len(set(used)) == 6 and all(0 <= p < 9 for p in used)
    assert (t.entries[0, 2:] == t.FREE).all() and (t.entries[1, 1:] == t.FREE).all()
    before = t.entries.copy(), t.lengths.copy(), list(t.free)
    for bad, error in (([48, 33, 0], ValueError),        # past a sequence's last position
                       ([33, 33, 0], MemoryError),       # more pages than are free
                       ([1, 1], ValueError), ([-1, 0, 0], ValueError)):
        with pytest.raises(error):
            t.extend(bad)
        assert (t.entries == before[0]).all() and (t.lengths == before[1]).all() and t.free == before[2]
    t.release(2)
    assert t.lengths.tolist() == [17, 15, 0] and len(t.free) == 6 and (t.entries[2] == t.FREE).all()
    t.extend([0, 0, 64])                                 # 50 positions are whole pages: 64
    assert len(t.free) == 2 and len(set(t.entries[t.entries != t.FREE].tolist())) == 7
    t.release(0), t.release(1), t.release(2)
    assert sorted(t.free) == list(range(9))
    t.release(1)                                         # an empty one: nothing
    assert len(t.free) == 9
    with pytest.raises(ValueError):
        PageTable(0, 1, 1, 1)


def test_row_types():
    from fe2o3_b200.kv_cache import _float_dtype
    assert _float_dtype(np.zeros(1, np.float32), None) == fe.DTYPE_F32
    assert _float_dtype(np.zeros(1, np.uint16), None) == fe.DTYPE_BF16
    assert _float_dtype((0, 4), fe.DTYPE_F32) == fe.DTYPE_F32
    with pytest.raises(TypeError):
        _float_dtype((0, 4), None)
    with pytest.raises(TypeError):
        _float_dtype(np.zeros(1, np.int32), None)


def test_rows_of_wider_storage():
    """Tensors say whether they are contiguous; addresses with a length do not."""
    import torch
    from fe2o3_b200.kv_cache import PagedKvCache, _contiguous
    f, h = torch.zeros(4, 2, 16), torch.zeros(4, 2, 16, dtype=torch.bfloat16)
    _contiguous(f, h, None, (0, 4), np.zeros(3))
    wide = torch.zeros(4, 3, 2, 16)
    with pytest.raises(ValueError):
        _contiguous(wide[:, 1])
    cache = PagedKvCache.__new__(PagedKvCache)           # (nothing of it is on a GPU before the rows are looked at)
    cache.kv_heads, cache.dim = 2, 16
    assert cache._rows(f, f, 4, None)["k_token_stride"] == 32
    for k, v in ((wide[:, 1], f), (f, wide[:, 2])):
        with pytest.raises(ValueError):
            cache._rows(k, v, 4, None)
    with pytest.raises(ValueError):
        cache.attention(wide[:, 0], f, 2)


def test_keys_and_values_of_unlike_types():
    import torch
    from fe2o3_b200.kv_cache import _pair_dtype
    f, h = torch.zeros(4, 2, 16), torch.zeros(4, 2, 16, dtype=torch.bfloat16)
    assert _pair_dtype(f, f, None) == fe.DTYPE_F32 and _pair_dtype(h, h, None) == fe.DTYPE_BF16
    assert _pair_dtype((0, 4), (0, 4), fe.DTYPE_BF16) == fe.DTYPE_BF16 and _pair_dtype(h, (0, 4), None) == fe.DTYPE_BF16
    with pytest.raises(TypeError):
        _pair_dtype(h, f, None)
    with pytest.raises(TypeError):
        _pair_dtype((0, 4), f, None)
