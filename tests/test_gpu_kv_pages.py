"""Page tables and slot maps planned on the GPU, against the host's book of pages and a plain walk over sequences and tokens."""
import numpy as np
import pytest

from test_gpu_kv_cache import gpu  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
FREE = 0xFFFFFFFF


class Book:
    """What the device should hold, sequence after sequence."""

    def __init__(self, batch, width, page, pages, seed=0):
        self.page, self.width = page, width
        self.table = np.full((batch, width), FREE, np.uint32)
        self.lengths = np.zeros(batch, np.uint32)
        self.stack = np.random.default_rng(seed).permutation(pages).astype(np.uint32)
        self.top = pages

    def step(self, counts, release=None):
        for b in range(len(self.lengths)):
            if release is not None and release[b]:
                for i in reversed(range(-(-int(self.lengths[b]) // self.page))):
                    self.stack[self.top] = self.table[b, i]
                    self.top += 1
                self.lengths[b] = 0
        each = counts is None   # a row for every sequence
        if each:
            counts = (self.lengths > 0).astype(np.int64)
        positions, slots, offsets = [], [], [0]
        for b, n in enumerate(counts):
            first, n = int(self.lengths[b]), int(n)
            for i in range(-(-first // self.page), -(-(first + n) // self.page)):
                self.top -= 1
                self.table[b, i] = self.stack[self.top]
            at = np.arange(first, first + n)
            positions.append(at)
            slots.append(self.table[b, at // self.page].astype(np.int64) * self.page + at % self.page)
            self.lengths[b] += n
            offsets.append(offsets[-1] + n)
            if each and not n:
                positions.append([0])
                slots.append([FREE])
        return np.concatenate(positions + [[]]).astype(np.int64), np.concatenate(slots + [[]]).astype(np.int64), np.array(offsets)


class Device:
    def __init__(self, gpu, book, tokens, in_place=True):  # noqa: F811
        self.fe, self.torch, self.ctx, self.stream = gpu
        up = lambda a: self.torch.from_numpy(np.array(a).view(np.int32)).cuda()  # noqa: E731
        self.up, self.book, self.tokens = up, book, tokens
        self.table, self.free, self.lengths, self.count = up(book.table), up(book.stack), up(book.lengths), up(np.array([book.top], np.uint32))
        new = lambda n: self.torch.full((n,), 77, dtype=self.torch.int32, device="cuda")  # noqa: E731
        self.next_lengths, self.next_count = (self.lengths, self.count) if in_place else (new(len(book.lengths)), new(1))
        self.offsets, self.positions, self.slots = new(len(book.lengths) + 1), new(tokens), new(tokens)

    def args(self, **kw):
        return {**dict(lengths=self.lengths, free_count=self.count, page_table=self.table, free_pages=self.free, next_lengths=self.next_lengths,
                       next_free_count=self.next_count, token_offsets=self.offsets, positions=self.positions, slots=self.slots,
                       batch=len(self.book.lengths), table_width=self.book.width, page_size=self.book.page, tokens=self.tokens), **kw}

    def step(self, counts=None, release=None, **kw):
        p = self.fe.prepare(self.ctx, "kv_pages_v1", counts=None if counts is None else self.up(np.asarray(counts, np.uint32)),
                            release=None if release is None else self.up(np.asarray(release, np.uint32)), **self.args(**kw))
        try:
            p.launch_and_wait(self.stream, 20000)
        finally:
            self.status = p.kernel_status
            p.destroy()

    def held(self):
        return {n: getattr(self, n).cpu().numpy().view(np.uint32).copy() for n in ("table", "free", "next_lengths", "next_count", "offsets", "positions", "slots")}

    def check(self, want):
        positions, slots, offsets = want
        got, b, n = self.held(), self.book, len(positions)
        assert (got["table"] == b.table).all() and (got["free"] == b.stack).all()
        assert (got["next_lengths"] == b.lengths).all() and got["next_count"][0] == b.top
        assert (got["offsets"] == offsets).all()
        assert (got["positions"][:n] == positions).all() and (got["positions"][n:] == 0).all()
        assert (got["slots"][:n] == slots).all() and (got["slots"][n:] == FREE).all()


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("batch,page,most,tokens", [(1, 16, 40, 64), (5, 1, 9, 45), (48, 16, 3, 160), (300, 7, 30, 9001), (33, 24, 400, 14000), (2000, 16, 3, 2001),
                                                    (1025, 16, 60, 70000), (2500, 64, 8, 20003), (1, 64, 50000, 50000)])
def test_steps(gpu, batch, page, most, tokens, in_place):  # noqa: F811
    """Prompts, single tokens, sequences that end and others that take their slots in the same step, tokens that do not fill the map."""
    rng = np.random.default_rng(batch + page)
    width = -(-3 * most // page) + 2
    book = Book(batch, width, page, batch * width + 3)
    d = Device(gpu, book, tokens, in_place)
    for step in range(6):
        release = None if step in (0, 3) else rng.random(batch) < 0.3
        counts = rng.integers(0, most + 1, batch) * (rng.random(batch) < 0.7)
        counts = np.minimum(counts, [max(0, width * page - (0 if release is not None and r else int(n))) for n, r in
                                     zip(book.lengths, release if release is not None else [0] * batch)])
        while counts.sum() > tokens:
            counts //= 2
        if step == 4:
            counts = None
        d.step(counts, release)
        d.check(book.step(counts, release))
        if not in_place:
            d.lengths.copy_(d.next_lengths)
            d.count.copy_(d.next_count)


def test_as_the_hosts_book(gpu):  # noqa: F811
    """The same pages in the same order as `PageTable` hands out."""
    from fe2o3_b200.kv_cache import PageTable
    rng = np.random.default_rng(3)
    host = PageTable(20, 300, 500, 16)
    book = Book(20, host.entries.shape[1], 16, 500)
    book.stack[:] = host.free
    d = Device(gpu, book, 4000)
    for step in range(8):
        gone = rng.random(20) < 0.2
        counts = rng.integers(0, 20, 20)
        for b in np.nonzero(gone)[0]:
            host.release(b)
        host.extend(counts)
        d.step(counts, gone)
        got = d.held()
        assert (got["next_lengths"] == host.lengths).all() and got["next_count"][0] == len(host.free)
        used = -(-host.lengths.astype(np.int64) // 16)
        for b in range(20):
            assert (got["table"][b, :used[b]] == host.entries[b, :used[b]]).all()
        assert (got["free"][:len(host.free)] == host.free).all()


def test_full_and_empty_batches(gpu):  # noqa: F811
    book = Book(3, 4, 8, 12)
    d = Device(gpu, book, 96)
    d.step([32, 32, 32])                                    # every page and every slot
    d.check(book.step([32, 32, 32]))
    assert book.top == 0
    d.step([32, 0, 5], [1, 0, 1])                           # all that came back goes out again
    d.check(book.step([32, 0, 5], [1, 0, 1]))
    d.step([0, 0, 0])
    d.check(book.step([0, 0, 0]))
    d.step([0, 0, 0], [1, 1, 1])
    d.check(book.step([0, 0, 0], [1, 1, 1]))
    assert book.top == 12
    d.step()                                                # no sequence at work
    d.check(book.step(None))
    empty = Device(gpu, Book(0, 4, 8, 5), 6)
    empty.step([], None)
    empty.check(empty.book.step([]))


@pytest.mark.parametrize("batch,tokens", [(4, 100), (4, 5000), (1100, 5000)])
def test_all_or_nothing(gpu, batch, tokens):  # noqa: F811
    """What does not fit is reported, and nothing but the step's own outputs changes."""
    fe = gpu[0]
    LENGTH, PAGES = 1, 7
    for in_place in (True, False):
        ref = Book(batch, 6, 8, 14)
        d = Device(gpu, ref, tokens, in_place)
        start, one = np.zeros(batch, np.int64), np.zeros(batch, np.int64)
        start[[0, 1, 3]] = 9, 8, 16
        d.step(start)
        d.check(ref.step(start))
        if not in_place:
            d.lengths.copy_(d.next_lengths)
            d.count.copy_(d.next_count)
        before, number = d.held(), np.arange(batch)
        for counts, release, status in ((one + 48 * (number == 0), None, LENGTH),             # past its row of the table
                                        (one + (1 << 31) * (number == 2), None, LENGTH),      # past 31 bits
                                        (one + 0xffffffff * (number < 2), None, LENGTH),
                                        (one + 24 * (number < 4), None, PAGES),               # 12 pages where 9 are free
                                        (one + 24 * (number < 4) + 8 * (number == 2), number == 1, PAGES)):   # 13 where 10 are
            with pytest.raises(fe.Fe2o3Error):
                d.step(counts, release)
            assert d.status == (LENGTH if counts.sum() > tokens else status)
            got = d.held()
            for n in ("table", "free"):
                assert (got[n] == before[n]).all(), n
            assert (got["next_lengths"] == ref.lengths).all() and got["next_count"][0] == ref.top
            assert (got["offsets"] == 0).all() and (got["positions"] == 0).all() and (got["slots"] == FREE).all()
    # more tokens than the map holds; without a map that is no matter
    d = Device(gpu, Book(2, 6, 8, 12), 10)
    with pytest.raises(fe.Fe2o3Error):
        d.step([6, 5])
    assert (d.held()["slots"] == FREE).all() and (d.held()["next_lengths"] == 0).all()
    d.step([6, 5], positions=None, slots=None)
    assert d.held()["next_lengths"].tolist() == [6, 5] and d.held()["offsets"].tolist() == [0, 6, 11]
    d.step([1, 1], positions=None, token_offsets=None)
    assert d.held()["slots"][:2].tolist() == [int(d.held()["table"][0, 0]) * 8 + 6, int(d.held()["table"][1, 0]) * 8 + 5]
    d.step([1, 1], slots=None, token_offsets=None)
    assert d.held()["positions"].tolist() == [7, 6] + [0] * 8


def test_what_the_state_holds_is_not_trusted(gpu):  # noqa: F811
    """A length beyond the table, more free pages than there are, page numbers that are none."""
    fe, torch, ctx, stream = gpu
    d = Device(gpu, Book(2, 3, 8, 6), 20)
    d.lengths.copy_(d.up(np.array([25, 0], np.uint32)))
    for release in (None, [1, 0]):
        with pytest.raises(fe.Fe2o3Error):
            d.step([0, 1], release)
        assert d.held()["next_lengths"].tolist() == [25, 0] and (d.held()["slots"] == FREE).all()
    d.lengths.zero_()
    d.count.fill_(7)
    with pytest.raises(fe.Fe2o3Error):
        d.step([0, 1])
    d.count.fill_(6)
    d.lengths.fill_(8)
    with pytest.raises(fe.Fe2o3Error):
        d.step([0, 0], [1, 1])                              # no room on the stack for pages that were never taken
    assert d.held()["next_count"][0] == 6
    d.lengths.zero_()
    d.free.fill_(1 << 30)
    with pytest.raises(fe.Fe2o3Error):
        d.step([3, 1])
    assert (d.held()["slots"] == FREE).all() and d.held()["positions"].tolist() == [0, 1, 2, 0] + [0] * 16
    p = fe.prepare(ctx, "kv_pages_v1", **d.args())
    p.launch(stream)
    stream.synchronize()
    ctx.take_kernel_status(stream)
    p.destroy()


def test_steps_replay_from_a_graph_and_run_on_another_stream(gpu):  # noqa: F811
    fe, torch, ctx, stream = gpu
    book = Book(40, 20, 16, 900)
    d = Device(gpu, book, 100)
    start = np.arange(40) % 5
    d.step(start)
    d.check(book.step(start))
    p = fe.prepare(ctx, "kv_pages_v1", **d.args())
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        p.launch(ctx.wrap_stream(side.cuda_stream))
    for _ in range(30):
        graph.replay()
        torch.cuda.synchronize()
        d.check(book.step(None))
    own = ctx.create_stream()
    p.launch(own)
    own.synchronize()
    d.check(book.step(None))
    p.destroy()
    assert ctx.take_kernel_status(stream) == 0


PATCHED = """
import struct, sys
sys.path[:0] = [{root!r}, {tests!r}]
import numpy as np, torch
import fe2o3_b200 as fe
from test_gpu_kv_pages import Book, Device
ctx = fe.GpuContext(0)
gpu = (fe, torch, ctx, ctx.default_stream())
book = Book({batch}, 300, 16, {batch} * 300)
d = Device(gpu, book, 5000)
counts = np.arange({batch}) % 4 * (5000 // {batch} // 8) + 1
p = fe.prepare(ctx, "kv_pages_v1", counts=d.up(counts.astype(np.uint32)), **d.args(positions=d.positions[:{first}], slots=d.slots[:{first}], tokens={first}))
p.patch_kernarg(188, struct.pack("<I", 5000))
p.launch_and_wait(gpu[3], 20000)
d.check(book.step(counts))
p.destroy()
print("patched plan is right")
"""


@pytest.mark.parametrize("batch,first", [(4, 64), (1000, 1000)])
def test_a_plan_patched_to_many_tokens(gpu, batch, first):  # noqa: F811
    """In a process of its own: what a prepare leaves behind for later launches stays with the process."""
    import os
    import subprocess
    import sys
    tests = os.path.dirname(os.path.abspath(__file__))
    done = subprocess.run([sys.executable, "-c", PATCHED.format(root=os.path.dirname(tests), tests=tests, batch=batch, first=first)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "patched plan is right" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("batch,most,tokens", [(3200, 9, 20003), (8191, 5, 30000), (8192, 1, 8192), (8192, 40, 100001)])
def test_the_largest_batches(gpu, batch, most, tokens, in_place):  # noqa: F811
    """More sequences than 48 KiB of shared memory hold, up to the most that are admitted."""
    test_steps(gpu, batch, 16, most, tokens, in_place)


@pytest.mark.parametrize("batch,tokens", [(5, 60), (700, 9000)])
def test_lengths_to_attend_to(gpu, batch, tokens):  # noqa: F811
    """The next lengths, with counts and without; zeros, and nothing else new, where a step does not fit."""
    fe, torch = gpu[:2]
    rng = np.random.default_rng(batch)
    for in_place in (True, False):
        book = Book(batch, 6, 8, 6 * batch)
        d = Device(gpu, book, tokens, in_place)
        attended = torch.full((batch,), 77, dtype=torch.int32, device="cuda")
        for counts, release in ((rng.integers(0, 12, batch), None), (None, None), (rng.integers(0, 9, batch), rng.random(batch) < 0.4), (np.full(batch, 49), None),
                                (None, rng.random(batch) < 0.4)):
            if counts is not None and counts.max() > 48:
                with pytest.raises(fe.Fe2o3Error):
                    d.step(counts, release, attended=attended)
                assert (attended == 0).all() and (d.held()["next_lengths"] == book.lengths).all()
                continue
            d.step(counts, release, attended=attended)
            d.check(book.step(counts, release))
            assert (attended.cpu().numpy() == book.lengths).all()
            if not in_place:
                d.lengths.copy_(d.next_lengths)
                d.count.copy_(d.next_count)


def test_packed_blocks_of_both_sizes(gpu):  # noqa: F811
    """The runtime adapter takes a block without its last slice, the lengths to attend to, as one where that is empty; no other size."""
    import ctypes as C
    import hashlib
    fe, torch, ctx, stream = gpu
    from fe2o3_b200._lib import LIB_PATH, lib
    with open(LIB_PATH, "rb") as f:
        image = f.read()
    exe, kid, nbytes, status = C.c_void_p(), C.c_uint32(), C.c_uint64(), C.c_uint32()
    digest = (C.c_uint8 * 32).from_buffer_copy(hashlib.sha256(image).digest())
    fe.check(lib.fe2o3_load_executable(ctx._h, image, C.c_uint64(len(image)), digest, C.byref(exe)))
    fe.check(lib.fe2o3_resolve_kernel(exe, b"kv_pages_v1", C.byref(kid), C.byref(nbytes)))
    assert nbytes.value == 208
    book = Book(7, 10, 8, 70)
    d = Device(gpu, book, 60)
    attended = torch.full((7,), 77, dtype=torch.int32, device="cuda")
    for size, counts in ((192, [5, 0, 9, 1, 8, 16, 3]), (208, [1, 2, 3, 4, 5, 6, 7]), (192, [0, 1, 0, 1, 0, 1, 0])):
        n = d.up(np.array(counts, np.uint32))
        args = fe.make_args("kv_pages_v1", counts=n, **d.args(**(dict(attended=attended) if size == 208 else {})))
        block = (C.c_uint8 * size).from_buffer_copy(bytes(args)[:size])
        for wrong in (191, 200):
            assert lib.fe2o3_launch_and_wait(exe, kid, None, block, C.c_uint64(wrong), stream._h, C.c_uint32(5000), C.byref(status)) == -5
        fe.check(lib.fe2o3_launch_and_wait(exe, kid, None, block, C.c_uint64(size), stream._h, C.c_uint32(5000), C.byref(status)))
        d.check(book.step(counts))
        if size == 208:
            assert (attended.cpu().numpy() == book.lengths).all()
    fe.check(lib.fe2o3_unload_executable(exe))
