"""The pages' bookkeeping on the device against its sequential form (oracle/paged.py), value by value."""
import numpy as np
import pytest

from helpers import seeded
from kandle_amd import Tensor
from kandle_amd import functional as F
from kandle_amd import _lib
from kandle_amd._lib import KandleHipError
from kandle_amd.graphs import HipGraph
from oracle import paged as op

pytestmark = pytest.mark.gpu


def i32(x):
    return Tensor(np.ascontiguousarray(x, np.int32), dtype="int32")


def same(got, want):
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g.numpy(), w)


def world(seed, rows, width, pages, page):
    """A table grown by random steps, with shared pages."""
    r = np.random.default_rng(seed)
    table, lens, refs = np.full((rows, width), -1), np.zeros(rows, np.int64), np.zeros(pages, np.int64)
    for _ in range(4):
        counts = r.integers(0, max(2, width * page // 6), size=rows)
        table, lens, refs, _, _ = op.pages_reserve(table, lens, refs, counts, page)
        parents = np.where(r.random(rows) < 0.1, -1, r.integers(0, rows, size=rows))
        table, lens, refs = op.pages_fork(table, lens, refs, parents)
    return r, table, lens, refs


@pytest.mark.parametrize("rows,width,pages,page", [(1, 1, 1, 16), (64, 128, 6000, 16), (64, 130, 6000, 16), (3, 4, 17000, 16), (4, 9, 40, 16), (70, 20, 900, 32), (300, 5, 3000, 16),
                                                   (1500, 3, 2500, 64), (5, 700, 9000, 16)])
def test_fork_and_reserve(hip, rows, width, pages, page):
    r, table, lens, refs = world(rows, rows, width, pages, page)
    for step in range(4):
        parents = r.integers(-1, rows + (step == 3), size=rows)
        want = op.pages_fork(table, lens, refs, parents)
        got = F.pages_fork(i32(table), i32(lens), i32(refs), i32(parents))
        same(got, want)
        counts = r.integers(-1, [2, page + 2, 3 * page, 2][step], size=rows)
        after = op.pages_reserve(*want, counts, page)
        moves, info = F.pages_reserve(*got, i32(counts), page)
        same([*got, moves, info], after)
        table, lens, refs = after[:3]


@pytest.mark.parametrize("rows,free,count", [(40, 0.02, 100), (40, 0.02, 33), (1100, 0.6, 80), (2048, 0.9, 60), (2048, 0.3, 40), (7, 0.0, 1)])
def test_reserve_from_a_large_pool(hip, rows, free, count):
    """Free pages few and far between, or behind the first thousands; enough of them or not; rows that are too long."""
    r = np.random.default_rng(rows + count)
    pages, width, page = 11000, 8, 16
    refs = (r.random(pages) >= free).astype(np.int64)
    lens = r.integers(0, 60, rows)
    table = np.where(np.arange(width) < -(-lens // page)[:, None], r.integers(0, pages, (rows, width)), -1)
    refs[table[table >= 0]] += 1                     # some are shared
    for counts in (r.integers(-1, count, rows), np.full(rows, 1), np.where(np.arange(rows) == rows - 1, 1000, 1)):
        want = op.pages_reserve(table, lens, refs, counts, page)
        t, n, f = i32(table), i32(lens), i32(refs)
        moves, info = F.pages_reserve(t, n, f, i32(counts), page)
        same([t, n, f, moves, info], want)


def test_the_last_sharer_keeps_the_tail_page(hip):
    table = np.array([[3, 1, -1], [3, 1, -1], [3, 1, -1], [5, 2, -1], [5, 2, -1]])
    lens, refs = np.array([20, 20, 20, 31, 31]), np.array([0, 3, 2, 3, 0, 2, 0, 0])
    for counts in ([1, 1, 1, 1, 1], [1, 0, 1, 0, 3], [0, 0, 1, 20, 0], [1, 1, 1, 1, 18], [0] * 5, [-3] * 5):
        t, n, f = i32(table), i32(lens), i32(refs)
        moves, info = F.pages_reserve(t, n, f, i32(counts), 16)
        same([t, n, f, moves, info], op.pages_reserve(table, lens, refs, counts, 16))


def test_reserve_is_all_or_nothing(hip):
    table, lens, refs = np.array([[0, -1, -1], [1, 2, -1]]), np.array([16, 30]), np.array([1, 1, 1, 0, 0])
    for counts, what in (([20, 20], (0, 0, 1)), ([33, 1], (0, 0, 1)), ([32, 18], (0, 1, 0)), ([33, 19], (0, 0, 2)), ([32, 2], (0, 0, 0))):
        t, n, f = i32(table), i32(lens), i32(refs)
        moves, info = F.pages_reserve(t, n, f, i32(counts), 16)
        want = op.pages_reserve(table, lens, refs, counts, 16)
        same([t, n, f, moves, info], want)
        assert what[2] == info.numpy()[2] and (what[1] > 0) == (info.numpy()[1] > 0)


def test_a_hole_in_the_tail_gets_a_page_and_no_copy(hip):
    table, lens, refs = np.array([[0, -1, -1], [-1, 2 ** 30, -1]]), np.array([20, 25]), np.array([1, 0, 0, 0])
    t, n, f = i32(table), i32(lens), i32(refs)
    moves, info = F.pages_reserve(t, n, f, i32([1, 8]), 16)
    same([t, n, f, moves, info], op.pages_reserve(table, lens, refs, [1, 8], 16))
    assert info.numpy().tolist() == [0, 0, 0] and t.numpy()[:, 1].tolist() == [1, 2]


def test_lengths_out_of_range_change_nothing_outside(hip):
    """Garbage on the device is refused by `info`, or ignored, and never addresses anything."""
    table, refs = np.array([[0, 1], [-7, 99]]), np.array([1, 1, 0])
    for lens, counts in (([2 ** 31 - 1, 40], [5, 2 ** 31 - 1]), ([-5, 33], [1, 1]), ([2 ** 31 - 1, 2 ** 31 - 1], [0, 0])):
        t, n, f = i32(table), i32(lens), i32(refs)
        moves, info = F.pages_reserve(t, n, f, i32(counts), 16)
        same([t, n, f, moves, info], op.pages_reserve(table, np.array(lens), refs, counts, 16) if max(counts) else
             (table, lens, refs, np.full((2, 2), -1), [0, 0, 0]))


@pytest.mark.parametrize("rows,width,pages", [(1, 4, 1), (3, 9, 41), (20, 30, 1500), (64, 70, 5003)])
def test_compact(hip, rows, width, pages):
    r = np.random.default_rng(pages)
    ids = r.permutation(pages)[: max(1, pages // 3)]
    table = np.full((rows, width), -1)
    flat = table.reshape(-1)
    flat[r.permutation(flat.size)[:min(len(ids), flat.size)]] = ids[:flat.size]
    table[-1] = table[0]                                       # shared pages
    table[0, -1] = 2 ** 30                                     # no page: stays as it is
    refs = op.count_refs(table, pages)
    got = F.pages_compact(i32(table), i32(refs))
    want = op.pages_compact(table, refs, max(1, pages // 2))
    same(got, want)
    again = F.pages_compact(got[0], got[1])
    assert again[3].numpy().tolist() == [0, int((refs > 0).sum())]
    same(again[:2], want[:2])


@pytest.mark.parametrize("dtype,planes,pages,shape", [("float32", (2, 2), 30, (2, 16, 64)), ("bfloat16", (), 50, (8, 16, 128)),
                                                      ("bfloat16", (3, 2), 9, (3, 32, 40)), ("float32", (1,), 7, (1, 16, 4))])
def test_copy(hip, dtype, planes, pages, shape):
    x, xh = seeded(81, (*planes, pages, *shape), dtype)
    ids = np.random.default_rng(pages).permutation(pages)
    n = pages // 3
    moves = np.stack([ids[:n], ids[n:2 * n]], 1)
    moves[0] = [ids[0], pages]                                 # outside the pool: skipped
    moves[1] = [-1, ids[n + 1]]
    for count in (n, 0, n + 100, -4, 2):
        y = F.clone(x)
        F.pages_copy(y, i32(moves), i32([count]))
        np.testing.assert_array_equal(y.numpy(), op.pages_copy(xh, moves, max(0, count)))


def test_copy_past_the_caches(hip):
    """Enough bytes for the copy's streaming form, in pages that are not whole pieces of it."""
    xh = np.random.default_rng(83).integers(0, 1 << 16, (5, 400, 8, 64, 120), dtype=np.uint16)
    x = Tensor(xh, dtype="bfloat16")
    ids = np.random.default_rng(84).permutation(400)
    moves = np.stack([ids[:150], ids[150:300]], 1)
    F.pages_copy(x, i32(moves), i32([150]))
    xh[:, moves[:, 1]] = xh[:, moves[:, 0]]
    np.testing.assert_array_equal(x.handle.raw_bits(), xh)


def test_a_beam_of_steps_replayed_from_a_graph(hip):
    """fork, reserve, copy of two steps (there and back between two sets of buffers) captured once, replayed with
    new parents, against the sequential form; what each row has written stays readable."""
    rows, width, pages, page = 6, 8, 60, 16
    r = np.random.default_rng(5)
    table, lens, refs, _, _ = op.pages_reserve(np.full((rows, width), -1), np.zeros(rows, np.int64), np.zeros(pages, np.int64),
                                               r.integers(1, 40, size=rows), page)
    pool, ph = seeded(83, (2, pages, 2, page, 8))
    a = [i32(table), i32(lens), i32(refs)]
    b = [i32(table), i32(lens), i32(refs)]
    p1, p2, ones = i32(np.zeros(rows)), i32(np.zeros(rows)), i32(np.ones(rows))
    m1, f1, m2, f2 = (F.zeros(s, "int32") for s in ((rows, 2), (3,), (rows, 2), (3,)))
    g = HipGraph()
    with g.capture():
        F.pages_fork(*a, p1, out=tuple(b))
        F.pages_reserve(*b, ones, page, out=(m1, f1))
        F.pages_copy(pool, m1, f1)
        F.pages_fork(*b, p2, out=tuple(a))
        F.pages_reserve(*a, ones, page, out=(m2, f2))
        F.pages_copy(pool, m2, f2)
    for step in range(5):
        for t, m, f in ((p1, m1, f1), (p2, m2, f2)):
            parents = r.integers(0, rows, size=rows)
            t.handle.storage.upload(parents.astype(np.int32))
            table, lens, refs = op.pages_fork(table, lens, refs, parents)
            table, lens, refs, moves, info = op.pages_reserve(table, lens, refs, np.ones(rows, np.int64), page)
            ph = op.pages_copy(ph, moves, info[0])
        g.replay()
        same([*a, m2, f2, pool], [table, lens, refs, moves, info, ph])
    g.dispose()


def test_refusals(hip):
    t, n, f, p = i32(np.zeros((2, 3))), i32([0, 0]), i32([0] * 5), i32([0, 1])
    with pytest.raises(KandleHipError, match="share memory"):
        F.pages_fork(t, n, f, p, out=(t, i32([0, 0]), i32([0] * 5)))
    with pytest.raises(KandleHipError, match="share memory"):
        F.pages_fork(t, n, f, p, out=(i32(np.zeros((2, 3))), i32([0, 0]), f))
    with pytest.raises(KandleHipError, match="share memory"):
        F.pages_compact(t, f, out=(t, i32([0] * 5), i32(np.zeros((2, 2))), i32([0, 0])))
    for size in (0, 8, 24, 8192):
        with pytest.raises(KandleHipError, match="page size"):
            F.pages_reserve(t, n, f, p, size)
    with pytest.raises(KandleHipError, match="at most 2048"):
        F.pages_reserve(i32(np.zeros((2049, 1))), i32(np.zeros(2049)), f, i32(np.zeros(2049)), 16)
    with pytest.raises(KandleHipError, match="multiple of 16"):
        F.pages_copy(F.zeros((4, 1, 1, 3)), i32([[0, 1]]), i32([1]))


def test_operands_that_share_memory_are_refused(hip):
    new = lambda *s: i32(np.zeros(s))  # noqa: E731
    t, n, f, p = new(2, 3), new(2), new(5), new(2)
    for lens in (n, p):
        with pytest.raises(KandleHipError, match="share memory"):
            F.pages_fork(t, n, f, p, out=(new(2, 3), lens, new(5)))
    with pytest.raises(KandleHipError, match="share memory"):
        F.pages_reserve(t, n, f, n, 16)
    both = new(7)
    with pytest.raises(KandleHipError, match="share memory"):
        F.pages_reserve(t, n, f, p, 16, out=(F.view(F.narrow(both, 0, 0, 4), (2, 2)), F.narrow(both, 0, 3, 3)))
    F.pages_reserve(t, n, f, p, 16, out=(F.view(F.narrow(both, 0, 0, 4), (2, 2)), F.narrow(both, 0, 4, 3)))
    with pytest.raises(KandleHipError, match="share memory"):
        F.pages_compact(t, f, out=(new(2, 3), f, new(2, 2), new(2)))


def test_tables_past_the_counters_are_refused(hip):
    a = i32(np.zeros(64))
    with pytest.raises(KandleHipError, match="2\\^31 entries"):   # refused on the host, whatever the pointers are
        _lib.call("kh_pages_reserve", a.handle.data_ptr(), 1 << 26, a.handle.data_ptr(), a.handle.data_ptr(), a.handle.data_ptr(), 64,
                  1 << 26, 64, 16, a.handle.data_ptr(), a.handle.data_ptr())
