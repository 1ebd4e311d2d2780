"""paged_attention and paged_kv_write against their float64 forms (oracle/paged.py), element by element within
the bound that oracle.paged.attention_bound counts."""
import numpy as np
import pytest

from helpers import dev, seeded
from kandle_amd import Tensor
from kandle_amd import functional as F
from kandle_amd import synthetic as syn
from kandle_amd._lib import KandleHipError
from kandle_amd.graphs import HipGraph
from oracle import paged as op

pytestmark = pytest.mark.gpu


def i32(x):
    return Tensor(np.ascontiguousarray(x, np.int32), dtype="int32")


class Cache:
    """Random pools and a shuffled page table for sequences of the given lengths."""

    def __init__(self, seed, dtype, lens, hkv, d, page, spare=3):
        self.dtype, self.page, self.lens = dtype, page, np.asarray(lens)
        count = -(-self.lens // page)
        pages = int(count.sum()) + spare
        ids = np.random.default_rng(seed).permutation(pages)
        self.table = np.full((len(lens), max(1, int(count.max(initial=0)) + 2)), -1, np.int64)
        at = 0
        for b, n in enumerate(count):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.k, self.kh = seeded(seed, (pages, hkv, page, d), dtype)
        self.v, self.vh = seeded(seed + 1, (pages, hkv, page, d), dtype)


def check(c, seed, news, hq, causal=True, scale=None, starts=True, **kw):
    """Runs the op for `news` new tokens per sequence and compares every row."""
    d = c.kh.shape[3]
    st = np.concatenate([[0], np.cumsum(news)])
    q, qh = seeded(seed, (int(st[-1]), hq, d), c.dtype)
    o = F.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lens), i32(st) if starts else None, scale=scale, is_causal=causal, **kw)
    compare(c, qh, o.numpy(), st, causal, scale)


def compare(c, qh, got, st, causal=True, scale=None, out=None):
    ref, a, smax = op.paged_attention(qh, c.kh, c.vh, c.table, c.lens, st, scale, causal, out)
    bound = op.attention_bound(c.dtype, ref, a, smax, qh.shape[2], int(c.lens.max(initial=1)))
    off = np.abs(got - ref)
    assert np.isfinite(got).all() and (off <= bound).all(), (float(np.nanmax(off / bound)), np.argwhere(~(off <= bound))[:5])


DTYPES = ("float32", "bfloat16")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page", [(4, 2, 128, 16), (16, 8, 128, 32), (5, 1, 64, 16), (8, 8, 64, 64), (40, 8, 128, 16),
                                           (24, 1, 128, 128), (34, 2, 64, 16)])
def test_one_token_per_sequence(hip, dtype, hq, hkv, d, page):
    c = Cache(1, dtype, [1, 15, 16, 17, 300, 1025, 2, 777], hkv, d, page)
    check(c, 3, [1] * 8, hq, starts=False, max_query_len=1, max_kv_len=1025)
    check(c, 4, [1] * 8, hq, starts=False)
    check(c, 5, [1] * 8, hq)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page,lens,news", [
    (4, 2, 128, 16, [1], [1]),
    (4, 2, 128, 16, [40, 64, 63, 65], [40, 1, 63, 2]),
    (16, 8, 128, 16, [333, 20, 700], [70, 20, 129]),
    (10, 2, 64, 32, [500, 131], [3, 131]),
    (3, 3, 128, 64, [260, 129], [260, 128]),
    (24, 2, 128, 16, [100, 350], [33, 17]),
    (34, 2, 64, 16, [77, 200], [5, 40]),
    (8, 8, 64, 16, [600, 1, 40], [300, 1, 0]),
    (4, 1, 128, 256, [1100], [513]),
    (4, 2, 128, 16, [7000], [300]),              # 256-row tiles
    (8, 2, 64, 32, [6500, 6300], [70, 100]),
    (2, 2, 128, 16, [2300, 9], [7, 9]),
])
def test_ragged_chunks(hip, dtype, hq, hkv, d, page, lens, news):
    c = Cache(7, dtype, lens, hkv, d, page)
    check(c, 9, news, hq)
    check(c, 10, news, hq, causal=False)
    check(c, 11, news, hq, max_query_len=max(news), max_kv_len=max(lens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("news", [[1, 1, 1], [3, 90, 1], [200, 40, 150]])
def test_evicted_pages_and_rows_that_see_nothing(hip, dtype, news):
    c = Cache(13, dtype, [400, 90, 333], 2, 128, 16)
    c.table[0, 1:9] = -1                       # a hole in the middle
    c.table[1, :] = -1                         # nothing left
    c.table[2, 0:3] = [-1, c.kh.shape[0], 2 ** 30]   # ids outside the pool are holes, too
    check(c, 15, news, 4)
    check(c, 16, news, 4, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_tokens_than_rows_and_empty_sequences(hip, dtype):
    c = Cache(17, dtype, [3, 0, 20], 2, 64, 16)
    check(c, 19, [8, 4, 0], 4)                 # the first five tokens, and a whole sequence, see no row
    check(c, 20, [8, 4, 0], 4, causal=False)
    check(c, 21, [0, 0, 0], 4)
    q = Tensor(np.zeros((0, 4, 64), np.float32), dtype=dtype)
    assert F.paged_attention(q, c.k, c.v, i32(np.zeros((0, 3))), i32(np.zeros(0)), i32([0])).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 1e-3])
def test_scales(hip, dtype, scale):
    c = Cache(23, dtype, [150, 70], 2, 64, 16)
    check(c, 25, [1, 70], 4, scale=scale)
    check(c, 26, [90, 3], 4, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("news", [[1, 1], [30, 100]])
def test_rows_outside_the_sequences_stay_and_limits_hold(hip, dtype, news):
    c = Cache(27, dtype, [200, 333], 2, 128, 16)
    st = np.concatenate([[0], np.cumsum(news)])
    tokens = int(st[-1]) + 5
    q, qh = seeded(29, (tokens, 4, 128), dtype)
    for limits in ({}, {"max_query_len": max(news), "max_kv_len": 333}):
        out, oh = seeded(31, (tokens, 4, 128), dtype)
        got = F.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lens), i32(st), out=out, **limits).numpy()
        np.testing.assert_array_equal(got[st[-1]:], oh[st[-1]:])
        compare(c, qh[:st[-1]], got[:st[-1]], st)
    # rows at or behind max_kv_len are not seen, tokens at or behind max_query_len not computed
    out, oh = seeded(33, (tokens, 4, 128), dtype)
    got = F.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lens), i32(st), is_causal=False, out=out, max_query_len=1,
                            max_kv_len=100).numpy()
    kept = np.ones(tokens, bool)
    kept[st[:-1]] = False
    np.testing.assert_array_equal(got[kept], oh[kept])
    for b in range(2):
        one = Cache(27, dtype, [200, 333], 2, 128, 16)
        one.table, one.lens = one.table[b:b + 1], np.array([100])
        compare(one, qh[st[b]:st[b] + 1], got[st[b]:st[b] + 1], np.array([0, 1]), causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("news,hq", [([1, 1], 4), ([16, 5], 4), ([40, 300], 4), ([40, 300], 24), ([200, 2], 8)])
@pytest.mark.parametrize("poison", [np.nan, np.inf, -np.inf])
def test_values_in_masked_places_do_not_matter(hip, dtype, news, hq, poison):
    """Rows behind the cached ones, pages of nobody, and later tokens' rows may hold anything."""
    c = Cache(35, dtype, [200, 333], 2, 128, 16)
    st = np.concatenate([[0], np.cumsum(news)])
    q, qh = seeded(37, (int(st[-1]), hq, 128), dtype)
    mine = [(c.table[b, p // 16], p % 16) for b in range(2) for p in range(c.lens[b])]
    k, v = np.full_like(c.kh, poison), np.full_like(c.vh, poison)
    for page, slot in mine:
        k[page, :, slot], v[page, :, slot] = c.kh[page, :, slot], c.vh[page, :, slot]
    run = lambda kk, vv: F.paged_attention(q, dev(kk, dtype), dev(vv, dtype), i32(c.table), i32(c.lens), i32(st)).numpy()  # noqa: E731
    compare(c, qh, run(k, v), st)
    # the last new token's own row of each sequence is for it alone (columns 5 and 70 of its value)
    for b in range(2):
        page, slot = c.table[b, (c.lens[b] - 1) // 16], (c.lens[b] - 1) % 16
        v[page, :, slot, [5, 70]] = poison
    got = run(k, v)
    last = st[1:] - 1
    early = np.setdiff1d(np.arange(st[-1]), last)
    ref, a, smax = op.paged_attention(qh, c.kh, c.vh, c.table, c.lens, st)
    bound = op.attention_bound(dtype, ref, a, smax, 128, 333)
    assert (np.abs(got - ref)[early] <= bound[early]).all()
    cols = np.setdiff1d(np.arange(128), [5, 70])
    assert (np.abs(got - ref)[last][..., cols] <= bound[last][..., cols]).all()
    seen = got[last][..., [5, 70]]
    assert np.isnan(seen).all() if np.isnan(poison) else (seen == poison).all()
    # a later token's key
    k[page, :, slot, 3] = poison
    got = run(k, v)
    early = np.setdiff1d(np.arange(st[-1]), last)
    assert (np.abs(got - ref)[early] <= bound[early]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_nan_query_stays_in_its_row(hip, dtype):
    c = Cache(39, dtype, [200, 333], 2, 64, 16)
    st = np.array([0, 40, 41])
    q, qh = seeded(41, (41, 4, 64), dtype)
    bad = np.array(qh)
    bad[17, 2, 9] = np.nan
    got = F.paged_attention(dev(bad, dtype), c.k, c.v, i32(c.table), i32(c.lens), i32(st)).numpy()
    assert np.isnan(got[17, 2]).all()
    ref, a, smax = op.paged_attention(qh, c.kh, c.vh, c.table, c.lens, st)
    rest = np.ones((41, 4), bool)
    rest[17, 2] = False
    assert (np.abs(got - ref) <= op.attention_bound(dtype, ref, a, smax, 64, 333))[rest].all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("news", [[1, 1], [50, 7], [200, 7]])
def test_large_scores(hip, dtype, news):
    """Scores of hundreds, growing along the sequence: the running maximum has to follow."""
    c = Cache(43, dtype, [500, 260], 2, 64, 16)
    k = np.array(c.kh)
    for b in range(2):
        for p in range(c.lens[b]):
            k[c.table[b, p // 16], :, p % 16] *= 0.05 * (1 + p)
    bits, c.kh = syn.bf16(k.astype(np.float32)) if dtype == "bfloat16" else (k, k.astype(np.float32))
    c.k = Tensor(bits, dtype=dtype) if dtype == "bfloat16" else dev(c.kh)
    check(c, 45, news, 4, scale=1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("news", [[1, 1, 1], [33, 100, 2]])
def test_strided_operands(hip, dtype, news):
    """Queries and outputs inside wider rows, pools with row-major heads, a table inside a wider one."""
    d, page, lens = 64, 16, np.array([300, 120, 31])
    c = Cache(47, dtype, lens, 3, d, page)
    pages = c.kh.shape[0]
    st = np.concatenate([[0], np.cumsum(news)])
    tokens = int(st[-1])
    wide, wh = seeded(49, (tokens, 20, d), dtype)                           # q heads 4..9 of 20
    q = F.narrow(wide, 1, 4, 6)
    out = F.narrow(F.zeros((tokens, 9, d), dtype), 1, 2, 6)
    kr = F.permute(dev(np.ascontiguousarray(c.kh.transpose(0, 2, 1, 3)), dtype), (0, 2, 1, 3))   # [pages, page, heads, d]
    both = F.zeros((pages, 2, 3, page, d), dtype)                           # values beside something else
    vv = F.narrow(both, 1, 1, 1)
    v = F.permute(vv, (0, 1, 2, 3, 4))
    v4 = Tensor(handle=type(v.handle).create_view(v.handle.storage, (pages, 3, page, d), dtype,
                                                  (v.strides[0], v.strides[2], v.strides[3], 1), v.offset))
    F.copy_(v4, c.v)
    table = F.narrow(i32(np.concatenate([np.full((3, 2), 1), c.table, np.full((3, 5), 2)], 1)), 1, 2, c.table.shape[1])
    F.paged_attention(q, kr, v4, table, i32(lens), i32(st), out=out)
    compare(c, wh[:, 4:10], out.numpy(), st)


@pytest.mark.parametrize("news", [[150, 2, 1], [300, 700, 1]])
def test_pools_with_the_heads_inside_the_rows(hip, news):
    """Equal strides of keys and values other than the usual: [pages, page size, heads, d] seen with heads first."""
    c = Cache(48, "bfloat16", [1300, 720, 31], 3, 128, 32)
    turn = lambda x: F.permute(dev(np.ascontiguousarray(x.transpose(0, 2, 1, 3)), "bfloat16"), (0, 2, 1, 3))  # noqa: E731
    c.k, c.v = turn(c.kh), turn(c.vh)
    check(c, 50, news, 6)
    check(c, 52, news, 6, causal=False)


def test_offsets_beyond_32_bits(hip):
    """A pool of 2^31 elements and more: pages at its far end."""
    page, d, pages = 16, 128, (1 << 20) + 5000
    k, v = F.zeros((pages, 1, page, d), "bfloat16"), F.zeros((pages, 1, page, d), "bfloat16")
    for lens, news in (([70, 500], [1, 1]), ([70, 500], [40, 30]), ([70, 500], [40, 300])):
        c = Cache(51, "bfloat16", lens, 1, d, page, spare=0)
        far = pages - c.kh.shape[0]
        for big, small in ((k, c.k), (v, c.v)):
            F.copy_(F.narrow(big, 0, far, c.kh.shape[0]), small)
        st = np.concatenate([[0], np.cumsum(news)])
        q, qh = seeded(53, (int(st[-1]), 2, d), "bfloat16")
        at = np.where(c.table >= 0, c.table + far, -1)
        compare(c, qh, F.paged_attention(q, k, v, i32(at), i32(c.lens), i32(st)).numpy(), st)
        rows, rh = seeded(55, (int(st[-1]), 1, d), "bfloat16")
        F.paged_kv_write(rows, rows, k, v, i32(at), i32(c.lens), i32(st))
        kp, vp = op.paged_kv_write(rh, rh, c.kh, c.vh, c.table, c.lens, st)
        np.testing.assert_array_equal(F.narrow(k, 0, far, c.kh.shape[0]).numpy(), kp)
        np.testing.assert_array_equal(F.narrow(v, 0, far, c.kh.shape[0]).numpy(), vp)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("news", [[1, 1, 1], [20, 300, 1]])
def test_repeats_and_graph_replays_are_the_same_bits(hip, dtype, news):
    """Two graphs that share the cache, replayed among eager calls; lengths read from the device at replay."""
    c = Cache(57, dtype, [900, 410, 77], 2, 128, 16)
    st = np.concatenate([[0], np.cumsum(news)])
    q, qh = seeded(59, (int(st[-1]), 8, 128), dtype)
    q2, q2h = seeded(61, (int(st[-1]), 8, 128), dtype)
    table, lens, starts = i32(c.table), i32(c.lens), i32(st)
    call = lambda x, **kw: F.paged_attention(x, c.k, c.v, table, lens, starts, **kw)  # noqa: E731
    want, want2 = call(q).numpy(), call(q2).numpy()
    compare(c, qh, want, st)
    g1, g2 = HipGraph(), HipGraph()
    with g1.capture():
        o1 = call(q)
    with g2.capture():
        o2 = call(q2)
    for _ in range(3):
        g1.replay()
        g2.replay()
        np.testing.assert_array_equal(call(q).numpy(), want)
        np.testing.assert_array_equal(o1.numpy(), want)
        np.testing.assert_array_equal(o2.numpy(), want2)
    shorter = np.maximum(c.lens - 37, np.asarray(news))
    lens.handle.storage.upload(shorter.astype(np.int32))
    g2.replay()
    c.lens = shorter
    compare(c, q2h, o2.numpy(), st)
    g1.dispose()
    g2.dispose()


@pytest.mark.parametrize("starts", [False, True])
def test_more_query_heads_than_a_tile_has_rows(hip, starts):
    """One token of 320 heads of one kv head: many packed rows with and without query starts."""
    c = Cache(62, "bfloat16", [700, 90, 1], 1, 64, 16)
    check(c, 64, [1, 1, 1], 320, starts=starts)
    if starts:
        check(c, 66, [3, 0, 1], 320)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,news,lens", [
    (1024, [512, 5], [600, 3000]),               # room for two full chunks, of which one is short
    (600, [300, 1, 0, 1], [300, 2000, 0, 1500]),
    (520, [1, 1], [2500, 1300]),
    (2000, [0, 200, 3], [0, 5000, 5000])])
def test_padded_batches(hip, dtype, tokens, news, lens):
    """The packed rows may have room for more tokens than the sequences use."""
    c = Cache(61, dtype, lens, 2, 128, 16)
    st = np.concatenate([[0], np.cumsum(news)])
    q, qh = seeded(63, (tokens, 4, 128), dtype)
    for most in (max(news), tokens // len(news), tokens):
        out, oh = seeded(65, (tokens, 4, 128), dtype)
        got = F.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lens), i32(st), out=out, max_query_len=most,
                                max_kv_len=max(lens)).numpy()
        np.testing.assert_array_equal(got[st[-1]:], oh[st[-1]:])
        if most >= max(news):
            compare(c, qh[:st[-1]], got[:st[-1]], st)


@pytest.mark.parametrize("lens,news", [([1200], [500]), ([1200, 901], [290, 210])])
def test_a_long_and_a_shorter_chunk(hip, lens, news):
    """Tiles that fill more than half of the chip: their keys in two chunks of different length."""
    c = Cache(75, "bfloat16", lens, 8, 64, 16)
    check(c, 77, news, 80, max_query_len=max(news), max_kv_len=1200)


def test_many_rows_of_pools_with_different_strides(hip):
    """Keys with the heads inside the rows, values with the rows inside the heads."""
    c = Cache(78, "bfloat16", [700, 90], 2, 128, 32)
    c.k = F.permute(dev(np.ascontiguousarray(c.kh.transpose(0, 2, 1, 3)), "bfloat16"), (0, 2, 1, 3))
    check(c, 79, [200, 1], 6)
    check(c, 80, [1, 90], 6)


def test_many_sequences(hip):
    """More sequences than are looked through at once, with gaps, lone tokens and chunks of many rows among them."""
    r = np.random.default_rng(67)
    news = np.where(r.random(700) < 0.3, 0, r.integers(1, 4, 700))
    news[[0, 255, 256, 511, 512, 699]] = [1, 150, 0, 140, 2, 133]
    lens = news + r.integers(0, 60, 700)
    c = Cache(69, "bfloat16", lens, 1, 64, 16)
    check(c, 71, news, 2)
    check(c, 72, news, 2, max_query_len=150, max_kv_len=int(lens.max()))


def test_refusals(hip):
    c = Cache(63, "float32", [40], 2, 64, 16)
    q = F.zeros((1, 4, 64))
    with pytest.raises(KandleHipError, match="page size"):
        F.paged_attention(q, F.zeros((3, 2, 24, 64)), F.zeros((3, 2, 24, 64)), i32(c.table), i32([40]))
    with pytest.raises(KandleHipError, match="head_dim"):
        F.paged_attention(F.zeros((1, 4, 96)), F.zeros((3, 2, 16, 96)), F.zeros((3, 2, 16, 96)), i32(c.table), i32([40]))
    with pytest.raises(KandleHipError, match="2\\^30"):
        F.paged_attention(q, F.zeros((1, 2, 4096, 64)), F.zeros((1, 2, 4096, 64)),
                          i32(np.zeros((1, 1 << 20))), i32([40]))
    with pytest.raises(KandleHipError, match="aligned"):
        F.paged_attention(F.narrow(F.zeros((1, 4, 66)), 2, 1, 64), c.k, c.v, i32(c.table), i32([40]))
    with pytest.raises(ValueError, match="max_kv_len"):
        F.paged_attention(q, c.k, c.v, i32(c.table), i32([40]), max_kv_len=-1)


# ---- the write ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,page,lens,news", [
    (8, 128, 16, [1, 16, 17, 400], [1, 1, 1, 1]),
    (2, 64, 32, [100, 64, 3], [100, 1, 3]),
    (3, 5, 16, [50, 20], [33, 20]),              # rows that are no multiple of 16 bytes
    (1, 128, 64, [700, 0, 9], [512, 0, 12]),     # more tokens than rows: the first three have no place
    (16, 128, 16, [90], [90]),
])
def test_write(hip, dtype, hkv, d, page, lens, news):
    c = Cache(65, dtype, lens, hkv, d, page)
    c.table[0, 0] = c.kh.shape[0] if len(lens) > 1 else c.table[0, 0]   # a row without a page is dropped
    st = np.concatenate([[0], np.cumsum(news)])
    k, kh = seeded(67, (int(st[-1]) + 2, hkv, d), dtype)                  # two rows behind the last sequence
    wide, wh = seeded(69, (int(st[-1]) + 2, hkv + 3, d), dtype)
    v = F.narrow(wide, 1, 2, hkv)
    F.paged_kv_write(k, v, c.k, c.v, i32(c.table), i32(c.lens), i32(st))
    kp, vp = op.paged_kv_write(kh, wh[:, 2:2 + hkv], c.kh, c.vh, c.table, c.lens, st)
    np.testing.assert_array_equal(c.k.numpy(), kp)
    np.testing.assert_array_equal(c.v.numpy(), vp)


def test_write_outside_the_table_is_dropped(hip):
    c = Cache(71, "float32", [40, 33], 2, 64, 16)
    k, kh = seeded(73, (2, 2, 64))
    lens = np.array([c.table.shape[1] * 16 + 1, 2 ** 31 - 1])
    F.paged_kv_write(k, k, c.k, c.v, i32(c.table), i32(lens))
    np.testing.assert_array_equal(c.k.numpy(), c.kh)
    np.testing.assert_array_equal(c.v.numpy(), c.vh)


def test_write_then_attend_in_a_captured_step(hip):
    """A decode loop's step on the device: write the new row, attend over all, lengths advanced between replays."""
    c = Cache(75, "bfloat16", [64, 30], 2, 64, 16)
    c.table[0, 4], c.table[1, 2] = c.kh.shape[0] - 1, c.kh.shape[0] - 2    # a page each for the rows to come
    table, lens = i32(c.table), i32(c.lens)
    q, k, v = (F.zeros((2, n, 64), "bfloat16") for n in (4, 2, 2))
    g = HipGraph()
    with g.capture():
        F.paged_kv_write(k, v, c.k, c.v, table, lens)
        o = F.paged_attention(q, c.k, c.v, table, lens)
    n = np.array(c.lens)
    for step in range(6):
        n = n + 1
        host = []
        for i, t in enumerate((q, k, v)):
            bits, vals = syn.bf16(syn.normal(100 + 3 * step + i, t.shape))
            t.handle.storage.upload(bits)
            host.append(vals)
        lens.handle.storage.upload(n.astype(np.int32))
        g.replay()
        c.kh, c.vh = op.paged_kv_write(host[1], host[2], c.kh, c.vh, c.table, n)
        c.lens = n
        compare(c, host[0], o.numpy(), np.array([0, 1, 2]))
    g.dispose()
