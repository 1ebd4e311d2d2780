"""Query starts and lengths that no program should pass (negative, falling, past the tokens, past the table): nothing
outside the operands is written, and where the starts only reach out of the tokens, what is inside is right.  (The places
that the kernels compute from them were checked on the host first, lane by lane.)"""
import numpy as np
import pytest

from helpers import seeded
from kandle_amd import Tensor
from kandle_amd import functional as F
from oracle import paged as op
from test_gpu_paged_attention import Cache, compare, i32

pytestmark = pytest.mark.gpu
TOP, LOW = 2 ** 31 - 1, -(2 ** 31)
BAD = {"falling": [90, 40, 400, 3, 700], "negative": [LOW, -3, -700, 650, LOW], "past": [TOP, TOP, 5, TOP, TOP],
       "all of it, twice": [0, 700, 0, 700, 0], "none": [700, 700, 700, 700, 700], "backwards": [700, 500, 300, 100, 0]}
LENS = {"fit": [400, 600, 333, 90], "wild": [TOP, LOW, -1, 10 ** 6]}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("starts", list(BAD))
def test_nothing_outside_is_written(hip, dtype, lens, starts):
    c = Cache(1, dtype, [400, 600, 333, 90], 2, 64, 16, spare=5)
    at, n = i32(BAD[starts]), i32(LENS[lens])
    wide, wh = seeded(3, (716, 4, 64), dtype)
    q, _ = seeded(5, (700, 4, 64), dtype)
    rows, _ = seeded(7, (700, 2, 64), dtype)
    for limits in ({}, {"max_query_len": 150, "max_kv_len": 500}, {"max_query_len": 1}):
        F.paged_attention(q, c.k, c.v, i32(c.table), n, at, out=F.narrow(wide, 0, 8, 700), **limits)
    got = wide.numpy()
    for part in (slice(0, 8), slice(708, 716)):
        np.testing.assert_array_equal(got[part], wh[part])
    np.testing.assert_array_equal(c.k.numpy(), c.kh)
    np.testing.assert_array_equal(c.v.numpy(), c.vh)
    F.paged_kv_write(rows, rows, c.k, c.v, i32(c.table), n, at)
    free = np.setdiff1d(np.arange(c.kh.shape[0]), c.table)
    assert len(free) == 5
    np.testing.assert_array_equal(c.k.numpy()[free], c.kh[free])
    np.testing.assert_array_equal(c.v.numpy()[free], c.vh[free])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("starts,lens", [([-5, 3, 7, TOP], [400, 90, 333]), ([LOW, 0, 300, 301], [40, 700, 333]),
                                         ([-1, 200, TOP, TOP], [400, TOP, 333]), ([0, 1, 2, 3], [TOP, 90, LOW])])
def test_starts_and_lengths_that_reach_out_are_cut(hip, dtype, starts, lens):
    tokens = 320
    c = Cache(9, dtype, [400, 720, 333], 2, 128, 16)
    q, qh = seeded(11, (tokens, 4, 128), dtype)
    out, oh = seeded(13, (tokens, 4, 128), dtype)
    got = F.paged_attention(q, c.k, c.v, i32(c.table), i32(lens), i32(starts), out=out).numpy()
    st = np.clip(starts, 0, tokens)
    np.testing.assert_array_equal(got[st[-1]:], oh[st[-1]:])
    c.lens = np.maximum(np.minimum(lens, 4000), 0)          # (rows behind the table are no rows)
    compare(c, qh, got, st, out=oh)
    rows, rh = seeded(15, (tokens, 2, 128), dtype)
    F.paged_kv_write(rows, rows, c.k, c.v, i32(c.table), i32(lens), i32(starts))
    kp, vp = op.paged_kv_write(rh, rh, c.kh, c.vh, c.table, np.array(lens), st)
    np.testing.assert_array_equal(c.k.numpy(), kp)
    np.testing.assert_array_equal(c.v.numpy(), vp)


def test_no_sequence_at_all(hip):
    q, pools = F.zeros((3, 4, 64)), F.zeros((2, 2, 16, 64))
    out, oh = seeded(17, (3, 4, 64))
    F.paged_attention(q, pools, pools, Tensor(np.zeros((0, 4), np.int32), dtype="int32"), i32(np.zeros(0)), i32([0]), out=out)
    np.testing.assert_array_equal(out.numpy(), oh)
