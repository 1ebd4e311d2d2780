"""Results that share memory with inputs are refused before anything is launched; views of one buffer that share none are
taken."""
import numpy as np
import pytest

from helpers import dev, seeded
from kandle_amd import Tensor
from kandle_amd import functional as F
from kandle_amd._lib import KandleHipError
from oracle import paged as op

pytestmark = pytest.mark.gpu
SHARED = pytest.raises(KandleHipError, match="share memory")


def i32(x):
    return Tensor(np.ascontiguousarray(x, np.int32), dtype="int32")


def view(t, shape, strides, offset, dtype="float32"):
    return Tensor(handle=type(t.handle).create_view(t.handle.storage, shape, dtype, strides, offset))


def test_attention_refuses_an_output_among_its_inputs(hip):
    q, kp, vp = F.zeros((2, 4, 64)), F.zeros((5, 2, 16, 64)), F.zeros((5, 2, 16, 64))
    table, lens, starts = i32([[0, 1], [2, 3]]), i32([20, 30]), i32([0, 1, 2])
    call = lambda out, q=q, **kw: F.paged_attention(q, kp, vp, table, lens, starts, out=out, **kw)  # noqa: E731
    with SHARED:
        call(q)
    for pool in (kp, vp):
        with SHARED:                              # rows of the last page
            call(view(pool, (2, 4, 64), (256, 64, 1), 4 * 2048 + 1536))
    wide = F.zeros((3, 4, 64))
    with SHARED:                                  # a token further
        call(F.narrow(wide, 0, 1, 2), F.narrow(wide, 0, 0, 2))
    rows = F.zeros((2, 9, 64))
    with SHARED:                                  # heads 0..3 and 3..6
        call(F.narrow(rows, 1, 3, 4), F.narrow(rows, 1, 0, 4))
    for small, n in ((table, 4), (lens, 2), (starts, 3)):
        big = F.zeros((600,), "int32")
        F.copy_(F.narrow(big, 0, 20, n), F.view(small, (n,)))
        part = view(big, small.shape, small.strides, 20, "int32")
        args = [part if t is small else t for t in (table, lens, starts)]
        with SHARED:
            F.paged_attention(q, kp, vp, *args, out=view(big, (2, 4, 64), (256, 64, 1), 0))


def test_heads_of_one_buffer_are_taken(hip):
    wide, wh = seeded(1, (2, 9, 64))
    kp, kh = seeded(2, (5, 2, 16, 64))
    table, lens = np.array([[0, 1], [2, 3]]), np.array([20, 30])
    F.paged_attention(F.narrow(wide, 1, 0, 4), kp, kp, i32(table), i32(lens), out=F.narrow(wide, 1, 4, 4))
    o, a, smax = op.paged_attention(wh[:, :4], kh, kh, table, lens)
    got = wide.numpy()
    assert (np.abs(got[:, 4:8] - o) <= op.attention_bound("float32", o, a, smax, 64, 30)).all()
    for part in (slice(0, 4), slice(8, 9)):
        np.testing.assert_array_equal(got[:, part], wh[:, part])


def test_write_refuses_pages_among_its_inputs(hip):
    k, kp, vp = F.zeros((2, 2, 64)), F.zeros((5, 2, 16, 64)), F.zeros((5, 2, 16, 64))
    table, lens = i32([[0, 1], [2, 3]]), i32([20, 30])
    for pool in (kp, vp):
        inside = view(pool, (2, 2, 64), (128, 64, 1), 4096)
        for pair in ((inside, k), (k, inside)):
            with SHARED:
                F.paged_kv_write(*pair, kp, vp, table, lens)
    with SHARED:                                  # two tensors into one pool
        F.paged_kv_write(k, F.zeros((2, 2, 64)), kp, kp, table, lens)
    both = F.zeros((9, 2, 16, 64))
    with SHARED:
        F.paged_kv_write(k, k, F.narrow(both, 0, 0, 5), F.narrow(both, 0, 4, 5), table, lens)
    with SHARED:
        F.paged_kv_write(k, k, kp, vp, table, lens, None, view(kp, (3,), (1,), 7, "int32"))


def test_pools_of_one_buffer_are_taken(hip):
    """Keys and values in turn per page, per head and per row, and one pool that is both."""
    (k, kh), (v, vh) = seeded(3, (2, 2, 64)), seeded(4, (2, 2, 64))
    table, lens = np.array([[0, 1], [2, 3]]), np.array([20, 30])
    for strides, apart in (((4096, 1024, 64, 1), 2048), ((4096, 2048, 64, 1), 1024), ((4096, 64, 256, 1), 128), ((4096, 128, 256, 1), 64)):
        pool = F.zeros((5, 4096))
        kp, vp = (view(pool, (5, 2, 16, 64), strides, at) for at in (0, apart))
        F.paged_kv_write(k, v, kp, vp, i32(table), i32(lens))
        want = op.paged_kv_write(kh, vh, np.zeros((5, 2, 16, 64)), np.zeros((5, 2, 16, 64)), table, lens)
        np.testing.assert_array_equal(kp.numpy(), want[0])
        np.testing.assert_array_equal(vp.numpy(), want[1])
    one = F.zeros((5, 2, 16, 64))
    F.paged_kv_write(k, k, one, one, i32(table), i32(lens))
    np.testing.assert_array_equal(one.numpy(), op.paged_kv_write(kh, kh, np.zeros((5, 2, 16, 64)), np.zeros((5, 2, 16, 64)), table, lens)[0])


def test_selection_refuses_results_among_the_logits(hip):
    x, s = F.zeros((2, 3, 10)), F.zeros((2, 3))
    new = lambda dtype="int32": F.zeros((2, 3), dtype)  # noqa: E731
    for i, dtype in enumerate(("float32", "int32", "int32")):
        out = [new("float32"), new(), new(), None]
        out[i] = view(x, (2, 3), (3, 1), 54, dtype)
        with SHARED:
            F.beam_select(x, s, 3, out=tuple(out))
    wide = dev(np.random.default_rng(5).normal(size=(2, 3, 16)).astype(np.float32))
    got = F.beam_select(F.narrow(wide, 2, 0, 10), s, 3)
    np.testing.assert_array_equal(got[1].numpy(), op.beam_select(wide.numpy()[:, :, :10], np.zeros((2, 3)), 3)[1])


def test_copy_refuses_moves_among_the_pages(hip):
    pages = F.zeros((4, 1, 16, 64))
    with SHARED:
        F.pages_copy(pages, view(pages, (2, 2), (2, 1), 4092, "int32"), i32([0]))
    with SHARED:
        F.pages_copy(pages, i32([[0, 1]]), view(pages, (1,), (1,), 5, "int32"))
