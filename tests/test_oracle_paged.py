"""The plain forms of the paged cache and beam search (oracle/paged.py) against closed forms and invariants, and
the refusals of the kernels' host side, which need no GPU."""
from types import SimpleNamespace as NS

import numpy as np
import pytest

from kandle_amd import kernels
from kandle_amd.tensor import contiguous_strides
from oracle import paged as op


def test_attention_of_equal_scores_is_the_mean_of_the_visible_rows():
    r = np.random.default_rng(0)
    kp, vp = np.zeros((4, 2, 16, 64)), r.normal(size=(4, 2, 16, 64))
    table = np.array([[2, -1, 0]])
    o, a, smax = op.paged_attention(r.normal(size=(3, 4, 64)), kp, vp, table, [40], [0, 3])
    for j in range(3):
        rows = np.concatenate([vp[2], vp[0][:, :38 + j - 32]], 1)     # positions 37 + j and before; page 1 is a hole
        np.testing.assert_allclose(o[j], np.repeat(rows.mean(1), 2, 0), atol=1e-14)
    assert (smax == 0).all() and (a >= np.abs(o) - 1e-15).all()
    o, _, _ = op.paged_attention(np.ones((2, 2, 64)), kp, vp, np.array([[1]]), [1], [0, 2])
    assert (o[0] == 0).all() and np.allclose(o[1], vp[1, :, 0])       # the first token has no row


def test_bookkeeping_keeps_the_counts_equal_to_the_tables():
    r = np.random.default_rng(1)
    page, rows, width, pages = 16, 9, 6, 60
    table, lens, refs = np.full((rows, width), -1), np.zeros(rows, np.int64), np.zeros(pages, np.int64)
    content = {}
    for step in range(60):
        counts = r.integers(0, 20, size=rows)
        t, n, rf, moves, info = op.pages_reserve(table, lens, refs, counts, page)
        if info[1] or info[2]:
            assert (t == table).all() and (n == lens).all() and info[0] == 0
        else:
            for s in range(rows):
                kept = (np.arange(width) < lens[s] // page) & (table[s] >= 0)
                assert (t[s][kept] == table[s][kept]).all()           # full pages stay where they are
                tail = t[s, lens[s] // page] if n[s] > lens[s] else -1
                assert tail < 0 or rf[tail] == 1                      # what a row writes to is its own
            table, lens, refs = t, n, rf
        np.testing.assert_array_equal(refs, op.count_refs(table, pages))
        parents = np.where(r.random(rows) < 0.2, -1, r.integers(0, rows, size=rows))
        table, lens, refs = op.pages_fork(table, lens, refs, parents)
        np.testing.assert_array_equal(refs, op.count_refs(table, pages))
        if step % 7 == 0:
            table, refs, moves, info = op.pages_compact(table, refs, pages // 2)
            np.testing.assert_array_equal(refs, op.count_refs(table, pages))
            assert (refs[:info[1]] > 0).all() and (refs[info[1]:] == 0).all()


def test_beam_select_is_a_sort_of_every_continuation():
    r = np.random.default_rng(2)
    x, s = r.normal(size=(2, 3, 11)), -r.random((2, 3))
    sc, tok, par, _ = op.beam_select(x, s, 5)
    every = (x - np.log(np.exp(x).sum(-1, keepdims=True)) + s[..., None]).reshape(2, -1)
    best = np.argsort(-every, axis=1)[:, :5]
    np.testing.assert_array_equal(par * 11 + tok, best)
    np.testing.assert_allclose(sc, np.take_along_axis(every, best, 1))
    sc, tok, par, fin = op.beam_select(x, s, 3, np.array([[1, 1, 1], [0, 1, 0]]), 4)
    assert (tok[0] == 4).all() and sorted(par[0]) == [0, 1, 2] and (fin[0] == 1).all()


def test_the_float64_forms_of_the_two_orders_agree():
    r = np.random.default_rng(3)
    x, s = np.round(r.normal(size=(1, 2, 3000)), 1), np.zeros((1, 2))   # many ties
    a = op.beam_select(x, s, 8)
    every = (x - (x.max(-1, keepdims=True) + np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)))).reshape(-1)
    order = sorted(range(6000), key=lambda i: (-every[i], i))[:8]
    np.testing.assert_array_equal(a[2][0] * 3000 + a[1][0], order)


# ---- refusals of the host side -----------------------------------------------------------------
class Fake(NS):
    """What the kernels' checks read of a tensor handle."""

    def __init__(self, shape, dtype="int32", strides=None):
        super().__init__(shape=tuple(shape), dtype=dtype, strides=tuple(strides or contiguous_strides(shape)), itemsize=4, kh_dtype=0)

    def is_contiguous(self):
        return self.strides == tuple(contiguous_strides(self.shape))

    def data_ptr(self):
        raise AssertionError("the call was not refused")


def _attention(**change):
    x = dict(query=Fake((3, 4, 64), "float32"), key_pages=Fake((5, 2, 16, 64), "float32"),
             value_pages=Fake((5, 2, 16, 64), "float32"), page_table=Fake((2, 3)), kv_lens=Fake((2,)),
             query_starts=Fake((3,)), output=Fake((3, 4, 64), "float32"), scale=1.0, is_causal=True)
    kernels.paged_attention(**{**x, **change})


@pytest.mark.parametrize("change,error", [
    ({"query": Fake((3, 4, 64), "bfloat16")}, TypeError),
    ({"output": Fake((3, 4, 64), "int32")}, TypeError),
    ({"query": Fake((4, 64), "float32")}, ValueError),
    ({"query": Fake((3, 4, 128), "float32")}, ValueError),
    ({"query": Fake((3, 4, 64), "float32", (256, 1, 4))}, ValueError),
    ({"output": Fake((2, 4, 64), "float32")}, ValueError),
    ({"value_pages": Fake((5, 2, 16, 128), "float32")}, ValueError),
    ({"key_pages": Fake((5, 3, 16, 64), "float32"), "value_pages": Fake((5, 3, 16, 64), "float32")}, ValueError),
    ({"key_pages": Fake((5, 0, 16, 64), "float32"), "value_pages": Fake((5, 0, 16, 64), "float32")}, ValueError),
    ({"page_table": Fake((2, 3), "float32")}, ValueError),
    ({"page_table": Fake((2, 3), "int32", (1, 2))}, ValueError),
    ({"page_table": Fake((2, 3), "int32", (2, 1))}, ValueError),
    ({"kv_lens": Fake((3,))}, ValueError),
    ({"kv_lens": Fake((2,), "float32")}, ValueError),
    ({"query_starts": Fake((2,))}, ValueError),
    ({"query_starts": None}, ValueError),
    ({"scale": float("nan")}, ValueError)])
def test_paged_attention_refuses(change, error):
    with pytest.raises(error):
        _attention(**change)
    with pytest.raises(AssertionError, match="not refused"):
        _attention()


def test_paged_write_and_bookkeeping_refuse():
    rows, pages = Fake((3, 2, 64), "float32"), Fake((5, 2, 16, 64), "float32")
    table, lens, starts = Fake((2, 3)), Fake((2,)), Fake((3,))
    for bad in ((Fake((3, 2, 64), "bfloat16"), rows, pages, pages, table, lens, starts),
                (rows, Fake((2, 2, 64), "float32"), pages, pages, table, lens, starts),
                (rows, rows, Fake((5, 2, 16, 32), "float32"), pages, table, lens, starts),
                (rows, rows, pages, pages, table, lens, None),
                (rows, rows, pages, pages, table, Fake((3,)), starts)):
        with pytest.raises((TypeError, ValueError)):
            kernels.paged_kv_write(*bad)
    refs, parents = Fake((7,)), Fake((2,))
    for bad in ((table, lens, Fake((7, 1)), parents, table, lens, refs), (table, lens, refs, Fake((3,)), table, lens, refs),
                (table, lens, refs, parents, Fake((2, 4)), lens, refs), (table, lens, refs, parents, table, lens, Fake((6,)))):
        with pytest.raises(ValueError):
            kernels.pages_fork(*bad)
    moves, info = Fake((2, 2)), Fake((3,))
    for bad in ((table, lens, refs, Fake((1,)), 16, moves, info), (table, lens, refs, parents, 16, Fake((3, 2)), info),
                (table, lens, refs, parents, 16, moves, Fake((2,)))):
        with pytest.raises(ValueError):
            kernels.pages_reserve(*bad)
    for bad in ((table, refs, table, refs, Fake((2, 2)), Fake((2,))), (table, refs, table, refs, Fake((3, 3)), Fake((2,))),
                (table, refs, table, refs, Fake((3, 2)), Fake((3,)))):
        with pytest.raises(ValueError):
            kernels.pages_compact(*bad)
    for bad in ((Fake((5, 2, 16), "float32"), moves, info), (Fake((5, 2, 16, 4), "float32", (128, 64, 1, 16)), moves, info),
                (pages, Fake((4,)), info), (pages, moves, Fake((0,))), (pages, moves, Fake((1,), "float32"))):
        with pytest.raises(ValueError):
            kernels.pages_copy(*bad)


def test_beam_select_refuses():
    x, s, f = Fake((2, 3, 50), "float32"), Fake((2, 3), "float32"), Fake((2, 3))
    good = (x, s, None, 3, None, s, f, f, None)
    with pytest.raises(AssertionError, match="not refused"):
        kernels.beam_select(*good)
    for i, bad in ((0, Fake((2, 3, 50))), (0, Fake((6, 50), "float32")), (0, Fake((2, 3, 50), "float32", (150, 1, 3))),
                   (1, Fake((2, 4), "float32")), (1, f), (2, f), (8, f), (3, 4), (5, f), (6, s), (7, Fake((2, 2)))):
        with pytest.raises((TypeError, ValueError)):
            kernels.beam_select(*good[:i], bad, *good[i + 1:])
    with pytest.raises(ValueError, match="eos_token_id"):
        kernels.beam_select(x, s, f, 3, None, s, f, f, f)


def test_caches_past_the_kernels_limits_are_refused():
    from kandle_amd.model_utils import PagedKVCache
    for sequences, rows in ((2049, 64), (2, (1 << 30) + 1)):
        with pytest.raises(ValueError, match="at most 2048 of 2\\^30"):
            PagedKVCache(2, 2, 64, 4, sequences, rows)
