"""beam_select against the sort of all continuations in float64 (oracle/paged.py).

Tokens, parents and flags are exact.  Scores: log sum exp from fp32 exponentials of arguments x - max (the rounding
of the argument, |x - max| u, weighs with the term's share; here |x - max| < 64) and fp32 sums of 8192 (42 additions on the way of a term), in all below
80 u absolute, and one rounding of the result: 2^-24 |score|.  u = 2^-24."""
import numpy as np
import pytest

from helpers import dev
from kandle_amd import Tensor
from kandle_amd import functional as F
from kandle_amd import synthetic as syn
from kandle_amd._lib import KandleHipError
from kandle_amd.graphs import HipGraph
from oracle import paged as op

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def logits_of(seed, shape, dtype, std=3.0):
    x = syn.normal(seed, shape, std)
    if dtype == "bfloat16":
        bits, vals = syn.bf16(x)
        return Tensor(bits, dtype="bfloat16"), vals
    return Tensor(x, dtype="float32"), x


def check(x, xh, scores, k=None, finished=None, eos=None):
    f = None if finished is None else Tensor(np.asarray(finished, np.int32), dtype="int32")
    s = np.asarray(scores, np.float32)
    got = F.beam_select(x, dev(s), k, f, eos)
    want = op.beam_select(xh, s, s.shape[1] if k is None else k, finished, eos)
    np.testing.assert_array_equal(got[2].numpy(), want[2])
    np.testing.assert_array_equal(got[1].numpy(), want[1])
    g, w = got[0].numpy().astype(np.float64), want[0]
    fin = np.isfinite(w)
    np.testing.assert_array_equal(np.isfinite(g), fin)
    assert (np.abs(g[fin] - w[fin]) <= 80 * U + U * np.abs(w[fin])).all()
    if finished is None:
        assert got[3] is None
    else:
        np.testing.assert_array_equal(got[3].numpy(), want[3])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("groups,beams,vocab,k", [
    (1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 2, 6), (1, 4, 1000, 4), (3, 5, 1023, 10), (2, 2, 1025, 64), (1, 8, 4096, 16), (2, 4, 5000, 4),
    (1, 4, 151936, 4), (2, 8, 151936, 8), (1, 64, 3001, 64), (1, 3, 33333, 7), (70, 2, 777, 2)])
def test_best_continuations(hip, dtype, groups, beams, vocab, k):
    x, xh = logits_of(groups + vocab, (groups, beams, vocab), dtype)
    check(x, xh, -20 * np.random.default_rng(vocab).random((groups, beams)), k)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [33, 100, 2060, 8200])
@pytest.mark.parametrize("k", [63, 64])
def test_as_many_as_lanes(hip, dtype, vocab, k):
    """k at and below the 64 lanes of a wave, the last wave's being mostly behind the row's end."""
    x, xh = logits_of(vocab + k, (1, 2, vocab), dtype)
    check(x, xh, np.array([[-1.5, -1.0]]), k)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_finished_beams_go_on_as_themselves(hip, dtype):
    x, xh = logits_of(3, (4, 5, 2000), dtype)
    s = -5 * np.random.default_rng(4).random((4, 5))
    fin = np.array([[0, 1, 0, 0, 1], [1, 1, 1, 1, 1], [0, 0, 0, 0, 0], [0, 0, 0, 0, 7]])
    s[3, 4] = -np.inf
    for eos in (0, 7, 1999):
        check(x, xh, s, None, fin, eos)
        check(x, xh, s, 2, fin, eos)
    xh = np.array(xh)
    xh[0, 0, 7] = 40.0                                        # a beam that ends now
    check(dev(xh, dtype), xh, s, None, fin, 7)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [40, 1500, 9000])
def test_ties_go_to_the_lower_beam_and_token(hip, dtype, vocab):
    r = np.random.default_rng(vocab)
    same = np.repeat(np.round(r.normal(size=(1, 1, vocab))).astype(np.float32), 4, 1)     # four equal beams of few values
    check(dev(same, dtype), same, np.zeros((1, 4)), 9)
    flat = np.zeros((2, 3, vocab), np.float32)
    flat[:, :, 1::2] = -0.0
    check(dev(flat, dtype), flat, np.array([[0, 0, 0], [0, -1, 0]]), 20)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_masked_and_broken_logits(hip, dtype):
    inf, nan = np.inf, np.nan
    _, xh = logits_of(5, (6, 2, 3000), dtype)
    x = np.array(xh)
    x[0, 0, 2:] = -inf                                        # two tokens allowed
    x[0, 1, :] = -inf                                         # none
    x[1, :, ::2] = nan                                        # as -inf
    x[2, 0, 77] = inf                                         # no finite sum: every continuation -inf
    x[3] = -inf
    x[4, 0, :] = nan
    x[5, 1, :] = np.finfo(np.float32).min if dtype == "float32" else -3.3895313892515355e38
    s = np.array([[-1, -2], [0, -1], [-1, -30], [0, 0], [-inf, -inf], [-3, nan]], np.float64)
    check(dev(x, dtype), x, s, 5)
    check(dev(x, dtype), x, np.full((6, 2), -inf), 7)
    first = np.full((6, 2), -inf)
    first[:, 0] = 0                                           # the first step: beams but one are not there yet
    check(dev(xh, dtype), xh, first, 4)


def test_large_and_small_values(hip):
    x = np.full((1, 2, 2500), 1e30, np.float32)
    x[0, 0, 5], x[0, 0, 9], x[0, 1, 3] = 2e30, 2e30, 3e38
    check(dev(x), x, np.zeros((1, 2)), 3)
    y = np.full((1, 1, 1300), -200.0, np.float32)
    y[0, 0, 1200] = 100.0
    check(dev(y), y, np.zeros((1, 1)), 3)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab,off", [(4097, 1), (2000, 3), (1030, 0), (151, 5)])
def test_strided_and_unaligned_rows(hip, dtype, vocab, off):
    wide, wh = logits_of(7, (2, 3, vocab + 9), dtype)
    x = F.narrow(wide, 2, off, vocab)
    check(x, wh[:, :, off:off + vocab], -np.random.default_rng(8).random((2, 3)))
    swapped = F.permute(x, (1, 0, 2))
    check(swapped, wh[:, :, off:off + vocab].transpose(1, 0, 2), -np.random.default_rng(9).random((3, 2)))


def test_graph_replays(hip):
    x, xh = logits_of(11, (3, 4, 20000), "float32")
    s = Tensor(np.zeros((3, 4), np.float32))
    f = Tensor(np.zeros((3, 4), np.int32), dtype="int32")
    g = HipGraph()
    with g.capture():
        out = F.beam_select(x, s, None, f, 7)
    r = np.random.default_rng(12)
    for _ in range(4):
        sh, fh = (-9 * r.random((3, 4))).astype(np.float32), (r.random((3, 4)) < 0.3).astype(np.int32)
        s.handle.storage.upload(sh)
        f.handle.storage.upload(fh)
        g.replay()
        want = op.beam_select(xh, sh, 4, fh, 7)
        np.testing.assert_array_equal(out[1].numpy(), want[1])
        np.testing.assert_array_equal(out[2].numpy(), want[2])
        eager = F.beam_select(x, s, None, f, 7)
        for a, b in zip(out, eager):
            np.testing.assert_array_equal(a.numpy(), b.numpy())
    g.dispose()


def test_refusals(hip):
    x, s = F.zeros((1, 2, 10)), F.zeros((1, 2))
    f = F.zeros((1, 2), "int32")
    for k in (0, 21, 65):
        with pytest.raises(KandleHipError, match="kh_beam_select"):
            F.beam_select(x, s, k)
    with pytest.raises(KandleHipError, match="may have finished"):
        F.beam_select(x, s, 3, f, 1)
    for eos in (-1, 10):
        with pytest.raises(KandleHipError, match="end token"):
            F.beam_select(x, s, 2, f, eos)
    with pytest.raises(KandleHipError, match="beams"):
        F.beam_select(F.zeros((1, 65, 10)), F.zeros((1, 65)), 2)


def test_results_in_place_of_inputs_are_refused(hip):
    x, s, f = F.zeros((1, 2, 10)), F.zeros((1, 2)), F.zeros((1, 2), "int32")
    new = lambda: F.zeros((1, 2), "int32")  # noqa: E731
    with pytest.raises(KandleHipError, match="share memory"):
        F.beam_select(x, s, 2, out=(s, new(), new(), None))
    with pytest.raises(KandleHipError, match="share memory"):
        F.beam_select(x, s, 2, f, 1, out=(F.zeros((1, 2)), new(), new(), f))
    same = new()
    with pytest.raises(KandleHipError, match="share memory"):
        F.beam_select(x, s, 2, out=(F.zeros((1, 2)), same, same, None))
