"""The order of beam_select where scores in float64 tie although logits differ: the lower beam, then the larger logit,
then the lower token (oracle/paged.py).  Tokens and parents are exact: logits are small multiples of powers of two or far
below half a step of the score, so no rounding of the kernel's sums decides."""
import numpy as np
import pytest

from helpers import dev
from kandle_amd import functional as F
from kandle_amd import synthetic as syn
from oracle import paged as op

pytestmark = pytest.mark.gpu
LOWEST = float(np.finfo(np.float32).min)


def check(x, xh, scores, k, finished=None, eos=None):
    s = np.asarray(scores, np.float32)
    finished = None if finished is None else np.asarray(finished, np.int32)
    f = None if finished is None else dev(finished, "int32")
    got = F.beam_select(x, dev(s), k, f, eos)
    want = op.beam_select(xh, s, k, finished, eos)
    np.testing.assert_array_equal(got[2].numpy(), want[2])
    np.testing.assert_array_equal(got[1].numpy(), want[1])
    w = want[0].astype(np.float32)      # (the scores are the beams' own, or -inf where that passes fp32)
    np.testing.assert_array_equal(np.isfinite(got[0].numpy()), np.isfinite(w))
    fin = np.isfinite(w)
    np.testing.assert_allclose(got[0].numpy()[fin], w[fin], rtol=2.0 ** -22, atol=80 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("score", [-1e20, -1e30, LOWEST, 1e25])
@pytest.mark.parametrize("vocab,off", [(50, 0), (8193, 0), (30000, 0), (30000, 3), (30000, 1)])
@pytest.mark.parametrize("k", [1, 2, 7, 64])
def test_scores_that_swallow_the_logits(hip, dtype, score, vocab, off, k):
    """Beams whose score so far is so large that every continuation has it: the largest logits of the lowest beam, from
    whatever run of the row, wherever the row starts."""
    xh = syn.normal(vocab + k, (2, 3, vocab + 4), 3.0)
    if dtype == "bfloat16":
        _, xh = syn.bf16(xh)
    x = F.narrow(dev(xh, dtype), 2, off, vocab)
    xh = xh[:, :, off:off + vocab]
    check(x, xh, np.full((2, 3), score), min(k, 3 * vocab))
    mixed = np.array([[score, -1.0, score], [-2.0, score, -1.5]])      # beside beams of ordinary scores
    if score < 0:
        check(x, xh, mixed, min(k, 3 * vocab))
    if k <= 3:
        check(x, xh, np.full((2, 3), score), k, [[0, 1, 0], [0, 0, 1]], 7)


@pytest.mark.parametrize("first,second", [(0, 1), (3, 700), (700, 3), (5, 9000), (9000, 5)])
@pytest.mark.parametrize("k", [1, 2, 3])
def test_logits_closer_than_half_a_step_of_the_score(hip, first, second, k):
    """Two logits that differ by 1e-20, in one run and in two: the larger one is chosen first, for every k."""
    x = np.full((1, 1, 10000), -30.0, np.float32)
    x[0, 0, first], x[0, 0, second] = 0.0, 1e-20
    check(dev(x), x, np.zeros((1, 1)), k)
    assert F.beam_select(dev(x), dev(np.zeros((1, 1), np.float32)), k)[1].numpy()[0, 0] == second


def test_many_equal_scores_of_few_logits(hip):
    """More candidates at one score than are ranked by counting."""
    r = np.random.default_rng(1)
    x = np.round(r.normal(size=(2, 2, 20000)) * 2).astype(np.float32)
    for k in (5, 64):
        check(dev(x), x, np.full((2, 2), -1e22), k)
