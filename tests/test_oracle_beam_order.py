"""The beam selection's plain form where different logits make one score."""
import numpy as np
import pytest

from oracle import paged as op


@pytest.mark.parametrize("k", [1, 2])
def test_the_larger_logit_of_a_tied_score_comes_first(k):
    x = np.array([[[0.0, 1e-20, -50.0]]])
    assert op.beam_select(x, np.zeros((1, 1)), k)[1][0].tolist() == [1, 0][:k]


def test_ties_go_to_the_lower_beam_then_the_larger_logit_then_the_lower_token():
    x = np.array([[[1.0, 3.0, 3.0, 2.0], [9.0, 1.0, 0.0, 0.0]]])
    for score in (-1e20, -1e30, 1e25):
        sc, tok, par, _ = op.beam_select(x, np.full((1, 2), score), 6)
        assert par[0].tolist() == [0, 0, 0, 0, 1, 1] and tok[0].tolist() == [1, 2, 3, 0, 0, 1] and (sc == score).all()
    sc, tok, par, _ = op.beam_select(x, np.array([[-np.inf, -1e20]]), 6)      # at -inf the logits count as equal
    assert par[0].tolist() == [1, 1, 1, 1, 0, 0] and tok[0].tolist() == [0, 1, 2, 3, 0, 1]
