"""paged_kv_write beside a reserve's info: the plain form, and the refusal of an info that is none."""
import numpy as np
import pytest

from kandle_amd import kernels
from oracle import paged as op
from test_oracle_paged import Fake


def test_a_reserve_that_lacked_pages_writes_nothing():
    k, pool = np.ones((1, 2, 4)), np.zeros((3, 2, 16, 4))
    for info, written in ((None, 1), ([0, 0, 0], 1), ([3, 0, 0], 1), ([0, 1, 0], 0), ([0, 0, 2], 0)):
        kp, vp = op.paged_kv_write(k, k, pool, pool, np.array([[2]]), [5], None, info)
        assert kp.sum() == vp.sum() == 8 * written and kp[2, :, 4].sum() == 8 * written


@pytest.mark.parametrize("info", [Fake((2,)), Fake((3,), "float32"), Fake((3, 1))])
def test_an_info_that_is_none_is_refused(info):
    rows, pages = Fake((3, 2, 64), "float32"), Fake((5, 2, 16, 64), "float32")
    good = (rows, rows, pages, pages, Fake((2, 3)), Fake((2,)), Fake((3,)))
    with pytest.raises(ValueError, match="info"):
        kernels.paged_kv_write(*good, info)
    with pytest.raises(AssertionError, match="not refused"):
        kernels.paged_kv_write(*good, Fake((3,)))
