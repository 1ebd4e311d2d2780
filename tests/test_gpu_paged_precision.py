"""How exact bfloat16 paged attention is, beyond the elementwise bound of the other tests (which one key left out of a
thousand would pass).

Few rows (up to 256 packed rows of a sequence): P is held in two bfloat16 parts, 2^-16 of it; the result is rounded once:
  |got - o| <= e + 2^-8 (|o| + e),  e = the float32 form's bound + 2^-16 sum p |v|.
Many rows: P is rounded once, as in the contiguous prefill.  A rounding to 8 bits is off by at most 2^-8 of the value,
uniformly, so by 2^-8 / sqrt(3) in the quadratic mean; those of P are independent and reach the normaliser, too:
  |got - o|_2 <= 2^-8 / sqrt(3) sqrt(sum o^2 (1 + sum p^2) + sum p^2 v^2) + |e|_2."""
import numpy as np
import pytest

from helpers import dev, seeded
from kandle_amd import functional as F
from oracle import paged as op
from test_gpu_paged_attention import Cache, i32

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


def run(c, seed, news, hq, **kw):
    st = np.concatenate([[0], np.cumsum(news)])
    q, qh = seeded(seed, (int(st[-1]), hq, c.kh.shape[3]), "bfloat16")
    got = F.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lens), i32(st), **kw).numpy().astype(np.float64)
    ref, a, smax = op.paged_attention(qh, c.kh, c.vh, c.table, c.lens, st)
    e = op.attention_bound("float32", ref, a, smax, qh.shape[2], int(c.lens.max()))
    return qh, st, got, ref, a, e


def tight(got, ref, a, e):
    e = e + 2.0 ** -16 * a
    return np.abs(got - ref) <= e + U * (np.abs(ref) + e)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,news,lens", [(4, [1, 1, 1, 1], [1, 40, 777, 2300]), (16, [1, 1], [3000, 64]), (4, [7, 1, 30], [500, 90, 31]),
                                          (8, [60, 1], [1500, 400])])
def test_few_rows_round_the_result_alone(hip, d, hq, news, lens):
    c = Cache(1, "bfloat16", lens, 2, d, 16)
    _, _, got, ref, a, e = run(c, 3, news, hq)
    assert tight(got, ref, a, e).all()


def test_single_tokens_beside_a_prompts_chunk_are_as_exact(hip):
    c = Cache(5, "bfloat16", [1500, 900, 31, 700], 2, 128, 16)
    _, st, got, ref, a, e = run(c, 7, [300, 1, 1, 20], 4)
    few = slice(st[1], None)
    assert tight(got, ref, a, e)[few].all()


@pytest.mark.parametrize("d,hq,hkv,news,lens", [(128, 4, 2, [150], [1200]), (64, 8, 2, [100, 300], [1000, 700]), (128, 2, 2, [400], [6500]),
                                                (128, 16, 8, [300, 1, 33], [900, 800, 70])])
def test_errors_of_many_rows_are_those_of_two_roundings(hip, d, hq, hkv, news, lens):
    c = Cache(9, "bfloat16", lens, hkv, d, 16)
    qh, st, got, ref, a, e = run(c, 11, news, hq)
    pv, pp = op.attention_spread(qh, c.kh, c.vh, c.table, c.lens, st)
    off, most = np.linalg.norm(got - ref), U / np.sqrt(3) * np.sqrt((ref ** 2 * (1 + pp[..., None])).sum() + pv.sum())
    assert off <= most + np.linalg.norm(e), (off, most)
    one = np.sqrt((pv.sum(-1) / len(ref)).sum())        # about what leaving one key out of each row would do
    assert one > 2 * most


@pytest.mark.parametrize("news,hq", [([1, 1], 4), ([30, 2], 4), ([1, 1], 34), ([300, 1], 4)])
def test_infinities_that_a_row_sees(hip, news, hq):
    """In the middle of the cache, where every row of a tile sees them: infinite columns, NaN where both signs meet, and all
    other columns as without them."""
    c = Cache(13, "bfloat16", [700, 500], 2, 128, 16)
    v = np.array(c.vh)
    for b, p, col, x in ((0, 33, 5, np.inf), (0, 200, 70, -np.inf), (0, 40, 9, np.inf), (0, 90, 9, -np.inf), (1, 100, 127, -np.inf),
                         (1, 17, 64, np.nan)):
        v[c.table[b, p // 16], :, p % 16, col] = x
    st = np.concatenate([[0], np.cumsum(news)])
    q, qh = seeded(15, (int(st[-1]), hq, 128), "bfloat16")
    got = F.paged_attention(q, c.k, dev(v, "bfloat16"), i32(c.table), i32(c.lens), i32(st)).numpy()
    ref, a, smax = op.paged_attention(qh, c.kh, c.vh, c.table, c.lens, st)
    bound = op.attention_bound("bfloat16", ref, a, smax, 128, 700)
    first, second = got[:st[1]], got[st[1]:]
    assert (first[..., 5] == np.inf).all() and (first[..., 70] == -np.inf).all() and np.isnan(first[..., 9]).all()
    assert (second[..., 127] == -np.inf).all() and np.isnan(second[..., 64]).all()
    for part, rest, cols in ((first, slice(0, st[1]), [5, 70, 9]), (second, slice(st[1], None), [127, 64])):
        kept = np.setdiff1d(np.arange(128), cols)
        assert (np.abs(part - ref[rest])[..., kept] <= bound[rest][..., kept]).all()
