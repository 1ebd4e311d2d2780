"""Whether two operands may share memory (csrc/spans.h), compiled for the host: never `apart` where a byte is common, and
apart for the layouts that programs use."""
import ctypes as C
import itertools
import os
import shutil
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kandle_amd", "csrc")
SOURCE = r"""
#include "spans.h"
extern "C" int apart(const int64_t* a, const int64_t* b) {
  auto span = [](const int64_t* x) {
    return kh::Span((const void*)x[0], x[1], x[2], x[5], x[3], x[6], x[4], x[7]);
  };
  return kh::apart(span(a), span(b));
}
"""


@pytest.fixture(scope="module")
def apart(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("spans")
    (d / "spans.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", str(d / "spans.so"), str(d / "spans.cpp")], check=True)
    lib = C.CDLL(str(d / "spans.so"))

    def call(a, b):
        return bool(lib.apart(*((C.c_int64 * 8)(*x) for x in (a, b))))
    return call


def taken(x):
    at, run, c, s = x[0], x[1], x[2:5], x[5:8]
    return {at + sum(i * t for i, t in zip(idx, s)) + r for idx in itertools.product(*(range(n) for n in c)) for r in range(run)}


def test_never_apart_where_a_byte_is_common(apart):
    r = np.random.default_rng(0)
    told = 0
    for _ in range(6000):
        a, b = ([int(1000 + r.integers(0, 60)), int(r.integers(0, 9)), *r.integers(0, 4, 3).tolist(),
                 *r.choice([-24, -8, 0, 1, 4, 6, 8, 12, 16, 24, 48], 3).tolist()] for _ in range(2))
        common = bool(taken(a) & taken(b))
        if apart(a, b):
            told += 1
            assert not common, (a, b)
        else:
            assert taken(a) and taken(b)      # (an empty operand shares nothing)
        assert apart(a, b) == apart(b, a)
    assert told > 1000


def test_apart_in_the_layouts_that_programs_use(apart):
    run = lambda at, n: [at, n, 1, 1, 1, 0, 0, 0]  # noqa: E731
    assert apart(run(1000, 8), run(1008, 8)) and not apart(run(1000, 8), run(1007, 8)) and apart(run(0, 8), run(0, 8))
    # heads of one [tokens, heads, d] buffer, d of 8 bytes: 0..3 and 4..5 of 6
    q, o, both = [1000, 8, 5, 4, 1, 48, 8, 0], [1032, 8, 5, 2, 1, 48, 8, 0], [1024, 8, 5, 3, 1, 48, 8, 0]
    assert apart(q, o) and not apart(q, both)
    # keys and values side by side: per page, per head inside the page's rows, and per row
    page, heads, rows, d = 4, 3, 5, 8
    size = 2 * heads * rows * d
    for k, v, inner in ((0, heads * rows * d, (rows * d, d)), (0, rows * d, (2 * rows * d, d)), (0, heads * d, (d, 2 * heads * d)),
                        (0, d, (2 * d, 2 * heads * d))):
        kp, vp = ([1000 + at, d, page, heads, rows, size, *inner] for at in (k, v))
        assert apart(kp, vp) and not apart(kp, kp)
        assert not taken(kp) & taken(vp)
    # layers one after the other, and steps near the limits of 64 bits
    assert apart([1000, 8, 1 << 40, 2, 1, 16, 8, 0], [1000 + (16 << 40), 8, 1, 1, 1, 0, 0, 0])
    assert not apart([1000, 8, 3, 1, 1, 1 << 62, 0, 0], [1000, 8, 3, 1, 1, 1 << 62, 0, 0])
