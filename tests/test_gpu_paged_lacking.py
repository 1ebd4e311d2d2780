"""A step whose reserve lacks pages, without a look at it in between: what is cached stays as it was, bit for bit, also in
pages that sequences share."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from helpers import seeded
from kandle_amd import Tensor
from kandle_amd import functional as F
from kandle_amd import synthetic as syn
from kandle_amd.graphs import HipGraph
from kandle_amd.model_utils import PagedKVCache, Qwen3Config, Qwen3ForCausalLM, init_qwen3_weights
from oracle import paged as op
from test_gpu_node_backend import ADDON, PKG, _ensure_dist

pytestmark = pytest.mark.gpu


def i32(x):
    return Tensor(np.ascontiguousarray(x, np.int32), dtype="int32")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d", [64, 5])
@pytest.mark.parametrize("info", [[0, 0, 0], [2, 0, 0], [0, 1, 0], [0, 0, 1], [0, 3, 2]])
def test_write_goes_by_the_reserves_info(hip, dtype, d, info):
    (k, kh), (v, vh) = seeded(1, (3, 2, d), dtype), seeded(2, (3, 2, d), dtype)
    (kp, kph), (vp, vph) = seeded(3, (6, 2, 16, d), dtype), seeded(4, (6, 2, 16, d), dtype)
    table, lens, starts = np.array([[4, 1], [2, -1]]), np.array([20, 7]), np.array([0, 2, 3])
    F.paged_kv_write(k, v, kp, vp, i32(table), i32(lens), i32(starts), i32(info))
    want = op.paged_kv_write(kh, vh, kph, vph, table, lens, starts, info)
    np.testing.assert_array_equal(kp.numpy(), want[0])
    np.testing.assert_array_equal(vp.numpy(), want[1])


def full_cache(spare):
    """Two sequences that share a page and a partly filled one, in a pool with `spare` free pages."""
    cache = PagedKVCache(1, 2, 64, 2 + spare, 3, 96, 16, "float32")
    cache.reserve([24, 0, 0])
    rows, _ = seeded(5, (24, 2, 64))
    F.paged_kv_write(rows, rows, *cache.layer(0), cache.page_table, cache.kv_lens, i32([0, 24, 24, 24]), cache.reserve_info)
    cache.fork([0, 0, -1])
    return cache


def state_of(cache):
    return [t.numpy().copy() for t in (cache.pages, *cache.state)]


@pytest.mark.parametrize("counts", [[1, 0, 0], [1, 1, 0], [9, 30, 0], [0, 1, 16]])
def test_an_unchecked_reserve_that_lacks_pages_loses_no_row(hip, counts):
    cache = full_cache(0)
    before = state_of(cache)
    cache.reserve(counts, check=False)
    n = np.concatenate([[0], np.cumsum(counts)])
    new, _ = seeded(7, (int(n[-1]), 2, 64))
    F.paged_kv_write(new, new, *cache.layer(0), cache.page_table, cache.kv_lens, i32(n), cache.reserve_info)
    for a, b in zip(before, state_of(cache)):
        np.testing.assert_array_equal(a, b)
    with pytest.raises(RuntimeError, match="pages are missing"):
        cache.check_info()
    cache.dispose()


def test_a_captured_step_that_lacks_pages_loses_no_row(hip):
    """Three replays with two free pages: the first takes both (a copied tail each, but for the last sharer), and so on
    until the pool is full; from then on nothing changes."""
    cache = full_cache(2)
    ones, (q, _), (new, _) = i32([1, 1, 0]), seeded(9, (2, 4, 64)), seeded(11, (2, 2, 64))
    starts = i32([0, 1, 2, 2])
    g = HipGraph()
    with g.capture():
        cache.enqueue_reserve(ones)
        F.paged_kv_write(new, new, *cache.layer(0), cache.page_table, cache.kv_lens, starts, cache.reserve_info)
        o = F.paged_attention(q, *cache.layer(0), cache.page_table, cache.kv_lens, starts)
    failed = 0
    for step in range(14):
        before = state_of(cache)
        g.replay()
        after = state_of(cache)
        if cache.reserve_info.numpy()[1]:
            failed += 1
            for a, b in zip(before, after):
                np.testing.assert_array_equal(a, b)
            with pytest.raises(RuntimeError, match="pages are missing"):
                cache.check_info()
        else:
            assert not failed and after[2].tolist() == [25 + step, 25 + step, 0]
    assert failed == 6                        # 24 rows and two pages: eight steps fill both tails, one more page is free
    o.dispose()
    g.dispose()
    cache.dispose()


def test_a_model_step_that_lacks_pages_loses_no_row(hip):
    """The step of a beam search on a pool that is too small, at the level of the model's own decode step."""
    cfg = Qwen3Config(vocab_size=500, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64)
    model = Qwen3ForCausalLM(cfg, init_qwen3_weights(cfg, seed=3, std=0.02), max_seq_len=64, activations="float32")
    cache = model.new_paged_cache(max_sequences=2, num_pages=2)
    prompt = [int(t) for t in syn.randint(40, (20,), 0, cfg.vocab_size)]
    model.forward_paged(prompt, [20, 0], cache).dispose()
    cache.fork([0, 0])
    before = state_of(cache)
    cache.enqueue_reserve(i32([1, 1]))
    model._paged_dev(i32([5, 6]), i32([20, 20]), None, None, cache, 1, 64).dispose()
    for a, b in zip(before, state_of(cache)):
        np.testing.assert_array_equal(a, b)
    cache.dispose()
    model.dispose()


def test_the_hosts_lengths_are_the_devices_after_a_reserve_that_lacked_pages(hip):
    cache = full_cache(1)
    cache.reserve([1, 0, 0], check=False)     # the free page
    cache.check_info()
    assert cache.lens.tolist() == cache.kv_lens.numpy().tolist() == [25, 24, 0]
    cache.reserve([8, 1, 5], check=False)     # two pages that are not there
    with pytest.raises(RuntimeError, match="2 pages are missing"):
        cache.check_info()
    assert cache.lens.tolist() == cache.kv_lens.numpy().tolist() == [25, 24, 0]
    cache.reserve([7, 8, 0])                  # the tails' room
    assert cache.lens.tolist() == cache.kv_lens.numpy().tolist() == [32, 32, 0]
    with pytest.raises(RuntimeError, match="1 pages are missing"):
        cache.reserve([0, 0, 3])
    assert cache.lens.tolist() == [32, 32, 0]
    cache.dispose()


@pytest.mark.parametrize("check", [False, True])
def test_a_reserve_that_lacked_pages_before_the_last_is_found(hip, check):
    """info is the last reserve's; one before it, which nobody looked at, shows in the lengths."""
    cache = full_cache(1)
    cache.reserve([0, 0, 17], check=False)    # two pages of one
    cache.reserve([1, 0, 0], check=False)     # the free one
    with pytest.raises(RuntimeError, match="before the last"):
        cache.reserve([1, 0, 0], check=True) if check else cache.check_info()
    assert cache.lens.tolist() == cache.kv_lens.numpy().tolist() == [25, 24, 0]
    cache.check_info()
    cache.reserve([1, 1, 0], check=False)
    cache.reserve([1, 1, 0], check=False)
    cache.fork([1, 0, 0])
    cache.check_info()
    assert cache.lens.tolist() == cache.kv_lens.numpy().tolist() == [26, 27, 27]
    cache.dispose()


SCRIPT = r"""
const m = require(process.argv[1]), addon = require(process.argv[2]);
m.HipBackend.create(0).then((b) => {
  const i32 = (shape, data) => m.HipTensorHandle.createNew(shape, 'int32', new Int32Array(data));
  const f32 = (shape, x) => m.HipTensorHandle.createNew(shape, 'float32', new Float32Array(shape.reduce((p, n) => p * n, 1)).fill(x));
  const write = b.operators.find('paged_kv_write'), out = [];
  for (const info of [undefined, i32([3], [1, 0, 0]), i32([3], [0, 2, 0]), i32([3], [0, 0, 1])]) {
    const kp = f32([2, 1, 16, 64], 0), rows = f32([1, 1, 64], 7);
    write(rows, rows, kp, f32([2, 1, 16, 64], 0), i32([1, 1], [1]), i32([1], [3]), null, info);
    const host = new ArrayBuffer(4 * kp.numel);
    addon.memcpyD2H(host, kp.ptr);
    out.push(new Float32Array(host).filter((x) => x === 7).length);
  }
  let refused = 0;
  const rows = f32([1, 1, 64], 7), pool = f32([2, 1, 16, 64], 0);
  try { write(rows, rows, pool, f32([2, 1, 16, 64], 0), i32([1, 1], [1]), i32([1], [3]), null, i32([2], [0, 0])); }
  catch (e) { refused = 1; }
  console.log(JSON.stringify({ out, refused }));
}).catch((e) => { console.error(e.stack); process.exit(1); });
"""


def test_write_goes_by_the_info_from_node(hip):
    if shutil.which("node") is None or not os.path.exists(ADDON):
        pytest.skip("node or the built addon is not available")
    _ensure_dist()
    run = subprocess.run(["node", "-e", SCRIPT, os.path.join(PKG, "dist", "index.js"), ADDON], capture_output=True, text=True,
                         timeout=100)
    assert run.returncode == 0, run.stderr
    assert json.loads(run.stdout.strip().splitlines()[-1]) == {"out": [64, 64, 0, 0], "refused": 1}
