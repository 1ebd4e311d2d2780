"""The paged cache's and the beam selection's kernels from Node, through the TypeScript HipBackend's registry: the
same results as the Python binding's, bit for bit."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from kandle_amd import Tensor
from kandle_amd import functional as F
from kandle_amd import synthetic as syn
from test_gpu_node_backend import ADDON, PKG, _ensure_dist

pytestmark = pytest.mark.gpu

SCRIPT = r"""
const fs = require('fs');
const m = require(process.argv[1]);
const dir = process.argv[2];
m.HipBackend.create(0).then((b) => {
  const reg = b.operators;
  const read = (name, shape, dtype) => {
    const buf = fs.readFileSync(dir + '/' + name);
    const ab = buf.buffer.slice(buf.byteOffset, buf.byteOffset + buf.length);
    return m.HipTensorHandle.createNew(shape, dtype, dtype === 'float32' ? new Float32Array(ab) : new Int32Array(ab));
  };
  const i32 = (shape) => m.HipTensorHandle.createNew(shape, 'int32');
  const f32 = (shape) => m.HipTensorHandle.createNew(shape, 'float32');
  const q = read('q', [3, 4, 64], 'float32'), k = read('k', [3, 2, 64], 'float32');
  const pool = read('pool', [2, 9, 2, 16, 64], 'float32');
  const half = (offset) => b.createTensorHandle({ storage: pool.storage, shape: [9, 2, 16, 64], dtype: 'float32', offset });
  const kp = half(0), vp = half(9 * 2048);
  const table = read('table', [3, 3], 'int32'), lens = read('lens', [3], 'int32'), refs = read('refs', [9], 'int32');
  const parents = read('parents', [3], 'int32'), counts = read('counts', [3], 'int32');
  const out = {};
  const t2 = i32([3, 3]), l2 = i32([3]), r2 = i32([9]), mv = i32([3, 2]), info = i32([3]);
  reg.find('pages_fork')(table, lens, refs, parents, t2, l2, r2);
  reg.find('pages_reserve')(t2, l2, r2, counts, 16, mv, info);
  reg.find('pages_copy')(pool, mv, info);
  reg.find('paged_kv_write')(k, k, kp, vp, t2, l2, null);
  const o = f32([3, 4, 64]);
  reg.find('paged_attention')(q, kp, vp, t2, l2, null, o, 0.125, true, 1);
  const t3 = i32([3, 3]), r3 = i32([9]), mv3 = i32([4, 2]), info3 = i32([2]);
  reg.find('pages_compact')(t2, r2, t3, r3, mv3, info3);
  const x = read('x', [1, 3, 500], 'float32'), s = read('s', [1, 3], 'float32'), fin = read('fin', [1, 3], 'int32');
  const os = f32([1, 3]), ot = i32([1, 3]), op = i32([1, 3]), of = i32([1, 3]);
  reg.find('beam_select')(x, s, fin, 3, 7, os, ot, op, of);
  const all = { t2, l2, r2, mv, info, pool, o, t3, r3, mv3, info3, os, ot, op, of };
  for (const name of Object.keys(all)) {
    const h = all[name];
    const host = new ArrayBuffer(4 * h.numel);
    require(process.argv[3]).memcpyD2H(host, h.ptr);
    fs.writeFileSync(dir + '/out_' + name, Buffer.from(host));
  }
  console.log(JSON.stringify({ ok: true }));
}).catch((e) => { console.error(e.stack); process.exit(1); });
"""


def test_kernels_from_node(hip, tmp_path):
    if shutil.which("node") is None or not os.path.exists(ADDON):
        pytest.skip("node or the built addon is not available")
    _ensure_dist()
    x = {"q": syn.normal(1, (3, 4, 64)), "k": syn.normal(2, (3, 2, 64)), "pool": syn.normal(3, (2, 9, 2, 16, 64)),
         "table": np.array([[4, 1, -1], [4, 2, -1], [7, -1, -1]]), "lens": np.array([30, 20, 16]),
         "refs": np.array([0, 1, 1, 0, 2, 0, 0, 1, 0]), "parents": np.array([0, 0, 2]), "counts": np.array([1, 1, 1]),
         "x": syn.normal(4, (1, 3, 500)), "s": np.array([[-1, -2, -1.5]]), "fin": np.array([[0, 0, 1]])}
    x = {n: v.astype(np.float32 if n in ("q", "k", "pool", "x", "s") else np.int32) for n, v in x.items()}
    for n, v in x.items():
        v.tofile(str(tmp_path / n))
    run = subprocess.run(["node", "-e", SCRIPT, os.path.join(PKG, "dist", "index.js"), str(tmp_path), ADDON],
                         capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and json.loads(run.stdout.strip().splitlines()[-1])["ok"], run.stderr
    t = {n: Tensor(v, dtype="float32" if v.dtype == np.float32 else "int32") for n, v in x.items()}
    t2, l2, r2 = F.pages_fork(t["table"], t["lens"], t["refs"], t["parents"])
    mv, info = F.pages_reserve(t2, l2, r2, t["counts"], 16)
    F.pages_copy(t["pool"], mv, info)
    kp, vp = (F.view(F.narrow(t["pool"], 0, i, 1), (9, 2, 16, 64)) for i in (0, 1))
    F.paged_kv_write(t["k"], t["k"], kp, vp, t2, l2)
    o = F.paged_attention(t["q"], kp, vp, t2, l2, max_query_len=1)
    t3, r3, mv3, info3 = F.pages_compact(t2, r2)
    os_, ot, op, of = F.beam_select(t["x"], t["s"], None, t["fin"], 7)
    assert info.numpy().tolist() == [1, 0, 0]
    for name, h in dict(t2=t2, l2=l2, r2=r2, mv=mv, info=info, pool=t["pool"], o=o, t3=t3, r3=r3, mv3=mv3, info3=info3, os=os_,
                        ot=ot, op=op, of=of).items():
        want = h.numpy()
        np.testing.assert_array_equal(np.fromfile(str(tmp_path / f"out_{name}"), want.dtype).reshape(want.shape), want, err_msg=name)
