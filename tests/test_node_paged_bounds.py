"""A paged cache whose table rows could hold more than a sequence may have, through
the Node addon: taken where maxEntries bounds it, as the library takes it."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

INDEX = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "webgllm_amd",
                     "node", "index.js")
SCRIPT = """
const A = require(process.argv[1]).addon
const wide = { pages: 9, pageSize: 1 << 20, ldTable: 2048, sequences: 2 }
const shape = { heads: 4, kvHeads: 2, headDim: 64 }
let refused = 0
try { A.pagedDecodeScratchBytes(wide, shape, 0) } catch (e) { refused++ }
console.log(refused, A.pagedDecodeScratchBytes(Object.assign({}, wide, { maxEntries: 5000 }), shape, 1))
"""


def test_wide_tables_under_a_bound():
    node = shutil.which("node")
    if node is None:
        pytest.skip("no node on this machine")
    from webgllm_amd import lib as L
    from webgllm_amd import ops
    p = subprocess.run([node, "-e", SCRIPT, INDEX], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stderr[-2000:]
    refused, size = map(int, p.stdout.split())
    d = L.PagedCacheDesc(None, None, 9, 1 << 20, None, 2048, 2, None, 5000)
    want = L.load().wg_paged_decode_scratch_bytes(C.byref(d), C.byref(ops.attn_shape(4, 2, 64)), 1)
    assert refused == 1 and size == want > 0
