"""The paged cache's calls of the Node N-API addon, run by Node itself
(tests/node/paged_test.js makes the assertions): scratch sizes and refused
arguments on the CPU; preparation, attention and eviction on the GPU against
the contiguous cache's calls."""
import ctypes as C
import json
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SCRIPT = os.path.join(ROOT, "tests", "node", "paged_test.js")
ADDON = os.path.join(ROOT, "webgllm_amd", "node", "webgllm_hip.node")


def _run(mode):
    node = shutil.which("node")
    if node is None:
        pytest.skip("no node on this machine")
    if not os.path.exists(ADDON):
        pytest.fail("webgllm_amd/node/webgllm_hip.node is not built (run __graft_entry__.build())")
    p = subprocess.run([node, SCRIPT, mode], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stderr[-4000:]
    return json.loads(p.stdout.strip().splitlines()[-1])


def test_sizes_and_refusals():
    from webgllm_amd import lib as L
    from webgllm_amd import ops
    out, lib = _run("cpu"), L.load()
    sh = ops.attn_shape(4, 2, 64)
    for i, (pages, wide) in enumerate([(9, 4), (9000, 4000)]):
        d = L.PagedCacheDesc(None, None, pages, 16, None, wide, 2, None, wide * 16)
        assert out["decode"][i] == lib.wg_paged_decode_scratch_bytes(C.byref(d), C.byref(sh), 0) > 0
        assert out["weights"][i] == lib.wg_paged_decode_scratch_bytes(C.byref(d), C.byref(sh), 1)
        assert out["prefill"][i] == lib.wg_paged_prefill_scratch_bytes(C.byref(d), C.byref(sh), 5)
        assert out["evict"][i] == lib.wg_paged_evict_scratch_bytes(C.byref(d))
    assert out["weights"][0] > out["decode"][0] and out["evict"][0] == 0 < out["evict"][1]


@pytest.mark.gpu
def test_two_sequences_in_pages(hip):
    assert _run("gpu")["kept"] == 36
