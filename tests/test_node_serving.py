"""Shared prefixes, adapters and several axes through the Node N-API addon, run
by Node itself (tests/node/serving_test.js makes the assertions): scratch sizes
and refused arguments on the CPU; on the GPU against the calls that share
nothing and sums in doubles."""
import ctypes as C
import json
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SCRIPT = os.path.join(ROOT, "tests", "node", "serving_test.js")
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
        for j, m in enumerate((2, 7)):
            assert out["shared"][i][j] == lib.wg_paged_shared_scratch_bytes(
                C.byref(d), C.byref(sh), m, 1)
    ad = L.AdaptersDesc(None, None, None, None, 3, 16, 64, 96, 2, (C.c_int32 * 4)(64, 32))
    one = L.AdaptersDesc(None, None, None, None, 1, 8, 4096, 64, 1, (C.c_int32 * 4)(64))
    assert out["adapter"] == [lib.wg_adapter_scratch_bytes(C.byref(ad), m) for m in (1, 50)]
    assert out["one"] == lib.wg_adapter_scratch_bytes(C.byref(one), 9) > 0


@pytest.mark.gpu
def test_against_the_calls_that_share_nothing(hip):
    assert _run("gpu")["rows"] == 3
