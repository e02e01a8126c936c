"""What wg_paged_attn_shared refuses where it runs as another call, on the CPU: under
its own name."""
import ctypes as C

import pytest

from tests.test_paged import F, _cache
from tests.test_serving import _shared
from webgllm_amd import lib as L


@pytest.mark.parametrize("M,rows", [(2, None), (100, F)])  # a token each; as prompts
@pytest.mark.parametrize("scratch,size", [(F, 64), (None, 1 << 40), (F + 8, 1 << 40)])
def test_scratch(M, rows, scratch, size):
    lib, sh = L.load(), L.AttnShape(8, 2, 64, 64, 1e-6, 0)
    c = _cache(pages=600, ld_table=256, max_entries=4096)
    assert lib.wg_paged_shared_scratch_bytes(C.byref(c), C.byref(sh), M, 1) > 64
    rc = _shared(lib, c, sh=sh, M=M, rows=rows, scratch=scratch, size=size)
    assert rc == -1 and L.last_error().startswith("wg_paged_attn_shared: scratch"), L.last_error()
