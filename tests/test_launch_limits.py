"""Calls whose launches would hold 2^32 threads in a dimension of the grid, on the
CPU: refused before the first launch, since a later one of the same call could not
rely on its results."""
import ctypes as C

import pytest

from tests.test_paged import F, _cache, _decode, _prefill
from tests.test_serving import _adapters, _add, _shared
from webgllm_amd import lib as L

FAR = dict(q=1 << 45, out=1 << 46, size=1 << 50)


def _heads(heads, kv_heads, hd=64):
    return L.AttnShape(heads, kv_heads, hd, hd, 1e-6, 0)


def _large(entries=4096, **more):
    return _cache(v=1 << 44, pages=600, ld_table=256, sequences=65535, max_entries=entries, **more)


@pytest.mark.parametrize("call,heads,entries,more", [
    (_shared, 256, 4096, dict(M=65535, groups=65535)),  # a row a sequence: the prefixes' blocks
    (_shared, 256, 4096, dict(M=131070, rows=F)),       # rows of several tokens: their own blocks
    (_shared, 2048, 64, dict(M=65535, groups=5)),       # a workgroup a unit
    (_shared, 512, 64, dict(M=131070, rows=F)),         # as prompts
    (_decode, 2048, 64, dict()), (_decode, 2048, 4096, dict()),
    (_prefill, 512, 64, dict(M=131070))])
def test_attention(call, heads, entries, more):
    lib, wide = L.load(), heads * 64
    strides = dict(ld=wide) if call is _prefill else dict(ldq=wide, ldo=wide)
    rc = call(lib, _large(entries), sh=_heads(heads, heads), **strides, **FAR, **more)
    assert rc == -1 and str(65535 if call is _decode else more["M"]) in L.last_error(), L.last_error()


@pytest.mark.parametrize("M", [1 << 30, 2 ** 31 - 1])
def test_adapters(M):
    lib = L.load()
    rc = _add(lib, _adapters(), M=M, rows=F, n=1, x=1 << 44, y=1 << 46, size=1 << 50)
    assert rc == -1 and f"{M} rows" in L.last_error(), L.last_error()
