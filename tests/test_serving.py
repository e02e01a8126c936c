"""Serving many requests together, on the CPU: which axis a frequency turns by
(csrc/paged_core.h, compiled by itself), and what the calls refuse before any
device work."""
import ctypes as C
import os
import subprocess

import pytest

from tests.test_paged import BAD_CACHES, CSRC, F, _cache
from webgllm_amd import lib as L


@pytest.fixture(scope="module")
def axis_of(tmp_path_factory):
    d = tmp_path_factory.mktemp("axes")
    src, so = d / "core.cpp", d / "core.so"
    src.write_text(f'#include "{CSRC}/paged_core.h"\n'
                   'extern "C" int axis(int axes, int inter, const int *n, int f) {\n'
                   '  wg::RopeAxes r = {axes, inter, {0, 0, 0, 0}};\n'
                   '  for (int a = 0; a < axes; a++) r.n[a] = n[a];\n'
                   '  return wg::rope_axis(r, f);\n}\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-o",
                    str(so), str(src)], check=True)
    core = C.CDLL(str(so))
    return lambda n, inter, f: core.axis(len(n), int(inter), (C.c_int * len(n))(*n), f)


@pytest.mark.parametrize("n", [[32], [16, 16], [8, 12, 12], [16, 24, 24], [0, 5, 3], [4, 0, 4],
                               [3, 1, 2, 2], [0, 0, 0, 7]])
def test_sections_one_after_another(axis_of, n):
    want = [a for a, k in enumerate(n) for _ in range(k)]
    assert [axis_of(n, False, f) for f in range(sum(n))] == want


@pytest.mark.parametrize("n", [[32], [16, 16], [12, 10, 10], [24, 20, 20], [11, 11, 10], [6, 0, 2],
                               [8, 8, 8, 8], [7, 3, 1, 1]])
def test_interleaved_sections(axis_of, n):
    """Each axis but the first has frequencies a, a + axes, a + 2 axes, .. as long
    as it has some; the first has all others."""
    P, k = sum(n), len(n)
    want = [0] * P
    for a in range(1, k):
        for i in range(n[a]):
            want[a + i * k] = a
    got = [axis_of(n, True, f) for f in range(P)]
    assert got == want and [got.count(a) for a in range(k)] == n


@pytest.mark.parametrize("n", [[8, 12, 12], [0, 16, 16], [0, 0, 32], [1, 1, 1, 29]])
def test_interleaved_sections_that_run_out_of_frequencies(axis_of, n):
    """Every axes-th frequency up to a section's end or the last, all others the
    first axis'."""
    P, k = sum(n), len(n)
    want = [f % k if f // k < n[f % k] else 0 for f in range(P)]
    assert [axis_of(n, True, f) for f in range(P)] == want


def _axes(lib, cache, sections=(8, 12, 12), inter=0, n=None, pos=F, ld_pos=3, sh=None, M=2,
          ldq=768, ldqo=512, rows=None, qkv=0x50000000, qo=0x40000000, axes=True, rope_rows=1025):
    sh = sh or L.AttnShape(8, 2, 64, 64, 1e-6, 0)
    ax = L.RopeAxes(len(sections) if n is None else n, inter, (C.c_int32 * 4)(*sections[:4]))
    return lib.wg_paged_head_prep_axes(qkv, M, ldq, C.byref(sh), None, None, F, rope_rows, pos,
                                       ld_pos, C.byref(ax) if axes else None, C.byref(cache), rows,
                                       qo, ldqo, None)


def _shared(lib, cache, sh=None, M=2, rows=None, starts=F, shared=F, groups=1, scratch=F,
            size=1 << 40, q=0x50000000, out=0x60000000, ldq=512, ldo=512):
    sh = sh or L.AttnShape(8, 2, 64, 64, 1e-6, 0)
    return lib.wg_paged_attn_shared(q, M, ldq, C.byref(sh), C.byref(cache), rows, starts, shared,
                                    groups, out, ldo, scratch, size, None)


def _adapters(**more):
    d = dict(a=F, b=0x10000000, rank=F, scale=F, slots=3, max_rank=16, K=64, N=96, parts=2,
             cols=(C.c_int32 * 4)(64, 32))
    return L.AdaptersDesc(**{**d, **more})


def _add(lib, ad, M=2, ldx=64, slot=F, rows=None, n=2, row_scale=None, y=0x60000000, ldy=96,
         scratch=F, size=1 << 40, x=0x50000000):
    return lib.wg_adapter_add(x, M, ldx, C.byref(ad) if ad is not None else None, slot, rows, n,
                              row_scale, y, ldy, scratch, size, None)


@pytest.mark.parametrize("fields,msg", BAD_CACHES)
@pytest.mark.parametrize("call", [_axes, _shared])
def test_bad_caches_are_refused(call, fields, msg):
    lib = L.load()
    assert call(lib, _cache(**fields)) == -1 and msg in L.last_error(), L.last_error()


@pytest.mark.parametrize("call,more,msg", [
    (_axes, dict(axes=False), "null"), (_axes, dict(pos=None), "null"),
    (_axes, dict(n=0), "0 axes"), (_axes, dict(sections=(8, 8, 8, 8, 0), n=5, ld_pos=5), "5 axes"),
    (_axes, dict(ld_pos=2), "of 2 positions"), (_axes, dict(sections=(8, 12, 11)), "31 frequencies"),
    (_axes, dict(sections=(33,), ld_pos=1), "33 frequencies"),
    (_axes, dict(sections=(40, -4, -4)), "a section of -4"),
    (_axes, dict(sections=(8, 12, 11), inter=1), "31 frequencies"),
    (_axes, dict(sections=(2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1)), "sections of"),
    (_axes, dict(sh=L.AttnShape(8, 2, 64, 32, 1e-6, 0)), "32 rotated dims"),
    (_axes, dict(M=3), "3 rows for 2 sequences"), (_axes, dict(ldq=767), "strides"),
    (_axes, dict(rope_rows=1024), "rope table"), (_axes, dict(qo=0x50000100), "overlaps"),
    (_axes, dict(sh=L.AttnShape(8, 2, 64, 64, 1e-6, 1)), "norm weights missing"),
    (_shared, dict(starts=None), "null"), (_shared, dict(shared=None), "null"),
    (_shared, dict(groups=0), "0 groups"), (_shared, dict(groups=3), "3 groups of 2"),
    (_shared, dict(M=3), "3 rows for 2 sequences"), (_shared, dict(M=0, rows=F), "0 rows"),
    (_shared, dict(sh=L.AttnShape(33, 1, 64, 64, 1e-6, 0)), "query heads"),
    (_shared, dict(sh=L.AttnShape(8, 2, 96, 96, 1e-6, 0)), "head_dim 96"),
    (_shared, dict(ldq=514), "16-byte aligned"), (_shared, dict(ldo=511), "strides"),
    (_shared, dict(out=0x50000000), "overlaps"), (_shared, dict(size=64), "scratch of 64"),
    (_shared, dict(scratch=None), "scratch"), (_shared, dict(scratch=F + 4), "16-byte aligned")])
def test_bad_arguments_are_refused(call, more, msg):
    lib = L.load()
    assert call(lib, _cache(), **more) == -1 and msg in L.last_error(), L.last_error()


@pytest.mark.parametrize("fields,msg", [
    (dict(a=None), "null"), (dict(b=None), "null"), (dict(rank=None), "null"),
    (dict(scale=None), "null"), (dict(slots=0), "0 adapters"), (dict(max_rank=12), "ranks up to 12"),
    (dict(max_rank=264), "ranks up to 264"), (dict(max_rank=0), "ranks up to 0"),
    (dict(K=60), "K 60"), (dict(K=0), "K 0"), (dict(K=2 ** 31 - 8), "up to 2^30"),
    (dict(N=2 ** 31 - 4, cols=(C.c_int32 * 4)(2 ** 30, 2 ** 30 - 4)), "up to 2^30"),
    (dict(parts=0), "0 parts"), (dict(parts=5), "5 parts"),
    (dict(N=92), "96 outputs of 92"), (dict(cols=(C.c_int32 * 4)(66, 30)), "66 outputs"),
    (dict(cols=(C.c_int32 * 4)(96, 0)), "0 outputs"), (dict(a=F + 8), "16-byte aligned"),
    (dict(b=0x10000004), "16-byte aligned")])
def test_bad_adapters_are_refused(fields, msg):
    lib = L.load()
    assert _add(lib, _adapters(**fields)) == -1 and msg in L.last_error(), L.last_error()


@pytest.mark.parametrize("more,msg", [
    (dict(x=None), "null"), (dict(slot=None), "null"), (dict(y=None), "null"),
    (dict(M=3), "3 rows of 2"), (dict(M=0, rows=F), "0 rows"), (dict(n=0, rows=F), "0 sequences"),
    (dict(n=65536, rows=F), "65536 sequences"), (dict(ldx=63), "strides"), (dict(ldy=95), "strides"),
    (dict(x=0x50000008), "16-byte aligned"), (dict(ldx=68), "16-byte aligned"),
    (dict(y=0x50000010), "overlaps"), (dict(size=8), "scratch of 8"), (dict(scratch=None), "scratch"),
    (dict(scratch=F + 8), "scratch")])
def test_bad_adapter_calls_are_refused(more, msg):
    lib = L.load()
    assert _add(lib, _adapters(), **more) == -1 and msg in L.last_error(), L.last_error()
    assert _add(lib, None) == -1 and "null" in L.last_error()


def test_scratch_sizes():
    lib = L.load()
    sh, long = L.AttnShape(8, 2, 64, 64, 1e-6, 0), _cache(pages=600, ld_table=256, max_entries=4096)
    sizes = [lib.wg_paged_shared_scratch_bytes(C.byref(long), C.byref(sh), M, 1) for M in (2, 3, 30)]
    assert 0 < sizes[0] and 0 < sizes[1] < sizes[2]
    # rows of several tokens as a prompt's: in a short cache, many a sequence
    for c, M in ((_cache(), 3), (long, 100)):
        assert lib.wg_paged_shared_scratch_bytes(C.byref(c), C.byref(sh), M, 1) == \
            lib.wg_paged_prefill_scratch_bytes(C.byref(c), C.byref(sh), M)
    assert lib.wg_paged_shared_scratch_bytes(None, C.byref(sh), 2, 1) == 0
    assert lib.wg_paged_shared_scratch_bytes(C.byref(_cache()), C.byref(sh), 2, 0) == 0
    assert lib.wg_adapter_scratch_bytes(C.byref(_adapters()), 5) >= 5 * 2 * 16 * 4
    assert lib.wg_adapter_scratch_bytes(None, 5) == 0
    assert lib.wg_adapter_scratch_bytes(C.byref(_adapters()), 0) == 0
