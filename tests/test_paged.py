"""The paged cache on the CPU: where entries lie and which a row sees
(csrc/paged_core.h, compiled by itself), and what the entry points refuse
before any device work."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from webgllm_amd import lib as L

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "webgllm_amd",
                    "csrc")


@pytest.fixture(scope="module")
def core(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    src, so = d / "core.cpp", d / "core.so"
    src.write_text(f'#include "{CSRC}/paged_core.h"\n'
                   'extern "C" int row(const int *table, int pages, int shift, int i) {\n'
                   '  wg::Paged c = {0, 0, table, 0, pages, shift, 0, 1, 1 << 30};\n'
                   '  return wg::paged_row(c, table, i);\n}\n'
                   'extern "C" int len(int n, int most) {\n'
                   '  wg::Paged c = {0, 0, 0, &n, 1, 0, 1, 1, most};\n'
                   '  return wg::paged_len(c, 0);\n}\n'
                   'extern "C" int span(int first, int last, int window, int sinks, int *out) {\n'
                   '  const wg::Span s = wg::paged_span(first, last, window, sinks);\n'
                   '  for (int t = 0; t < s.count; t++) out[t] = wg::span_entry(s, t);\n'
                   '  return s.count;\n}\n'
                   'extern "C" int sees(int i, int j, int window, int sinks) {\n'
                   '  return wg::paged_sees(i, j, window, sinks);\n}\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-o",
                    str(so), str(src)], check=True)
    return C.CDLL(str(so))


def test_rows_of_pages(core):
    table = np.array([3, 0, -1, 5, 6, 2 ** 31 - 1, -2 ** 31], dtype=np.int32)
    t = table.ctypes.data_as(C.c_void_p)
    for shift in (0, 4, 10):
        for page, want in enumerate((3, 0, None, 5, None, None, None)):  # pages 0 .. 5
            for off in {0, (1 << shift) - 1}:
                got = core.row(t, 6, shift, (page << shift) + off)
                assert got == (-1 if want is None else (want << shift) + off)
    big = np.array([(1 << 27) - 1], dtype=np.int32)  # the largest row: 2^31 - 1 less one
    assert core.row(big.ctypes.data_as(C.c_void_p), 1 << 27, 4, 14) == 2 ** 31 - 2


def test_lengths_are_cut(core):
    assert [core.len(n, 100) for n in (-2 ** 31, -1, 0, 1, 100, 101, 2 ** 31 - 1)] == \
        [0, 0, 0, 1, 100, 100, 100]


@pytest.mark.parametrize("window", [0, 1, 2, 5, 30, 31, 2 ** 31 - 1])
@pytest.mark.parametrize("sinks", [0, 1, 4, 29, 2 ** 31 - 1])
def test_spans_hold_what_rows_see(core, window, sinks):
    out = (C.c_int * 64)()
    for first, last in ((0, 0), (29, 29), (7, 29), (0, 29)):
        n = core.span(first, last, window, sinks, out)
        got = list(out[:n])
        assert got == sorted(set(got)) and all(0 <= j <= last for j in got)
        seen = {j for i in range(first, last + 1) for j in range(last + 1)
                if core.sees(i, j, window, sinks)}
        want = {j for i in range(first, last + 1) for j in range(i + 1)
                if not window or j < sinks or j > i - window}
        assert seen == want and seen <= set(got)
        if first == last:
            assert seen == set(got)


F = 0x100000  # fake device addresses: the calls fail before any launch


def _cache(**more):
    d = dict(k=F, v=0x10000000, pages=8, page_size=16, table=F, ld_table=4, sequences=2, lens=F,
             max_entries=64)
    return L.PagedCacheDesc(**{**d, **more})


BAD_CACHES = [(dict(k=None), "null cache"), (dict(table=None), "null cache"),
              (dict(lens=None), "null cache"), (dict(k=F + 8), "16-byte aligned"),
              (dict(page_size=24), "a power of two"), (dict(page_size=0), "a power of two"),
              (dict(pages=0), "fewer than 2^31"), (dict(pages=1 << 27), "fewer than 2^31"),
              (dict(sequences=0), "0 sequences"), (dict(sequences=65536), "65536 sequences"),
              (dict(max_entries=65), "65 entries"), (dict(max_entries=0), "0 entries"),
              (dict(ld_table=1 << 30, max_entries=(1 << 30) + 1), "entries a sequence"),
              (dict(v=F + 16), "overlap")]


def _prep(lib, cache, sh=None, M=2, ldq=768, ldqo=512, rows=None, qo=0x40000000, rope_rows=1025,
          norm=None, qkv=0x50000000):
    sh = sh or L.AttnShape(8, 2, 64, 64, 1e-6, 0)
    return lib.wg_paged_head_prep(qkv, M, ldq, C.byref(sh), norm, norm, F, rope_rows, None,
                                  C.byref(cache), rows, qo, ldqo, None)


def _decode(lib, cache, sh=None, ldq=512, ldo=512, window=0, sinks=0, weights=None, ldw=0,
            scratch=F, size=1 << 40, q=0x50000000, out=0x60000000):
    sh = sh or L.AttnShape(8, 2, 64, 64, 1e-6, 0)
    return lib.wg_paged_attn_decode(q, ldq, C.byref(sh), C.byref(cache), window, sinks, weights,
                                    ldw, out, ldo, scratch, size, None)


def _prefill(lib, cache, sh=None, M=4, rows=F, window=0, sinks=0, scratch=F, size=1 << 40,
             q=0x50000000, out=0x60000000, ld=512):
    sh = sh or L.AttnShape(8, 2, 64, 64, 1e-6, 0)
    return lib.wg_paged_attn_prefill(q, M, ld, C.byref(sh), C.byref(cache), rows, window, sinks,
                                     out, ld, scratch, size, None)


def _evict(lib, cache, to=None, kv_dim=128, keep=32, sinks=4, recent=8, weights=0x50000000,
           ldw=64, lens=F, tow=0x60000000, ldtw=32, kept=F, ldk=32, scratch=F, size=1 << 40):
    to = to or _cache()
    return lib.wg_paged_evict(C.byref(cache), kv_dim, weights, ldw, keep, sinks, recent,
                              C.byref(to), lens, tow, ldtw, kept, ldk, scratch, size, None)


@pytest.mark.parametrize("fields,msg", BAD_CACHES)
@pytest.mark.parametrize("call", [_prep, _decode, _prefill, _evict])
def test_bad_caches_are_refused(call, fields, msg):
    lib = L.load()
    assert call(lib, _cache(**fields)) == -1 and msg in L.last_error(), L.last_error()
    if call is _evict and "lens" not in fields:  # (the new lengths are an argument)
        rc = call(lib, _cache(), to=_cache(**fields))
        assert rc == -1 and ("(to)" in L.last_error() or "sequences" in L.last_error())


@pytest.mark.parametrize("call,more,msg", [
    (_prep, dict(M=3), "3 rows for 2 sequences"), (_prep, dict(M=0, rows=F), "0 rows"),
    (_prep, dict(ldq=767), "strides"), (_prep, dict(ldqo=511), "strides"),
    (_prep, dict(rope_rows=1024), "rope table"), (_prep, dict(qo=0x50000100), "overlaps"),
    (_prep, dict(sh=L.AttnShape(8, 2, 64, 64, 1e-6, 1)), "norm weights missing"),
    (_prep, dict(sh=L.AttnShape(8, 3, 64, 64, 1e-6, 0)), "query heads"),
    (_prep, dict(sh=L.AttnShape(8, 2, 60, 60, 1e-6, 0)), "head_dim"),
    (_prep, dict(sh=L.AttnShape(8, 2, 64, 65, 1e-6, 0)), "rotated dims"),
    (_decode, dict(sh=L.AttnShape(65, 1, 64, 64, 1e-6, 0)), "query heads"),
    (_decode, dict(sh=L.AttnShape(8, 2, 96, 96, 1e-6, 0)), "head_dim 96"),
    (_decode, dict(window=-1), "window"), (_decode, dict(sinks=-1), "sinks"),
    (_decode, dict(ldq=514), "16-byte aligned"), (_decode, dict(q=0x50000004), "16-byte aligned"),
    (_decode, dict(ldo=511), "strides"), (_decode, dict(out=0x50000000), "overlaps"),
    (_decode, dict(weights=F, ldw=63), "weights of 63"),
    (_decode, dict(weights=F, ldw=64, size=0), "scratch of 0"),
    (_decode, dict(weights=F, ldw=64, scratch=F + 4), "16-byte aligned"),
    (_prefill, dict(sh=L.AttnShape(33, 1, 64, 64, 1e-6, 0)), "query heads"),
    (_prefill, dict(rows=None), "row_start"), (_prefill, dict(M=0), "0 rows"),
    (_prefill, dict(window=-5), "window"),
    (_evict, dict(kv_dim=12), "a multiple of 8"), (_evict, dict(keep=0), "kept"),
    (_evict, dict(sinks=30), "30 sinks and 8 recent entries of 32"),
    (_evict, dict(sinks=-1), "sinks"), (_evict, dict(recent=-1), "recent"),
    (_evict, dict(ldw=63), "strides"), (_evict, dict(ldk=31), "strides"),
    (_evict, dict(ldtw=31), "strides"), (_evict, dict(tow=0x50000010), "overlaps"),
    (_evict, dict(weights=None), "null"), (_evict, dict(kept=None), "null"),
    (_evict, dict(lens=None), "null"),
    (_evict, dict(to=_cache(sequences=1)), "2 sequences to 1"),
    (_evict, dict(to=_cache(max_entries=31)), "room for 31 entries of 32")])
def test_bad_arguments_are_refused(call, more, msg):
    lib = L.load()
    assert call(lib, _cache(), **more) == -1 and msg in L.last_error(), L.last_error()


def test_scratch_follows_the_cache():
    lib = L.load()
    sh = L.AttnShape(8, 2, 64, 64, 1e-6, 0)
    plain, summed = (lib.wg_paged_decode_scratch_bytes(C.byref(_cache()), C.byref(sh), w)
                     for w in (0, 1))
    assert summed >= plain + 2 * 8 * 64 * 4  # the scores of every head
    assert lib.wg_paged_decode_scratch_bytes(None, C.byref(sh), 1) == 0
    assert lib.wg_paged_prefill_scratch_bytes(None, None, 4) == 0
    assert lib.wg_paged_evict_scratch_bytes(None) == 0
