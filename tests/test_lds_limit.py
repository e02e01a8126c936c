"""Kernels' raised LDS limits (csrc/lds_limit.h, compiled by itself): whatever the
order of the sizes asked for, the one set last holds every launch."""
import ctypes as C
import itertools
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "webgllm_amd",
                    "csrc")


@pytest.fixture(scope="module")
def limits(tmp_path_factory):
    d = tmp_path_factory.mktemp("lds")
    src, so = d / "limits.cpp", d / "limits.so"
    src.write_text(f'#include "{CSRC}/lds_limit.h"\n'
                   'extern "C" void *make() { return new wg::LdsLimits; }\n'
                   'extern "C" int above(void *l, const void *k, int dev, int n) {\n'
                   '  return static_cast<wg::LdsLimits *>(l)->above(k, dev, n);\n}\n'
                   'extern "C" void set(void *l, const void *k, int dev, int n) {\n'
                   '  static_cast<wg::LdsLimits *>(l)->set(k, dev, n);\n}\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-o",
                    str(so), str(src)], check=True)
    lib = C.CDLL(str(so))
    lib.make.restype = C.c_void_p
    lib.above.argtypes = lib.set.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int]
    lib.set.restype = None
    return lib


def test_limits_only_rise(limits):
    sizes = (66, 74, 99)
    for order in itertools.product(sizes, repeat=4):
        l, now = limits.make(), {}  # the attribute, as the device holds it
        for i, n in enumerate(order):
            for at in ((1, 0), (1, 1), (2, 0)) if i % 2 else ((1, 0),):  # (kernel, device)
                if limits.above(l, *at, n):
                    now[at] = n
                    limits.set(l, *at, n)
                assert now[at] >= n, (order, at)
    l = limits.make()
    limits.set(l, 1, 0, 99)
    assert not limits.above(l, 1, 0, 99) and not limits.above(l, 1, 0, 74)
    assert limits.above(l, 1, 1, 74) and limits.above(l, 2, 0, 74)
