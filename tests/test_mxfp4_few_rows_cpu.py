"""Which form of the few-rows kernel each size takes (csrc/mxfp4_tiles.hpp, compiled here): the GPU tests name every form, and
no form is built that no call takes."""
import ctypes
import itertools
import os
import re
import subprocess

import pytest

import test_gpu_mxfp4_few_rows as gpu
from lux3d_fused import _lib

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "candle-3d_amd", "csrc")
KIND = {"fp4": 0, "2byte": 1, "f32": 2}


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("mxfp4_few_rows")
    src, so = out / "few.cpp", out / "few.so"
    src.write_text('#include "mxfp4_tiles.hpp"\n'
                   'using namespace lux3d;\n'
                   'extern "C" int64_t below(int kind, int64_t m, int64_t n, int64_t k, int gated) {\n'
                   '  return mx_choose((MxKind)kind, m, n, k, gated).rows;\n}\n'
                   'extern "C" void few(int two, int64_t m, int64_t n, int64_t k, int gated, int *o) {\n'
                   '  const MxFewTile f = mx_few_tile(two, m, n, k, gated);\n'
                   '  o[0] = f.rows, o[1] = f.cols, o[2] = f.waves;\n}\n')
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-shared", "-fPIC", "-I", CSRC, "-o", str(so), str(src)], check=True)
    dll = ctypes.CDLL(str(so))
    dll.below.argtypes = [ctypes.c_int] + [ctypes.c_int64] * 3 + [ctypes.c_int]
    dll.below.restype = ctypes.c_int64
    dll.few.argtypes = [ctypes.c_int] + [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.c_void_p]
    return dll


def form(lib, two, gated, m, k, n):
    o = (ctypes.c_int * 3)()
    lib.few(int(two), m, n, k, int(gated), o)
    return tuple(o)


MS, KS = (1, 15, 16, 17, 100), (32, 480, 512, 992, 1024, 1536, 6112, 6144, 8192, 65536)
NS = (1, 77, 2048, 8191, 8192, 16383, 16384, 24575, 24576, 32000, 200000)


def forms(lib, two, gated, most):
    return {form(lib, two, gated, m, k, n) for m, k, n in itertools.product([m for m in MS if m <= most], KS, NS)}


def test_few_rows_tests_reach_the_forms_they_name(lib):
    for mt, nt, nw, two, gated, m, k, n in gpu.FEW:
        assert form(lib, two, gated, m, k, n) == (mt, nt, nw), (mt, nt, nw, two, gated, m, k, n)
        for kind in ("2byte",) if two else ("f32", "fp4"):
            assert lib.below(KIND[kind], m, n, k, int(gated)) == 0, (kind, gated, m, k, n)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("two", [False, True])
def test_every_form_is_named(lib, two, gated):
    assert forms(lib, two, gated, 100) == {t[:3] for t in gpu.FEW if t[3:5] == (two, gated)}


def test_every_built_form_is_taken(lib):
    """The names of the kernels in the library, by their template arguments: x's type (void: packed), x in 4 bits, gated, the
    form. Plain x of more than 16 rows that enters in 4 bits is packed first."""
    with open(_lib.LIB_PATH, "rb") as f:
        names = set(re.findall(rb"mx_rows_kernelI(?:NS_\d+(\w+?)E|(v))Lb([01])ELb([01])ELi(\d+)ELi(\d+)ELi(\d+)E", f.read()))
    built = {((x or v).decode(), int(fp4), int(gated), int(mt), int(nt), int(nw)) for x, v, fp4, gated, mt, nt, nw in names}
    taken = set()
    for x, fp4, gated in itertools.product(("BF16", "F16", "F32", "v"), (0, 1), (0, 1)):
        if x == "v" and not fp4:
            continue
        for f in forms(lib, x in ("BF16", "F16") and not fp4, gated, 16 if fp4 and x != "v" else 100):
            taken.add((x, fp4, gated, *f))
    assert built == taken, (built - taken, taken - built)
