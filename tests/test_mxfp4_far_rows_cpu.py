"""When the linears on 4-bit weights leave the kernel of many rows because its offsets would pass 32 bits (csrc/mxfp4_tiles.hpp,
compiled here): the sizes of the GPU tests of far rows, and the borders."""
import ctypes
import os
import subprocess

import pytest

import test_gpu_mxfp4_far_rows as gpu

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "candle-3d_amd", "csrc")
KIND = {"fp4": 0, "2byte": 1, "f32": 2}


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("mxfp4_far_rows")
    src, so = out / "far.cpp", out / "far.so"
    src.write_text('#include "mxfp4_tiles.hpp"\n'
                   'using namespace lux3d;\n'
                   'extern "C" int64_t below(int kind, int64_t m, int64_t n, int64_t k, int gated) {\n'
                   '  return mx_choose((MxKind)kind, m, n, k, gated).rows;\n}\n'
                   'extern "C" int fits(int kind, int64_t ldx, int64_t xs_rows, int64_t n, int64_t k, int64_t ldy) {\n'
                   '  return mx_gemm_fits((MxKind)kind, ldx, xs_rows, n, k, ldy);\n}\n')
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-shared", "-fPIC", "-I", CSRC, "-o", str(so), str(src)], check=True)
    dll = ctypes.CDLL(str(so))
    dll.below.argtypes = [ctypes.c_int] + [ctypes.c_int64] * 3 + [ctypes.c_int]
    dll.below.restype = ctypes.c_int64
    dll.fits.argtypes = [ctypes.c_int] + [ctypes.c_int64] * 5
    return dll


def test_rows_far_apart_leave_the_tiles(lib):
    """What the kernel of many rows would take with rows close, and cannot address so far apart."""
    for kind, gated, m, k, n, x_apart, y_apart in gpu.FAR:
        assert lib.below(KIND[kind], m, n, k, int(gated)) > 0, (kind, gated, m, k, n)
        assert lib.fits(KIND[kind], k, m, n, k, n) and not lib.fits(KIND[kind], x_apart or k, m, n, k, y_apart or n)
    for kind, eb in (("2byte", 2), ("f32", 4)):  # the last row apart that fits, and the next
        most = ((2 ** 31 - 1) // 256 - 64) // eb
        assert lib.fits(KIND[kind], most, 40, 64, 64, 64) and not lib.fits(KIND[kind], most + 1, 40, 64, 64, 64)
        assert lib.fits(KIND[kind], 64, 40, 64, 64, 2 ** 21 - 1) and not lib.fits(KIND[kind], 64, 40, 64, 64, 2 ** 21)
    rows = (2 ** 31 - 1) // 4  # four scale bytes a row
    assert lib.fits(KIND["fp4"], 32, rows, 64, 32, 64) and not lib.fits(KIND["fp4"], 32, rows + 1, 64, 32, 64)
    assert lib.fits(KIND["f32"], 32, 40, rows, 32, 64) and not lib.fits(KIND["f32"], 32, 40, rows + 1, 32, 64)
