"""The kernel and tile that each size of the 4-bit linears' GPU tile tests takes: the dispatch's own choice
(csrc/mxfp4_tiles.hpp, compiled here), so that a change of its costs cannot leave a tile untested."""
import ctypes
import itertools
import os
import subprocess

import pytest

import test_gpu_mxfp4_tiles as gpu

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "candle-3d_amd", "csrc")
KIND = {"fp4": 0, "2byte": 1, "f32": 2}


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("mxfp4_tiles")
    src, so = out / "tiles.cpp", out / "tiles.so"
    src.write_text('#include "mxfp4_tiles.hpp"\n'
                   'using namespace lux3d;\n'
                   'extern "C" void choose(int kind, int64_t m, int64_t n, int64_t k, int gated, int64_t *o) {\n'
                   '  const MxChoice c = mx_choose((MxKind)kind, m, n, k, gated);\n'
                   '  o[0] = c.tile.rows, o[1] = c.tile.cols, o[2] = c.tile.groups, o[3] = c.rows;\n}\n'
                   'extern "C" int few_tiles(int two, int64_t n, int64_t k, int gated) { return mx_few_tiles(two, n, k, gated); }\n')
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-shared", "-fPIC", "-I", CSRC, "-o", str(so), str(src)], check=True)
    dll = ctypes.CDLL(str(so))
    dll.choose.argtypes = [ctypes.c_int] + [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.c_void_p]
    dll.few_tiles.argtypes = [ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
    return dll


def choose(lib, kind, gated, m, k, n):
    o = (ctypes.c_int64 * 4)()
    lib.choose(KIND[kind], m, n, k, int(gated), o)
    return tuple(o)


def test_tile_tests_reach_the_tiles_they_name(lib):
    for kind, gated, rows, cols, groups, split, m, k, n in gpu.TILES:
        r, c, g, below = choose(lib, kind, gated, m, k, n)
        assert (r, c, g, below != m) == (rows, cols, groups, split) and below > 0, (kind, gated, m, k, n, r, c, g, below)
    for gated, m, k, n in gpu.STAY:
        r, c, g, below = choose(lib, "fp4", gated, m, k, n)
        assert (r, c) == (256, 256) and -(-below // 256) * -(-n // (128 if gated else 256)) > 256, (gated, m, k, n, r, c, below)
    for kind, gated, m, k, n in [("f32" if t[0] == "f32" else "2byte", False, *t[1:]) for t in gpu.PLAIN_REST] + [("fp4", *t) for t in gpu.PACKED_REST]:
        assert 0 < choose(lib, kind, gated, m, k, n)[3] < m, (kind, gated, m, k, n)
    for tiles, two, gated, n, k in gpu.WIDE:
        assert lib.few_tiles(int(two), n, k, int(gated)) == tiles, (tiles, two, gated, n, k)


def test_every_choice_is_named(lib):
    """Over the whole range no tile comes up that the GPU tests do not name, and what a tile leaves over is a few rows."""
    named = {t[:6] for t in gpu.TILES}
    sizes = [17, 31, 33, 64, 65, 100, 129, 250, 257, 400, 515, 777, 1029, 1500, 2049, 2500, 4098, 6000, 9001, 16392, 40000]
    for kind, gated, m, k, n in itertools.product(KIND, (False, True), sizes, [32, 64, 96, 128, 352, 384, 416, 512, 1024, 1536, 2048, 4096, 8192],
                                                  [1, 17, 64, 130, 300, 777, 1536, 2048, 3001, 4096, 8192, 9216, 20000]):
        r, c, g, below = choose(lib, kind, gated, m, k, n)
        if below == 0:
            assert (r, c) == (16, 16)
            continue
        assert (kind, gated, r, c, g, below != m) in named, (kind, gated, m, k, n, r, c, g, below)
        assert below == m or (below % r == 0 and 1 <= m - below <= 16)
        assert not (kind == "fp4" and r == 256 and k < 512)


def test_few_rows_take_no_tile(lib):
    for kind, gated, m, k, n in itertools.product(KIND, (False, True), range(1, 17), (32, 1024, 8192), (1, 4096, 32000)):
        assert choose(lib, kind, gated, m, k, n)[3] == 0


def test_sizes_at_the_ends(lib):
    """The largest numbers of rows and columns leave costs finite and a choice."""
    for kind, gated in itertools.product(KIND, (False, True)):
        for m, k, n in ((2 ** 31, 32, 1), (2 ** 24, 8192, 2 ** 24), (17, 2 ** 20, 2 ** 20)):
            r, c, g, below = choose(lib, kind, gated, m, k, n)
            assert 0 <= below <= m and r > 0
