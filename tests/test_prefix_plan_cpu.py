"""How lux3d_sdpa_shared_prefix cuts its work (csrc/prefix_plan.hpp, compiled here): every row meets every key block once,
no workgroup is without work, the parts have the workspace that is asked for."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "candle-3d_amd", "csrc")
NAMES = ("joint", "ks", "tile", "own_tile", "prefix_tiles", "prefix_run", "prefix_runs", "own_tiles", "own_run", "own_runs",
         "parts", "wgs", "values")


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    out = tmp_path_factory.mktemp("prefix_plan")
    src, lib = out / "plan.cpp", out / "plan.so"
    src.write_text('#include "prefix_plan.hpp"\n'
                   'extern "C" void plan(const int64_t *a, int64_t *r) {\n'
                   '  const auto s = lux3d::prefix_plan(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7] != 0);\n'
                   '  const int64_t v[] = {s.joint, s.ks, s.tile, s.own_tile, s.prefix_tiles, s.prefix_run, s.prefix_runs,\n'
                   '                       s.own_tiles, s.own_run, s.own_runs, s.parts, s.wgs,\n'
                   '                       lux3d::prefix_workspace(s, a[0], a[1], a[3], a[6])};\n'
                   '  for (int i = 0; i < 13; ++i) r[i] = v[i];\n'
                   '}\n')
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", CSRC, "-o", str(lib), str(src)], check=True)
    fn = ctypes.CDLL(str(lib)).plan

    def get(*a):
        args, r = (ctypes.c_int64 * 8)(*a), (ctypes.c_int64 * 13)()
        fn(args, r)
        return dict(zip(NAMES, r))
    return get


def blocks(n):
    return (n + 63) // 64


def runs_cover(run, runs, n):
    """`runs` runs of `run` blocks are all n of them, none empty."""
    assert run >= 1 and runs * run >= n and (runs == 0 or (runs - 1) * run < max(n, 1)), (run, runs, n)


def check(plan, b, h, hkv, n, p, ls, d, f32):
    s = plan(b, h, hkv, n, p, ls, d, int(f32))
    rows, what = n * (h // hkv), (b, h, hkv, n, p, ls, d, f32, s)
    if s["joint"]:
        assert s["tile"] * s["ks"] == 128 and not (f32 and s["ks"] > 1), what
        assert s["own_tiles"] * s["tile"] >= rows > (s["own_tiles"] - 1) * s["tile"], what
        runs_cover(s["own_run"], s["own_runs"], blocks(p) + blocks(ls))
        assert s["parts"] == s["own_runs"] >= 1, what
        assert s["wgs"] == b * hkv * s["own_tiles"] * s["own_runs"], what
    else:
        assert s["tile"] == 128 and s["own_tile"] == (128 if f32 else 64), what
        assert s["prefix_tiles"] * 128 >= b * rows > (s["prefix_tiles"] - 1) * 128, what
        assert s["own_tiles"] * s["own_tile"] >= rows > (s["own_tiles"] - 1) * s["own_tile"], what
        runs_cover(s["prefix_run"], s["prefix_runs"], blocks(p))
        assert (s["prefix_runs"] == 0) == (p == 0), what
        if p == 0 and ls == 0:  # one item a row tile still writes the zeros
            assert s["own_runs"] == 1, what
        else:
            runs_cover(s["own_run"], s["own_runs"], blocks(ls))
            assert (s["own_runs"] == 0) == (ls == 0), what
        assert s["parts"] == s["prefix_runs"] + s["own_runs"] >= 1, what
        assert s["wgs"] == hkv * (s["prefix_tiles"] * s["prefix_runs"] + b * s["own_tiles"] * s["own_runs"]), what
    assert s["values"] == (s["parts"] * b * h * n * (d + 2) if s["parts"] > 1 else 0), what
    # the number of a part is part of its place in the workspace, and a workgroup's is 32-bit
    assert s["wgs"] < 2 ** 31, what
    return s


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_small_and_edge_sizes(plan, d, f32):
    for b in (1, 2, 9):
        for h, hkv in ((1, 1), (8, 2), (16, 16)):
            for n in (1, 2, 31, 32, 33, 64, 127, 128, 129, 700):
                for p in (0, 1, 63, 64, 65, 1029, 20000):
                    for ls in (0, 1, 64, 65, 999):
                        check(plan, b, h, hkv, n, p, ls, d, f32)


def test_drawn_sizes(plan):
    r = random.Random(5)
    kinds = set()
    for _ in range(20000):
        g, hkv = r.choice([1, 2, 4, 8]), r.choice([1, 2, 4, 8, 16])
        n = int(2 ** r.uniform(0, 13))
        s = check(plan, r.randint(1, 128), g * hkv, hkv, n, r.choice([0, int(2 ** r.uniform(0, 20))]),
                  r.choice([0, int(2 ** r.uniform(0, 15))]), r.choice([64, 128]), r.random() < 0.3)
        kinds.add((s["joint"], s["ks"], s["parts"] > 1))
    assert kinds == {(1, 1, False), (1, 1, True), (1, 2, False), (1, 2, True), (0, 1, False), (0, 1, True)}
