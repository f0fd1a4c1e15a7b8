"""The GPU tests of the shared-prefix attention's merge reach each of its forms (csrc/prefix_plan.hpp, compiled here)."""
import ctypes
import os
import subprocess

import pytest

pytest.importorskip("torch")

import test_gpu_prefix_merge as cases  # noqa: E402
from test_prefix_plan_cpu import CSRC, plan  # noqa: E402, F401 (fixture)


@pytest.fixture(scope="module")
def groups(tmp_path_factory):
    out = tmp_path_factory.mktemp("prefix_merge")
    src, lib = out / "merge.cpp", out / "merge.so"
    src.write_text('#include "prefix_plan.hpp"\n'
                   'extern "C" int groups(int64_t parts, int64_t rows) { return lux3d::prefix_merge_groups(parts, rows); }\n')
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", CSRC, "-o", str(lib), str(src)], check=True)
    fn = ctypes.CDLL(str(lib)).groups
    fn.argtypes = [ctypes.c_int64] * 2
    return fn


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
def test_sizes_reach_each_form(plan, groups, d, f32):  # noqa: F811
    def form(case):
        b, h, hkv, n, p, ls, _ = case
        parts = plan(b, h, hkv, n, p, ls, d, f32)["parts"]
        assert parts > 1, case
        return groups(parts, b * h * n)
    assert {form(c) for c in cases.MANY} == {0}
    assert {form(c) for c in cases.SOME} == {4}
    assert {form(c) for c in cases.FEW} == {1}
    # the prefix alone: in one run, and in several
    alone = {plan(*c[:6], d, f32)["parts"] > 1 for c in cases.ALONE}
    assert alone == {False, True}


def test_rule(groups):
    assert [groups(*a) for a in ((2, 4095), (2, 4096), (8, 4096), (9, 4096), (32, 10 ** 6), (33, 1), (33, 10 ** 6))] == \
        [4, 1, 1, 4, 4, 0, 0]
