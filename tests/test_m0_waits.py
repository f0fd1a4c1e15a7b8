"""The build check on the wait states of the direct global -> LDS loads (candle-3d_amd/check_m0.py, check_waits): one
between the scalar write of m0 and the load, five between a vector instruction's SGPR and the load, over every path. On
small assembly texts, and on the device assembly that the build wrote."""
import os
import re
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "candle-3d_amd")
sys.path.insert(0, PKG)
import check_m0  # noqa: E402


def asm(*ins):
    return "\t;;#ASMSTART\n" + "".join(f"\t{i}\n" for i in ins) + "\t;;#ASMEND\n"


LOAD = asm("s_mov_b32 m0, s8", "s_nop 0", "buffer_load_dwordx4 v146, s[0:3], s9 offen lds")


def write(tmp_path, body):
    p = tmp_path / "k.s"
    p.write_text("_Z6kernelv:                              ; @_Z6kernelv\n" + body + "\ts_endpgm\n")
    return str(p)


def test_loads_with_their_waits_pass(tmp_path):
    p = write(tmp_path, LOAD + "\tv_mov_b32 v0, 0\n" + LOAD.replace("dwordx4", "dword"))
    assert check_m0.check_waits(p) == [] and check_m0.check(p) == ([], 1, 2)
    assert check_m0.main(["check_m0.py", p]) == 0


def test_a_load_right_behind_its_m0_fails_the_build(tmp_path):
    p = write(tmp_path, LOAD + asm("s_mov_b32 m0, s8", "buffer_load_dwordx4 v146, s[0:3], s9 offen lds"))
    bad = check_m0.check_waits(p)
    assert len(bad) == 1 and "0 wait states between m0" in bad[0]
    assert check_m0.main(["check_m0.py", p]) == 1


@pytest.mark.parametrize("name", ["s9", "s2"])
@pytest.mark.parametrize("between,ok", [("", False), ("\tv_mov_b32 v0, 0\n", False), ("\ts_nop 1\n", False),
                                        ("\ts_nop 2\n", True), ("\tv_mov_b32 v0, 0\n" * 3, True),
                                        (".LBB0_1:\n\tv_mov_b32 v0, 0\n", False)])
def test_vector_writes_of_the_loads_sgprs(tmp_path, name, between, ok):
    """The block's own s_mov and s_nop are two of the five wait states."""
    bad = check_m0.check_waits(write(tmp_path, f"\tv_readfirstlane_b32 {name}, v4\n" + between + LOAD))
    assert (bad == []) == ok and all("a vector instruction's SGPR" in b for b in bad)


@pytest.mark.parametrize("ins,ok", [("s_mov_b32 s9, s20", True), ("v_cmp_gt_i32_e64 s[2:3], v0, v1", False),
                                    ("v_add_co_u32_e64 v3, s[0:1], v0, v1", False), ("v_readfirstlane_b32 s8, v4", True),
                                    ("v_cmp_gt_i32_e64 s[4:5], v0, s9", True)])
def test_which_writes_count(tmp_path, ins, ok):
    assert (check_m0.check_waits(write(tmp_path, f"\t{ins}\n" + LOAD)) == []) == ok


def test_writes_on_another_path(tmp_path):
    """A loop's back edge and a branch around the wait lead to the load, too."""
    loop = ".LBB0_1:\n" + LOAD + "\tv_mov_b32 v0, 0\n\tv_readlane_b32 s3, v1, 2\n\ts_cbranch_scc1 .LBB0_1\n"
    assert check_m0.check_waits(write(tmp_path, loop))
    body = "\tv_readlane_b32 s3, v1, 2\n\ts_cbranch_vccz .LBB0_2\n\ts_nop 4\n.LBB0_2:\n" + LOAD
    assert check_m0.check_waits(write(tmp_path, body))
    body = "\tv_readlane_b32 s3, v1, 2\n\ts_branch .LBB0_2\n\ts_nop 4\n.LBB0_2:\n\ts_mov_b32 s3, 0\n" + LOAD
    assert check_m0.check_waits(write(tmp_path, body)) == []


def test_the_built_assembly_has_every_wait():
    mk = open(os.path.join(PKG, "Makefile")).read()
    srcs = re.search(r"^M0_SRCS\s*=\s*(.*)$", mk, flags=re.M).group(1).split()
    paths = [os.path.join(PKG, "_build", os.path.basename(s)[:-4] + ".s") for s in srcs]
    if not all(os.path.exists(p) for p in paths):
        pytest.skip("no build here (the device assembly is written by make)")
    for p in paths:
        assert check_m0.check_waits(p) == []
        text = open(p).read()
        assert len(re.findall(r"s_mov_b32 m0, s\d+\n\ts_nop 0\n\tbuffer_load_dword(?:x4)? .* offen lds", text)) == \
            check_m0.check(p)[2] > 0
