"""The build's check of saved registers: it finds a save where lanes may be off in a few lines of assembly that hold one, and nothing in the
assembly of the library as it was built."""
import os

import pytest

from quant_flash_attn_amd import build, save_check

TO_ACC, TO_SCRATCH = "v_accvgpr_write_b32 a5, v28", "scratch_store_dword off, v28, off offset:4"


def _found(tmp_path, *lines):
    out = ["_Zkernel:", *(line if line.endswith(":") else "\t" + line for line in lines), "\ts_endpgm", "\t\t.amdhsa_private_segment_fixed_size 0"]
    path = tmp_path / "k.s"
    path.write_text("\n".join(out) + "\n")
    return len(save_check.check(str(path)))


@pytest.mark.parametrize("save", [TO_ACC, TO_SCRATCH, "scratch_store_dwordx2 off, v[27:28], off", "scratch_store_dword off, a3, off"])
def test_a_save_where_a_branch_joins(tmp_path, save):
    """As it was found: at the join, in front of the instruction that turns the other lanes on."""
    branch = ["s_and_saveexec_b64 s[2:3], vcc", "s_cbranch_execz .LBB0_2", "v_mov_b32_e32 v1, 0", ".LBB0_2:"]
    assert _found(tmp_path, save) == 0
    assert _found(tmp_path, *branch, save, "s_or_b64 exec, exec, s[2:3]") == 1
    assert _found(tmp_path, *branch, "s_or_b64 exec, exec, s[2:3]", save) == 0
    assert _found(tmp_path, *branch[:2], save, *branch[2:], "s_or_b64 exec, exec, s[2:3]") == 1


def test_what_is_made_and_saved_under_one_mask(tmp_path):
    lines = ["s_and_saveexec_b64 s[2:3], vcc", "v_mov_b32_e32 v28, 1", TO_ACC, "s_or_b64 exec, exec, s[2:3]"]
    assert _found(tmp_path, *lines) == 0
    assert _found(tmp_path, lines[1], lines[0], *lines[2:]) == 1
    assert _found(tmp_path, lines[0], "s_cbranch_scc1 .LBB0_1", lines[1], ".LBB0_1:", *lines[2:]) == 1   # made on one of two paths


def test_masks_that_are_all_lanes(tmp_path):
    inside = ["s_and_saveexec_b64 s[4:5], vcc", "s_or_b64 exec, exec, s[4:5]"]
    off = "s_and_saveexec_b64 s[2:3], vcc"
    assert _found(tmp_path, off, *inside, "s_or_b64 exec, exec, s[2:3]", TO_ACC) == 0
    assert _found(tmp_path, off, *inside, TO_ACC) == 1                                                     # the inner branch alone has joined
    assert _found(tmp_path, off, "s_mov_b64 s[8:9], s[2:3]", "s_mov_b64 s[2:3], 0", "s_mov_b64 exec, s[8:9]", TO_ACC) == 0
    assert _found(tmp_path, off, "s_mov_b64 s[2:3], 0", "s_or_b64 exec, exec, s[2:3]", TO_ACC) == 1     # what it held is gone
    assert _found(tmp_path, off, "s_add_u32 s3, s6, s7", "s_or_b64 exec, exec, s[2:3]", TO_ACC) == 1
    spilled = ["v_writelane_b32 v90, s2, 4", "v_writelane_b32 v90, s3, 5", "s_mov_b64 s[2:3], 0", "v_readlane_b32 s6, v90, 4", "v_readlane_b32 s7, v90, 5"]
    assert _found(tmp_path, off, *spilled, "s_or_b64 exec, exec, s[6:7]", TO_ACC) == 0
    assert _found(tmp_path, off, *spilled[:-1], "v_readlane_b32 s7, v90, 4", "s_or_b64 exec, exec, s[6:7]", TO_ACC) == 1   # one half twice
    assert _found(tmp_path, "s_mov_b64 s[0:1], exec", "s_and_b64 s[2:3], s[0:1], vcc", "s_mov_b64 exec, s[2:3]", TO_ACC, "s_mov_b64 exec, s[0:1]", TO_ACC) == 1
    assert _found(tmp_path, "s_and_b64 exec, exec, vcc", TO_ACC, "s_mov_b64 exec, -1", TO_ACC) == 1


def test_paths_that_meet(tmp_path):
    """All lanes are on where they are on every path, and a loop that lanes leave one by one ends with some off."""
    assert _found(tmp_path, "s_cbranch_scc1 .LBB0_1", "s_and_b64 exec, exec, vcc", ".LBB0_1:", TO_ACC) == 1
    loop = [".LBB0_1:", "s_andn2_b64 exec, exec, s[6:7]", "s_cbranch_execnz .LBB0_1"]
    assert _found(tmp_path, "s_mov_b64 s[0:1], exec", *loop, TO_ACC, "s_mov_b64 exec, s[0:1]", TO_ACC) == 1
    assert _found(tmp_path, ".LBB0_1:", TO_ACC, "s_and_b64 exec, exec, vcc", "s_cbranch_execnz .LBB0_1") == 1   # on the second way round
    other = ["s_and_saveexec_b64 s[2:3], vcc", "s_xor_b64 s[2:3], exec, s[2:3]", "s_or_saveexec_b64 s[4:5], s[2:3]", TO_ACC]
    assert _found(tmp_path, *other) == 1   # not followed: counts as off


@pytest.mark.parametrize("src", build.NO_SPARE)
def test_the_library_as_built(src):
    asm = build.assembly_path(src)
    if not os.path.exists(asm):
        pytest.skip("the library's assembly is not there: it stays in the build folder of the machine that built it")
    assert save_check.check(asm) == []
    assert open(asm).read().count("_kernel") > 0
