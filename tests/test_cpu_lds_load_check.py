"""The static check of loads into LDS (qtpytorch_amd/csrc/check_lds_loads.py) on
synthetic assembly with planted mistakes, and on the source whose loads are inline
assembly."""
import os
import shutil

import pytest

from qtpytorch_amd.csrc import check_lds_loads as ck

LOAD = "\tbuffer_load_dwordx4 v1, s[4:7], 0 offen lds\n"


def run(body):
    n, problems = ck.check_asm("_Z4kernv:\n" + body + "\ts_endpgm\n.Lfunc_end0:\n")
    assert n == body.count(" lds\n")
    return problems


def test_m0_needs_one_state():
    assert len(run("\t;;#ASMSTART\n\ts_mov_b32 m0, s2\n" + LOAD + "\t;;#ASMEND\n")) == 1
    assert run("\ts_mov_b32 m0, s2\n\ts_nop 0\n" + LOAD) == []
    assert run("\ts_mov_b32 m0, s2\n\tv_add_u32_e32 v1, v1, v2\n" + LOAD) == []


def test_a_scalar_that_a_vector_instruction_wrote_needs_five():
    write = "\tv_readfirstlane_b32 s5, v9\n"
    m0 = "\ts_mov_b32 m0, s2\n\ts_nop 0\n"  # two of them
    assert len(run(write + m0 + LOAD)) == 1
    assert len(run(write + "\ts_nop 1\n" + m0 + LOAD)) == 1
    assert run(write + "\ts_nop 2\n" + m0 + LOAD) == []
    assert run(write.replace("s5", "s8") + m0 + LOAD) == []
    assert len(run("\tv_cmp_eq_u32_e64 s[6:7], v1, v2\n" + m0 + LOAD)) == 2
    assert len(run("\tv_add_co_u32 v3, s[4:5], v1, v2\n" + m0 + LOAD)) == 2
    assert run(write + "\ts_mov_b32 s5, s9\n" + m0 + LOAD) == []  # written again by a scalar instruction


def test_paths_across_blocks():
    late = "\ts_mov_b32 m0, s2\n\ts_cbranch_scc1 .LBB0_1\n\ts_nop 4\n.LBB0_1:\n" + LOAD
    assert run(late) == []  # the branch is one state
    loop = ".LBB0_1:\n" + LOAD + "\tv_readfirstlane_b32 s6, v9\n\ts_cbranch_scc1 .LBB0_1\n"
    assert len(run(loop)) == 1
    assert run(loop.replace("\ts_cbranch", "\ts_nop 3\n\ts_cbranch")) == []
    assert run("\tv_readfirstlane_b32 s6, v9\n\ts_branch .LBB0_2\n.LBB0_1:\n" + LOAD + ".LBB0_2:\n") == []


def test_loads_into_registers_are_not_meant():
    assert run("\ts_mov_b32 m0, s2\n\tbuffer_load_dwordx4 v[0:3], v1, s[4:7], 0 offen\n") == []


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="needs hipcc")
def test_source_passes():
    from qtpytorch_amd.csrc import build as b

    n, problems = ck.check_source(os.path.join(os.path.dirname(ck.__file__), "mxk_mxfp4_gemm.hip"), b.hipcc(),
                                  b.HIPCC_FLAGS)
    assert n > 500
    assert problems == []
