"""The build's guard against reads of a register too soon behind a write of half of it (phyai_amd/csrc/check_fused_asm.py)."""

from __future__ import annotations

import importlib.util
import os

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "phyai_amd", "csrc")


@pytest.fixture(scope="module")
def guard():
    spec = importlib.util.spec_from_file_location("check_fused_asm", os.path.join(CSRC, "check_fused_asm.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


SDWA = "v_max_u32_sdwa v7, v9, v8 dst_sel:WORD_1 dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:DWORD"
UPPER = "v_cvt_pk_fp8_f32 v7, v1, v2 op_sel:[0,0,1]"


@pytest.mark.parametrize("code,found", [
    (SDWA, "writes a part"),
    (SDWA + "|s_nop 7|v_div_scale_f32 v8, s[2:3], s4, s4, v7", "writes a part"),
    ("v_max_u32_sdwa v7, v9, v8 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:WORD_1 src1_sel:DWORD|v_mov_b32_e32 v1, v7", None),
    # a vector or matrix instruction one and two wait states later
    (UPPER + "|v_add_u32_e32 v3, v4, v7", "reads half"),
    (UPPER + "|v_mov_b32_e32 v3, v4|v_add_u32_e32 v3, v7, v4", "reads half"),
    (UPPER + "|s_nop 0|v_mfma_f32_16x16x128_f8f6f4 v[18:21], v[10:17], v[0:7], 0", "reads half"),
    (UPPER + "|s_nop 1|v_mfma_f32_16x16x128_f8f6f4 v[18:21], v[10:17], v[0:7], 0", None),
    (UPPER + "|v_mov_b32_e32 v3, v4|s_mov_b32 s1, s2|v_add_u32_e32 v3, v7, v4", None),
    # the register written anew, another one, the lower half, a store
    (UPPER + "|v_mov_b32_e32 v7, v4", None),
    (UPPER + "|v_add_u32_e32 v3, v8, v4", None),
    ("v_cvt_pk_fp8_f32 v7, v1, v2|v_cvt_pk_fp8_f32 v7, v3, v4 op_sel:[0,0,1]", None),
    (UPPER + "|ds_write_b64 v0, v[6:7]", None),
    # by way of a branch and round a loop
    (UPPER + "|s_branch L0|s_nop 7|<L0>:|v_add_u32_e32 v3, v7, v4", "reads half"),
    ("<L0>:|v_add_u32_e32 v3, v7, v4|" + UPPER + "|s_cbranch_scc0 L0", "reads half"),
    ("<L0>:|v_add_u32_e32 v3, v7, v4|" + UPPER + "|s_nop 0|s_cbranch_scc0 L0", None),
])
def test_planted_half_writes_are_caught(guard, code, found):
    text = "<_Zkernel>:\n" + "".join((t if t.startswith("<") else "\t" + t + "      // 00000000: 0") + "\n" for t in code.split("|")) + "\ts_endpgm   // 0\n"
    bad, functions, _ = guard.check_disassembly(text)
    assert functions == 1
    assert not bad if found is None else len(bad) == 1 and found in bad[0], bad


def test_no_kernel_of_the_library_has_one(guard):
    """Written against the library before its weight quantizers were mended: two kernels of it had the SDWA form, one wait state
    in front of the division that reads it."""
    library = os.path.join(guard.LIB, "libphyai_fp8.so")
    if not os.path.exists(library) or not os.path.exists(guard.OBJDUMP):
        pytest.skip("no built library or no disassembler here")
    bad = [p for text in guard.disassemble(library) for f in guard.functions_of(text) for p in guard.half_problems(f)]
    assert not bad, "\n".join(bad[:20])
