"""The check of 64-bit shifts by a vector register (rknpu2_matmul_open_amd/audit_waits.py): on pieces of disassembly, and on the built library."""
import os

import pytest

from rknpu2_matmul_open_amd import audit_waits, build


def _function(*lines, name="_Z6kernelv"):
    return "0000000000001000 <%s>:\n" % name + "".join("\t%s // 000000001000: 00000000\n" % line for line in lines) + "\ts_endpgm\n"


def _found(*lines):
    violations, functions = audit_waits.audit_shifts_text(_function(*lines))
    assert functions == 1
    return len(violations)


@pytest.mark.parametrize("shift", ["v_lshlrev_b64", "v_lshrrev_b64", "v_ashrrev_i64"])
def test_an_amount_in_the_last_register_of_a_block_is_found(shift):
    assert _found("v_mov_b32_e32 v103, v0", shift + " v[100:101], v103, v[100:101]") == 1
    assert _found("v_mov_b32_e32 v103, v0", shift + " v[100:101], v103, v[100:101]", "v_mov_b32_e32 v104, 0") == 0      # (the register behind is the wave's)
    assert _found("v_mov_b32_e32 v103, v0", shift + " v[100:101], v103, v[100:101]", "global_load_dwordx4 v[104:107], v[2:3], off") == 0
    assert _found(shift + " v[100:101], v102, v[100:101]") == 0                                                        # (so it is of a begun block)
    assert _found(shift + " v[100:101], s7, v[100:101]", "v_mov_b32_e32 v103, v0") == 0
    assert _found(shift + " v[102:103], 3, v[102:103]") == 0
    # ahead of accumulators, blocks are of four
    assert _found("v_mov_b32_e32 v99, v0", shift + " v[96:97], v99, v[96:97]") == 0
    assert _found("v_mov_b32_e32 v99, v0", shift + " v[96:97], v99, v[96:97]", "v_accvgpr_write_b32 a0, v1") == 1


def test_each_function_is_looked_at_by_itself():
    bad = _function("v_lshlrev_b64 v[4:5], v7, v[4:5]", name="_Z3badv")
    text = _function("v_mov_b32_e32 v200, 0", name="_Z5otherv") + bad + _function("v_add_f32_e32 v9, v8, v7", name="_Z4lastv")
    violations, functions = audit_waits.audit_shifts_text(text)
    assert functions == 3 and len(violations) == 1 and violations[0].startswith("_Z3badv: `v_lshlrev_b64 v[4:5], v7, v[4:5]`")


def test_the_built_library_has_none():
    if not os.path.exists(build.LIB) or not os.path.exists(os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")):
        pytest.skip("needs the built library and llvm-objdump")
    violations, functions = audit_waits.audit_shifts(build.LIB)
    assert functions > 400 and not violations, violations
