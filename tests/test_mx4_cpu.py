"""The MX4 boundary without a GPU: the header, the exports and their bindings, refusals that come ahead of any device work, and what
the dispatch decides, which is arithmetic."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

from rknpu2_matmul_open_amd import capi
from tests import mx4_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INC = os.path.join(ROOT, "include")


@pytest.fixture(scope="module")
def lib():
    return capi.load_library()


def test_header_compiles_as_c99(tmp_path):
    src = tmp_path / "h.c"
    src.write_text('#include "rk_npu_mx4.h"\nint main(void) { return 0; }\n')
    subprocess.check_call(["gcc", "-std=c99", "-pedantic", "-Wall", "-Werror", "-I", INC, "-c", str(src), "-o", str(tmp_path / "o.o")])


def test_library_exports_what_the_header_declares(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(INC, "rk_npu_mx4.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(rk_npu_[a-z0-9_]+)\s*\(", text))
    assert len(declared) >= 15
    assert all(hasattr(lib, n) for n in declared)
    assert set(capi.MX4_SYMBOLS) == declared


def test_struct_layouts_match_the_c_compiler(tmp_path):
    lines, want = [], []
    for name, cls in (("rk_npu_mx4_weight_config", capi.MX4WeightConfig), ("rk_npu_block_norm_args", capi.BlockNormArgs)):
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        want.append(C.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (name, field))
            want.append(getattr(cls, field).offset)
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "rk_npu_mx4.h"\nint main(void) { %s return 0; }\n' % " ".join(lines))
    subprocess.check_call(["gcc", "-I", INC, str(src), "-o", str(tmp_path / "s")])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert got == want


def test_refusals_without_a_context(lib):
    some = C.c_void_p(4096)
    bad = capi.RK_NPU_ERR_PARAM
    assert lib.rk_npu_mx4_quantize_device(None, 0, 1, 32, some, 32, some, some) == bad
    assert lib.rk_npu_mx4_dequantize_device(None, 0, 1, 32, some, some, some, 32) == bad
    assert lib.rk_npu_mx4_run_device(None, None, 1, 0, some, 32, 0, some, 32) == bad
    assert lib.rk_npu_mx4_run_swiglu_device(None, None, 1, 0, some, 32, 0, some, 32) == bad
    assert lib.rk_npu_mx4_stage_device(None, 1, 0, some, 32) == bad
    assert lib.rk_npu_mx4_run_staged_device(None, None, 0, some, 32) == bad
    assert lib.rk_npu_mx4_run_ffn_device(None, None, None, None, 1, 0, some, 32, 0, some, 32) == bad
    args = capi.BlockNormArgs()
    lib.rk_npu_block_norm_args_init(C.byref(args), 3, 64)
    assert (args.struct_size, args.rows, args.D) == (C.sizeof(args), 3, 64)
    assert (args.residual_scale, args.branch_scale) == (1.0, 1.0) and abs(args.eps - 1e-6) < 1e-12
    assert lib.rk_npu_block_norm_device(None, C.byref(args)) == bad
    assert lib.rk_npu_mx4_run_ffn_block_device(None, None, None, None, C.byref(args), some, None) == bad
    assert lib.rk_npu_mx4_weights_query(None, None, None) == bad
    config = capi.MX4WeightConfig(32, 32, 0)
    assert not lib.rk_npu_mx4_weights_create(None, C.byref(config), some, some)
    assert not lib.rk_npu_mx4_workspace_create(None, 1, 32, 32)
    lib.rk_npu_mx4_weights_free(None)
    lib.rk_npu_mx4_workspace_free(None)


def _route(lib, M, N, K, swiglu):
    out = [C.c_int(0) for _ in range(4)]
    lib.rkh_mx4_route(M, N, K, swiglu, *[C.byref(x) for x in out])
    return [x.value for x in out]


@pytest.mark.parametrize("swiglu", [0, 1])
def test_route_covers_every_row_and_column_and_its_scratch_is_what_the_parts_need(lib, swiglu):
    lib.rkh_mx4_scratch_bytes.restype = lib.rkh_mx4_scratch_most.restype = C.c_size_t
    rng = np.random.default_rng(3)
    for _ in range(3000):
        M, N, K = (int(np.exp(rng.uniform(0, np.log(top)))) for top in (9000, 40000, 40000))
        kernel, rows, columns, parts = _route(lib, M, N, K, swiglu)
        assert rows > 0 and columns % 16 == 0 and 1 <= parts <= max(1, -(-K // 512)), (M, N, K)
        if kernel == 0:
            assert M <= rows and parts == 1
        else:
            assert rows % 32 == 0 and columns % 32 == 0
            assert not swiglu or columns % 128 == 0 # whole gate / up pairs in each wave
        places = 2 * (-(-N // 32) * 32) if swiglu else -(-N // 32) * 32
        tiles = -(-M // rows) * -(-places // columns)
        want = tiles * parts * rows * columns * 4 if parts > 1 else 0
        assert lib.rkh_mx4_scratch_bytes(M, N, K, swiglu) == want, (M, N, K)
        assert want <= lib.rkh_mx4_scratch_most(M, K), (M, N, K)


def test_reference_of_the_format():
    """The oracle itself: its codes are what the definition says at every border between two values and beside it."""
    borders = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    down = [0, 1, 1, 2, 2, 4, 4]    # ties: 0 | 0.5 -> 0, 0.5 | 1 -> 1, 1 | 1.5 -> 1, 1.5 | 2 -> 2, 2 | 3 -> 2, 3 | 4 -> 4, 4 | 6 -> 4
    x = np.zeros((1, 32))
    x[0, 0] = 4.0                   # scale 1
    x[0, 1:8] = borders
    x[0, 8:15] = np.nextafter(borders, 10)
    x[0, 15:22] = np.nextafter(borders, 0)
    got = ref.round_trip(x)[0]
    assert list(got[1:8]) == down
    assert list(got[8:15]) == [0.5, 1, 1.5, 2, 3, 4, 6]
    assert list(got[15:22]) == [0, 0.5, 1, 1.5, 2, 3, 4]
    assert ref.quantize(np.full((1, 32), 7.99))[1][0, 0] == 127 and ref.round_trip(np.full((1, 32), 7.99))[0, 0] == 6
    codes, scales = ref.exact_rows(np.random.default_rng(1), 5, 70)
    again = ref.quantize(ref.values(codes, scales, 70))
    live = ref.values(codes, scales, 96).reshape(5, 96)
    assert np.array_equal(again[1], scales) and np.array_equal(ref.values(*again, 96), live)


def test_audit_sees_sums_in_accumulation_registers():
    """A product from asm whose sum is moved before it is through is reported, in either half of the registers."""
    from rknpu2_matmul_open_amd import audit_waits

    def kernel(behind):
        return "\n".join(["_Z14mx4_big_kernelv:", "\tv_mov_b32_e32 v1, 0", ";;#ASMSTART",
                          "\tv_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[8:11], v[12:15], a[4:7], v20, v21 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4",
                          ";;#ASMEND"] + behind + ["\ts_endpgm", ".Lfunc_end0:"])
    move = "\tv_accvgpr_read_b32 v30, a5"
    assert len(audit_waits.audit_text(kernel([move]))[0]) == 1
    assert len(audit_waits.audit_text(kernel(["\ts_nop 7", move]))[0]) == 1
    assert audit_waits.audit_text(kernel(["\ts_nop 7", "\ts_nop 7", move])) == ([], 1)
    assert audit_waits.audit_text(kernel(["\tv_accvgpr_read_b32 v30, a8"])) == ([], 1)


def test_wrappers_refuse_host_tensors_and_odd_layouts():
    import torch

    from rknpu2_matmul_open_amd import ops
    with pytest.raises(ValueError):
        ops._mx4_rows(torch.zeros(4, 32))
    with pytest.raises(ValueError):
        ops._channel(torch.zeros(32), 32, "weight")

    class OnDevice:  # (what the wrappers look at)
        def __init__(self, t):
            self.t, self.dtype, self.shape, self.is_cuda = t, t.dtype, t.shape, True
            self.stride, self.data_ptr = t.stride, t.data_ptr
    kind, _, ld = ops._mx4_rows(OnDevice(torch.zeros(4, 40, dtype=torch.bfloat16)[:, :32]))
    assert (kind, ld) == (capi.MX4_BF16, 40)
    assert ops._mx4_rows(OnDevice(torch.zeros(1, 32)))[2] == 32
    for bad in (torch.zeros(4, 32).t(), torch.zeros(32), torch.zeros(4, 64)[:, ::2]):
        with pytest.raises(ValueError):
            ops._mx4_rows(OnDevice(bad))
    with pytest.raises(TypeError):
        ops._mx4_rows(OnDevice(torch.zeros(4, 32, dtype=torch.float64)))


def test_wrappers_refuse_short_weights_and_results_of_other_rows_than_the_staged():
    import torch

    from rknpu2_matmul_open_amd import ops

    class Session:  # (nothing is called before the checks)
        lib = domain = None
    for codes, scales in ((np.zeros((4, 31), np.uint8), np.zeros((4, 2), np.uint8)), (np.zeros((4, 32), np.uint8), np.zeros((4, 1), np.uint8)),
                          (np.zeros((4, 32), np.int8), np.zeros((4, 2), np.uint8)), (np.zeros((4, 64), np.uint8)[:, ::2], np.zeros((4, 2), np.uint8))):
        with pytest.raises(ValueError):
            ops.MX4Weights(Session, 40, 4, codes, scales)
    ws = ops.MX4Workspace.__new__(ops.MX4Workspace)
    ws.K, ws.staged = 40, 5

    class Weights:
        N, gate_up = 64, False

    class Out:
        def __init__(self, t):
            self.dtype, self.shape, self.is_cuda, self.stride, self.data_ptr = t.dtype, t.shape, True, t.stride, t.data_ptr
    for rows in (4, 6, 0):
        with pytest.raises(ValueError):
            ws.run_staged(Weights, Out(torch.zeros(rows, 64)))
