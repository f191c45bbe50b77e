"""The boundary of G4 layers and of the heads' norm and rotation without a GPU: headers, exports and bindings, refusals ahead of any device work,
and what the dispatch decides, which is arithmetic."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

from rknpu2_matmul_open_amd import audit_waits, capi
from tests import g4_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INC = os.path.join(ROOT, "include")
HEADERS = ("rk_npu_g4.h", "rk_npu_heads.h")


@pytest.fixture(scope="module")
def lib():
    return capi.load_library()


@pytest.mark.parametrize("header", HEADERS)
def test_headers_compile_as_c99(tmp_path, header):
    src = tmp_path / "h.c"
    src.write_text('#include "%s"\nint main(void) { return 0; }\n' % header)
    subprocess.check_call(["gcc", "-std=c99", "-pedantic", "-Wall", "-Werror", "-I", INC, "-c", str(src), "-o", str(tmp_path / "o.o")])


def test_library_exports_what_the_headers_declare(lib):
    declared = set()
    for header in HEADERS:
        text = re.sub(r"/\*.*?\*/", "", open(os.path.join(INC, header)).read(), flags=re.S)
        declared |= set(re.findall(r"\b(rk_npu_[a-z0-9_]+)\s*\(", text))
    assert len(declared) >= 10
    assert all(hasattr(lib, n) for n in declared)
    assert set(capi.G4_SYMBOLS) == declared


def test_struct_layouts_match_the_c_compiler(tmp_path):
    lines, want = [], []
    for name, cls in (("rk_npu_g4_weight_config", capi.G4WeightConfig), ("rk_npu_heads_args", capi.HeadsArgs)):
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        want.append(C.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (name, field))
            want.append(getattr(cls, field).offset)
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "rk_npu_g4.h"\n#include "rk_npu_heads.h"\nint main(void) { %s return 0; }\n' % " ".join(lines))
    subprocess.check_call(["gcc", "-I", INC, str(src), "-o", str(tmp_path / "s")])
    assert [int(x) for x in subprocess.check_output([str(tmp_path / "s")]).split()] == want


def test_refusals_without_a_context(lib):
    some, bad = C.c_void_p(4096), capi.RK_NPU_ERR_PARAM
    assert lib.rk_npu_g4_run_device(None, None, 1, 1, some, 32, 0, some, 32) == bad
    assert lib.rk_npu_g4_run_swiglu_device(None, None, 1, 1, some, 32, 0, some, 32) == bad
    assert lib.rk_npu_g4_weights_query(None, None, None) == bad
    config = capi.G4WeightConfig(32, 32, 32, 0, capi.MX4_F16)
    assert not lib.rk_npu_g4_weights_create(None, C.byref(config), some, some, None)
    assert not lib.rk_npu_g4_weights_create_device(None, C.byref(config), some, some, None)
    assert not lib.rk_npu_g4_workspace_create(None, 1, 32, 32)
    lib.rk_npu_g4_weights_free(None)
    lib.rk_npu_g4_workspace_free(None)
    a = capi.HeadsArgs()
    lib.rk_npu_heads_args_init(C.byref(a), 3, 64)
    assert (a.struct_size, a.rows, a.head_dim, a.rotary_dim, a.norm, a.axes, a.rotation_scale) == (C.sizeof(a), 3, 64, 64, 1, 1, 1.0) and abs(a.eps - 1e-6) < 1e-12
    assert lib.rk_npu_heads_norm_rotate_device(None, C.byref(a)) == bad
    lib.rk_npu_heads_args_init(None, 3, 64)


def _route(lib, M, N, K, gpb, swiglu):
    out = [C.c_int(0) for _ in range(4)]
    lib.rkh_g4_route(M, N, K, gpb, swiglu, *[C.byref(x) for x in out])
    return [x.value for x in out]


@pytest.mark.parametrize("swiglu", [0, 1])
def test_route_covers_every_row_and_column_and_its_scratch_is_what_the_parts_need(lib, swiglu):
    lib.rkh_g4_scratch_bytes.restype = lib.rkh_g4_scratch_most.restype = C.c_size_t
    rng = np.random.default_rng(3)
    seen = set()
    for _ in range(4000):
        M, N, K = (int(np.exp(rng.uniform(0, np.log(top)))) for top in (9000, 40000, 40000))
        gpb = int(rng.choice([1, 2, 4]))
        kernel, rows, columns, parts = _route(lib, M, N, K, gpb, swiglu)
        places = 2 * (-(-N // 32) * 32) if swiglu else -(-N // 64) * 64
        seen.add((kernel, rows, parts > 1))
        assert rows > 0 and 1 <= parts <= max(1, -(-K // 128) // 2), (M, N, K)
        if kernel == 0:
            assert M <= 16 == rows and parts == 1 and places % columns == 0 and (not swiglu or columns % 32 == 0)
            assert lib.rkh_g4_scratch_bytes(M, N, K, gpb, swiglu) == 0
            continue
        assert M > 16 and rows in (32, 64, 128, 256) and columns == 128
        tiles = -(-M // rows) * -(-places // columns)
        want = tiles * parts * rows * columns * 4 if parts > 1 else 0
        assert lib.rkh_g4_scratch_bytes(M, N, K, gpb, swiglu) == want, (M, N, K)
        # what a workspace of as many rows has, and one of more
        assert want <= lib.rkh_g4_scratch_most(M, K) <= lib.rkh_g4_scratch_most(M + 5, K), (M, N, K)
    assert {(0, 16, False), (1, 32, False), (1, 32, True), (1, 64, False), (1, 64, True), (1, 128, True), (1, 256, False), (1, 256, True)} <= seen, seen


def test_the_shapes_that_are_tested_take_every_kernel(lib):
    def reached(shapes, swiglu):
        out = set()
        for M, N, K, group in shapes:
            kernel, rows, columns, parts = _route(lib, M, N, K, {0: 1, 64: 2}.get(group % 128, 4), swiglu)
            out.add((rows, parts > 1) if kernel else (columns, min(M, 5) if columns > 16 else 0))
        return out
    tiles = {(rows, False) for rows in (32, 64, 128, 256)}
    assert tiles | {(32, True), (64, True), (16, 0), (32, 4), (64, 5)} <= reached(ref.SHAPES, 0)
    assert tiles | {(32, True), (64, True), (32, 1), (32, 4), (64, 5)} <= reached(ref.SWIGLU, 1)


def test_audit_counts_a_product_in_between_for_its_passes():
    def kernel(behind):
        return "\n".join(["_Z14g4_tile_kernelv:", "\tv_mov_b32_e32 v1, 0", ";;#ASMSTART", "\tv_mfma_f32_32x32x16_f16 v[32:47], a[8:11], v[12:15], v[32:47]", ";;#ASMEND"] +
                         behind + ["\ts_endpgm", ".Lfunc_end0:"])
    other, read = "\tv_mfma_f32_32x32x16_f16 v[64:79], a[8:11], v[12:15], 0", "\tv_fmac_f32_e32 v100, v33, v101"
    assert len(audit_waits.audit_text(kernel([read]))[0]) == 1
    assert len(audit_waits.audit_text(kernel([other, read]))[0]) == 1
    assert audit_waits.audit_text(kernel([other, other, read])) == ([], 1)
    assert len(audit_waits.audit_text(kernel([other.replace("32x32x16", "16x16x32"), other, read]))[0]) == 1


def test_reference_of_the_format():
    """The oracle itself, on a matrix written out."""
    code = np.array([[0, 15, 8, 9], [1, 2, 3, 4]])
    assert ref.pack(code).tolist() == [[0xf0, 0x98], [0x21, 0x43]]
    assert ref.pack(code[:, :3]).tolist() == [[0xf0, 0x08], [0x21, 0x03]]
    scales, zeros = np.array([[0.5, 2.0], [1.0, 4.0]]), np.array([[1, 9], [0, 255]])
    assert ref.weights(code, scales, None, 2).tolist() == [[-4, 3.5, 0, 2], [-7, -6, -20, -16]]
    assert ref.weights(code, scales, zeros, 2).tolist() == [[-0.5, 7, -2, 0], [1, 2, -1008, -1004]]
    x = np.arange(1.0, 7.0).reshape(1, 1, 6)
    assert np.allclose(ref.rotate(x, np.array([[1]]), [np.pi / 2, np.pi], [0, 0], False), [[[-3, -2, 1, -4, 5, 6]]])
    assert np.allclose(ref.rotate(x, np.array([[0], [1]]), [np.pi / 2, np.pi], [0, 1], True), [[[1, 2, -3, -4, 5, 6]]])
    assert np.allclose(ref.head_norm(x, np.full(6, 2.0), 0.0), 2 * x / np.sqrt(91 / 6))
