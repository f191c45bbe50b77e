"""Which tensors the heads' host layer takes, without a GPU: rk_heads.cpp compiled with heads_calls_cpu.cpp, against integers of any size."""
import os
import subprocess

import numpy as np
import pytest

from rknpu2_matmul_open_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "rknpu2_matmul_open_amd", "csrc")


@pytest.fixture(scope="module")
def answers(tmp_path_factory):
    exe = tmp_path_factory.mktemp("heads") / "heads_calls"
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-I" + CSRC, "-I" + os.path.join(ROOT, "include"),
                           "-o", str(exe), os.path.join(ROOT, "tests", "heads_calls_cpu.cpp"), os.path.join(CSRC, "rk_heads.cpp")])

    def ask(cases):
        text = "\n".join(" ".join(map(str, c)) for c in cases)
        done = subprocess.run([str(exe)], input=text, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=120)
        assert done.returncode == 0, done.stderr
        return [tuple(map(int, line.split())) for line in done.stdout.split("\n") if line]
    return ask


TAKEN, REFUSED = (0, 1), (capi.RK_NPU_ERR_PARAM, 0)


def test_strides_whose_extent_passes_64_bits_are_refused(answers):
    """2^25 rows 2^39 values apart are 2^64 values: nothing, in 64 bits."""
    assert answers([((1 << 25) + 1, 2, 16, 1 << 39, 1 << 40), ((1 << 24) + 1, 3, 16, 1 << 40, 1 << 40), ((1 << 26) + 1, 2, 64, 1 << 38, 1 << 39), (2 ** 31 - 16, 1 << 20, 512, 1 << 40, 1 << 40),
                    (1 << 20, 1 << 20, 1, 1 << 40, 1 << 40), ((1 << 17) + 1, 2, 16, 1 << 39, 1 << 40)]) == [REFUSED] * 6


def test_tensors_are_taken_where_their_rows_and_heads_lie_apart(answers):
    rng = np.random.default_rng(5)
    size = lambda top: int(np.exp2(rng.uniform(0, top)))  # noqa: E731
    cases, want = [], []
    for _ in range(4000):
        rows, heads, dim = size(30.9), size(19.9), min(512, size(9.1))
        row, head = size(62), size(62)
        if rng.random() < 0.6: # (near the edge between the layouts)
            if rng.random() < 0.5:
                head = dim + size(12) - 1
                row = (heads - 1) * head + dim + int(rng.integers(-2, 3))
            else:
                row = dim + size(12) - 1
                head = (rows - 1) * row + dim + int(rng.integers(-2, 3))
        apart = ((rows == 1 or row >= dim) and (heads == 1 or head >= dim) and
                 (rows == 1 or heads == 1 or row >= (heads - 1) * head + dim or head >= (rows - 1) * row + dim))
        values = max(((rows - 1) * row if rows > 1 else 0) + ((heads - 1) * head if heads > 1 else 0) + dim, rows * row if rows > 1 else 0, heads * head if heads > 1 else 0)
        if apart and 1 << 40 < max(row if rows > 1 else 0, head if heads > 1 else 0):
            continue # (a stride of its own limit)
        if apart and 1 << 55 < values <= 1 << 57:
            continue
        cases.append((rows, heads, dim, row, head))
        want.append(TAKEN if apart and values <= 1 << 55 else REFUSED)
    assert want.count(TAKEN) > 400 and want.count(REFUSED) > 400
    got = answers(cases)
    assert got == want, next((c, g, w) for c, g, w in zip(cases, got, want) if g != w)
