"""On which device the G4 and heads calls launch, without a GPU: rk_g4.cpp and rk_heads.cpp compiled with device_calls_cpu.cpp, which takes the place of the HIP side."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "rknpu2_matmul_open_amd", "csrc")


def test_nothing_is_launched_where_the_contexts_device_cannot_be_made_current(tmp_path):
    exe = tmp_path / "device_calls"
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-rdynamic", "-I" + CSRC, "-I" + os.path.join(ROOT, "include"), "-o", str(exe),
                           os.path.join(ROOT, "tests", "device_calls_cpu.cpp")] + [os.path.join(CSRC, f) for f in ("rk_core.cpp", "rk_g4.cpp", "rk_heads.cpp")] +
                          ["-Wl,--unresolved-symbols=ignore-all,-z,lazy", "-lpthread", "-ldl"])  # (what no checked call reaches)
    done = subprocess.run([str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
    assert done.returncode == 0, done.stdout
