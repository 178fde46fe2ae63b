"""The index arithmetic of the 8-bit kernels, compiled for the host from the header that the kernels include."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_index_arithmetic_of_the_kernels_on_the_host(tmp_path):
    exe = tmp_path / "q8_tiling_test"
    build = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined", "-fno-omit-frame-pointer",
                            f"-I{ROOT / 'librecuda_b200' / 'csrc' / 'kernels'}", str(ROOT / "tests" / "cpp" / "q8_tiling_test.cpp"), "-o", str(exe)],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "8-bit tiling ok" in run.stdout, (run.stdout + run.stderr)[-3000:]
