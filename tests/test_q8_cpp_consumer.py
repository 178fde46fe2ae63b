"""A C++ program that uses the 8-bit operators through <librecuda.h>: compiled and linked here without a GPU, run on one."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
LIBDIR = ROOT / "librecuda_b200" / "lib"


def build(tmp_path) -> Path:
    exe = tmp_path / "q8_consumer_test"
    done = subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-O1", f"-I{ROOT / 'include'}",
                           str(ROOT / "tests" / "cpp" / "q8_consumer_test.cpp"), f"-L{LIBDIR}", "-ldriverapi", f"-Wl,-rpath,{LIBDIR}", "-o", str(exe)],
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-3000:]
    return exe


def test_the_program_compiles_and_links(tmp_path):
    assert build(tmp_path).exists()


def test_the_kernel_header_is_plain_c(tmp_path):
    src = tmp_path / "c.c"
    src.write_text('#include "lcb200_kernels.h"\nint main(void) { lcbCacheQ8 c = {0}; return lcb_pack_q8(c.k_codes, c.k_scales, 0, 0, LCB_F32, 0, 0, 0); }\n')
    done = subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'include'}", "-c", str(src), "-o", str(tmp_path / "c.o")],
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr


@pytest.mark.gpu
def test_the_program_runs(tmp_path):
    run = subprocess.run([str(build(tmp_path))], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "8-bit operators ok" in run.stdout, (run.stdout + run.stderr)[-3000:]
