"""What Await says about the sticky device error word: a wait that gave up and an index out of range are told apart."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_the_words_for_every_bit(tmp_path):
    exe = tmp_path / "error_word_test"
    build = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined", "-fno-omit-frame-pointer",
                            f"-I{ROOT / 'librecuda_b200' / 'csrc' / 'driverapi'}", str(ROOT / "tests" / "cpp" / "error_word_test.cpp"), "-o", str(exe),
                            "-pthread"], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "error word ok" in run.stdout, (run.stdout + run.stderr)[-3000:]


SCRIPT = """
import sys
sys.path.insert(0, {root!r})
import numpy as np
from librecuda_b200 import api
context = api.Context(0, api.CU_CTX_SCHED_YIELD)
stream = api.Stream()
codes, scales, k, slots = (api.DeviceBuffer(4096) for _ in range(4))
stream.memcpy(slots, np.array([1 << 40], np.int64).view(np.uint8), 8)
stream.memset_d8(k, 0, 4096)
stream.cache_write_q8(api.CacheQ8(codes.ptr, scales.ptr, None, None, 2, 4, 1, 32, 0, 0), (k, 32, 32), None, api.F32, slots, 1)
stream.commence()
try:
    stream.await_()
except api.LibreCudaError as e:
    print("status", e.status)
"""


@pytest.mark.gpu
def test_await_names_an_index_out_of_range():
    run = subprocess.run([sys.executable, "-c", SCRIPT.format(root=str(ROOT))], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    assert "status" in run.stdout
    assert "device error word 4" in run.stderr and "out of range" in run.stderr and "bounded wait" not in run.stderr
