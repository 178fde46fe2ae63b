"""The cache operators in two CUDA contexts on one device, neither of them the runtime's own: each context has its kernels and its error
word, and a bad index in one is found there."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

SCRIPT = """
import ctypes, sys
sys.path.insert(0, {root!r})
import numpy as np
from librecuda_b200 import _native as N
lib = N.lib
cu = ctypes.CDLL("libcuda.so.1")

def ok(rc):
    assert rc == 0, rc

ok(cu.cuInit(0))
contexts = []
for _ in range(2):
    c = ctypes.c_void_p()
    ok(cu.cuCtxCreate_v2(ctypes.byref(c), 0, 0))
    contexts.append(c)

def device(array):
    p = ctypes.c_uint64()
    ok(cu.cuMemAlloc_v2(ctypes.byref(p), ctypes.c_size_t(array.nbytes)))
    ok(cu.cuMemcpyHtoD_v2(p, array.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(array.nbytes)))
    return p.value

def error_word():
    w = ctypes.c_uint()
    ok(lib.lcb_device_error_word(ctypes.byref(w)))
    return w.value

state = []
for c in contexts:
    ok(cu.cuCtxSetCurrent(c))
    codes, scales = np.full(8 * 32, 0xC5, np.uint8), np.full(8, 0xC5, np.uint8)
    state.append(dict(codes=device(codes), scales=device(scales), k=device(np.ones((2, 32), np.float32)), good=device(np.array([1, 6], np.int64)),
                      bad=device(np.array([8, 3], np.int64))))
order = [(0, "good"), (1, "good"), (1, "bad"), (0, "good"), (0, "bad"), (1, "good"), (1, "bad"), (0, "bad")]
expected = [0, 0]
for which, slots in order:
    s = state[which]
    ok(cu.cuCtxSetCurrent(contexts[which]))
    cache = N.CacheQ8(s["codes"], s["scales"], None, None, 2, 4, 1, 32, 0, 0)
    ok(lib.lcb_cache_write_q8(cache, s["k"], 32, 32, None, 0, 0, 0, s[slots], 2, None))
    assert error_word() == (4 if slots == "bad" else 0), (which, slots)
    assert error_word() == 0
    ok(cu.cuCtxSetCurrent(contexts[1 - which]))
    assert error_word() == 0
for c, s in zip(contexts, state):
    ok(cu.cuCtxSetCurrent(c))
    got = np.zeros(8 * 32, np.uint8)
    ok(cu.cuMemcpyDtoH_v2(got.ctypes.data_as(ctypes.c_void_p), ctypes.c_uint64(s["codes"]), ctypes.c_size_t(got.nbytes)))
    rows = got.reshape(8, 32)
    assert all((rows[i] == (0x78 if i in (1, 3, 6) else 0xC5)).all() for i in range(8)), rows[:, 0]
print("contexts ok")
"""


def test_two_contexts_on_one_device():
    run = subprocess.run([sys.executable, "-c", SCRIPT.format(root=str(ROOT))], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "contexts ok" in run.stdout, (run.stdout + run.stderr)[-3000:]
