"""lcb_preload brings the 8-bit kernels onto the device: the first call of a process does not load them."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

SCRIPT = """
import sys, time
sys.path.insert(0, {root!r})
import torch
from librecuda_b200 import _native as N
x = torch.zeros(64, 1024, device="cuda")
codes, scales = (torch.zeros(64, n, dtype=torch.uint8, device="cuda") for n in (1024, 32))
slots, pool = torch.zeros(1, dtype=torch.int64, device="cuda"), [torch.zeros(1 << 16, dtype=torch.uint8, device="cuda") for _ in range(2)]
cache = N.CacheQ8(pool[0].data_ptr(), pool[1].data_ptr(), None, None, 4, 4, 4, 256, 0, 0)
stream = torch.cuda.current_stream().cuda_stream
torch.cuda.synchronize()
assert N.lib.lcb_preload() == 0
calls = [lambda: N.lib.lcb_pack_q8(codes.data_ptr(), scales.data_ptr(), x.data_ptr(), 1024, 0, 64, 1024, stream),
         lambda: N.lib.lcb_cache_write_q8(cache, x.data_ptr(), 1024, 256, None, 0, 0, 0, slots.data_ptr(), 1, stream)]
for call in calls:
    t = time.perf_counter()
    assert call() == 0
    print((time.perf_counter() - t) * 1e6)
torch.cuda.synchronize()
"""


def test_the_first_call_after_a_preload_loads_nothing():
    # loading the kernels of one source takes 3 ms, a first call without it 50 us; the best of three processes, since a
    # machine may be busy
    best = [1e9, 1e9]
    for _ in range(3):
        run = subprocess.run([sys.executable, "-c", SCRIPT.format(root=str(ROOT))], capture_output=True, text=True, timeout=300)
        assert run.returncode == 0, run.stderr[-2000:]
        best = [min(a, float(b)) for a, b in zip(best, run.stdout.split())]
    assert max(best) < 1000, best
