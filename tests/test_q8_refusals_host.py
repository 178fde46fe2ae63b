"""Calls of the 8-bit operators that are refused because no launch could carry them out, without a GPU.  Each runs in a process
of its own: a call that ends its process fails only its own case."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

CALLS = """
import sys
sys.path.insert(0, {root!r})
from librecuda_b200 import _native as N
rows, cols = {rows}, {cols}
p = [i << 20 for i in range(1, 10)]
wide = lambda i: (p[i], cols + 32)
print(N.lib.lcb_pack_q8(p[0], p[1], *wide(2), {kind}, rows, cols, None),
      N.lib.lcb_unpack_q8(*wide(2), {kind}, p[0], p[1], rows, cols, None),
      N.lib.lcb_silu_mul_pack_q8(*wide(0), *p[1:5], *wide(5), *wide(6), {kind}, rows, cols, None),
      N.lib.lcb_silu_mul_grad_q8(*wide(0), *wide(1), *wide(2), *wide(3), *p[4:8], {kind}, rows, cols, None))
"""


# parts of 2048 values: 2^32 of them, a few more, and just too many for a grid of 2^31 - 1
@pytest.mark.parametrize("kind", [0, 2])
@pytest.mark.parametrize("rows,cols", [(2, 1 << 43), (2, (1 << 43) + 2048), (2, 1 << 44), (3, (1 << 43) + 1), (1 << 8, 1 << 42)])
def test_rows_of_more_parts_than_a_grid_has(rows, cols, kind):
    run = subprocess.run([sys.executable, "-c", CALLS.format(root=str(ROOT), rows=rows, cols=cols, kind=kind)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, f"the process ended with {run.returncode}: {run.stderr[-500:]}"
    assert run.stdout.split() == ["1"] * 4


CACHES = """
import sys
sys.path.insert(0, {root!r})
from librecuda_b200 import api
p = [i << 20 for i in range(1, 10)]
cache = api.CacheQ8(*p[:4], {pages}, {page}, {heads}, {dim}, {dim}, 0)
stride = {heads} * {dim}
print(api.lib.lcb_cache_write_q8(cache, p[4], 0, 0, p[5], 0, 0, 0, p[6], {tokens}, None),
      api.lib.lcb_cache_read_q8(cache, p[4], stride, {dim}, p[5], stride, {dim}, 0, p[6], 1, p[7], p[8], {tokens}, 1, 1, None))
"""


@pytest.mark.parametrize("pages,page,heads,dim,tokens", [(1, 16, 8, 128, 1 << 31), (1, 16, 1024, 1, 1 << 27), (1, 1, 1 << 20, 1, 1 << 20), (1, 1, 1, 1, 1 << 40)])
def test_more_tokens_or_sequences_than_a_grid_has(pages, page, heads, dim, tokens):
    run = subprocess.run([sys.executable, "-c", CACHES.format(root=str(ROOT), pages=pages, page=page, heads=heads, dim=dim, tokens=tokens)],
                         capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, f"the process ended with {run.returncode}: {run.stderr[-500:]}"
    assert run.stdout.split() == ["1", "1"]
