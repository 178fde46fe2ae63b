"""Recorded 8-bit operators refuse host memory in the place of every single operand, and shapes that no launch takes.  Each call is
first recorded as it should be, with a buffer of its own for every operand, and accepted; then one operand is replaced."""
import numpy as np
import pytest

from librecuda_b200 import api

pytestmark = pytest.mark.gpu
BYTES = 1 << 16
ROWS, COLS = 8, 64


def status_of(call):
    try:
        call()
    except api.LibreCudaError as e:
        return e.status
    return api.SUCCESS


def cache_of(p):
    return api.CacheQ8(*(api._ptr(x) for x in p), 4, 4, 2, 64, 64, 0)


# name -> (operands, call(stream, operands, rows, cols)); every operand is a pointer
OPERATORS = {
    "pack": (3, lambda s, p, rows, cols: s.pack_q8(p[:2], (p[2], cols), api.F32, rows, cols)),
    "unpack": (3, lambda s, p, rows, cols: s.unpack_q8((p[0], cols), p[1:], api.F32, rows, cols)),
    "gated unit": (7, lambda s, p, rows, cols: s.silu_mul_pack_q8((p[0], cols), p[1:3], p[3:5], (p[5], cols), (p[6], cols), api.F32, rows, cols)),
    "gradient": (8, lambda s, p, rows, cols: s.silu_mul_grad_q8((p[0], cols), (p[1], cols), (p[2], cols), p[3:5], p[5:7], api.F32, rows, cols, h=(p[7], cols))),
    "gradient without h": (7, lambda s, p, rows, cols: s.silu_mul_grad_q8((p[0], cols), (p[1], cols), (p[2], cols), p[3:5], p[5:7], api.F32, rows, cols)),
    "cache write": (7, lambda s, p, rows, cols: s.cache_write_q8(cache_of(p[:4]), (p[4], 128, 64), (p[5], 128, 64), api.F16, p[6], rows)),
    "cache read": (9, lambda s, p, rows, cols: s.cache_read_q8(cache_of(p[:4]), (p[4], 128, 64), (p[5], 128, 64), api.F16, p[6], 2, p[7], p[8], 1, rows, rows)),
}


@pytest.fixture()
def buffers(stream):
    # zeros are a valid slot, page, length and first row, and slots 0..7 for the write are set below
    made = [api.DeviceBuffer(BYTES) for _ in range(9)]
    for b in made:
        stream.memset_d8(b, 0, BYTES)
    stream.run()
    yield made
    for b in made:
        b.free()


@pytest.mark.parametrize("name", list(OPERATORS))
def test_host_memory_is_refused_for_every_operand(stream, buffers, name):
    count, call = OPERATORS[name]
    if name == "cache write":
        stream.memcpy(buffers[6], np.arange(ROWS, dtype=np.int64).view(np.uint8), 8 * ROWS)
        stream.run()
    pageable, pinned = np.zeros(BYTES, np.uint8), api.PinnedBuffer(BYTES)
    assert status_of(lambda: call(stream, buffers[:count], ROWS, COLS)) == api.SUCCESS
    for i in range(count):
        for host in (pageable, pinned.array):
            operands = list(buffers[:count])
            operands[i] = host
            assert status_of(lambda: call(stream, operands, ROWS, COLS)) == api.ERROR_INVALID_VALUE, (i, host is pageable)
    stream.run()  # the first call runs, the refused ones left nothing behind
    assert api.device_error_word() == 0
    pinned.array = None
    pinned.free()


@pytest.mark.parametrize("name", ["pack", "unpack", "gated unit", "gradient"])
def test_shapes_that_no_launch_takes_are_refused_when_recorded(stream, buffers, name):
    count, call = OPERATORS[name]
    for rows, cols in ((2, 1 << 43), (3, (1 << 43) + 1), (1 << 40, 64)):
        assert status_of(lambda: call(stream, buffers[:count], rows, cols)) == api.ERROR_INVALID_VALUE, (rows, cols)
    stream.run()


def test_more_tokens_than_a_launch_takes_are_refused_when_recorded(stream, buffers):
    _, call = OPERATORS["cache write"]
    assert status_of(lambda: call(stream, buffers[:7], 1 << 40, 0)) == api.ERROR_INVALID_VALUE
    stream.run()
