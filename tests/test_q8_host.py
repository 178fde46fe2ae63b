"""The 8-bit operators without a GPU: what they refuse, what they take as nothing to do, the division that turns a unit
index into a row, and the 64-bit restatement itself against hand-computed values."""
import ctypes as C
import random

import numpy as np
import pytest

import q8_oracle as q8
from librecuda_b200 import _native as N
from librecuda_b200 import api

lib = N.lib
A = 1 << 20  # an address that nothing reads: every call here is refused, or has nothing to do
B, D, E, F, G = (A * i for i in range(2, 7))
BIG = 1 << 62


def cache(**over):
    fields = dict(k_codes=A, k_scales=B, v_codes=D, v_scales=E, pages=4, page_tokens=16, heads=2, k_dim=64, v_dim=64, order=0)
    fields.update(over)
    return api.CacheQ8(**fields)


def write(c=None, k=A, kts=128, khs=64, v=A, vts=128, vhs=64, kind=2, slots=A, tokens=3):
    return lib.lcb_cache_write_q8(cache() if c is None else c, k, kts, khs, v, vts, vhs, kind, slots, tokens, None)


def read(c=None, k=A, kts=128, khs=64, v=B, vts=128, vhs=64, kind=2, table=A, stride=2, lengths=A, first=A, n=2, longest=32, rows=64):
    return lib.lcb_cache_read_q8(cache() if c is None else c, k, kts, khs, v, vts, vhs, kind, table, stride, lengths, first, n, longest,
                                 rows, None)


BAD_CACHES = [dict(pages=0), dict(page_tokens=0), dict(heads=0), dict(k_dim=0), dict(order=2), dict(order=-1), dict(k_codes=None),
              dict(k_scales=None), dict(v_codes=None), dict(v_scales=None), dict(v_dim=0), dict(pages=BIG, page_tokens=4),
              dict(k_dim=2**64 - 1), dict(heads=BIG), dict(v_dim=BIG)]


@pytest.mark.parametrize("over", BAD_CACHES, ids=str)
def test_a_bad_cache_is_refused(over):
    assert write(cache(**over)) == 1
    assert read(cache(**over)) == 1


@pytest.mark.parametrize("over", [dict(k=None), dict(v=None), dict(slots=None), dict(kind=3), dict(kind=-1), dict(k=A + 1), dict(v=A + 1),
                                  dict(k=A + 2, kind=0), dict(slots=A + 4), dict(kts=BIG, tokens=9), dict(khs=2**63), dict(tokens=BIG)], ids=str)
def test_a_bad_cache_write_is_refused(over):
    assert write(**over) == 1


@pytest.mark.parametrize("over", [dict(k=None), dict(v=None), dict(table=None), dict(lengths=None), dict(first=None), dict(kind=7),
                                  dict(k=A + 1), dict(table=A + 2), dict(lengths=A + 1), dict(first=A + 4), dict(longest=33),
                                  dict(stride=0), dict(longest=1 << 31, stride=1 << 40), dict(n=BIG), dict(rows=0), dict(rows=BIG),
                                  dict(khs=63), dict(kts=127), dict(kts=0), dict(khs=0), dict(vts=64, vhs=64),
                                  dict(kts=64, khs=64 * 63)], ids=str)
def test_a_bad_cache_read_is_refused(over):
    assert read(**over) == 1


def test_both_orders_of_output_rows_are_told_from_overlapping_ones():
    # heads outermost is a layout of its own; one row fewer between the heads and rows would overlap.  What passes
    # the checks comes back with the error of a machine without a device, or needs one: only refusals run here.
    assert read(kts=64, khs=64 * 64 - 1, vts=64, vhs=64 * 64) == 1
    assert read(kts=64, khs=64 * 64, vts=64, vhs=64 * 64 - 1) == 1


def test_a_cache_call_with_nothing_to_do_returns_at_once():
    assert write(tokens=0, k=None, v=None, slots=None) == 0
    assert read(n=0, k=None, v=None, table=None, lengths=None, first=None) == 0
    assert read(longest=0, k=None, v=None) == 0
    assert write(cache(pages=0), tokens=0) == 1  # a bad descriptor is refused all the same
    assert write(tokens=0, kind=5) == 1
    assert lib.lcb_cache_write_q8(None, A, 1, 1, A, 1, 1, 0, A, 1, None) == 1


def pack(codes=A, scales=B, x=D, stride=100, kind=2, rows=3, cols=100):
    return lib.lcb_pack_q8(codes, scales, x, stride, kind, rows, cols, None)


def unpack(y=A, stride=100, kind=2, codes=B, scales=D, rows=3, cols=100):
    return lib.lcb_unpack_q8(y, stride, kind, codes, scales, rows, cols, None)


@pytest.mark.parametrize("over", [dict(codes=None), dict(scales=None), dict(x=None), dict(kind=3), dict(kind=-1), dict(x=A + 1),
                                  dict(x=A + 2, kind=0), dict(rows=BIG), dict(cols=BIG, rows=4), dict(cols=2**64 - 1, rows=1),
                                  dict(stride=BIG)], ids=str)
def test_a_bad_pack_is_refused(over):
    assert pack(**over) == 1


@pytest.mark.parametrize("over", [dict(codes=None), dict(scales=None), dict(y=None), dict(kind=9), dict(y=A + 1), dict(stride=99),
                                  dict(stride=0), dict(rows=BIG), dict(cols=BIG, rows=4)], ids=str)
def test_a_bad_unpack_is_refused(over):
    assert unpack(**over) == 1


def silu(h=A, hs=100, gc=B, gs=D, uc=E, us=F, g=G, gst=100, u=G, ust=100, kind=2, rows=3, cols=100):
    return lib.lcb_silu_mul_pack_q8(h, hs, gc, gs, uc, us, g, gst, u, ust, kind, rows, cols, None)


def grad(dg=A, dgs=100, du=B, dus=100, h=D, hs=100, dh=E, dhs=100, gc=A, gs=A, uc=A, us=A, kind=2, rows=3, cols=100):
    return lib.lcb_silu_mul_grad_q8(dg, dgs, du, dus, h, hs, dh, dhs, gc, gs, uc, us, kind, rows, cols, None)


@pytest.mark.parametrize("over", [dict(h=None), dict(gc=None), dict(gs=None), dict(uc=None), dict(us=None), dict(g=None), dict(u=None),
                                  dict(kind=3), dict(h=A + 1), dict(g=A + 1), dict(u=A + 1), dict(hs=99), dict(rows=BIG)], ids=str)
def test_a_bad_silu_mul_pack_is_refused(over):
    assert silu(**over) == 1


@pytest.mark.parametrize("over", [dict(dg=None), dict(du=None), dict(dh=None), dict(gc=None), dict(gs=None), dict(uc=None), dict(us=None),
                                  dict(kind=-1), dict(dg=A + 1), dict(du=A + 1), dict(dh=A + 1), dict(h=A + 1), dict(dgs=99), dict(dus=0),
                                  dict(hs=50), dict(cols=BIG)], ids=str)
def test_a_bad_silu_mul_grad_is_refused(over):
    assert grad(**over) == 1


def test_outputs_at_one_address_are_refused():
    assert pack(codes=B) == 1 and pack(x=A) == 1 and unpack(y=B) == 1 and unpack(codes=D) == 1
    assert silu(gc=A) == 1 and silu(uc=B) == 1 and silu(us=D) == 1
    assert grad(du=A) == 1 and grad(h=A) == 1 and grad(h=B) == 1
    assert write(cache(v_codes=A)) == 1 and write(cache(v_scales=B)) == 1 and write(cache(k_scales=A)) == 1
    assert read(v=A) == 1


def test_an_empty_matrix_is_nothing_to_do():
    for empty in (dict(rows=0), dict(cols=0)):
        assert pack(codes=None, scales=None, x=None, **empty) == 0
        assert unpack(codes=None, scales=None, y=None, **empty) == 0
        assert silu(h=None, g=None, **empty) == 0
        assert grad(dh=None, gc=None, **empty) == 0
        assert pack(kind=4, **empty) == 1


def test_the_magic_number_division_is_exact():
    # quotient = high half of n * floor((2^64 - 1) / d), or one more
    rng = random.Random(5)
    ds = [1, 2, 3, 7, 32, 96, 1001, 2**31 - 1, 2**32, 2**40 + 12345, 2**62] + [rng.randrange(1, 2 ** rng.randrange(1, 63)) for _ in range(300)]
    for d in ds:
        magic = (2**64 - 1) // d
        for n in [0, 1, d - 1, d, d + 1, 2 * d - 1, 2**63, 2**64 - 1] + [rng.randrange(2 ** rng.randrange(1, 65)) for _ in range(30)]:
            q = (n * magic) >> 64
            q += n - q * d >= d
            assert q == n // d, (n, d)


def test_the_restatement_knows_the_format():
    assert q8.CODE_VALUES[0x7E] == 448 and q8.CODE_VALUES[1] == 2.0 ** -9 and q8.CODE_VALUES[0x38] == 1 and q8.CODE_VALUES[0xB8] == -1
    x = np.zeros((1, 33))
    x[0, :4] = [448, -1.0625, np.inf, np.nan]  # 1.0625 is half a step from 1 and 1.125: to the even code
    x[0, 32] = 2.0 ** -140
    codes, scales = q8.pack(x)
    assert scales.tolist() == [[127, 0]]
    assert codes[0, :5].tolist() == [0x7E, 0xB8, 0x7F, 0x7F, 0] and codes[0, 32] == 0  # 2^-140 / 2^-127 is below half the smallest code
    assert q8.scale_bytes(np.array([0.0, 448.0, np.nextafter(448, 500), 449 * 2.0 ** 119, 1.75 * 2.0 ** -119, 2.0 ** -149])).tolist() == [0, 127, 128, 246, 0, 0]
    assert q8.unpack(codes, scales)[0, 1] == -1.0


def test_recorded_operations_need_a_stream():
    c = cache()
    calls = [lib.libreCuPackQ8(A, A, A, 100, 2, 3, 100, None, False), lib.libreCuUnpackQ8(A, 100, 2, A, A, 3, 100, None, False),
             lib.libreCuSiluMulPackQ8(A, 100, A, A, A, A, A, 100, A, 100, 2, 3, 100, None, False),
             lib.libreCuSiluMulGradQ8(A, 100, A, 100, None, 0, A, 100, A, A, A, A, 2, 3, 100, None, False),
             lib.libreCuCacheWriteQ8(c, A, 128, 64, A, 128, 64, 2, A, 3, None, False),
             lib.libreCuCacheReadQ8(c, A, 128, 64, A, 128, 64, 2, A, 2, A, A, 2, 32, 64, None, False)]
    assert calls == [api.ERROR_INVALID_VALUE] * 6
