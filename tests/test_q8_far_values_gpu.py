"""The gated unit and its gradient at gates far below zero, where exp(-gate) nears the largest 32-bit number, beside factors
that bring the products back into range.

Error bounds.  With u = 2^-24, the sigmoid is good to 12 u of itself where it is a normal number (the bound that
test_q8_gpu.py derives).  Below 2^-126 it is held in steps of 2^-149, so it is off by half a step more; g * s, the product
with a factor and the sum in dgate stay below 29 u = 2^-19 of the terms' size.  Below -88.7228, where exp(-g) is beyond the
largest 32-bit number, the sigmoid is 0: it is below 2^-128 there, and that times the factors is what a product lacks."""
import numpy as np
import pytest
import torch

import q8_oracle as q8
from librecuda_b200 import api

lib = api.lib
pytestmark = pytest.mark.gpu
KINDS = ["f32", "bf16", "f16"]
FORMS = [(4, 512, 0), (4, 1416, 0), (3, 511, 0), (5, 67, 0), (5, 67, 1), (1, 96, 1)]  # rows, columns, offset: every access form
LIMIT = -88.7228  # ln of the largest 32-bit number


def current():
    return torch.cuda.current_stream().cuda_stream


def ok(rc):
    api.lcb_check(rc, "8-bit operator")


def device(values, kind, offset):
    flat = torch.zeros(offset + values.size + 64, dtype=q8.TORCH_TYPES[kind], device="cuda")
    m = flat[offset:offset + values.size].view(values.shape)
    m.copy_(torch.from_numpy(values).float())  # float32 holds every value exactly, so the type rounds once
    return m


def packed(rows, cols):
    return [torch.zeros(rows, n, dtype=torch.uint8, device="cuda") for n in (cols, q8.groups(cols))]


def half_step(want, kind):
    info = torch.finfo(q8.TORCH_TYPES[kind])
    return info.eps / 2 * np.abs(want) + float(info.smallest_normal) * info.eps / 2


def within(got, want, bound):
    off = np.abs(got.double().cpu().numpy() - want)
    worst = np.max(off / bound)
    assert worst <= 1.0, f"error is {worst:.3f} of its bound"


def lost(g, factors):
    """What a product with the sigmoid may lack: half a step of a subnormal, or the whole of what is beyond the range."""
    return np.where(g < LIMIT, 2.0 ** -128, 2.0 ** -149) * factors


def far_gates(rng, shape, top):
    """(gates from -91 to -86 in steps of the type, factors as large as they may be)"""
    g = -88.5 + 2.5 * (2 * rng.random(shape) - 1)
    g[rng.random(shape) < 0.2] = -88.0
    g[rng.random(shape) < 0.1] = -88.7
    g[rng.random(shape) < 0.1] = -87.5
    g[rng.random(shape) < 0.05] = -1000.0
    g[rng.random(shape) < 0.05] = 3.0
    return g, rng.choice([-1.0, 1.0], shape) * top * (0.25 + 0.25 * rng.random(shape))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,offset", FORMS)
def test_the_gated_unit_at_far_gates(rows, cols, offset, kind):
    rng = np.random.default_rng(cols)
    g, u = far_gates(rng, (rows, cols), 2.0 ** 15 if kind == "f16" else 2.0 ** 120)
    gm, um = device(g, kind, offset), device(u, kind, offset)
    g, u = gm.double().cpu().numpy(), um.double().cpu().numpy()
    hm = device(np.zeros((rows, cols)), kind, offset)
    packs = packed(rows, cols) + packed(rows, cols)
    ok(lib.lcb_silu_mul_pack_q8(hm.data_ptr(), cols, *(p.data_ptr() for p in packs), gm.data_ptr(), cols, um.data_ptr(), cols, q8.TYPE_CODES[kind],
                                rows, cols, current()))
    want = q8.silu_mul(g, u)
    if kind == "f16":  # 3 * 2^15 rounds to infinity there
        fine = np.abs(want) < 65504
        assert bool((hm.double().cpu().numpy()[~fine] == np.sign(want[~fine]) * np.inf).all())
        hm = torch.where(torch.from_numpy(fine).cuda(), hm, 0)
        want = np.where(fine, want, 0)
    within(hm, want, 2.0 ** -20 * np.abs(want) + lost(g, np.abs(g * u)) + half_step(want, kind))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,offset", FORMS)
def test_the_gradient_at_far_gates(rows, cols, offset, kind):
    rng = np.random.default_rng(cols + 1)
    g, u = far_gates(rng, (rows, cols), 2.0 ** 60)
    g[g < -500] = -448.0  # codes of one group reach 2^-14 of its largest value; -88 = -1.375 * 64 is one of them
    (gc, gs), (uc, us) = q8.pack(g), q8.pack(u)
    g, u = q8.unpack(gc, gs), q8.unpack(uc, us)
    d = rng.choice([-1.0, 1.0], g.shape) * (2.0 ** 10 if kind == "f16" else 2.0 ** 50) * (1 + rng.random(g.shape))
    dm = device(d, kind, offset)
    d = dm.double().cpu().numpy()
    ins = [torch.from_numpy(v).cuda() for v in (gc, gs, uc, us)]
    dg, du, hm = (device(np.zeros((rows, cols)), kind, offset) for _ in range(3))
    ok(lib.lcb_silu_mul_grad_q8(dg.data_ptr(), cols, du.data_ptr(), cols, hm.data_ptr(), cols, dm.data_ptr(), cols, *(t.data_ptr() for t in ins),
                                q8.TYPE_CODES[kind], rows, cols, current()))
    by_g, by_u, terms = q8.silu_mul_grad(g, u, d)
    h = q8.silu_mul(g, u)
    near = g < 0  # at 3 the products with 2^60 are beyond f16
    assert int((g == -88).sum()) > 10
    for got, want, size, factors in ((dg, by_g, terms, np.abs(d * u) * (1 + np.abs(g))), (du, by_u, np.abs(by_u), np.abs(d * g)), (hm, h, np.abs(h), np.abs(g * u))):
        at = near if kind == "f16" else np.ones_like(near)
        want = np.where(at, want, 0)
        got = torch.where(torch.from_numpy(at).cuda(), got, 0)
        within(got, want, 2.0 ** -19 * size + lost(g, factors) + half_step(want, kind))
