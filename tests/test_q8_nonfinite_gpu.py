"""Infinities, NaN, overflow and extreme scales in the gated unit and its gradient, in every type and access form: a bad
value shows where it stands, with its sign, and changes nothing beside it.

Error bounds of the finite values: those of test_q8_gpu.py (2^-20 of h and dup, 2^-19 of dgate's terms), and what numbers
below 2^-126 lose, half a step of 2^-149 of the sigmoid, of g * s, of their sum in dgate and of dh * u, each times what it is
multiplied with afterwards.  Below g = -88.7228 the sigmoid is 0 in 32 bits; it is below 2^-128 there."""
import numpy as np
import pytest
import torch

import q8_oracle as q8
from librecuda_b200 import api

lib = api.lib
pytestmark = pytest.mark.gpu
KINDS = ["f32", "bf16", "f16"]
FORMS = [(6, 512, 0), (6, 1416, 0), (6, 511, 0), (6, 1100, 1), (9, 67, 0), (9, 67, 1), (1, 96, 1), (1, 1000, 0)]  # rows, columns, offset


def current():
    return torch.cuda.current_stream().cuda_stream


def ok(rc):
    api.lcb_check(rc, "8-bit operator")


def device(values, kind, offset):
    flat = torch.zeros(offset + values.size + 64, dtype=q8.TORCH_TYPES[kind], device="cuda")
    m = flat[offset:offset + values.size].view(values.shape)
    m.copy_(torch.from_numpy(values.astype(np.float32)))
    return m


def rounded(x, kind):
    """to 32 bits and then to the type: what passes the largest number becomes infinite"""
    with np.errstate(over="ignore"):
        return torch.from_numpy(x.astype(np.float32)).to(q8.TORCH_TYPES[kind])


def compare(got, want, bound, kind):
    got, expected = got.cpu().double().numpy(), rounded(want, kind).double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(expected)), np.argwhere(np.isnan(got) != np.isnan(expected))[:5]
    far = np.isinf(expected)
    assert np.array_equal(got[far], expected[far])
    fine = np.isfinite(expected)
    info = torch.finfo(q8.TORCH_TYPES[kind])
    half = info.eps / 2 * np.abs(want[fine]) + float(info.smallest_normal) * info.eps / 2
    worst = np.max(np.abs(got[fine] - want[fine]) / (bound[fine] + half), initial=0.0)
    assert worst <= 1.0, f"error is {worst:.3f} of its bound"


def lost(g):
    """of a product with the sigmoid, for each unit of what it is multiplied with"""
    return np.where(g < -88.7228, 2.0 ** -128, 2.0 ** -149)


def sprinkle(rng, x, values, share):
    for v in values:
        x[rng.random(x.shape) < share] = v


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,offset", FORMS)
def test_the_gated_unit(rows, cols, offset, kind):
    rng = np.random.default_rng(rows * cols)
    g, u = (rng.standard_normal((rows, cols)) * 4 for _ in range(2))
    g[0], u[0] = np.clip(g[0], -20, 20), np.clip(u[0], -20, 20)
    sprinkle(rng, g, (np.inf, -np.inf, np.nan, 0.0, -0.0, 300.0, -300.0, 3e4, -3e4), 0.02)
    sprinkle(rng, u, (np.inf, -np.inf, np.nan, 0.0, 300.0, -300.0), 0.02)
    if rows > 1:
        g[1], u[1] = 300.0, np.where(rng.random(cols) < 0.5, 250.0, -250.0)  # 75000: beyond f16 only
    if kind != "f16":
        sprinkle(rng, g, (3e38, -3e38, 1e30), 0.01)
        sprinkle(rng, u, (3e38, -3e38), 0.01)
    g[np.isinf(u) & (g < -80)] = -3.0  # there the sign of 0 * infinity would depend on the width of the arithmetic
    gm, um = device(g, kind, offset), device(u, kind, offset)
    g, u = gm.double().cpu().numpy(), um.double().cpu().numpy()
    hm = device(np.zeros((rows, cols)), kind, offset)
    packs = [torch.zeros(rows, n, dtype=torch.uint8, device="cuda") for n in (cols, q8.groups(cols)) * 2]
    ok(lib.lcb_silu_mul_pack_q8(hm.data_ptr(), cols, *(p.data_ptr() for p in packs), gm.data_ptr(), cols, um.data_ptr(), cols, q8.TYPE_CODES[kind],
                                rows, cols, current()))
    with np.errstate(invalid="ignore", over="ignore"):
        want = q8.silu_mul(g, u)
        bound = 2.0 ** -20 * np.abs(want) + lost(g) * np.abs(g * u) + 2.0 ** -149 * (1 + np.abs(u))
    compare(hm, want, bound, kind)
    for p, w in zip(packs, (*q8.pack(g), *q8.pack(u))):
        assert np.array_equal(p.cpu().numpy(), w)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,offset", FORMS)
def test_the_gradient(rows, cols, offset, kind):
    rng = np.random.default_rng(rows + cols)
    gc, uc = (rng.integers(0, 256, (rows, cols), dtype=np.uint8) for _ in range(2))  # every code, both NaN codes among them
    n = q8.groups(cols)
    gs = rng.choice(np.arange(0, 247, dtype=np.uint8), (rows, n))
    gs[rng.random((rows, n)) < 0.6] = 120  # magnitudes up to 3.5
    us = rng.integers(0, 188, (rows, n), dtype=np.uint8)  # up to 448 * 2^60
    us[rng.random((rows, n)) < 0.5] = 122
    g, u = q8.unpack(gc, gs), q8.unpack(uc, us)
    d = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-20, 15 if kind == "f16" else 50, (rows, 1))
    d[0] = rng.standard_normal(cols)
    sprinkle(rng, d, (0.0, np.nan), 0.02)
    for v in (np.inf, -np.inf):
        d[(rng.random(d.shape) < 0.05) & (np.abs(g) < 30)] = v
    dm = device(d, kind, offset)
    d = dm.double().cpu().numpy()
    ins = [torch.from_numpy(v).cuda() for v in (gc, gs, uc, us)]
    dg, du, hm = (device(np.zeros((rows, cols)), kind, offset) for _ in range(3))
    ok(lib.lcb_silu_mul_grad_q8(dg.data_ptr(), cols, du.data_ptr(), cols, hm.data_ptr(), cols, dm.data_ptr(), cols, *(t.data_ptr() for t in ins),
                                q8.TYPE_CODES[kind], rows, cols, current()))
    with np.errstate(invalid="ignore", over="ignore"):
        by_g, by_u, terms = q8.silu_mul_grad(g, u, d)
        h = q8.silu_mul(g, u)
        step = 2.0 ** -149
        compare(dg, by_g, 2.0 ** -19 * terms + lost(g) * np.abs(d * u) * (1 + np.abs(g)) + step * (2 + np.abs(d * u)), kind)
        compare(du, by_u, 2.0 ** -20 * np.abs(by_u) + lost(g) * np.abs(d * g) + step * (1 + np.abs(d)), kind)
        compare(hm, h, 2.0 ** -20 * np.abs(h) + lost(g) * np.abs(g * u) + step * (1 + np.abs(u)), kind)
