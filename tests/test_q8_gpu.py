"""The 8-bit operators on the GPU against their 64-bit restatement: bytes of packed rows exactly, read-back values exactly
(one rounding of an exact value), the gated unit and its gradients to bounds counted in roundings.

Error bounds.  The kernels work in 32 bits (unit u = 2^-24).  exp is good to 2 ulp of its result (2^-22 = 4 u) plus 2 u of its
argument's rounding, 1 + e adds u, the quotient at most 4 u, a product u.  So sigmoid and 1 - sigmoid are good to
(6 + 1 + 4 + 1) u = 12 u, g * sigmoid to 13 u, h and dup to 14 u, below 2^-20.  dgate is a sum of two terms, the larger
chain sigmoid, g * sigmoid, * (1 - sigmoid), the sum and two products: 13 + 12 + 1 + 3 = 29 u of the terms' size, below
2^-19.  The result is rounded to its type by at most eps / 2 of itself, or half its smallest subnormal.  Below
exp(-87) the sigmoid itself is subnormal or zero in 32 bits: 2^-126 of the factors is added for that."""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import q8_oracle as q8
from librecuda_b200 import api

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent
lib = api.lib
KINDS = ["f32", "f16", "bf16"]
GUARD = 0xC5


def current():
    return torch.cuda.current_stream().cuda_stream


def ok(rc):
    api.lcb_check(rc, "8-bit operator")


def guarded_bytes(n, offset=0):
    """A byte range of n inside a larger one filled with the guard byte, `offset` bytes off a 256-byte boundary."""
    whole = torch.full((n + 512,), GUARD, dtype=torch.uint8, device="cuda")
    return whole, whole[256 + offset:256 + offset + n]


def guards_intact(whole, part):
    at = part.data_ptr() - whole.data_ptr()
    out = torch.cat((whole[:at], whole[at + part.numel():]))
    return bool((out == GUARD).all())


def wide(values, kind, gap=0, offset=0):
    """A matrix of the type with rows `gap` elements apart, `offset` elements behind an aligned address."""
    rows, cols = values.shape
    flat = torch.full((offset + rows * (cols + gap) + 64,), 7.0, dtype=q8.TORCH_TYPES[kind], device="cuda")
    m = flat[offset:offset + rows * (cols + gap)].view(rows, cols + gap)[:, :cols]
    m.copy_(values)
    return flat, m


def special_values(rows, cols, kind, seed=0):
    """Random rows of many magnitudes, with zeros, ties, largest values, subnormals, infinities and NaN among them."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-12, 12, (rows, 1))
    x[rng.random((rows, cols)) < 0.05] = 0.0
    x[rng.random((rows, cols)) < 0.05] *= 2.0 ** -12
    x[rng.random((rows, cols)) < 0.03] = 1.0625   # halfway between codes at some scales
    x[rng.random((rows, cols)) < 0.03] = -1.1875
    x[rng.random((rows, cols)) < 0.02] = 1.75     # 448 at a power of two
    info = torch.finfo(q8.TORCH_TYPES[kind])
    if rows > 4:
        x[1] = 0.0
        x[1, ::2] = -0.0
        x[2, rng.random(cols) < 0.1] = np.inf
        x[2, rng.random(cols) < 0.1] = np.nan
        x[2, rng.random(cols) < 0.1] = -np.inf
        x[3, rng.random(cols) < 0.2] = info.max
        x[3, rng.random(cols) < 0.2] = -info.max
        x[4] = info.smallest_normal * rng.standard_normal(cols) * 0.1
    if rows > 5:
        x[5] = rng.choice([np.inf, np.nan, -np.inf], cols)  # a row that has no finite value
    return torch.from_numpy(x).to(torch.float32).to(q8.TORCH_TYPES[kind])


SHAPES = [(1, 1), (1, 31), (3, 32), (2, 33), (7, 64), (5, 80), (6, 96), (9, 128), (1, 4096), (129, 1001), (33, 1416), (300, 256), (8, 8200)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_pack_gives_the_bytes_of_the_definition(kind, rows, cols):
    values = special_values(rows, cols, kind, rows + cols)
    want_codes, want_scales = q8.pack(values.double().numpy())
    for gap, offset, byte_offset in ((0, 0, 0), (16, 0, 0), (8, 8, 8), (3, 0, 0), (0, 1, 1), (5, 3, 7)):
        _, src = wide(values, kind, gap, offset)
        all_codes, codes = guarded_bytes(rows * cols, byte_offset)
        all_scales, scales = guarded_bytes(rows * q8.groups(cols), byte_offset)
        ok(lib.lcb_pack_q8(codes.data_ptr(), scales.data_ptr(), src.data_ptr(), src.stride(0), q8.TYPE_CODES[kind], rows, cols, current()))
        assert np.array_equal(scales.cpu().numpy().reshape(rows, -1), want_scales), (gap, offset)
        assert np.array_equal(codes.cpu().numpy().reshape(rows, -1), want_codes), (gap, offset)
        assert guards_intact(all_codes, codes) and guards_intact(all_scales, scales), (gap, offset)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_unpack_gives_the_values_of_all_codes_and_scales(kind, rows, cols):
    rng = np.random.default_rng(rows * 7 + cols)
    codes = rng.integers(0, 256, (rows, cols), dtype=np.uint8)
    scales = rng.integers(0, 247, (rows, q8.groups(cols)), dtype=np.uint8)
    want = q8.rounded(q8.unpack(codes, scales), kind)
    for gap, offset, byte_offset in ((0, 0, 0), (16, 0, 0), (8, 8, 8), (3, 0, 1), (0, 1, 0), (5, 3, 7)):
        _, c = guarded_bytes(rows * cols, byte_offset)
        _, s = guarded_bytes(rows * q8.groups(cols), byte_offset)
        c.copy_(torch.from_numpy(codes).flatten())
        s.copy_(torch.from_numpy(scales).flatten())
        flat, dst = wide(torch.zeros(rows, cols), kind, gap, offset)
        before = flat.clone()
        ok(lib.lcb_unpack_q8(dst.data_ptr(), dst.stride(0), q8.TYPE_CODES[kind], c.data_ptr(), s.data_ptr(), rows, cols, current()))
        got = dst.cpu()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0)), (gap, offset)
        dst.zero_()
        assert torch.equal(flat, before), "bytes between the rows changed"


@pytest.mark.parametrize("kind", KINDS)
def test_a_round_trip_is_off_by_one_rounding_at_most(kind):
    # |value - x| <= 2^-4 |x| (half a step of e4m3) or half the smallest step of the group's scale, 2^-10 s; then the type's own
    rows, cols = 64, 1024
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-8, 8, (rows, 1))).to(q8.TORCH_TYPES[kind]).cuda()
    codes, scales = (torch.empty(rows, n, dtype=torch.uint8, device="cuda") for n in (cols, q8.groups(cols)))
    y = torch.empty_like(x)
    ok(lib.lcb_pack_q8(codes.data_ptr(), scales.data_ptr(), x.data_ptr(), cols, q8.TYPE_CODES[kind], rows, cols, current()))
    ok(lib.lcb_unpack_q8(y.data_ptr(), cols, q8.TYPE_CODES[kind], codes.data_ptr(), scales.data_ptr(), rows, cols, current()))
    s = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    off, size = (y.double() - x.double()).abs(), x.double().abs()
    assert bool((off <= 2.0 ** -4 * size + 2.0 ** -10 * s).all())


def half_step(want, kind):
    info = torch.finfo(q8.TORCH_TYPES[kind])
    return info.eps / 2 * np.abs(want) + float(info.smallest_normal) * info.eps / 2


def check_close(got, want, bound):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isfinite(got), np.isfinite(want))
    fine = np.isfinite(want)
    off = np.abs(got - want)[fine]
    worst = np.max(off / bound[fine]) if off.size else 0.0
    assert worst <= 1.0, f"error is {worst:.3f} of its bound"


def gate_values(rows, cols, seed):
    rng = np.random.default_rng(seed)
    g, u, d = (rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-3, 5, (rows, 1)) for _ in range(3))
    g[rng.random(g.shape) < 0.02] = 0.0
    g[rng.random(g.shape) < 0.02] = -95.0
    g[rng.random(g.shape) < 0.02] = 95.0
    g[rng.random(g.shape) < 0.02] = -20.0
    g[rng.random(g.shape) < 0.02] = -1.2785  # where the derivative changes its sign
    return g, u, d


LAYOUTS = [(0, 0, 0), (16, 0, 0), (8, 8, 8), (3, 1, 5)]
UNIT_SHAPES = [(1, 1), (2, 33), (7, 96), (5, 80), (3, 1416), (33, 2731), (130, 512)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", UNIT_SHAPES)
def test_silu_mul_pack(kind, rows, cols):
    g64, u64, _ = gate_values(rows, cols, rows + cols)
    g, u = (torch.from_numpy(v).to(q8.TORCH_TYPES[kind]) for v in (g64, u64))
    g64, u64 = g.double().numpy(), u.double().numpy()
    want = q8.silu_mul(g64, u64)
    bound = 2.0 ** -20 * np.abs(want) + np.abs(g64 * u64) * 2.0 ** -126 + half_step(want, kind)
    packs = [q8.pack(g64), q8.pack(u64)]
    for gap, offset, byte_offset in LAYOUTS:
        (_, gm), (_, um), (flat, hm) = (wide(v, kind, gap, offset) for v in (g, u, torch.zeros(rows, cols)))
        before = flat.clone()
        outs = [[guarded_bytes(n, byte_offset) for n in (rows * cols, rows * q8.groups(cols))] for _ in range(2)]
        ok(lib.lcb_silu_mul_pack_q8(hm.data_ptr(), hm.stride(0), *(part.data_ptr() for pair in outs for _, part in pair), gm.data_ptr(), gm.stride(0),
                                    um.data_ptr(), um.stride(0), q8.TYPE_CODES[kind], rows, cols, current()))
        check_close(hm, want, bound)
        for pair, wants in zip(outs, packs):
            for (whole, part), w in zip(pair, wants):
                assert np.array_equal(part.cpu().numpy().reshape(rows, -1), w)
                assert guards_intact(whole, part)
        hm.zero_()
        assert torch.equal(flat, before)


@pytest.mark.parametrize("again", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", UNIT_SHAPES)
def test_silu_mul_grad(kind, rows, cols, again):
    g64, u64, d64 = gate_values(rows, cols, rows * 3 + cols)
    (gc, gs), (uc, us) = q8.pack(g64), q8.pack(u64)
    g64, u64 = q8.unpack(gc, gs), q8.unpack(uc, us)
    d = torch.from_numpy(d64).to(q8.TORCH_TYPES[kind])
    d64 = d.double().numpy()
    dgate, dup, terms = q8.silu_mul_grad(g64, u64, d64)
    h = q8.silu_mul(g64, u64)
    tiny = 2.0 ** -126
    bounds = [2.0 ** -19 * terms + np.abs(d64 * u64) * (1 + np.abs(g64)) * tiny + half_step(dgate, kind),
              2.0 ** -20 * np.abs(dup) + np.abs(d64 * g64) * tiny + half_step(dup, kind),
              2.0 ** -20 * np.abs(h) + np.abs(g64 * u64) * tiny + half_step(h, kind)]
    for gap, offset, byte_offset in LAYOUTS:
        ins = []
        for v in (gc, gs, uc, us):
            _, part = guarded_bytes(v.size, byte_offset)
            part.copy_(torch.from_numpy(v).flatten())
            ins.append(part)
        _, dm = wide(d, kind, gap, offset)
        outs = [wide(torch.zeros(rows, cols), kind, gap, offset) for _ in range(3)]
        before = [flat.clone() for flat, _ in outs]
        (dg, du, hm) = (m for _, m in outs)
        ok(lib.lcb_silu_mul_grad_q8(dg.data_ptr(), dg.stride(0), du.data_ptr(), du.stride(0), hm.data_ptr() if again else None, hm.stride(0),
                                    dm.data_ptr(), dm.stride(0), *(p.data_ptr() for p in ins), q8.TYPE_CODES[kind], rows, cols, current()))
        check_close(dg, dgate, bounds[0])
        check_close(du, dup, bounds[1])
        if again:
            check_close(hm, h, bounds[2])
        else:
            assert bool((hm == 0).all())
        for (flat, m), b in zip(outs, before):
            m.zero_()
            assert torch.equal(flat, b)


def test_gradients_agree_with_differences():
    # central differences of the 64-bit unit at the checkpoint's values: their own error is h^2 / 6 of the third derivative
    # (below 1 for silu) times |u|, and 2^-53 |unit| / h
    rows, cols, h = 5, 160, 2.0 ** -13
    rng = np.random.default_rng(8)
    (gc, gs), (uc, us) = (q8.pack(rng.standard_normal((rows, cols)) * 3) for _ in range(2))
    g, u = q8.unpack(gc, gs), q8.unpack(uc, us)
    d = rng.standard_normal((rows, cols)).astype(np.float32).astype(np.float64)
    dev = [torch.from_numpy(v).cuda() for v in (gc, gs, uc, us)]
    dh = torch.from_numpy(d).float().cuda()
    dg, du = torch.empty_like(dh), torch.empty_like(dh)
    ok(lib.lcb_silu_mul_grad_q8(dg.data_ptr(), cols, du.data_ptr(), cols, None, 0, dh.data_ptr(), cols, *(t.data_ptr() for t in dev), 0,
                                rows, cols, current()))
    by_g = d * (q8.silu_mul(g + h, u) - q8.silu_mul(g - h, u)) / (2 * h)
    by_u = d * (q8.silu_mul(g, u + h) - q8.silu_mul(g, u - h)) / (2 * h)
    size = np.abs(d) * (1 + np.abs(u)) * (1 + np.abs(g))
    bound = size * (h * h / 6 + 2.0 ** -50 / h + 2.0 ** -19)
    assert np.all(np.abs(dg.double().cpu().numpy() - by_g) <= bound)
    assert np.all(np.abs(du.double().cpu().numpy() - by_u) <= bound)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(40, 512), (40, 70), (40, 1001), (40, 1416), (1, 5003), (6000, 600), (2000, 1003)])
def test_outputs_may_be_the_rows_of_an_input(rows, cols, kind):
    code = q8.TYPE_CODES[kind]
    g, u, d = (torch.randn(rows, cols, device="cuda").to(q8.TORCH_TYPES[kind]) for _ in range(3))
    packs = [torch.empty(rows, n, dtype=torch.uint8, device="cuda") for n in (cols, q8.groups(cols)) * 2]
    ptrs = [p.data_ptr() for p in packs]

    def forward(h, g, u):
        ok(lib.lcb_silu_mul_pack_q8(h.data_ptr(), cols, *ptrs, g.data_ptr(), cols, u.data_ptr(), cols, code, rows, cols, current()))

    def backward(dg, du, dh):
        ok(lib.lcb_silu_mul_grad_q8(dg.data_ptr(), cols, du.data_ptr(), cols, None, 0, dh.data_ptr(), cols, *ptrs, code, rows, cols, current()))

    h, dg, du = (torch.empty_like(g) for _ in range(3))
    forward(h, g, u)
    kept = [p.clone() for p in packs]
    backward(dg, du, d)
    same = g.clone()
    forward(same, same, u)
    assert torch.equal(same, h) and all(torch.equal(a, b) for a, b in zip(packs, kept))
    same = d.clone()
    backward(same, du, same)
    assert torch.equal(same, dg)


def test_a_broadcast_input_row_is_read_again_for_every_row():
    cols = 192
    x = torch.randn(1, cols, device="cuda").half()
    codes, scales = torch.empty(9, cols, dtype=torch.uint8, device="cuda"), torch.empty(9, 6, dtype=torch.uint8, device="cuda")
    ok(lib.lcb_pack_q8(codes.data_ptr(), scales.data_ptr(), x.data_ptr(), 0, 1, 9, cols, current()))
    want = q8.pack(x.double().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), np.repeat(want[0], 9, 0)) and np.array_equal(scales.cpu().numpy(), np.repeat(want[1], 9, 0))


# ---- paged cache ---------------------------------------------------------------------------------------------------

class Cache:
    def __init__(self, pages, page, heads, k_dim, v_dim, heads_first):
        self.shape = (pages, heads, page) if heads_first else (pages, page, heads)
        self.pages, self.page, self.heads, self.dims, self.heads_first = pages, page, heads, (k_dim, v_dim), heads_first
        self.parts = [torch.full((*self.shape, n), GUARD, dtype=torch.uint8, device="cuda")
                      for d in self.dims if d for n in (d, q8.groups(d))]
        ptrs = [p.data_ptr() for p in self.parts] + [None] * (4 - len(self.parts))
        self.c = api.CacheQ8(*ptrs, pages, page, heads, k_dim, v_dim, api.CACHE_HEADS_FIRST if heads_first else api.CACHE_TOKENS_FIRST)

    def by_slot(self, part):
        """[slots, heads, n] on the host"""
        x = self.parts[part].cpu().numpy()
        if self.heads_first:
            x = x.transpose(0, 2, 1, 3)
        return x.reshape(self.pages * self.page, self.heads, -1)


def qkv(tokens, heads, dims, kind, seed):
    """k and v as slices of one wide projection, their 64-bit values beside them."""
    n = heads * sum(dims)
    x = special_values(tokens, n, kind, seed).cuda()
    k = x[:, :heads * dims[0]].unflatten(1, (heads, dims[0]))
    v = x[:, heads * dims[0]:].unflatten(1, (heads, dims[1])) if dims[1] else None
    return k, v


def cache_write(cache, k, v, slots, kind):
    vs = (v.data_ptr(), v.stride(0), v.stride(1)) if v is not None else (None, 0, 0)
    return lib.lcb_cache_write_q8(cache.c, k.data_ptr(), k.stride(0), k.stride(1), *vs, q8.TYPE_CODES[kind], slots.data_ptr(), slots.numel(), current())


def cache_read(cache, k, v, table, lengths, first, longest, kind, rows=None):
    vs = (v.data_ptr(), v.stride(0), v.stride(1)) if v is not None else (None, 0, 0)
    return lib.lcb_cache_read_q8(cache.c, k.data_ptr(), k.stride(0), k.stride(1), *vs, q8.TYPE_CODES[kind], table.data_ptr(), table.stride(0),
                                 lengths.data_ptr(), first.data_ptr(), lengths.numel(), longest, k.shape[0] if rows is None else rows, current())


GEOMETRIES = [(16, 8, 128, 128), (16, 1, 64, 64), (7, 3, 80, 96), (64, 2, 192, 128), (1, 5, 65, 33), (24, 4, 40, 256), (32, 1, 576, 0), (8, 2, 1, 31)]


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page,heads,k_dim,v_dim", GEOMETRIES)
def test_cache_write_fills_the_named_slots_only(page, heads, k_dim, v_dim, kind, heads_first):
    for tokens in (1, 2, 19, 150):
        pages = -(-tokens // page) + 3
        cache = Cache(pages, page, heads, k_dim, v_dim, heads_first)
        k, v = qkv(tokens, heads, (k_dim, v_dim), kind, tokens)
        rng = np.random.default_rng(tokens)
        slots = rng.permutation(pages * page)[:tokens]
        skipped = rng.random(tokens) < (0.3 if tokens > 2 else 0)
        slots[skipped] = -1 - rng.integers(0, 2**40, int(skipped.sum()))
        ok(cache_write(cache, k, v, torch.from_numpy(slots).cuda(), kind))
        for side, x in enumerate((k, v) if v is not None else (k,)):
            codes, scales = q8.pack(x.double().cpu().numpy())
            for part, new in ((2 * side, codes), (2 * side + 1, scales)):
                want = np.full((pages * page, heads, new.shape[-1]), GUARD, np.uint8)
                want[slots[~skipped]] = new[~skipped]
                assert np.array_equal(cache.by_slot(part), want), (tokens, part)
    assert api.device_error_word() == 0


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page,heads,k_dim,v_dim", GEOMETRIES)
def test_cache_read_returns_the_sequences_and_leaves_other_rows(page, heads, k_dim, v_dim, kind, heads_first):
    rng = np.random.default_rng(page + heads)
    lengths = np.array([5, 0, 1, page, page + 1, 3 * page - 1, 2 * page, 70], np.int32)
    longest = int(lengths.max())
    per = -(-longest // page)
    pages = per * len(lengths) + 2
    cache = Cache(pages, page, heads, k_dim, v_dim, heads_first)
    for i, p in enumerate(cache.parts):
        p.copy_(torch.from_numpy(rng.integers(0, 247 if i % 2 else 256, p.shape, dtype=np.uint8)))
    table = rng.permutation(pages)[:per * len(lengths)].reshape(len(lengths), per).astype(np.int32)
    table[3, 0] = table[4, 0]  # a page that two sequences share
    for b, n in enumerate(lengths):
        table[b, -(-int(n) // page):] = rng.integers(-2**31, 2**31 - 1)  # entries that no position needs are never looked at
    ragged = np.concatenate(([0], np.cumsum(lengths)[:-1])).astype(np.int64)
    padded = np.arange(len(lengths), dtype=np.int64) * longest
    for first, rows, order in ((ragged, int(lengths.sum()) + 3, "thd"), (padded, len(lengths) * longest, "thd"), (ragged, int(lengths.sum()) + 3, "htd")):
        outs, wants = [], []
        for side, d in enumerate(d for d in (k_dim, v_dim) if d):
            shape = (rows, heads, d) if order == "thd" else (heads, rows, d)
            out = torch.full(shape, 5.0, dtype=q8.TORCH_TYPES[kind], device="cuda")
            outs.append(out if order == "thd" else out.transpose(0, 1))
            want = torch.full((rows, heads, d), 5.0, dtype=q8.TORCH_TYPES[kind])
            values = q8.rounded(q8.unpack(cache.by_slot(2 * side), cache.by_slot(2 * side + 1)), kind)
            for b, n in enumerate(lengths):
                at = np.arange(n)
                want[first[b]:first[b] + n] = values[table[b, at // page].astype(np.int64) * page + at % page]
            wants.append(want)
        t, ln, f = (torch.from_numpy(v).cuda() for v in (table, lengths, first))
        ok(cache_read(cache, outs[0], outs[1] if len(outs) > 1 else None, t, ln, f, longest, kind))
        for got, want in zip(outs, wants):
            got = got.cpu()
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
    assert api.device_error_word() == 0


def test_indices_out_of_range_are_skipped_and_reported(ctx):
    page, heads, dim = 16, 2, 64
    cache = Cache(4, page, heads, dim, dim, False)
    assert api.device_error_word() == 0
    k, v = qkv(6, heads, (dim, dim), "f32", 1)
    k, v = k.nan_to_num(0, 0, 0).contiguous(), v.nan_to_num(0, 0, 0).contiguous()
    slots = torch.tensor([0, 64, 3, 2**62, -1, 63], device="cuda")
    ok(cache_write(cache, k, v, slots, "f32"))
    assert api.device_error_word() == 4 and api.device_error_word() == 0
    codes, _ = q8.pack(k.double().cpu().numpy())
    got = cache.by_slot(0)
    for t, s in ((0, 0), (2, 3), (5, 63)):
        assert np.array_equal(got[s], codes[t])
        got[s] = GUARD
    assert (got == GUARD).all()

    for i, p in enumerate(cache.parts):
        p.fill_(127 if i % 2 else 0x38)  # ones
    good_table, good_lengths, good_first = [[0, 1], [2, 3]], [20, 17], [0, 20]
    cases = [("table", [[0, 4], [2, 3]], {*range(0, 16), *range(20, 37)}), ("table", [[0, 1], [-1, 3]], {*range(20), 36}),
             ("lengths", [33, 17], {*range(32), *range(32, 37)}), ("lengths", [-1, 17], {*range(20, 37)}),
             ("first", [0, 30], {*range(20), *range(30, 40)}), ("first", [-5, 20], {*range(0, 15), *range(20, 37)}),
             ("first", [2**63 - 1, 20], {*range(20, 37)}), ("first", [-2**63, 20], {*range(20, 37)})]
    for name, value, want_rows in cases:
        args = {"table": good_table, "lengths": good_lengths, "first": good_first, name: value}
        out_k, out_v = (torch.full((40, heads, dim), -3.0, device="cuda") for _ in range(2))
        ok(cache_read(cache, out_k, out_v, torch.tensor(args["table"], dtype=torch.int32, device="cuda"),
                      torch.tensor(args["lengths"], dtype=torch.int32, device="cuda"), torch.tensor(args["first"], device="cuda"), 32, "f32"))
        assert api.device_error_word() == 4, (name, value)
        for out in (out_k, out_v):
            written = set(torch.nonzero((out != -3.0).all(-1).all(-1)).flatten().tolist())
            assert written == want_rows, (name, value)
            assert bool((out[list(set(range(40)) - want_rows)] == -3.0).all())


def test_offsets_beyond_32_bits():
    # a pool of keys and values above 4 GiB each, the last pages in use; one matrix row that starts beyond 4 GiB
    page, heads, dim = 64, 8, 128
    pages = (5 << 30) // (page * heads * dim)
    for heads_first in (False, True):
        cache = Cache(pages, page, heads, dim, dim, heads_first)
        tokens = 130
        k, v = qkv(tokens, heads, (dim, dim), "bf16", 4)
        slots = torch.arange(pages * page - tokens, pages * page, device="cuda")
        ok(cache_write(cache, k, v, slots, "bf16"))
        table = torch.arange(pages - 3, pages, dtype=torch.int32, device="cuda").view(1, 3)
        lengths, first = torch.tensor([3 * page], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
        out_k, out_v = (torch.zeros(3 * page, heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        ok(cache_read(cache, out_k, out_v, table, lengths, first, 3 * page, "bf16"))
        for out, x in ((out_k, k), (out_v, v)):
            want = q8.rounded(q8.unpack(*q8.pack(x.double().cpu().numpy())), "bf16")
            got = out[3 * page - tokens:].cpu()
            assert torch.equal(got.nan_to_num(nan=9.0), want.nan_to_num(nan=9.0))
        for p in cache.parts:
            untouched = p[:pages - 3].flatten()
            assert int((untouched != GUARD).sum()) == 0
        del cache, p, untouched
        torch.cuda.empty_cache()
    rows, cols, stride = 3, 96, 3 << 29  # bf16 rows 3 GiB apart
    x = torch.zeros((rows - 1) * stride + cols, dtype=torch.bfloat16, device="cuda")
    m = torch.as_strided(x, (rows, cols), (stride, 1))
    m.copy_(torch.randn(rows, cols))
    codes, scales = (torch.empty(rows, n, dtype=torch.uint8, device="cuda") for n in (cols, 3))
    ok(lib.lcb_pack_q8(codes.data_ptr(), scales.data_ptr(), m.data_ptr(), stride, 2, rows, cols, current()))
    want = q8.pack(m.double().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])
    torch.cuda.empty_cache()


# ---- streams, graphs, the recorded API -------------------------------------------------------------------------------

def test_a_decoding_step_replayed_from_a_graph_sees_new_inputs():
    page, heads, dim = 16, 4, 128
    cache = Cache(6, page, heads, dim, dim, False)
    x = torch.zeros(2, 2 * heads * dim, dtype=torch.bfloat16, device="cuda")
    k, v = x[:, :heads * dim].unflatten(1, (heads, dim)), x[:, heads * dim:].unflatten(1, (heads, dim))
    slots = torch.zeros(2, dtype=torch.int64, device="cuda")
    table = torch.tensor([[0, 1], [3, 2]], dtype=torch.int32, device="cuda")
    lengths, first = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([0, 32], device="cuda")
    out_k, out_v = (torch.zeros(64, heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def step():
        ok(cache_write(cache, k, v, slots, "bf16"))
        ok(cache_read(cache, out_k, out_v, table, lengths, first, 32, "bf16"))

    slots.fill_(-1)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    seen = []
    for t in range(20):
        new = torch.randn(2, 2 * heads * dim, generator=torch.Generator().manual_seed(t)).bfloat16()
        x.copy_(new)
        seen.append(new)
        slots.copy_(torch.tensor([t, (3 if t < page else 2) * page + t % page]))
        lengths.fill_(t + 1)
        graph.replay()
        for b in range(2):
            for out, lo in ((out_k, 0), (out_v, heads * dim)):
                rows = torch.stack([s[b, lo:lo + heads * dim] for s in seen]).view(t + 1, heads, dim)
                want = q8.rounded(q8.unpack(*q8.pack(rows.double().numpy())), "bf16")
                assert torch.equal(out[32 * b:32 * b + t + 1].cpu(), want)
                assert bool((out[32 * b + t + 1:32 * b + 32] == 0).all())
    assert api.device_error_word() == 0


def test_the_first_call_of_a_process_may_be_captured(tmp_path):
    script = tmp_path / "first.py"
    script.write_text(f"""
import sys
sys.path[:0] = [{str(ROOT)!r}, {str(ROOT / "tests")!r}]
import torch
import q8_oracle as q8
from librecuda_b200 import api
x = torch.randn(100, 256, device="cuda")
codes, scales = (torch.zeros(100, n, dtype=torch.uint8, device="cuda") for n in (256, 8))
pool = [torch.zeros(128 * 256, dtype=torch.uint8, device="cuda") for _ in range(2)]
slots = torch.arange(100, device="cuda")
cache = api.CacheQ8(pool[0].data_ptr(), pool[1].data_ptr(), None, None, 8, 16, 1, 256, 0, 0)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    stream = torch.cuda.current_stream().cuda_stream
    assert api.lib.lcb_pack_q8(codes.data_ptr(), scales.data_ptr(), x.data_ptr(), 256, 0, 100, 256, stream) == 0
    assert api.lib.lcb_cache_write_q8(cache, x.data_ptr(), 256, 256, None, 0, 0, 0, slots.data_ptr(), 100, stream) == 0
graph.replay()
torch.cuda.synchronize()
want = q8.torch_pack(x)
assert torch.equal(codes, want[0]) and torch.equal(scales, want[1]) and torch.equal(pool[0][:25600].view(100, 256), want[0])
print("first call captured")
""")
    run = subprocess.run([sys.executable, str(script)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "first call captured" in run.stdout, run.stderr[-2000:]


def test_two_streams_at_once_give_what_each_gives_alone():
    rows, cols = 2000, 4096
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [torch.randn(rows, cols, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    outs = [[torch.empty(rows, n, dtype=torch.uint8, device="cuda") for n in (cols, cols // 32)] for _ in range(4)]
    torch.cuda.synchronize()
    for round_ in range(3):
        for i in (0, 1):
            ok(lib.lcb_pack_q8(*(o.data_ptr() for o in outs[i]), xs[i].data_ptr(), cols, 2, rows, cols, streams[i].cuda_stream))
    torch.cuda.synchronize()
    for i in (0, 1):
        ok(lib.lcb_pack_q8(*(o.data_ptr() for o in outs[2 + i]), xs[i].data_ptr(), cols, 2, rows, cols, current()))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[i], outs[2 + i]))
