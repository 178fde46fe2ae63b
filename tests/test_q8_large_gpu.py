"""The 8-bit operators at sizes where a CTA takes several passes and a read several tiles, where rows lie side by side in a CTA,
share it, or are cut into lines, with a last tile that is only part full.  Compared byte for byte with a restatement in torch, which
is itself compared with the 64-bit one."""
import numpy as np
import pytest
import torch

import q8_oracle as q8
from librecuda_b200 import api

lib = api.lib


def test_the_two_restatements_agree():
    rng = np.random.default_rng(0)
    x = torch.from_numpy((rng.standard_normal((200, 100)) * 2.0 ** rng.integers(-60, 60, (200, 1))).astype(np.float32))
    x[3, 5], x[4, 6], x[5, 7], x[6], x[7, :40] = float("inf"), float("nan"), -float("inf"), 0.0, 1.75
    x[8, 0], x[9] = torch.finfo(torch.float32).max, 2.0 ** -140
    codes, scales = q8.torch_pack(x)
    want = q8.pack(x.double().numpy())
    assert np.array_equal(codes.numpy(), want[0]) and np.array_equal(scales.numpy(), want[1])
    assert np.array_equal(q8.torch_unpack(codes, scales).numpy(), q8.unpack(*want), equal_nan=True)


def current():
    return torch.cuda.current_stream().cuda_stream


def ok(rc):
    api.lcb_check(rc, "8-bit operator")


def matrix(rows, cols, dtype, gap, offset, fill=None):
    flat = torch.full((offset + rows * (cols + gap) + 64,), 3.0, dtype=dtype, device="cuda")
    m = flat[offset:offset + rows * (cols + gap)].view(rows, cols + gap)[:, :cols]
    if fill is not None:
        m.copy_(fill)
    return flat, m


def values(rows, cols, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=gen) * torch.exp2(torch.randint(-9, 9, (rows, 1), device="cuda", generator=gen))
    x.view(-1)[::9973] = float("nan")
    x.view(-1)[::7919] = float("inf")
    return x.to(dtype)


# (rows, cols, gap, offset): dense and cut into lines; strided, in chunks; side by side; 16-byte accesses; any address; one long row
# with and without a part of a group at its end
LARGE = [(5000, 1024, 0, 0), (2003, 2080, 32, 0), (3001, 4112, 16, 0), (40001, 96, 32, 0), (50021, 80, 0, 0), (9001, 1416, 0, 0), (20011, 200, 8, 8),
         (9001, 1001, 0, 0), (30011, 65, 3, 1), (4001, 2731, 2, 0), (1, 9_000_000, 0, 0), (1, 9_000_017, 0, 0), (1, 5_000_003, 0, 3), (70001, 32, 0, 0),
         (90001, 1, 0, 0), (30001, 32, 0, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,gap,offset", LARGE)
def test_large_matrices(rows, cols, gap, offset, kind):
    dtype = q8.TORCH_TYPES[kind]
    code = q8.TYPE_CODES[kind]
    x = values(rows, cols, dtype, rows)
    _, src = matrix(rows, cols, dtype, gap, offset, x)
    packs = [[torch.full((rows * n + 64,), 0xC5, dtype=torch.uint8, device="cuda") for n in (cols, q8.groups(cols))] for _ in range(2)]
    ptrs = [p.data_ptr() for pair in packs for p in pair]
    ok(lib.lcb_pack_q8(*ptrs[:2], src.data_ptr(), src.stride(0), code, rows, cols, current()))
    want = q8.torch_pack(x)
    for p, w in zip(packs[0], want):
        assert torch.equal(p[:w.numel()].view_as(w), w)
        assert bool((p[w.numel():] == 0xC5).all())
    flat, dst = matrix(rows, cols, dtype, gap, offset)
    before = flat.clone()
    ok(lib.lcb_unpack_q8(dst.data_ptr(), dst.stride(0), code, *ptrs[:2], rows, cols, current()))
    top = torch.finfo(dtype).max
    back = q8.torch_unpack(*want).clamp(-top, top).float().to(dtype)
    assert torch.equal(dst.nan_to_num(nan=0.0), back.nan_to_num(nan=0.0)) and torch.equal(dst.isnan(), back.isnan())
    dst.copy_(before[offset:offset + rows * (cols + gap)].view(rows, cols + gap)[:, :cols])
    assert torch.equal(flat, before)

    # the gated unit; infinities and NaN taken out of its inputs here, see the smaller tests
    gate, up, d = (values(rows, cols, torch.float32, rows + i).nan_to_num(0, 0, 0).clamp(-30, 30).to(dtype) for i in range(3))
    (_, gm), (_, um), (_, dm), (flat_h, hm), (flat_g, dg), (flat_u, du) = (
        matrix(rows, cols, dtype, gap, offset, v) for v in (gate, up, d, None, None, None))
    befores = [f.clone() for f in (flat_h, flat_g, flat_u)]
    ok(lib.lcb_silu_mul_pack_q8(hm.data_ptr(), hm.stride(0), *ptrs, gm.data_ptr(), gm.stride(0), um.data_ptr(), um.stride(0), code, rows, cols, current()))
    wants = [q8.torch_pack(v) for v in (gate, up)]
    for pair, w2 in zip(packs, wants):
        for p, w in zip(pair, w2):
            assert torch.equal(p[:w.numel()].view_as(w), w)
            assert bool((p[w.numel():] == 0xC5).all())
    half = torch.finfo(dtype).eps / 2
    tiny = float(torch.finfo(dtype).smallest_normal) * half

    def close(got, want, terms, units):  # units of 2^-24 of the terms, and the type's rounding (bounds as in the smaller tests)
        off = (got.double() - want).abs()
        assert bool((off <= units * 2.0 ** -24 * terms + half * want.abs() + tiny + 2.0 ** -120 * (1 + terms)).all())

    g64, u64, d64 = gate.double(), up.double(), d.double()
    h = g64 * torch.sigmoid(g64) * u64
    close(hm, h, h.abs(), 16)
    g64, u64 = (q8.torch_unpack(*w) for w in wants)
    s, q = torch.sigmoid(g64), torch.sigmoid(-g64)
    ok(lib.lcb_silu_mul_grad_q8(dg.data_ptr(), dg.stride(0), du.data_ptr(), du.stride(0), hm.data_ptr(), hm.stride(0), dm.data_ptr(), dm.stride(0), *ptrs,
                                code, rows, cols, current()))
    close(dg, d64 * u64 * s * (1 + g64 * q), (d64 * u64).abs() * s * (1 + g64.abs() * q), 32)
    close(du, d64 * g64 * s, (d64 * g64 * s).abs(), 16)
    close(hm, g64 * s * u64, (g64 * s * u64).abs(), 16)
    for flat, before in zip((flat_h, flat_g, flat_u), befores):  # between the rows nothing changed
        inside = torch.zeros(flat.numel(), dtype=torch.bool, device="cuda")
        inside[offset:offset + rows * (cols + gap)].view(rows, cols + gap)[:, :cols] = True
        assert torch.equal(flat[~inside], before[~inside])


@pytest.mark.gpu
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("kind,heads,k_dim,v_dim,page", [("bf16", 2, 64, 64, 16), ("f16", 1, 72, 72, 24), ("f32", 2, 33, 64, 64), ("bf16", 3, 65, 65, 7),
                                                         ("bf16", 40, 128, 64, 8)])
def test_large_caches(kind, heads, k_dim, v_dim, page, heads_first):
    dtype, code, gen = q8.TORCH_TYPES[kind], q8.TYPE_CODES[kind], torch.Generator(device="cuda").manual_seed(heads)
    few = heads * (k_dim + v_dim) > 1000
    sequences, longest = (20, 1500) if few else (300, 2047)
    lengths = torch.randint(0, longest + 1, (sequences,), generator=gen, device="cuda")
    lengths[:4] = torch.tensor([longest, 0, 1, longest - 1])
    total, per = int(lengths.sum()), -(-longest // page)
    pages = per * sequences + 3
    table = torch.randperm(pages, generator=gen, device="cuda")[:per * sequences].view(sequences, per).int()
    first = lengths.cumsum(0) - lengths
    which = torch.repeat_interleave(lengths)
    position = torch.arange(total, device="cuda") - first[which]
    slots = table[which, position // page].long() * page + position % page
    order = torch.randperm(total, generator=gen, device="cuda")  # tokens arrive in any order, some without a slot
    tokens = torch.cat((order, torch.zeros(1000, dtype=torch.long, device="cuda")))
    where = torch.cat((slots[order], torch.full((1000,), -1, device="cuda")))
    shape = (pages, heads, page) if heads_first else (pages, page, heads)
    parts = [torch.full((*shape, n), 0xC5, dtype=torch.uint8, device="cuda") for d in (k_dim, v_dim) for n in (d, q8.groups(d))]
    cache = api.CacheQ8(*(p.data_ptr() for p in parts), pages, page, heads, k_dim, v_dim, api.CACHE_HEADS_FIRST if heads_first else 0)
    rows = [values(total, heads * d, dtype, d).view(total, heads, d) for d in (k_dim, v_dim)]
    k, v = (r[tokens].contiguous() for r in rows)
    ok(lib.lcb_cache_write_q8(cache, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), code, where.data_ptr(),
                              tokens.numel(), current()))
    used = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    used[slots] = True
    for side, r in enumerate(rows):
        for p, w in zip(parts[2 * side:2 * side + 2], q8.torch_pack(r)):
            by_slot = (p.transpose(1, 2) if heads_first else p).reshape(pages * page, heads, -1)
            assert torch.equal(by_slot[slots], w)
            assert bool((by_slot[~used] == 0xC5).all())
    outs = [torch.full((total + 5, heads, d), 3.0, dtype=dtype, device="cuda") for d in (k_dim, v_dim)]
    ok(lib.lcb_cache_read_q8(cache, outs[0].data_ptr(), outs[0].stride(0), outs[0].stride(1), outs[1].data_ptr(), outs[1].stride(0),
                             outs[1].stride(1), code, table.data_ptr(), per, lengths.int().data_ptr(), first.data_ptr(), sequences, longest,
                             total + 5, current()))
    top = torch.finfo(dtype).max
    for out, r in zip(outs, rows):
        want = q8.torch_unpack(*q8.torch_pack(r)).clamp(-top, top).float().to(dtype)
        assert torch.equal(out[:total].nan_to_num(nan=0.0), want.nan_to_num(nan=0.0)) and torch.equal(out[:total].isnan(), want.isnan())
        assert bool((out[total:] == 3.0).all())
    assert api.device_error_word() == 0


@pytest.mark.gpu
def test_a_bound_far_above_the_lengths():
    # the grid is sized for max_length; sequences this short use one page of it each
    sequences, longest, page, dim = 4096, 1 << 20, 1024, 32
    gen = torch.Generator(device="cuda").manual_seed(5)
    lengths = torch.randint(0, 41, (sequences,), generator=gen, device="cuda")
    lengths[7] = 1024
    total = int(lengths.sum())
    first = lengths.cumsum(0) - lengths
    table = torch.full((sequences, longest // page), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.randperm(sequences, generator=gen, device="cuda").int()
    codes = torch.randint(0, 127, (sequences, page, 1, dim), generator=gen, device="cuda", dtype=torch.uint8)
    scales = torch.randint(100, 140, (sequences, page, 1, 1), generator=gen, device="cuda", dtype=torch.uint8)
    cache = api.CacheQ8(codes.data_ptr(), scales.data_ptr(), None, None, sequences, page, 1, dim, 0, 0)
    out = torch.full((total + 1, 1, dim), 3.0, device="cuda")
    ok(lib.lcb_cache_read_q8(cache, out.data_ptr(), dim, dim, None, 0, 0, 0, table.data_ptr(), table.stride(0), lengths.int().data_ptr(), first.data_ptr(),
                             sequences, longest, total + 1, current()))
    which = torch.repeat_interleave(lengths)
    position = torch.arange(total, device="cuda") - first[which]
    at = table[which, 0].long()
    assert torch.equal(out[:total], q8.torch_unpack(codes[at, position], scales[at, position]).float())
    assert bool((out[total] == 3).all()) and api.device_error_word() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("order", [api.CACHE_TOKENS_FIRST, api.CACHE_HEADS_FIRST])
def test_slots_beyond_32_bits(order):
    page, pages = 1 << 16, (1 << 16) + 3
    codes = torch.full((pages * page * 2,), 0xC5, dtype=torch.uint8, device="cuda")
    scales = torch.full((pages * page * 2,), 0xC5, dtype=torch.uint8, device="cuda")
    cache = api.CacheQ8(codes.data_ptr(), scales.data_ptr(), None, None, pages, page, 2, 1, 0, order)
    slots = torch.tensor([0, 5, page - 1, 2**32 - 1, 2**32, 2**32 + 70_000, pages * page - 1, -2**40], device="cuda")
    x = torch.arange(1, 17, device="cuda", dtype=torch.float32).view(8, 2, 1)
    ok(lib.lcb_cache_write_q8(cache, x.data_ptr(), 2, 1, None, 0, 0, 0, slots.data_ptr(), 8, current()))
    want = q8.torch_pack(x)
    for t in range(7):
        p, o = int(slots[t]) // page, int(slots[t]) % page
        for h in range(2):
            row = (p * 2 + h) * page + o if order else (p * page + o) * 2 + h
            assert int(codes[row]) == int(want[0][t, h, 0]) and int(scales[row]) == int(want[1][t, h, 0])
    assert sum(int((c != 0xC5).sum()) for c in codes.chunk(8)) == 14
    assert api.device_error_word() == 0
    # the last page read back
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda")
    lengths, first = torch.tensor([page], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.long, device="cuda")
    codes.view(pages, -1)[pages - 1] = torch.where(codes.view(pages, -1)[pages - 1] == 0xC5, 0, codes.view(pages, -1)[pages - 1])
    out = torch.zeros(page, 2, device="cuda")
    ok(lib.lcb_cache_read_q8(cache, out.data_ptr(), 2, 1, None, 0, 0, 0, table.data_ptr(), 1, lengths.data_ptr(), first.data_ptr(), 1, page, page, current()))
    assert out[-1].tolist() == [13.0, 14.0] and int((out != 0).sum()) == 2
    del codes, scales
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_rows_beyond_32_bits():
    rows = 2**32 + 1000
    x = torch.ones(rows, dtype=torch.bfloat16, device="cuda")
    for lo in (0, 2**31 - 40, 2**32 - 40, rows - 100):
        x[lo:lo + 100] = torch.arange(100, device="cuda", dtype=torch.bfloat16) - 50
    codes, scales = torch.zeros(rows, dtype=torch.uint8, device="cuda"), torch.zeros(rows, dtype=torch.uint8, device="cuda")
    ok(lib.lcb_pack_q8(codes.data_ptr(), scales.data_ptr(), x.data_ptr(), 1, 2, rows, 1, current()))
    for lo in range(0, rows, 1 << 28):
        c, s = q8.torch_pack(x[lo:lo + (1 << 28)].view(-1, 1))
        assert torch.equal(codes[lo:lo + (1 << 28)], c.view(-1)) and torch.equal(scales[lo:lo + (1 << 28)], s.view(-1))
        del c, s
    x.zero_()
    ok(lib.lcb_unpack_q8(x.data_ptr(), 1, 2, codes.data_ptr(), scales.data_ptr(), rows, 1, current()))
    kept = q8.torch_unpack(*q8.torch_pack((torch.arange(100, device="cuda") - 50).view(-1, 1))).view(-1).bfloat16()  # e4m3 keeps four bits
    for lo in (0, 2**31 - 40, 2**32 - 40, rows - 100):
        assert torch.equal(x[lo:lo + 100], kept)
    assert float(x[1000:2**31 - 1000:65537].min()) == 1.0
    del x, codes, scales
    torch.cuda.empty_cache()
