"""The 8-bit operators as recorded stream operations, together with the copies they are used beside: a checkpoint that is moved to
pinned host memory and back before the backward pass, pages of a cache that are copied and read through another table, and
the rules of a recorded operation (order, refusals, reports of bad indices at Await)."""
import numpy as np
import pytest
import torch

import q8_oracle as q8
from librecuda_b200 import api
from gpu_util import to_device, to_host

pytestmark = pytest.mark.gpu


def as_bytes(t):
    return t.contiguous().view(torch.uint8).numpy().reshape(-1)


def upload(stream, t):
    data = as_bytes(t)
    d = api.DeviceBuffer(data.size)
    to_device(stream, d, data)
    return d


def download(stream, d, dtype, shape):
    return torch.from_numpy(to_host(stream, d, int(np.prod(shape)) * dtype.itemsize)).view(dtype).view(shape)


def within(got, want, terms, units):
    half = torch.finfo(got.dtype).eps / 2
    return bool((np.abs(got.double().numpy() - want) <= units * 2.0 ** -24 * terms + half * np.abs(want) + 1e-30).all())


@pytest.mark.parametrize("rows,cols", [(64, 1024), (37, 333)])
def test_a_checkpoint_goes_to_the_host_and_back_before_the_backward_pass(stream, rows, cols):
    gen = torch.Generator().manual_seed(rows)
    gate, up, dh = (torch.randn(rows, cols, generator=gen).bfloat16() for _ in range(3))
    n, m = rows * cols, rows * q8.groups(cols)
    d_gate, d_up, d_dh = (upload(stream, t) for t in (gate, up, dh))
    h, dgate, dup, h2 = (api.DeviceBuffer(2 * n) for _ in range(4))
    packs = [(api.DeviceBuffer(n), api.DeviceBuffer(m)) for _ in range(2)]
    hosts = [[api.PinnedBuffer(b.nbytes) for b in pair] for pair in packs]
    # one recorded list: forward, checkpoint to the host, its device memory used for something else, back, backward
    stream.silu_mul_pack_q8((h, cols), packs[0], packs[1], (d_gate, cols), (d_up, cols), api.BF16, rows, cols)
    for pair, host in zip(packs, hosts):
        for b, p in zip(pair, host):
            stream.memcpy(p.array, b, b.nbytes)
            stream.memset_d8(b, 0x5A, b.nbytes)
            stream.memcpy(b, p.array, b.nbytes)
    stream.silu_mul_grad_q8((dgate, cols), (dup, cols), (d_dh, cols), packs[0], packs[1], api.BF16, rows, cols, h=(h2, cols))
    stream.run()
    wants = [q8.pack(t.double().numpy()) for t in (gate, up)]
    for host, want in zip(hosts, wants):
        for p, w in zip(host, want):
            assert np.array_equal(p.array, w.reshape(-1))
    got = [download(stream, b, torch.bfloat16, (rows, cols)) for b in (h, dgate, dup, h2)]
    want = q8.silu_mul(gate.double().numpy(), up.double().numpy())
    assert within(got[0], want, np.abs(want), 16)
    g, u = (q8.unpack(*w) for w in wants)
    by_g, by_u, terms = q8.silu_mul_grad(g, u, dh.double().numpy())
    again = q8.silu_mul(g, u)
    assert within(got[1], by_g, terms, 32) and within(got[2], by_u, np.abs(by_u), 16) and within(got[3], again, np.abs(again), 16)
    for host in hosts:
        for p in host:
            p.array = None
            p.free()
    for b in (d_gate, d_up, d_dh, h, dgate, dup, h2, *packs[0], *packs[1]):
        b.free()


def test_a_copy_behind_a_pack_sees_what_it_wrote(stream):
    # an ordered copy may load before the kernel in front of it has drained, unless that kernel writes its source: the stream has to
    # know what the operators write.  Two different inputs in turn, so that a stale source would show.
    rows, cols = 4096, 2048
    gen = torch.Generator().manual_seed(1)
    xs = [torch.randn(rows, cols, generator=gen).bfloat16() for _ in range(2)]
    dev = [upload(stream, x) for x in xs]
    wants = [q8.torch_pack(x) for x in xs]
    codes, scales, copy_c, copy_s = (api.DeviceBuffer(rows * n) for n in (cols, cols // 32) * 2)
    wide, copy_w = api.DeviceBuffer(2 * rows * cols), api.DeviceBuffer(2 * rows * cols)
    for i in range(12):
        stream.pack_q8((codes, scales), (dev[i % 2], cols), api.BF16, rows, cols)
        stream.memcpy(copy_c, codes, rows * cols)
        stream.memcpy(copy_s, scales, rows * cols // 32)
        stream.unpack_q8((wide, cols), (copy_c, copy_s), api.BF16, rows, cols)
        stream.memcpy(copy_w, wide, 2 * rows * cols)
        stream.run()
        c, s = wants[i % 2]
        assert np.array_equal(to_host(stream, copy_c, rows * cols), c.numpy().reshape(-1))
        assert np.array_equal(to_host(stream, copy_s, rows * cols // 32), s.numpy().reshape(-1))
        assert torch.equal(download(stream, copy_w, torch.bfloat16, (rows, cols)), q8.torch_unpack(c, s).to(torch.bfloat16))
    for b in (*dev, codes, scales, copy_c, copy_s, wide, copy_w):
        b.free()


@pytest.mark.parametrize("order", [api.CACHE_TOKENS_FIRST, api.CACHE_HEADS_FIRST])
def test_pages_are_copied_and_read_through_another_table(stream, order):
    pages, page, heads, dim, tokens = 8, 16, 3, 64, 40
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn(tokens, heads, dim, generator=gen).half() for _ in range(2))
    old, new = [4, 1, 6], [2, 0, 7]
    slots = torch.tensor([old[t // page] * page + t % page for t in range(tokens)])
    d_k, d_v, d_slots = (upload(stream, t) for t in (k, v, slots))
    sizes = [page * heads * dim, page * heads * 2] * 2  # bytes of a page in each part
    parts = [api.DeviceBuffer(pages * n) for n in sizes]
    cache = api.CacheQ8(*(p.ptr for p in parts), pages, page, heads, dim, dim, order)
    table, lengths, first = upload(stream, torch.tensor([new], dtype=torch.int32)), upload(stream, torch.tensor([tokens], dtype=torch.int32)), \
        upload(stream, torch.tensor([2], dtype=torch.int64))
    outs = [api.DeviceBuffer(2 * (tokens + 4) * heads * dim) for _ in range(2)]
    for p in parts:
        stream.memset_d8(p, 0xEE, p.nbytes)
    for o in outs:
        stream.memset_d16(o, 0x4200, o.nbytes // 2)  # 3.0
    stream.cache_write_q8(cache, (d_k, heads * dim, dim), (d_v, heads * dim, dim), api.F16, d_slots, tokens)
    cache.pages = 0  # the recorded call has its own copy of the descriptor
    for p, n in zip(parts, sizes):
        for a, b in zip(old, new):
            stream.memcpy(p.view(b * n), p.view(a * n), n)
            stream.memset_d8(p.view(a * n), 0, n)
    cache.pages = pages
    stream.cache_read_q8(cache, (outs[0], heads * dim, dim), (outs[1], heads * dim, dim), api.F16, table, 3, lengths, first, 1, tokens, tokens + 4)
    stream.run()
    for o, x in zip(outs, (k, v)):
        got = download(stream, o, torch.float16, (tokens + 4, heads, dim))
        want = q8.rounded(q8.unpack(*q8.pack(x.double().numpy())), "f16")
        assert torch.equal(got[2:tokens + 2], want)
        assert bool((got[:2] == 3).all()) and bool((got[tokens + 2:] == 3).all())
    for b in (d_k, d_v, d_slots, table, lengths, first, *parts, *outs):
        b.free()


def test_async_packs_are_joined_by_the_next_ordered_operation(stream):
    rows, cols = 512, 1024
    gen = torch.Generator().manual_seed(3)
    xs = [torch.randn(rows, cols, generator=gen) for _ in range(6)]
    dev = [upload(stream, x) for x in xs]
    packs = [(api.DeviceBuffer(rows * cols), api.DeviceBuffer(rows * cols // 32)) for _ in xs]
    outs = [api.DeviceBuffer(4 * rows * cols) for _ in xs]
    for d, p in zip(dev, packs):
        stream.pack_q8(p, (d, cols), api.F32, rows, cols, async_=True)
    for p, o in zip(packs, outs):
        stream.unpack_q8((o, cols), p, api.F32, rows, cols)
    stream.run()
    for x, o in zip(xs, outs):
        assert torch.equal(download(stream, o, torch.float32, (rows, cols)), q8.torch_unpack(*q8.torch_pack(x)).float())
    for b in (*dev, *outs, *(b for p in packs for b in p)):
        b.free()


def status_of(call):
    try:
        call()
    except api.LibreCudaError as e:
        return e.status
    return api.SUCCESS


def test_recorded_operations_refuse_what_the_kernels_would_and_host_memory(stream):
    a, b, c = (api.DeviceBuffer(1 << 16) for _ in range(3))
    host = np.zeros(1 << 16, np.uint8)
    bad = api.ERROR_INVALID_VALUE
    assert status_of(lambda: stream.pack_q8((a, b), (c, 64), 7, 8, 64)) == bad
    assert status_of(lambda: stream.pack_q8((a, b), (host, 64), api.F32, 8, 64)) == bad
    assert status_of(lambda: stream.pack_q8((host, b), (c, 64), api.F32, 8, 64)) == bad
    assert status_of(lambda: stream.unpack_q8((c, 63), (a, b), api.F32, 8, 64)) == bad
    assert status_of(lambda: stream.silu_mul_pack_q8((c, 64), (a, host), (a, b), (c, 64), (c, 64), api.F16, 8, 64)) == bad
    assert status_of(lambda: stream.silu_mul_grad_q8((c, 64), (c, 64), (c, 64), (a, b), (a, b), api.F16, 8, 64, h=(host, 64))) == bad
    cache = api.CacheQ8(a.ptr, b.ptr, None, None, 4, 4, 2, 64, 0, 0)
    slots = b
    assert status_of(lambda: stream.cache_write_q8(cache, (c, 128, 64), None, api.F16, host, 3)) == bad
    assert status_of(lambda: stream.cache_read_q8(cache, (c, 128, 64), None, api.F16, b, 2, b, b, 1, 9, 9)) == bad  # 9 > 2 pages of 4
    assert status_of(lambda: stream.cache_write_q8(cache, (c, 128, 64), None, api.F16, slots, 0)) == api.SUCCESS
    stream.run()  # nothing of the refused calls was recorded
    for x in (a, b, c):
        x.free()


def test_a_bad_slot_is_reported_once_by_await(stream):
    dim, heads = 32, 1
    cache_parts = [api.DeviceBuffer(4096), api.DeviceBuffer(4096)]
    cache = api.CacheQ8(cache_parts[0].ptr, cache_parts[1].ptr, None, None, 2, 4, heads, dim, 0, 0)
    k = upload(stream, torch.ones(2, dim))
    for slots, status in (([1, 8], api.ERROR_UNKNOWN), ([1, 7], api.SUCCESS), ([-1, -1], api.SUCCESS), ([2**40, 0], api.ERROR_UNKNOWN), ([0, 1], api.SUCCESS)):
        s = upload(stream, torch.tensor(slots))
        stream.cache_write_q8(cache, (k, dim, dim), None, api.F32, s, 2)
        stream.commence()
        assert status_of(stream.await_) == status
        s.free()
    for b in (*cache_parts, k):
        b.free()
