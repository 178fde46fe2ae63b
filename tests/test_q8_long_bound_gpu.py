"""Reads whose bound on the lengths is the largest there is, in caches whose tokens take many CTAs each."""
import pytest
import torch

import q8_oracle as q8
from librecuda_b200 import api

lib = api.lib


@pytest.mark.gpu
@pytest.mark.parametrize("order", [api.CACHE_TOKENS_FIRST, api.CACHE_HEADS_FIRST])
@pytest.mark.parametrize("heads,k_dim,v_dim,kind", [(1024, 1, 3, "bf16"), (300, 40, 33, "f32"), (1024, 16, 16, "f16")])
def test_the_largest_bound_on_the_lengths(heads, k_dim, v_dim, kind, order):
    page, pages, longest = 4096, 4, 2**31 - 1
    gen = torch.Generator(device="cuda").manual_seed(heads + k_dim)
    shape = (pages, page, heads) if order == api.CACHE_TOKENS_FIRST else (pages, heads, page)
    parts = [torch.randint(0, hi, (*shape, n), generator=gen, device="cuda", dtype=torch.uint8)
             for d in (k_dim, v_dim) for n, hi in ((d, 127), (q8.groups(d), 134))]
    cache = api.CacheQ8(*(p.data_ptr() for p in parts), pages, page, heads, k_dim, v_dim, order)
    lengths = [0, 5, 4100, 1]
    table = torch.full((len(lengths), 1 << 19), -1, dtype=torch.int32, device="cuda")
    table[1, 0], table[2, 0], table[2, 1], table[3, 0] = 2, 3, 0, 1
    first = [0, 0, 5, 4105]
    rows = 4108
    outs = [torch.full((rows, heads, d), 3.0, dtype=q8.TORCH_TYPES[kind], device="cuda") for d in (k_dim, v_dim)]
    lens, firsts = torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.tensor(first, device="cuda")
    rc = lib.lcb_cache_read_q8(cache, outs[0].data_ptr(), heads * k_dim, k_dim, outs[1].data_ptr(), heads * v_dim, v_dim, q8.TYPE_CODES[kind],
                               table.data_ptr(), table.stride(0), lens.data_ptr(), firsts.data_ptr(), len(lengths), longest, rows,
                               torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert api.device_error_word() == 0
    top = torch.finfo(q8.TORCH_TYPES[kind]).max
    for side, out in enumerate(outs):
        codes, scales = (p if order == api.CACHE_TOKENS_FIRST else p.transpose(1, 2) for p in parts[2 * side:2 * side + 2])
        for b, n in enumerate(lengths):
            for at in range(0, n, page):
                p, count = int(table[b, at // page]), min(page, n - at)
                want = q8.torch_unpack(codes[p, :count].contiguous(), scales[p, :count].contiguous()).clamp(-top, top).float().to(out.dtype)
                assert torch.equal(out[first[b] + at:first[b] + at + count], want), (side, b, at)
        assert bool((out[4106:] == 3.0).all())
