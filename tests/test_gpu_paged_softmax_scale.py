"""Softmax scales from float32's smallest to its largest through the C ABI, over keys whose scores are all 0: every row is the mean of the values it
attends to, with keys left out before and behind."""
import ctypes
import math

import pytest
import torch

import sparseattention_amd as sa
from sparseattention_amd import _native

pytestmark = pytest.mark.gpu


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("scale", [1.5e-45, 1e-38, 1e-20, 1e-9, 0.1, 1e5, 3e38])
@pytest.mark.parametrize("block_scale", [2.0 ** -96, 1.0, 2.0 ** 119])
@pytest.mark.parametrize("Hq,Sq,window", [(2, 3, 0), (2, 1, 40), (8, 8, 70)])
def test_scores_of_zero(gpu, scale, block_scale, Hq, Sq, window):
    H, D, n, pages = 2, 64, 203, 4
    g = torch.Generator(device=gpu).manual_seed(0)
    cache = sa.empty_paged_cache(pages, H, D, page_size=64, device=gpu)
    table, lens = ints([[3, 1, 0, 2]], gpu), ints([n], gpu)
    v = torch.randn(1, H, n, D, generator=g, device=gpu).bfloat16()
    sa.paged_cache_append(cache, torch.zeros_like(v), v, table, ints([0], gpu))
    cache.k_scales.fill_(block_scale)
    held = sa.paged_cache_gather(cache, table, lens, length=n)[1].double().cpu()
    q = torch.randn(1, Hq, Sq, D, generator=g, device=gpu).bfloat16()
    o, lse = torch.empty_like(q), torch.empty(1, Hq, Sq, device=gpu)
    lib, S = _native.load(), lambda t: _native.strides(t.stride())  # noqa: E731
    c = _native.PagedCacheStruct(cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scales.data_ptr(), cache.v_scales.data_ptr(), pages, H, 64, D, D)
    need = lib.sa_decode_paged_workspace_bytes(1, Hq, H, Sq, D, pages, 64)
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    _native.check(lib.sa_sparse_attention_decode_paged(
        q.data_ptr(), S(q), ctypes.byref(c), table.data_ptr(), S(table), lens.data_ptr(), None, pages, o.data_ptr(), S(o), *[None] * 10, 0, 1, Hq, Sq,
        window, 0, scale, ws.data_ptr(), need, lse.data_ptr(), S(lse), torch.cuda.current_stream().cuda_stream))
    for head in range(Hq):
        for i in range(Sq):
            end = n - Sq + i + 1
            seen = held[0, head * H // Hq, max(end - window, 0) if window else 0:end]
            # weights of 1: sums in float32, one rounding of the result
            want, size = seen.mean(0), seen.abs().mean(0)
            assert ((o[0, head, i].double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + (len(seen) + 8) * 2.0 ** -24 * size).all()
            assert abs(float(lse[0, head, i]) - math.log(len(seen))) <= 2.0 ** -20 * math.log(len(seen))
