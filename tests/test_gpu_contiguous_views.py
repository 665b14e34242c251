"""Tensors that are contiguous, but lie at an address or have strides in dimensions of size 1 that the kernels do not take: the results are
those of an ordinary copy, to the bit."""
import pytest
import torch

import sparseattention_amd as sa

pytestmark = pytest.mark.gpu


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def shifted(x):
    """x two bytes behind a 16-byte boundary."""
    flat = torch.empty(x.numel() + 8, dtype=x.dtype, device=x.device)
    view = flat[1:1 + x.numel()].view(x.shape)
    view.copy_(x)
    assert view.is_contiguous() and view.data_ptr() % 16 == 2
    return view


def odd_stride(x):
    """x [1, ...] with an odd stride in its first dimension."""
    n = x.numel()
    view = torch.empty(n + 8, dtype=x.dtype, device=x.device).as_strided(x.shape, (n + 3, *x.stride()[1:]))
    view.copy_(x)
    assert view.is_contiguous() and view.stride(0) % 8 and view.data_ptr() % 16 == 0
    return view


@pytest.mark.parametrize("made", [shifted, odd_stride])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_paged(gpu, made, dtype):
    H, D, n = 2, 64, 45
    g = torch.Generator(device=gpu).manual_seed(0)
    k, v = (torch.randn(1, H, n, D, generator=g, device=gpu).to(dtype) for _ in range(2))
    q = torch.randn(1, 2 * H, 3, D, generator=g, device=gpu).to(dtype)
    table, lens = ints([[1, 0]], gpu), ints([n], gpu)
    outs = []
    for as_is in (lambda x: x, made):
        cache = sa.empty_paged_cache(2, H, D, page_size=32, device=gpu)
        sa.paged_cache_append(cache, as_is(k), as_is(v), table, ints([0], gpu))
        outs.append((cache.k, cache.v, sa.sparse_attention_decode_paged(as_is(q), cache, table, lens)))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("made", [shifted, odd_stride])
def test_dense(gpu, made):
    g = torch.Generator(device=gpu).manual_seed(1)
    k, v, q = (torch.randn(1, 2, n, 64, generator=g, device=gpu).bfloat16() for n in (256, 256, 128))
    mask = (torch.arange(256, device=gpu)[None] <= torch.arange(128, device=gpu)[:, None] + 128)[None, None].expand(1, 2, 128, 256)
    assert torch.equal(sa.sparse_attention(made(q), made(k), made(v), mask, 128, 32), sa.sparse_attention(q, k, v, mask, 128, 32))
    few, seen = q[:, :, :4].contiguous(), mask[:, :, :4]
    assert torch.equal(sa.sparse_attention_decode(made(few), made(k), made(v), seen, 32), sa.sparse_attention_decode(few, k, v, seen, 32))
