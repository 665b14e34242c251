"""What the paged cache holds beyond fp16's 65504, read back as fp16 and attended to by fp16 queries: 61440 whatever the scale of its block."""
import pytest
import torch

import sparseattention_amd as sa
from paged_reference import attention, tolerances

pytestmark = pytest.mark.gpu


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def in_fp16(x):
    return torch.where(x.abs() > 65504.0, torch.sign(x) * 61440.0, x)


@pytest.mark.parametrize("e", list(range(7, 29)) + [40, 119])
@pytest.mark.parametrize("D", [64, 256])
def test_every_code(gpu, e, D):
    cache = sa.empty_paged_cache(1, 1, D, page_size=32, device=gpu)
    codes = torch.arange(256, dtype=torch.uint8, device=gpu).repeat(D // 8)
    for t in (cache.k, cache.v):
        t.copy_(codes.view(t.shape))
    for t in (cache.k_scales, cache.v_scales):
        t.fill_(2.0 ** e)
    args = cache, ints([[0]], gpu), ints([32], gpu)
    for wide, got in zip(sa.paged_cache_gather(*args), sa.paged_cache_gather(*args, dtype=torch.float16)):
        want, got = in_fp16(wide.double()), got.double()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and int(torch.isnan(got).sum()) == 32 * D // 128
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("size", [1.0e5, 2.0 ** 30 * 3, 1.0e10, 1.0e20, 2.0 ** 127])
def test_tokens(gpu, size):
    """bf16 tokens, one large in a block of small ones."""
    D = 128
    x = torch.ones(1, 1, 64, D, dtype=torch.bfloat16, device=gpu)
    x[0, 0, 3], x[0, 0, 40] = size, -size
    x[0, 0, 5], x[0, 0, 6] = float("nan"), 7000.0
    cache = sa.empty_paged_cache(1, 1, D, page_size=64, device=gpu)
    table, n = ints([[0]], gpu), ints([64], gpu)
    sa.paged_cache_append(cache, x, x, table, ints([0], gpu))
    for wide, got in zip(sa.paged_cache_gather(cache, table, n), sa.paged_cache_gather(cache, table, n, dtype=torch.float16)):
        assert (got[0, 0, 3] == 61440.0).all() and (got[0, 0, 40] == -61440.0).all() and torch.isnan(got[0, 0, 5]).all()
        assert torch.equal(got.double().nan_to_num(0.0), in_fp16(wide.double()).nan_to_num(0.0))


@pytest.mark.parametrize("e", [8, 21, 22, 23, 24, 25, 119])
@pytest.mark.parametrize("D,G,Sq", [(64, 2, 3), (128, 1, 1), (128, 4, 8), (256, 5, 4)])
def test_attention(gpu, e, D, G, Sq):
    """Blocks of that scale beside ordinary ones, codes of every kind, some at keys that rows leave out."""
    H, n = 2, 250
    g = torch.Generator(device=gpu).manual_seed(e)
    cache = sa.empty_paged_cache(4, H, D, page_size=64, device=gpu)
    table, lens = ints([[2, 0, 3, 1]], gpu), ints([n], gpu)
    k, v = (torch.randn(1, H, 256, D, generator=g, device=gpu).half() for _ in range(2))
    sa.paged_cache_append(cache, k, v, table, ints([0], gpu))
    codes = torch.randint(0, 256, cache.v[2].shape, generator=g, device=gpu, dtype=torch.uint8)
    cache.v[2] = torch.where((codes & 0x7F) == 0x7F, codes & 0x80, codes)
    cache.v_scales[2] = 2.0 ** e
    q = torch.randn(1, H * G, Sq, D, generator=g, device=gpu).half()
    K, V = (t.double().cpu() for t in sa.paged_cache_gather(cache, table, lens, dtype=torch.float16))
    wide = sa.paged_cache_gather(cache, table, lens)[1].double().cpu()
    assert float(wide.abs().max()) > 65504.0 and torch.equal(V, in_fp16(wide))
    see = torch.rand(1, H, Sq, 256, generator=torch.Generator().manual_seed(1)) < 0.5
    see[..., n:] = False
    last = n - Sq + torch.arange(Sq)[:, None]
    for mask in (None, see):
        o = sa.sparse_attention_decode_paged(q, cache, table, lens, None if mask is None else mask.to(gpu)).double().cpu()
        for h in range(H):
            s = torch.arange(256) <= last if mask is None else mask[0, h]
            rows = q[0, h * G:(h + 1) * G].double().cpu().reshape(G * Sq, D)
            want = attention(rows, K[0, h], V[0, h], s.repeat(G, 1))
            tol, _ = tolerances(*want, n, 61440.0, D, torch.float16)
            got = o[0, h * G:(h + 1) * G].reshape(G * Sq, D)
            assert float(((got - want[0]).abs() - tol).max()) <= 0.0
