"""Scores of 10^9 and more, of either sign, whose float32 steps are many powers of two of a weight: each row has one key that outweighs all others
entirely, so it gives that key's values as they are held."""
import math

import pytest
import torch

import sparseattention_amd as sa

pytestmark = pytest.mark.gpu


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("D,G,Sq", [(64, 3, 2), (128, 4, 8), (256, 1, 1)])
@pytest.mark.parametrize("n", [9, 300, 9001])
@pytest.mark.parametrize("dtype,q_size,k_size", [(torch.float16, 2000.0, 2.0 ** 13), (torch.bfloat16, 2000.0, 2.0 ** 13), (torch.bfloat16, 1.0e7, 2.0 ** 19),
                                                 (torch.bfloat16, 1.0e13, 2.0 ** 70)])
def test_one_key_outweighs_all(gpu, D, G, Sq, n, dtype, q_size, k_size):
    H = 2
    g = torch.Generator(device=gpu).manual_seed(n)
    k = torch.full((1, H, n, D), 2.0 * k_size, device=gpu)
    most, least = n // 3, n // 2
    k[:, :, most], k[:, :, least] = 4.0 * k_size, k_size
    v = torch.randn(1, H, n, D, generator=g, device=gpu)
    pages = -(-n // 64)
    cache = sa.empty_paged_cache(pages, H, D, page_size=64, device=gpu)
    table, lens = torch.arange(pages, dtype=torch.int32, device=gpu)[None], ints([n], gpu)
    sa.paged_cache_append(cache, k.to(dtype), v.to(dtype), table, ints([0], gpu))
    held = sa.paged_cache_gather(cache, table, lens, length=n, dtype=dtype)[1]
    # one query value per row (sums of D equal products are exact), rows of both signs
    q = q_size * (1.0 + torch.rand(1, H * G, Sq, 1, generator=g, device=gpu))
    q = (q * torch.where(torch.rand(q.shape, generator=g, device=gpu) < 0.5, -1.0, 1.0)).to(dtype).expand(1, H * G, Sq, D).contiguous()
    see = torch.ones(1, 1, Sq, 64 * pages, dtype=torch.bool, device=gpu)
    for mask in (None, see):
        rows = ints([n + Sq - 1 if mask is None else n], gpu)  # (every row sees both keys)
        if mask is None and n + Sq - 1 > 64 * pages:
            continue
        if mask is None:
            sa.paged_cache_append(cache, k[:, :, :1].expand(1, H, Sq, D).to(dtype), v[:, :, :1].expand(1, H, Sq, D).to(dtype), table, lens)
        o, lse = sa.sparse_attention_decode_paged(q, cache, table, rows, mask, return_lse=True)
        for head in range(H * G):
            for i in range(Sq):
                x = float(q[0, head, i, 0])
                want = held[0, head // G, most if x > 0 else least]
                assert torch.equal(o[0, head, i], want)
                score = x * (4.0 if x > 0 else 1.0) * k_size * math.sqrt(D)
                # (three roundings: to the score, by the scale, back from powers of two)
                assert abs(float(lse[0, head, i]) - score) <= 4 * 2.0 ** -24 * abs(score)
