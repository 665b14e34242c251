"""verify_drafts where a part of a row, as a workgroup sums it, is longer than a thread's four values and no multiple of them: V and B that cut rows into parts of 5, 6, 7, 9, 10, 13 ...
times 1024.  The checks are test_gpu_verify's."""
import pytest
import torch

import sparseattention_amd as sa
from test_gpu_verify import TYPES, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("B,n,V", [(64, 2, 151936), (48, 2, 128256), (96, 2, 50257), (32, 2, 200000), (64, 2, 100000), (512, 2, 50257), (128, 2, 90001), (32, 4, 151936), (1100, 2, 9300),
                                   (1024, 3, 5000), (1030, 2, 31000)])
def test_sizes(gpu, dtype, drawn, B, n, V):
    p, tokens, u, parents, q = make(B + n + V, B, n, V, TYPES[dtype], drawn, sharp=2.0, wide=V % 2 == 0)
    check(p, tokens, u, parents, q)
    u[:, 1:] = 0.9999  # (after rejections, if anything)
    u[:, 0] = torch.linspace(0.0, 1.0 - 2.0 ** -24, B, device="cuda")  # (from the first token to the last)
    check(p, tokens, u, parents, q)


@pytest.mark.parametrize("B,V,each", [(64, 151936, 10240), (32, 151936, 5120), (64, 100000, 7168), (96, 50257, 5120), (1024, 31000, 31744)])
def test_rejected_tokens_stay_out(gpu, B, V, each):
    """A rejected token with most of the row's probability behind a border of 32 of its part, and the tokens around it left: none of the rejected comes out."""
    g = torch.Generator(device="cuda").manual_seed(V)
    border = 32 * torch.randint(1, each // 32, (B,), generator=g, device="cuda") + each * torch.randint(0, (V - 1) // each + 1, (B,), generator=g, device="cuda")
    border = border.clamp(max=(V - 64) // 32 * 32)
    p = torch.zeros(B, 4, V, device="cuda")
    p.scatter_(2, (border[:, None] + torch.arange(-6, 8, device="cuda"))[:, None].expand(B, 4, 14), 0.01)
    rejected = border[:, None] + torch.arange(3, device="cuda")  # (the first three bits of a word)
    p.scatter_(2, rejected[:, None].expand(B, 4, 3), 0.2)
    tokens = torch.cat([torch.zeros(B, 1, dtype=torch.int64, device="cuda"), rejected], 1)
    u = torch.full((B, 4), 0.9999, device="cuda")
    u[:, 0] = torch.rand(B, generator=g, device="cuda")
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda").expand(B, 4)
    path, accepted, token = check(p, tokens, u, parents)
    assert (accepted == 1).all() and not (token[:, None] == rejected).any()


def test_distribution(gpu):
    """Counts of 200000 draws among 5000 tokens, which a part of 5120 holds, by hundreds of tokens: within 5 standard deviations (a chance of 6e-7 each, 50 of them)."""
    B, V, g = 200000, 5000, torch.Generator(device="cuda").manual_seed(31)
    p = torch.softmax(torch.randn(V, generator=g, device="cuda"), 0)
    u = torch.rand(B, 2, generator=g, device="cuda")
    tokens = torch.randint(V, (B, 2), generator=g, device="cuda")
    path, accepted, token = sa.verify_drafts(p.expand(B, 2, V), tokens, u)
    first = torch.where(accepted > 1, tokens[:, 1], token)
    count = torch.bincount(first, minlength=V).view(50, 100).sum(1).double().cpu()
    want = p.double().cpu().view(50, 100).sum(1) / p.double().sum().cpu()
    assert ((count - B * want).abs() <= 5 * torch.sqrt(B * want * (1 - want))).all(), count - B * want
