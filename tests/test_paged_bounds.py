"""How far what the paged cache holds is from the tokens: the bounds that PagedCache states, on the 64-bit restatement that its kernels equal to the
bit."""
import random

import pytest
import torch

from paged_reference import Sequence


def scales(s, n):
    return torch.tensor([2.0 ** s.exps[t // 32] for t in range(n)], dtype=torch.float64)[:, None]


@pytest.mark.parametrize("seed", range(6))
def test_stored_at_once(seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(96, 64, generator=g) * torch.exp2(torch.randint(-30, 30, (96, 64), generator=g).float())).bfloat16()
    s = Sequence(64)
    s.append(x)
    x = x.double()
    assert ((s.x - x).abs() <= torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 * scales(s, 96))).all()


@pytest.mark.parametrize("seed", range(12))
def test_stored_one_by_one(seed):
    """Tokens that grow on the way, so that what is held is rounded again and again."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    s, xs, size = Sequence(64), [], 1.0
    for _ in range(64):
        x = (torch.randn(1, 64, generator=g) * size * torch.exp2(-8 * torch.rand(1, 64, generator=g))).bfloat16()
        s.append(x)
        xs.append(x.double())
        size *= 2.0 ** rng.choice([0, 0, 1, 1, 2, -1])
    x = torch.cat(xs)
    assert ((s.x - x).abs() < 2.0 ** -4 * x.abs() + 2.0 ** -9 * scales(s, 64)).all()


def test_a_block_that_grows_exceeds_the_bound_of_one_rounding():
    """1.8203125 behind which tokens double: the second bound is needed, and holds."""
    s, x = Sequence(64), torch.full((1, 64), 1.8203125, dtype=torch.float64)
    s.append(x)
    for i in range(1, 31):
        s.append(torch.full((1, 64), 2.0 ** i, dtype=torch.float64) * 1.5)
        off, scale = float((s.x[0] - x[0]).abs().max()), 2.0 ** s.exps[0]
        assert off < 2.0 ** -4 * 1.8203125 + 2.0 ** -9 * scale
        if s.exps[0] == 7:
            assert off == 2.0 - 1.8203125 > max(2.0 ** -4 * 1.8203125, 2.0 ** -10 * scale)


def test_the_largest_scale():
    top = torch.finfo(torch.bfloat16).max
    s = Sequence(64)
    s.append(torch.tensor([[top, -top, 2.9e38, 1.0] * 16], dtype=torch.bfloat16))
    assert s.exps == [119] and s.x[0, 0] == 448 * 2.0 ** 119 == -s.x[0, 1]
    assert 0.12 < 1 - float(s.x[0, 0]) / top < 0.13 and abs(float(s.x[0, 2]) - 2.9e38) <= 2.0 ** -4 * 2.9e38
