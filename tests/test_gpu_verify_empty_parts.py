"""verify_drafts on rows most of whose parts are empty, where running sums over parts differ by a rounding between a part with probability and an empty one behind it."""
import pytest
import torch

from test_gpu_verify import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("behind", [4, 5, 7, 20, 63])
@pytest.mark.parametrize("place", [0, 700, 2047])
def test_an_empty_part_has_no_token(gpu, behind, place):
    """Parts of 2048 values, of which a tree of sums makes 2^-53 + 2^-53 + 1 up to part 2 as 1, (2^-53 + 2^-53) + (1 + 0) up to part 3 as 1 + 2^-52; half of the whole lies between."""
    p = torch.zeros(1, 1, 1 << 17, device="cuda")
    at = 2048 * torch.tensor([0, 1, 2, behind], device="cuda") + place
    p[0, 0, at] = torch.tensor([2.0 ** -53, 2.0 ** -53, 1.0, 1.0], device="cuda")
    path, accepted, token = check(p, torch.zeros(1, 1, dtype=torch.int64, device="cuda"), torch.full((1, 1), 0.5, device="cuda"))
    assert int(token) in at[2:].tolist()


def test_few_tokens_left(gpu):
    """What a cut of all but the likeliest tokens leaves: some tens of 131072, and numbers at the borders of their running sums."""
    g = torch.Generator(device="cuda").manual_seed(41)
    B, V = 64, 131072
    p = torch.zeros(B, 1, V, device="cuda")
    at = torch.randint(V, (B, 30), generator=g, device="cuda").sort(1).values
    p[:, 0].scatter_(1, at, torch.rand(B, 30, generator=g, device="cuda") ** 8)
    sums = torch.cumsum(p[:, 0].double(), 1)
    u = (sums.gather(1, at[torch.arange(B), torch.arange(B) % 30][:, None]) / sums[:, -1:]).float().clamp(max=1.0 - 2.0 ** -24)
    for step in (-1.0, 0.0, 1.0):
        check(p, torch.zeros(B, 1, dtype=torch.int64, device="cuda"), (u + step * 2.0 ** -24).clamp(0.0, 1.0 - 2.0 ** -24))
