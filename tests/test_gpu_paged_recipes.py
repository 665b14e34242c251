"""The calls that the module's documentation shows, run as they stand there, with grouped heads and without."""
import textwrap

import pytest
import torch

import sparseattention_amd as sa
from sparseattention_amd import paged_cache
from test_gpu_paged_decode import check, ints, queries

pytestmark = pytest.mark.gpu


def recipes():
    """The indented blocks of the module's docstring."""
    blocks, lines = [], []
    for line in paged_cache.__doc__.splitlines() + [""]:
        if line.startswith("    "):
            lines.append(line)
        elif lines:
            blocks.append(textwrap.dedent("\n".join(lines)))
            lines = []
    return blocks


@pytest.mark.parametrize("G", [1, 4])
def test_a_step_and_a_chunk(gpu, G):
    step, chunk = recipes()
    B, H, D, P, n = 2, 2, 64, 32, 128
    g = torch.Generator(device=gpu).manual_seed(0)
    cache = sa.empty_paged_cache(B * 8, H, D, page_size=P, device=gpu)
    page_table = torch.arange(B * 8, dtype=torch.int32, device=gpu).view(B, 8)
    held = [77, 128]
    k, v = (torch.randn(B, H, 128, D, generator=g, device=gpu).bfloat16() for _ in range(2))
    sa.paged_cache_append(cache, k, v, page_table, ints([0] * B, gpu), ints(held, gpu))
    lens = ints(held, gpu)
    # a chunk of 128 rows behind what the sequences hold
    k, v = (torch.randn(B, H, n, D, generator=g, device=gpu).bfloat16() for _ in range(2))
    at = torch.arange(8 * P, device=gpu)
    mask = (at <= lens[:, None, None] + torch.arange(n, device=gpu)[:, None])[:, None].expand(B, H * G, n, 8 * P)
    names = dict(vars(sa), cache=cache, page_table=page_table, lens=lens, n=n, k=k, v=v, q=queries(B, H * G, n, D, torch.bfloat16, 1, gpu), mask=mask,
                 BLOCK_Q=128, BLOCK_K=32)
    exec(chunk, names)
    o, q = names["o"], names["q"]
    for i in (0, 77, n - 1):  # (that row alone from the pages; bound of the prompt kernels' parity)
        row = sa.sparse_attention_decode_paged(q[:, :, i:i + 1], cache, page_table, lens + i + 1)
        assert float((o[:, :, i:i + 1].float() - row.float()).abs().max()) < 2e-2
    # and a step of one token
    lens = lens + n - 5
    k, v = (torch.randn(B, H, 1, D, generator=g, device=gpu).bfloat16() for _ in range(2))
    q = queries(B, H * G, 1, D, torch.bfloat16, 2, gpu)
    names = dict(vars(sa), cache=cache, page_table=page_table, lens=lens, k=k, v=v, q=q)
    exec(step, names)
    check(cache, page_table, (lens + 1).tolist(), q, names["o"])
