"""Batches of so many sequences, or lists, that a launch in front finds where each begins: with several tiles of query rows per K/V head, windows,
padding, sequences of nothing; against the 64-bit reference."""
import pytest
import torch

import sparseattention_amd as sa
from test_gpu_paged_decode import check, ints, make, masks, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,H,G,D,P,Sq,top,window,dtype", [
    (257, 2, 5, 64, 32, 8, 200, None, torch.bfloat16),     # 40 rows of a K/V head: two tiles
    (300, 1, 9, 128, 32, 8, 150, 40, torch.float16),       # three
    (520, 2, 4, 64, 64, 16, 90, 33, torch.bfloat16),
    (4100, 1, 11, 64, 32, 3, 70, None, torch.float16),     # units by more than 64 x 64
    (270, 1, 34, 256, 64, 1, 130, None, torch.bfloat16),
    (300, 2, 1, 128, 32, 1, 260, 100, torch.bfloat16),
])
def test_sequences(gpu, B, H, G, D, P, Sq, top, window, dtype):
    lens = [(37 * b) % top if b % 7 else 0 for b in range(B)]
    lens[B // 2] = 20 * top  # (one is many pieces)
    counts = [(b * 5) % (Sq + 1) for b in range(B)]
    cache, table = make(B, H, D, P, lens, dtype, 50, gpu)
    q = queries(B, H * G, Sq, D, dtype, 51, gpu)
    for c in (None, counts):
        args = {"window": window, "counts": None if c is None else ints(c, gpu)}
        o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), return_lse=True, **args)
        check(cache, table, lens, q, o, lse, counts=c, window=window)


def test_all_of_nothing(gpu):
    cache, table = make(400, 2, 64, 32, [40] * 400, torch.bfloat16, 52, gpu)
    q = queries(400, 10, 8, 64, torch.bfloat16, 53, gpu)
    for lens, counts in (([0] * 400, None), ([40] * 400, [0] * 400), ([40] * 399 + [0], [0] * 399 + [3])):
        o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), counts=None if counts is None else ints(counts, gpu), return_lse=True)
        assert not o.any() and (lse == -float("inf")).all()


@pytest.mark.parametrize("kind", ["tiles", "rows", "none", "all"])
@pytest.mark.parametrize("B,H,G,D,P,Sq,Sk,dtype", [(23, 3, 5, 64, 32, 8, 320, torch.bfloat16), (70, 1, 3, 128, 64, 16, 192, torch.float16),
                                                   (9, 8, 40, 64, 32, 1, 256, torch.bfloat16), (33, 2, 3, 256, 32, 12, 96, torch.bfloat16)])
def test_lists(gpu, kind, B, H, G, D, P, Sq, Sk, dtype):
    lens = [(Sk - 7, Sk // 2 + 3, 0, Sk)[b % 4] for b in range(B)]
    counts = [(Sq, 0, Sq - 1, 1)[b % 4 if b % 3 else 0] for b in range(B)]
    cache, table = make(B, H, D, P, lens, dtype, 54, gpu, width=Sk // P + 1)
    q = queries(B, H * G, Sq, D, dtype, 55, gpu)
    see = masks(kind, B, H, Sq, Sk, P, 56)
    md = sa.compute_mask_kernel(see.to(gpu), Sq, P)
    for c in (None, counts):
        o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), mask_metadata=md, counts=None if c is None else ints(c, gpu), return_lse=True)
        check(cache, table, lens, q, o, lse, see=see, counts=c)


def test_few_and_many_are_alike(gpu):
    """A batch of 300, and the same sequences by 100, which find their pieces themselves (cut elsewhere, so not alike to the bit)."""
    B, Sq, D = 300, 8, 64
    lens = [(91 * b) % 700 for b in range(B)]
    cache, table = make(B, 2, D, 32, lens, torch.bfloat16, 57, gpu)
    q = queries(B, 10, Sq, D, torch.bfloat16, 58, gpu)
    n = ints(lens, gpu)
    whole = sa.sparse_attention_decode_paged(q, cache, table, n, window=300)
    check(cache, table, lens, q, whole, window=300)
    for at in (0, 100, 200):
        part = slice(at, at + 100)
        o = sa.sparse_attention_decode_paged(q[part], cache, table[part], n[part], window=300)
        check(cache, table[part], lens[part], q[part], o, window=300)
