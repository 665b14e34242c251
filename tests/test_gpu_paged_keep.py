"""paged_cache_keep: what the cache holds afterwards, to the bit, against the rule for its scales and roundings in 64 bits."""
import math

import pytest
import torch

import sparseattention_amd as sa
from paged_reference import EXP_MIN, exponent_of, held_at

pytestmark = pytest.mark.gpu


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(seed, B, H, D, P, lens, n, spread=3.0, dtype=torch.bfloat16):
    """Sequences of lens[b] tokens and n drafts behind them, with magnitudes that differ from token to token."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = max(1, -(-(max(lens) + n) // P)) + 1
    cache = sa.empty_paged_cache(B * width + 2, H, D, page_size=P)
    table = torch.randperm(B * width + 2, generator=g, device="cuda")[:B * width].int().view(B, width)
    m = max(lens) + n
    x = [(torch.randn(B, H, m, D, generator=g, device="cuda") * torch.exp(spread * torch.randn(B, H, m, 1, generator=g, device="cuda"))).to(dtype) for _ in range(2)]
    start = torch.zeros(B, dtype=torch.int32, device="cuda")
    sa.paged_cache_append(cache, *x, table, start, counts=ints(*lens))
    for b, a in enumerate(lens):  # (behind what is held, as a step stores them)
        sa.paged_cache_append(cache, *(t[b:b + 1, :, a:a + n] for t in x), table[b:b + 1], ints(a))
    return cache, table


def held(cache, table):
    """k and v [B,H,tokens,D] in 64 bits and the blocks' exponents [B,H,blocks] (0 where there is no page)."""
    n = table.shape[1] * cache.page_size
    values = [t.double().cpu() for t in sa.paged_cache_gather(cache, table, ints(*[n] * len(table)))]
    ok = (table >= 0) & (table < cache.num_pages)
    exps = []
    for s in (cache.k_scales, cache.v_scales):
        e = torch.round(torch.log2(s[torch.where(ok, table, 0).long()].clamp(min=2.0 ** EXP_MIN)))  # [B, pages, H, per]
        exps.append(e.permute(0, 2, 1, 3).flatten(2).long().cpu())
    return values, exps, ok.cpu()


def expect(x, exps, ok, per_page, length, path, n):
    """One head's tokens [N,D] and exponents after the call: the rows [0, length + len(path)) that are defined."""
    x, exps = x.clone(), exps.clone()
    N = x.shape[0]
    there = lambda t: t < N and bool(ok[t // per_page])  # noqa: E731
    moves = {length + i: length + s for i, s in enumerate(path) if 0 <= s < n and there(length + s) and there(length + i)}
    out, end = x.clone(), min(length + len(path), N)
    for block in range(length // 32, (end + 31) // 32):
        lo, hi = block * 32, min(block * 32 + 32, end)
        rows = list(range(lo, hi))
        come = [moves.get(t, t) for t in rows]
        if not there(lo) or come == rows:
            continue
        foreign = [s for t, s in zip(rows, come) if s // 32 != block]
        e = int(exps[block]) if len(foreign) < len(rows) else EXP_MIN
        if foreign:
            e = max(e, exponent_of(x[foreign]))
        out[lo:hi] = held_at(x[come], e)
        exps[block] = e
    return out[:end], exps


def check(cache, table, lens, paths, n, accepted=None):
    B = len(lens)
    before, exps, ok = held(cache, table)
    path = torch.full((B, n), -1, dtype=torch.int32)
    for b, q in enumerate(paths):
        path[b, :len(q)] = torch.tensor(q, dtype=torch.int32)
    count = [len(q) for q in paths] if accepted is None else accepted
    sa.paged_cache_keep(cache, table, ints(*lens), path.cuda(), ints(*count))
    after, exps_after, _ = held(cache, table)
    for i in range(2):
        for b in range(B):
            m = min(max(count[b], 0), n)
            for h in range(cache.num_heads):
                want, e = expect(before[i][b, h], exps[i][b, h], ok[b], cache.page_size, max(lens[b], 0), path[b, :m].tolist(), n)
                got = after[i][b, h, :len(want)]
                assert torch.equal(torch.nan_to_num(got, 1e300), torch.nan_to_num(want, 1e300)), (i, b, h)
                blocks = -(-len(want) // 32)
                live = ok[b].repeat_interleave(cache.page_size // 32)[:blocks]
                assert torch.equal(exps_after[i][b, h, :blocks][live], e[:blocks][live]), (i, b, h)


def paths_of(seed, B, n):
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(B):
        k = int(torch.randint(1, n + 1, (1,), generator=g))
        out.append([0] + sorted((torch.randperm(n - 1, generator=g)[:k - 1] + 1).tolist()) if n > 1 else [0])
    return out


@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("P", [32, 64, 256])
@pytest.mark.parametrize("n", [1, 2, 8, 33, 64])
def test_paths(gpu, D, P, n):
    lens = [0, 1, 17, 31, 32, 33, 63, 100]
    cache, table = make(n, 8, 2, D, P, lens, n)
    check(cache, table, lens, paths_of(n + D, 8, n), n)


@pytest.mark.parametrize("spread", [0.0, 1.0, 12.0])
def test_scales_that_grow_and_shrink(gpu, spread):
    """Tokens from blocks of far larger and far smaller scales."""
    lens = [0, 20, 31, 5]
    cache, table = make(1, 4, 2, 64, 32, lens, 64, spread)
    check(cache, table, lens, [[0, 63], [0, 30, 40, 50, 60], [1, 33, 34, 63], [40, 41, 42]], 64)
    cache, table = make(2, 4, 2, 64, 32, lens, 64, spread)
    cache.k_scales[table[:, 1].long()] *= 2.0 ** 20
    cache.v_scales[table[:, 2].long()] *= 2.0 ** -30
    check(cache, table, lens, paths_of(3, 4, 64), 64)


def test_every_code(gpu):
    """All codes, NaN among them, from one block to another: as they are where the scales agree, and across the largest distance of scales."""
    for e0, e1 in ((0, 0), (3, 0), (0, 3), (119, -96), (-96, 119), (7, -9)):
        cache = sa.empty_paged_cache(3, 1, 256, page_size=32)
        table = ints(0, 1)[None]
        for t in (cache.k, cache.v):
            t.copy_(torch.randint(0, 256, t.shape, device="cuda", dtype=torch.uint8))
        for s in (cache.k_scales, cache.v_scales):
            s[0], s[1], s[2] = 2.0 ** e0, 2.0 ** e1, 1.0
        check(cache, table, [16], [[0, 20, 21, 2, 45, 3]], 46)


def test_orders_and_repeats(gpu):
    """Nodes in any order, one for several places: all are read before any is written."""
    lens = [10, 30]
    cache, table = make(4, 2, 2, 64, 32, lens, 40)
    check(cache, table, lens, [[5, 4, 3, 2, 1, 0], [39, 39, 0, 0, 20]], 40)


def test_entries_that_are_none(gpu):
    lens, n = [25, 0, 31, 7, -4], 20
    cache, table = make(5, 5, 2, 64, 32, [max(x, 0) for x in lens], n)
    check(cache, table, lens, [[0, -1, 5, 20, 6], [1 << 30, 3, -(1 << 31)], [], [0, 1, 2], [3, 4]], n)
    check(cache, table, lens, [[4, 5, 6], [1, 2], [9], [3], [2]], n, accepted=[-1, 0, 1, 1, 2])
    path = ints(*range(1, 20), 0)[None].expand(5, 20)
    before = cache.k.clone()
    sa.paged_cache_keep(cache, table, ints(*lens), path, ints(0, 0, 0, 0, 0))
    assert torch.equal(cache.k, before)
    identity = ints(*range(20))[None].expand(5, 20)
    sa.paged_cache_keep(cache, table, ints(*lens), identity, ints(20, 3, 99, 0, 20))
    assert torch.equal(cache.k, before)


def test_pages_that_do_not_exist(gpu):
    lens, n = [20, 50, 60], 64
    cache, table = make(6, 3, 2, 64, 32, lens, n)
    table[0, 1], table[1, 2], table[2, 3] = -1, cache.num_pages, -9
    spare = torch.ones(cache.num_pages, dtype=torch.bool, device="cuda")
    spare[table[(table >= 0) & (table < cache.num_pages)].long()] = False
    before = cache.v[spare].clone()
    check(cache, table, lens, [[0, 20, 30, 44], list(range(0, 64, 2)), [1, 40, 50]], n)
    assert torch.equal(cache.v[spare], before)
    short = table[:, :2].contiguous()  # (drafts and places past the table)
    check(cache, short, [20, 50, 2 ** 31 - 1], [[0, 5, 60], [1, 2, 30], [3, 4]], n)


def test_no_other_page_changes(gpu):
    lens = [40, 90]
    cache, table = make(7, 2, 3, 64, 32, lens, 30)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)]
    sa.paged_cache_keep(cache, table, ints(*lens), ints(*([0, 10, 20] + [-1] * 27))[None].expand(2, 30), ints(3, 3))
    touched = table[[0, 1], [1, 2]].long().tolist()
    for a, b in zip(before, (cache.k, cache.v, cache.k_scales, cache.v_scales)):
        changed = (a != b).flatten(1).any(1).nonzero().flatten().tolist()
        assert set(changed) <= set(touched)


def test_captured_and_replayed(gpu):
    lens, n = ints(30, 3), 12
    cache, table = make(8, 2, 2, 64, 32, [60, 60], n)
    path, accepted = ints(0, 3, 5, 11, *[-1] * 8)[None].repeat(2, 1), ints(4, 2)
    pristine = [t.clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)]
    tensors = (cache.k, cache.v, cache.k_scales, cache.v_scales)
    step = lambda: sa.paged_cache_keep(cache, table, lens, path, accepted)  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        results = []
        for way in (graph.replay, step):
            for t, x in zip(tensors, pristine):
                t.copy_(x)
            way()
            torch.cuda.synchronize()
            results.append([t.clone() for t in tensors])
        assert all(torch.equal(a, b) for a, b in zip(*results)), i
        lens += 9
        path[:, 1:4] = ints(2 + i, 6 + i, 8 + i)


def test_refusals(gpu):
    cache, table = make(9, 2, 2, 64, 32, [4, 4], 5)
    path, lens = torch.zeros(2, 5, dtype=torch.int32, device="cuda"), ints(4, 4)
    for bad in (dict(path=path.long()), dict(path=path[:1]), dict(path=path[0]), dict(path=path.cpu()), dict(path=torch.zeros(2, 65, dtype=torch.int32, device="cuda")),
                dict(accepted=lens[:1]), dict(accepted=lens.long()), dict(lens=lens[:1])):
        with pytest.raises(ValueError):
            sa.paged_cache_keep(cache, table, **{**dict(lens=lens, path=path, accepted=lens), **bad})
    sa.paged_cache_keep(cache, table, lens, path[:, :0], lens)
