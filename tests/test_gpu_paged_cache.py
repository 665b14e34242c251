"""The paged cache's own operators against the 64-bit reference of paged_reference.py.  What is stored, read back, copied and moved
is defined to the bit, so every comparison is for equality."""
import pytest
import torch

import sparseattention_amd as sa
from paged_reference import Sequence

pytestmark = pytest.mark.gpu


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def tables(B, width, pool, seed, dev):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pool, generator=g)[:B * width].view(B, width).to(torch.int32).to(dev)


def same(got, want):
    """Equal, NaN where NaN."""
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def check_held(cache, table, lens, seqs, dtype=torch.bfloat16):
    """seqs[b][h][0 or 1]: Sequence of K or V."""
    k, v = sa.paged_cache_gather(cache, table, lens, dtype=dtype)
    n = table.shape[1] * cache.page_size
    for which, got in enumerate((k, v)):
        want = torch.zeros(got.shape, dtype=torch.float64)
        for b, heads in enumerate(seqs):
            for h, pair in enumerate(heads):
                x = pair[which].x[:n]
                want[b, h, :len(x)] = x
        same(got, want)


def values(shape, seed, dev, dtype, grow=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(1.5 * torch.randn(shape[:-1] + (1,), generator=g))
    if grow:
        x = x * torch.exp2(grow * torch.arange(shape[2]).float())[:, None]
    return x.to(dtype).to(dev)


@pytest.mark.parametrize("D,P,dtype", [(64, 32, torch.float16), (128, 64, torch.bfloat16), (256, 128, torch.bfloat16),
                                       (80, 64, torch.float16), (128, 256, torch.bfloat16), (36, 32, torch.bfloat16)])
@pytest.mark.parametrize("steps", [(1, 1, 1, 30, 1, 40), (33, 31, 1), (70, 5), (32, 64, 1)])
def test_appends_in_steps(gpu, D, P, dtype, steps):
    """Ragged counts, starts and ends inside blocks, scales that grow while a block fills; what lies behind stays as it was."""
    B, H, width = 3, 2, 2 + 128 // P
    cache = sa.empty_paged_cache(B * width + 2, H, D, page_size=P, device=gpu)
    cache.k.fill_(0x7F)  # NaN codes everywhere: nothing of what a page held before may show
    cache.v.fill_(0xFF)
    cache.k_scales.fill_(2.0 ** 60)
    cache.v_scales.fill_(2.0 ** 60)
    table = tables(B, width, B * width + 2, 0, gpu)
    seqs = [[(Sequence(D), Sequence(D)) for _ in range(H)] for _ in range(B)]
    lens = [0] * B
    for i, S in enumerate(steps):
        counts = [S, max(S - 3, 0), S // 2]
        k, v = values((B, H, S, D), 10 * i, gpu, dtype, 0.2), values((B, H, S, D), 10 * i + 1, gpu, dtype, -0.1)
        sa.paged_cache_append(cache, k, v, table, ints(lens, gpu), None if i == 0 and S == 1 else ints(counts, gpu))
        if i == 0 and S == 1:
            counts = [S] * B
        for b in range(B):
            for h in range(H):
                seqs[b][h][0].append(k[b, h, :counts[b]])
                seqs[b][h][1].append(v[b, h, :counts[b]])
        lens = [a + c for a, c in zip(lens, counts)]
        check_held(cache, table, ints(lens, gpu), seqs)
    unused = sorted(set(range(B * width + 2)) - {int(p) for b in range(B) for p in table[b, :-(-lens[b] // P)].tolist()})
    assert (cache.k[unused] == 0x7F).all() and (cache.v[unused] == 0xFF).all() and (cache.k_scales[unused] == 2.0 ** 60).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_value_in_a_block_of_its_size(gpu, dtype):
    """All finite values of the type next to each power of two that sets their block's scale, and NaN and infinities among them."""
    D, P = 64, 64
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.float16 if dtype == torch.float16 else torch.bfloat16)
    x = bits.view(1, 32, 32, D)  # 32 heads of one block of 2048 values: codes of one sign and exponent range together
    cache = sa.empty_paged_cache(2, 32, D, page_size=P, device=gpu)
    table = ints([[1]], gpu)
    sa.paged_cache_append(cache, x.to(gpu), x.flip(1).contiguous().to(gpu), table, ints([0], gpu))
    seqs = [[(Sequence(D), Sequence(D)) for _ in range(32)]]
    for h in range(32):
        seqs[0][h][0].append(x[0, h])
        seqs[0][h][1].append(x[0, 31 - h])
    check_held(cache, table, ints([32], gpu), seqs)


def test_extremes_of_the_scale(gpu):
    D = 64
    rows = [torch.full((1, D), 0.0), torch.full((1, D), 1e-38), torch.full((1, D), 3.38e38), torch.full((1, D), 448.0), torch.full((1, D), 450.0),
            torch.full((1, D), float("inf")), torch.full((1, D), float("nan"))]
    cache = sa.empty_paged_cache(1, len(rows), D, page_size=32, device=gpu)
    x = torch.stack(rows)[None].to(torch.bfloat16).to(gpu)
    sa.paged_cache_append(cache, x, -x, ints([[0]], gpu), ints([0], gpu))
    seqs = [[(Sequence(D), Sequence(D)) for _ in rows]]
    for h in range(len(rows)):
        seqs[0][h][0].append(x[0, h])
        seqs[0][h][1].append(-x[0, h])
    check_held(cache, ints([[0]], gpu), ints([1], gpu), seqs)
    # a zero block that takes something, a large one that takes something small
    y = torch.full((1, len(rows), 1, D), 3.0, dtype=torch.bfloat16, device=gpu)
    sa.paged_cache_append(cache, y, y, ints([[0]], gpu), ints([1], gpu))
    for h in range(len(rows)):
        seqs[0][h][0].append(y[0, h])
        seqs[0][h][1].append(y[0, h])
    check_held(cache, ints([[0]], gpu), ints([2], gpu), seqs)


def test_layouts_of_new_tokens_and_tables(gpu):
    """[B,S,H,D] storage, rows that are views of wider ones, unaligned views, a table of every second column, lengths with a stride."""
    B, H, S, D, P = 2, 3, 45, 64, 32
    base = values((B, S, H, D + 8), 1, gpu, torch.bfloat16)
    odd = values((B, H, S, D + 3), 2, gpu, torch.bfloat16)
    wide = torch.full((B, 8), -1, dtype=torch.int32, device=gpu)
    wide[:, ::2] = tables(B, 4, 20, 3, gpu)
    lens = torch.zeros(B, 2, dtype=torch.int32, device=gpu)[:, 0]
    for k, v in ((base[..., :D].transpose(1, 2), odd[..., 1:D + 1]), (odd[..., 2:D + 2], base[..., 8:].transpose(1, 2)),
                 (base[:1, :, :1, :D].transpose(1, 2).expand(B, H, S, D), odd[:, :1, :, :D].expand(B, H, S, D))):
        cache = sa.empty_paged_cache(20, H, D, page_size=P, device=gpu)
        sa.paged_cache_append(cache, k, v, wide[:, ::2], lens)
        seqs = [[(Sequence(D), Sequence(D)) for _ in range(H)] for _ in range(B)]
        for b in range(B):
            for h in range(H):
                seqs[b][h][0].append(k[b, h])
                seqs[b][h][1].append(v[b, h])
        check_held(cache, wide[:, ::2], ints([S] * B, gpu), seqs)


def test_what_has_no_page_is_not_stored(gpu):
    """Entries outside the pool, tokens past the table, negative lengths and counts; the pool's other pages stay as they were."""
    D, P, H = 64, 32, 2
    cache = sa.empty_paged_cache(4, H, D, page_size=P, device=gpu)
    x = values((3, H, 100, D), 5, gpu, torch.bfloat16)
    table = ints([[0, -1, 4], [1 << 30, 1, -(1 << 31)], [2, 2, 2]], gpu)
    sa.paged_cache_append(cache, x, x, table, ints([0, 0, 96], gpu), ints([100, 100, 100], gpu))
    seqs = [[(Sequence(D), Sequence(D)) for _ in range(H)] for _ in range(3)]
    for h in range(H):
        for which in range(2):
            seqs[0][h][which].append(x[0, h, :32])
            s = Sequence(D)
            s.append(x[1, h, 32:64])
            seqs[1][h][which].x = torch.cat([torch.zeros(32, D, dtype=torch.float64), s.x])
    check_held(cache, table, ints([96, 96, 0], gpu), seqs)
    assert not cache.k[2:].any() and not cache.v_scales[2:].any()
    before = cache.k.clone()
    sa.paged_cache_append(cache, x, x, table, ints([5, -7, 2 ** 31 - 1], gpu), ints([-3, 0, 50], gpu))
    assert torch.equal(cache.k, before)
    sa.paged_cache_append(cache, x[:1], x[:1], ints([[3, 3]], gpu), ints([-7], gpu), ints([20], gpu))  # (from 0 on)
    s = Sequence(D)
    s.append(x[0, 0, :20])
    same(sa.paged_cache_gather(cache, ints([[3]], gpu), ints([20], gpu))[0][0, 0, :20], s.x)


@pytest.mark.parametrize("e", [-96, -24, -1, 7, 8, 9, 20, 21, 22, 23, 24, 25, 40, 119])
def test_every_code_in_fp16(gpu, e):
    cache = sa.empty_paged_cache(1, 1, 64, page_size=32, device=gpu)
    codes = torch.arange(256, dtype=torch.uint8, device=gpu).repeat(8)
    for t in (cache.k, cache.v):
        t.copy_(codes.view(t.shape))
    for t in (cache.k_scales, cache.v_scales):
        t.fill_(2.0 ** e)
    args = cache, ints([[0]], gpu), ints([32], gpu)
    for wide, got in zip(sa.paged_cache_gather(*args), sa.paged_cache_gather(*args, dtype=torch.float16)):
        wide = wide.double()
        held = torch.unique(wide[wide.abs() <= 65504.0].abs())
        want = torch.where(wide.abs() > 65504.0, torch.sign(wide) * held.max(), wide)
        same(got, (torch.round(want * 2.0 ** 24) * 2.0 ** -24 if e < 0 else want).half())


def test_lengths_far_out_of_range(gpu):
    """Lengths below 0 count as 0, down to the type's lowest; those past the table as what it has place for."""
    D, P, H = 64, 32, 1
    cache = filled(12, H, D, P, 30, gpu)
    table = ints([[0, 1, 2], [3, 4, 5], [6, 7, 8]], gpu)
    lens = ints([-(1 << 31), 2 ** 31 - 1, -1], gpu)
    k, v = sa.paged_cache_gather(cache, table, lens)
    whole = sa.paged_cache_gather(cache, table, ints([0, 96, 0], gpu))
    same(k, whole[0]), same(v, whole[1])
    assert not k[0].any() and not v[2].any()
    new, n = sa.paged_cache_fork(cache, table, lens, ints([0, 1, 2], gpu), ints([9, 10, 11], gpu))
    assert n.tolist() == [0, 96, 0] and new.tolist() == [[-1] * 3, [3, 4, 5], [-1] * 3]
    pages, count = sa.paged_cache_free_pages(cache, table, lens)
    assert int(count) == 9 and pages[:9].tolist() == [0, 1, 2, 6, 7, 8, 9, 10, 11]
    new, used = sa.paged_cache_compact(cache, table, lens)
    assert int(used) == 3 and new.tolist() == [[-1] * 3, [0, 1, 2], [-1] * 3]  # (3, 4, 5 to the free 0, 1, 2)
    got = sa.paged_cache_gather(cache, new, lens)
    same(got[0], whole[0]), same(got[1], whole[1])


def test_what_fp16_does_not_hold(gpu):
    """Read back as fp16, what the cache holds beyond its 65504 (65504 itself is held as 65536) becomes 61440, the largest code within the
    type, and what is below its normal numbers is rounded (to even) to its steps of 2^-24."""
    D, P = 64, 32
    cache = sa.empty_paged_cache(1, 1, D, page_size=P, device=gpu)
    x = torch.zeros(1, 1, 32, D, dtype=torch.bfloat16, device=gpu)
    x[0, 0, 0] = 2.0 ** 17
    x[0, 0, 1] = -2.0 ** 16
    x[0, 0, 2] = -448.0
    x[0, 0, 3] = float("nan")
    sa.paged_cache_append(cache, x, x, ints([[0]], gpu), ints([0], gpu))
    for got in sa.paged_cache_gather(cache, ints([[0]], gpu), ints([32], gpu), dtype=torch.float16):
        assert (got[0, 0, 0] == 61440.0).all() and (got[0, 0, 1] == -61440.0).all() and (got[0, 0, 2] == -448.0).all()
        assert torch.isnan(got[0, 0, 3]).all() and not got[0, 0, 4:].any()
    x[0, 0, 0] = 1.0 * 2.0 ** -14
    x[0, 0, 1] = -1.125 * 2.0 ** -22  # (4.5 steps of 2^-24: 4)
    x[0, 0, 2] = 1.0 * 2.0 ** -25     # (half a step: 0)
    x[0, 0, 3] = 1.5 * 2.0 ** -24     # (1.5 steps: 2)
    cache = sa.empty_paged_cache(1, 1, D, page_size=P, device=gpu)
    sa.paged_cache_append(cache, x, x, ints([[0]], gpu), ints([0], gpu))
    held = sa.paged_cache_gather(cache, ints([[0]], gpu), ints([32], gpu))[0].double()
    for got in sa.paged_cache_gather(cache, ints([[0]], gpu), ints([32], gpu), dtype=torch.float16):
        same(got, torch.round(held * 2.0 ** 24) * 2.0 ** -24)


def test_empty_calls(gpu):
    cache = sa.empty_paged_cache(4, 2, 64, page_size=32, device=gpu)
    none = torch.empty(0, dtype=torch.int32, device=gpu)
    x = torch.empty(0, 2, 3, 64, dtype=torch.bfloat16, device=gpu)
    empty_table = torch.empty(0, 2, dtype=torch.int32, device=gpu)
    sa.paged_cache_append(cache, x, x, empty_table, none)
    sa.paged_cache_append(cache, x.new_empty(1, 2, 0, 64), x.new_empty(1, 2, 0, 64), ints([[0]], gpu), ints([0], gpu))
    assert sa.paged_cache_gather(cache, empty_table, none)[0].shape == (0, 2, 64, 64)
    assert sa.paged_cache_gather(cache, ints([[0]], gpu), ints([9], gpu), length=0)[1].shape == (1, 2, 0, 64)
    sa.paged_cache_copy(cache, none, none)
    assert sa.paged_cache_fork(cache, ints([[0]], gpu), ints([9], gpu), none, none)[0].shape == (0, 1)
    table, used = sa.paged_cache_compact(cache, empty_table, none)
    assert table.shape == (0, 2) and used.item() == 0
    pages, count = sa.paged_cache_free_pages(cache, empty_table, none)
    assert pages.tolist() == [0, 1, 2, 3] and count.item() == 4
    assert sa.sparse_attention_decode_paged(x, cache, empty_table, none).shape == (0, 2, 3, 64)


def filled(pool, H, D, P, seed, dev):
    """A pool of random codes and scales."""
    g = torch.Generator(device=dev).manual_seed(seed)
    cache = sa.empty_paged_cache(pool, H, D, page_size=P, device=dev)
    for t in (cache.k, cache.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device=dev, dtype=torch.uint8))
    for t in (cache.k_scales, cache.v_scales):
        t.copy_(torch.exp2(torch.randint(-20, 20, t.shape, generator=g, device=dev).float()))
    return cache


def parts(cache):
    return cache.k, cache.v, cache.k_scales, cache.v_scales


@pytest.mark.parametrize("H,D,P", [(1, 64, 32), (3, 128, 64), (2, 256, 256)])
def test_copy(gpu, H, D, P):
    cache = filled(12, H, D, P, 0, gpu)
    want = [t.clone() for t in parts(cache)]
    src, dst = [0, 1, -1, 2, 12, 0, 3, 5, 1, 99], [6, 7, 8, 7, 9, 8, -1, 5, 10, 7]
    for s, d in zip(src, dst):
        if 0 <= s < 12 and 0 <= d < 12:
            for t in want:
                t[d] = t[s]
    sa.paged_cache_copy(cache, ints(src, gpu), ints(dst, gpu))
    for got, w in zip(parts(cache), want):
        assert torch.equal(got, w)


@pytest.mark.parametrize("H", [2, 5])
def test_copy_of_many(gpu, H):
    n = 700
    cache = filled(2 * n, H, 64, 32, 1, gpu)
    order = torch.randperm(2 * n, generator=torch.Generator().manual_seed(2)).to(torch.int32).to(gpu)
    src, dst = order[:n], order[n:].clone()
    dst[:300] = dst[300:600]  # named again
    want = [t.clone() for t in parts(cache)]
    for t in want:
        t[dst[300:].long()] = t[src[300:].long()]
    sa.paged_cache_copy(cache, src, dst)
    for got, w in zip(parts(cache), want):
        assert torch.equal(got, w)


def plain_fork(cache, table, lens, parents, new_pages):
    """(table, lens, copies) of a fork: copies are (source, destination, blocks) that take place, in order."""
    P, width = cache.page_size, len(table[0])
    rows, out, copies = [], [], {}
    for i, b in enumerate(parents):
        n = min(max(lens[b], 0), width * P) if 0 <= b < len(table) else 0
        full, tail = divmod(n, P)
        row = table[b][:full] if n else []
        if tail:
            old, new = table[b][full], new_pages[i]
            ok = 0 <= new < cache.num_pages and 0 <= old < cache.num_pages and old != new
            if ok:
                copies[new] = (old, -(-tail // 32))
            row = row + [new if ok else old]
        rows.append(row + [-1] * (width - len(row)))
        out.append(n)
    return rows, out, copies


def test_fork(gpu):
    P, width = 64, 4
    cache = filled(40, 3, 64, P, 3, gpu)
    table = [[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11], [12, -1, 99, 13]]
    lens = [130, 128, 0, 200]
    parents = [0, 0, 1, 2, 3, 4, -1, 0, 3, 0, 2]
    new_pages = [20, 21, 22, 23, 24, 25, 26, -1, 40, 20, 21]
    lens[3] = 256 + 5  # longer than the table: as long as the table
    rows, out, copies = plain_fork(cache, table, lens, parents, new_pages)
    want = [t.clone() for t in parts(cache)]
    for new, (old, blocks) in copies.items():
        for t in want:
            t[new, :, :blocks] = t[old, :, :blocks]
    new_table, new_lens = sa.paged_cache_fork(cache, ints(table, gpu), ints(lens, gpu), ints(parents, gpu), ints(new_pages, gpu))
    assert new_table.tolist() == rows and new_lens.tolist() == out
    for got, w in zip(parts(cache), want):
        assert torch.equal(got, w)


def test_fork_of_many(gpu):
    P, width, B, n = 32, 3, 6, 900
    cache = filled(2000, 5, 64, P, 31, gpu)
    table = torch.arange(B * width).view(B, width).tolist()
    lens = [70, 33, 1, 0, 96, 64]
    parents = [(7 * i) % 8 - 1 for i in range(n)]
    new_pages = [100 + (i if i % 9 else i // 2) for i in range(n)]  # some of them twice
    rows, out, copies = plain_fork(cache, table, lens, parents, new_pages)
    want = [t.clone() for t in parts(cache)]
    for t in want:
        t[list(copies)] = t[[old for old, _ in copies.values()]]  # (a page is one block)
    new_table, new_lens = sa.paged_cache_fork(cache, ints(table, gpu), ints(lens, gpu), ints(parents, gpu), ints(new_pages, gpu))
    assert new_table.tolist() == rows and new_lens.tolist() == out
    for got, w in zip(parts(cache), want):
        assert torch.equal(got, w)


@pytest.mark.parametrize("pool,B,width,P", [(1, 1, 1, 32), (31, 2, 3, 64), (33, 5, 6, 32), (1000, 7, 60, 32), (40000, 33, 700, 64), (1 << 20, 64, 512, 32),
                                            (8193, 5000, 1, 32), (20000, 3, 2500, 32), (16385, 40, 1024, 64)])
def test_compact_and_free(gpu, pool, B, width, P):
    g = torch.Generator().manual_seed(pool)
    H, D = 1, 64
    many = pool > 2000
    if many:  # (codes of few distinct values: the comparison is of page numbers written into the pages)
        cache = sa.empty_paged_cache(pool, H, D, page_size=P, device=gpu)
        cache.k_scales.copy_(torch.arange(pool, device=gpu).view(pool, 1, 1).expand_as(cache.k_scales))
        cache.v_scales.copy_(cache.k_scales + 0.5)
        cache.k.view(torch.int32).copy_(torch.arange(pool, device=gpu, dtype=torch.int32).view(pool, 1, 1, 1).expand_as(cache.k.view(torch.int32)))
        cache.v.copy_(cache.k)
    else:
        cache = filled(pool, H, D, P, 5, gpu)
    table = torch.randint(-2, pool + 2, (B, width), generator=g, dtype=torch.int32)
    lens = torch.randint(-5, width * P + 40, (B,), generator=g, dtype=torch.int32)
    lens[0] = width * P
    used = (torch.arange(width)[None] * P) < lens[:, None]
    named = table[used & (table >= 0) & (table < pool)].unique().tolist()
    L = len(named)
    pages, count = sa.paged_cache_free_pages(cache, table.to(gpu), lens.to(gpu))
    free = torch.ones(pool, dtype=torch.bool)
    free[named] = False
    free = free.nonzero()[:, 0].tolist()
    assert count.item() == pool - L and pages.tolist() == free + [-1] * L
    holes, movers = [p for p in free if p < L], [p for p in named if p >= L]
    assert len(holes) == len(movers)
    before = [t.clone() for t in parts(cache)]
    for t in before:
        if holes:
            t[holes] = t[movers]
    given = table.to(gpu)
    new_table, n = sa.paged_cache_compact(cache, given, lens.to(gpu))
    assert n.item() == L and torch.equal(given.cpu(), table)
    to = torch.arange(pool, dtype=torch.int32)
    to[movers] = torch.tensor(holes, dtype=torch.int32)
    ok = used & (table >= 0) & (table < pool)
    assert torch.equal(new_table.cpu(), torch.where(ok, to[table.clamp(0, pool - 1).long()], -1))
    for got, w in zip(parts(cache), before):
        assert torch.equal(got, w)


def test_more_than_4_gib_of_codes(gpu):
    """Offsets past 32 bits, in the pool's bytes and in the rows read back."""
    P, H, D = 256, 16, 128
    pool = (5 << 30) // (P * H * D)
    cache = sa.empty_paged_cache(pool, H, D, page_size=P, device=gpu)
    x = values((1, H, 300, D), 7, gpu, torch.bfloat16)
    table = ints([[pool - 1, pool - 2]], gpu)
    sa.paged_cache_append(cache, x, x, table, ints([0], gpu))
    s = Sequence(D)
    s.append(x[0, H - 1])
    k, v = sa.paged_cache_gather(cache, table, ints([300], gpu), length=300)
    same(k[0, H - 1], s.x)
    same(v[0, H - 1], s.x)
    sa.paged_cache_copy(cache, ints([pool - 1], gpu), ints([3], gpu))
    assert torch.equal(cache.v[3], cache.v[pool - 1]) and cache.v[3].any()
    q = torch.randn(1, H, 1, D, device=gpu).to(torch.bfloat16)
    a = sa.sparse_attention_decode_paged(q, cache, table, ints([300], gpu))
    b = sa.sparse_attention_decode_paged(q, cache, ints([[3, pool - 2]], gpu), ints([300], gpu))
    assert torch.equal(a, b) and a.abs().sum() > 0


def test_refusals(gpu):
    cache = sa.empty_paged_cache(4, 2, 64, page_size=32, device=gpu)
    table, lens = ints([[0, 1]], gpu), ints([0], gpu)
    x = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16, device=gpu)
    for k, v in ((x[:, :1], x[:, :1]), (x, x[:, :, :2]), (x[..., :32], x[..., :32]), (x[0], x[0]), (x.cpu(), x), (x.expand(2, 2, 3, 64), x.expand(2, 2, 3, 64))):
        with pytest.raises(ValueError):
            sa.paged_cache_append(cache, k, v, table, lens)
    for k, v in ((x.float(), x.float()), (x, x.half())):
        with pytest.raises(TypeError):
            sa.paged_cache_append(cache, k, v, table, lens)
    for t, n in ((table.long(), lens), (table, lens.long()), (table.cpu(), lens), (table, lens.cpu()), (table[0], lens), (table, lens[0]), (table[:, :0], lens),
                 (table, ints([0, 0], gpu))):
        for call in (lambda: sa.paged_cache_append(cache, x, x, t, n), lambda: sa.paged_cache_gather(cache, t, n),
                     lambda: sa.paged_cache_compact(cache, t, n), lambda: sa.paged_cache_free_pages(cache, t, n),
                     lambda: sa.paged_cache_fork(cache, t, n, lens, lens), lambda: sa.sparse_attention_decode_paged(x, cache, t, n)):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(TypeError):
        sa.paged_cache_gather(cache, table, lens, dtype=torch.float32)
    with pytest.raises(ValueError):
        sa.paged_cache_gather(cache, table, lens, length=-1)
    with pytest.raises(ValueError):
        sa.paged_cache_copy(cache, ints([0, 1], gpu), ints([2], gpu))
    with pytest.raises(ValueError):
        sa.paged_cache_fork(cache, table, lens, ints([0, 0], gpu), ints([2], gpu))
    for bad in (dict(k=cache.k[:, :, :, :1024]), dict(v=cache.v[:2]), dict(k_scales=cache.k_scales.double()), dict(v_scales=cache.v_scales.cpu()), dict(head_dim=65),
                dict(k=cache.k.to(torch.int8))):
        with pytest.raises(ValueError):
            sa.paged_cache_gather(sa.PagedCache(**{**cache.__dict__, **bad}), table, lens)
