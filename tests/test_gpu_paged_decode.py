"""sparse_attention_decode_paged against a 64-bit attention over what the cache holds (read back by paged_cache_gather, which
test_gpu_paged_cache.py holds to the bit), within bounds counted in paged_reference.tolerances."""
import pytest
import torch

import sparseattention_amd as sa
from paged_reference import attention, tolerances

pytestmark = pytest.mark.gpu


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def make(B, H, D, P, lens, dtype, seed, dev, width=None, stale=True):
    """A cache that holds lens[b] tokens of every sequence, its other codes NaN."""
    width = width or max(1, -(-max(lens) // P))
    g = torch.Generator(device=dev).manual_seed(seed)
    pool = B * width + 3
    cache = sa.empty_paged_cache(pool, H, D, page_size=P, device=dev)
    if stale:
        for t in (cache.k, cache.v):
            t.fill_(0x7F)
        for t in (cache.k_scales, cache.v_scales):
            t.fill_(2.0 ** 100)
    table = torch.randperm(pool, generator=g, device=dev)[:B * width].view(B, width).to(torch.int32)
    n = max(1, max(lens))
    k, v = (torch.randn(B, H, n, D, generator=g, device=dev) * torch.exp(torch.randn(1, H, n, 1, generator=g, device=dev)) for _ in range(2))
    sa.paged_cache_append(cache, k.to(dtype), v.to(dtype), table, torch.zeros(B, dtype=torch.int32, device=dev), ints(lens, dev))
    return cache, table


def queries(B, Hq, Sq, D, dtype, seed, dev, size=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (size * torch.randn(B, Hq, Sq, D, generator=g, device=dev)).to(dtype)


def check(cache, table, lens, q, o, lse=None, see=None, counts=None, window=None):
    """see: bool [B,H,Sq,Sk] or None for causal rows."""
    B, Hq, Sq, D = q.shape
    H, n = cache.num_heads, table.shape[1] * cache.page_size
    k, v = (t.double().cpu() for t in sa.paged_cache_gather(cache, table, ints([n] * B, q.device)))
    ok = ((table >= 0) & (table < cache.num_pages)).cpu().repeat_interleave(cache.page_size, 1)
    assert o.shape == q.shape and o.dtype == q.dtype
    for b in range(B):
        m = min(max(lens[b], 0), n)
        rows = Sq if counts is None else min(max(counts[b], 0), Sq)
        for h in range(H):
            at = torch.arange(m)
            if see is None:
                last = m - rows + torch.arange(Sq)[:, None]
                s = at <= last
                if window is not None:
                    s = s & (at > last - window)
            else:
                s = torch.zeros(Sq, m, dtype=torch.bool)
                got = see[b, h, :, :m].cpu()
                s[:, :got.shape[1]] = got
            s = s & ok[b, :m]
            s[rows:] = False
            G = Hq // H
            qq = q[b, h * G:(h + 1) * G].double().cpu().reshape(G * Sq, D)
            want, wl, size, arg = attention(qq, k[b, h, :m], v[b, h, :m], s.repeat(G, 1))
            vmax = float(v[b, h, :m].nan_to_num(0.0).abs().max()) if m else 0.0
            tol, tol_l = tolerances(want, wl, size, arg, m, vmax, D, q.dtype)
            got = o[b, h * G:(h + 1) * G].double().cpu().reshape(G * Sq, D)
            assert torch.equal(torch.isnan(got), torch.isnan(want)), (b, h)
            off = ((got - want).abs() - tol).nan_to_num(0.0)
            assert float(off.max()) <= 0.0, (b, h, float(off.max()), float((got - want).abs().nan_to_num(0.0).max()))
            if lse is not None:
                gl = lse[b, h * G:(h + 1) * G].double().cpu().reshape(-1)
                dead = ~s.any(-1).repeat(G)
                assert (gl[dead] == -float("inf")).all() and (got[dead] == 0).all()
                off = ((gl - wl).abs() - tol_l)[~dead].nan_to_num(0.0)
                assert off.numel() == 0 or float(off.max()) <= 0.0, (b, h, float(off.max()))


@pytest.mark.parametrize("B,H,G,D,P,Sq,lens,dtype", [
    (1, 1, 1, 64, 32, 1, [1], torch.bfloat16),
    (4, 2, 1, 128, 64, 1, [0, 1, 31, 32], torch.bfloat16),
    (5, 2, 4, 128, 32, 1, [33, 64, 65, 300, 1000], torch.float16),
    (3, 1, 7, 64, 128, 5, [4, 5, 777], torch.bfloat16),
    (2, 3, 2, 256, 64, 3, [100, 515], torch.float16),
    (2, 2, 8, 128, 256, 32, [20, 700], torch.bfloat16),
    (2, 2, 3, 80, 64, 2, [129, 3], torch.bfloat16),
    (1, 1, 2, 36, 32, 2, [70], torch.float16),
    (1, 2, 4, 128, 64, 1, [20011], torch.bfloat16),
    (1, 1, 1, 64, 32, 17, [9000], torch.float16),
    (1, 1, 2, 64, 64, 3, [131077], torch.bfloat16),  # (a plane of more than 64 parts)
    (40, 8, 1, 64, 64, 1, [37 * i % 1501 for i in range(40)], torch.bfloat16),
    (130, 1, 3, 64, 32, 1, [53 * i % 200 for i in range(130)], torch.float16),
    (300, 8, 1, 64, 32, 1, [7 * i % 90 for i in range(300)], torch.bfloat16),
    (256, 3, 1, 64, 32, 1, [31 * i % 400 for i in range(256)], torch.float16),
    (1300, 1, 2, 64, 32, 1, [11 * i % 70 for i in range(1300)], torch.bfloat16),
    (6, 2, 5, 128, 64, 32, [900, 33, 0, 400, 2500, 1], torch.bfloat16),
])
def test_causal(gpu, B, H, G, D, P, Sq, lens, dtype):
    cache, table = make(B, H, D, P, lens, dtype, 0, gpu)
    q = queries(B, H * G, Sq, D, dtype, 1, gpu)
    o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), return_lse=True)
    check(cache, table, lens, q, o, lse)
    assert torch.equal(sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu)), o)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 1000, 1 << 40])
@pytest.mark.parametrize("Sq,G", [(1, 1), (6, 2), (32, 2)])
def test_window(gpu, window, Sq, G):
    lens = [3, 500, 129]
    cache, table = make(3, 2, 64, 32, lens, torch.bfloat16, 2, gpu)
    q = queries(3, 2 * G, Sq, 64, torch.bfloat16, 3, gpu)
    o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), window=window, return_lse=True)
    check(cache, table, lens, q, o, lse, window=window)


def test_padded_batch(gpu):
    """Rows behind counts, lengths past the table and below 0, counts out of range."""
    lens, counts = [70, 70, 70, 200, -3, 64, 2 ** 31 - 1], [3, 0, 1, 2, 3, 100, -1]
    cache, table = make(7, 2, 128, 32, [128] * 7, torch.bfloat16, 4, gpu)
    q = queries(7, 6, 3, 128, torch.bfloat16, 5, gpu)
    for window in (None, 40):
        o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), counts=ints(counts, gpu), window=window, return_lse=True)
        check(cache, table, lens, q, o, lse, counts=counts, window=window)
    # a NaN that rows of padding meet
    k = torch.full((7, 2, 1, 128), float("nan"), dtype=torch.bfloat16, device=gpu)
    sa.paged_cache_append(cache, k, k, table, ints([2] * 7, gpu))
    for window in (None, 40):
        o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), counts=ints(counts, gpu), window=window, return_lse=True)
        check(cache, table, lens, q, o, lse, counts=counts, window=window)
    cache, table = make(7, 2, 128, 32, [128] * 7, torch.bfloat16, 4, gpu)
    seen = torch.rand(7, 2, 3, 128, generator=torch.Generator().manual_seed(0)) < 0.5
    o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), seen.to(gpu), counts=ints(counts, gpu), return_lse=True)
    check(cache, table, lens, q, o, lse, see=seen, counts=counts)


def masks(kind, B, H, Sq, Sk, P, seed):
    g = torch.Generator().manual_seed(seed)
    tiles = torch.rand(B, H, 1, Sk // P, generator=g)
    m = (tiles < 0.4).repeat_interleave(P, -1).expand(B, H, Sq, Sk).clone()
    mixed = (tiles > 0.7).repeat_interleave(P, -1).expand(B, H, Sq, Sk)
    m = m | (mixed & (torch.rand(B, H, Sq, Sk, generator=g) < 0.5))
    if kind == "rows":
        m[:, :, ::2] = False  # rows without a key
    if kind == "none":
        m[:] = False
    if kind == "all":
        m[:] = True
    return m


@pytest.mark.parametrize("kind", ["tiles", "rows", "none", "all"])
@pytest.mark.parametrize("B,H,G,D,P,Sq,Sk,dtype", [(2, 2, 1, 128, 32, 1, 320, torch.bfloat16), (2, 3, 2, 64, 64, 5, 1024, torch.float16),
                                                   (1, 2, 4, 128, 128, 32, 512, torch.bfloat16), (2, 1, 3, 256, 256, 2, 768, torch.bfloat16),
                                                   (3, 2, 5, 128, 32, 9, 4096, torch.float16), (70, 3, 1, 64, 32, 2, 192, torch.bfloat16),
                                                   (24, 40, 1, 64, 32, 1, 96, torch.float16), (420, 3, 1, 64, 32, 1, 64, torch.bfloat16)])
def test_lists(gpu, kind, B, H, G, D, P, Sq, Sk, dtype):
    lens = [(Sk - 7, Sk // 2 + 3, Sk)[b % 3] for b in range(B)]
    cache, table = make(B, H, D, P, lens, dtype, 6, gpu, width=Sk // P + 1)
    q = queries(B, H * G, Sq, D, dtype, 7, gpu)
    see = masks(kind, B, H, Sq, Sk, P, 8)
    o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), see.to(gpu), return_lse=True)
    check(cache, table, lens, q, o, lse, see=see)
    md = sa.compute_mask_kernel(see.to(gpu), Sq, P)
    o2, lse2 = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), mask_metadata=md, return_lse=True)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    # one plane for the batch or the heads, by stride 0
    for shared in (see[:1, :1], see[:, :1], see[:1]):
        wide = shared.to(gpu).expand(B, H, Sq, Sk)
        o = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), shared.to(gpu))
        check(cache, table, lens, q, o, see=wide)


def test_terms(gpu):
    """Lists from a formula: sink keys and a window, no mask tensor."""
    B, H, Sq, P, Sk = 2, 2, 4, 64, 2048
    lens = [Sk, Sk - 100]
    cache, table = make(B, H, 128, P, lens, torch.bfloat16, 9, gpu)
    q = queries(B, 4 * H, Sq, 128, torch.bfloat16, 10, gpu)
    terms = [sa.causal_term(window=300, offset=Sk - Sq), sa.block_term(k_range=(0, 40))]
    md = sa.compute_mask_terms(terms, B, H, Sq, Sk, Sq, P, device=gpu)
    see = sa.materialize_mask_terms(terms, B, Sq, Sk).expand(B, H, Sq, Sk)
    o = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), mask_metadata=md)
    check(cache, table, lens, q, o, see=see)


def test_nan_and_infinity_reach_who_attends_to_them(gpu):
    """NaN in K and V, before, inside and behind what rows see; the rows that do not see it are as without it."""
    B, H, G, Sq, P, D = 1, 2, 2, 4, 64, 64
    for dtype in (torch.bfloat16, torch.float16):
        for at, in_k in ((3, True), (3, False), (126, True), (126, False), (127, False), (125, False)):
            g = torch.Generator(device=gpu).manual_seed(at)
            k, v = (torch.randn(B, H, 128, D, generator=g, device=gpu).to(dtype) for _ in range(2))
            (k if in_k else v)[0, 1, at, 5] = float("nan") if at % 2 else float("inf")
            cache = sa.empty_paged_cache(3, H, D, page_size=P, device=gpu)
            table = ints([[2, 0]], gpu)
            sa.paged_cache_append(cache, k, v, table, ints([0], gpu))
            q = queries(B, H * G, Sq, D, dtype, 11, gpu)
            for lens in ([128], [127], [126], [60]):
                for window in (None, 2):
                    o = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), window=window)
                    check(cache, table, lens, q, o, window=window)
            see = torch.ones(B, H, Sq, 128, dtype=torch.bool)
            see[:, :, 1::2, at] = False
            o = sa.sparse_attention_decode_paged(q, cache, table, ints([128], gpu), see.to(gpu))
            check(cache, table, [128], q, o, see=see)
            see[..., at] = False
            o = sa.sparse_attention_decode_paged(q, cache, table, ints([128], gpu), see.to(gpu))
            assert torch.isfinite(o).all()


def test_pages_that_are_none(gpu):
    lens = [300, 300]
    cache, table = make(2, 2, 128, 64, lens, torch.bfloat16, 12, gpu)
    table[0, 1], table[0, 4], table[1, :] = -1, cache.num_pages, 1 << 30
    q = queries(2, 4, 3, 128, torch.bfloat16, 13, gpu)
    o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), return_lse=True)
    check(cache, table, lens, q, o, lse)
    assert not o[1].any()


def test_lists_out_of_range(gpu):
    """Indices that are no tile are refused by the wrapper, once per state of the lists."""
    cache, table = make(1, 2, 64, 32, [256], torch.bfloat16, 14, gpu)
    q = queries(1, 2, 1, 64, torch.bfloat16, 15, gpu)
    mask = torch.ones(1, 2, 1, 256, dtype=torch.bool, device=gpu)
    md = sa.compute_mask_kernel(mask, 1, 32)
    md.unmasked_kv_ids[0, 0, 0, 3] = 8
    with pytest.raises(ValueError):
        sa.sparse_attention_decode_paged(q, cache, table, ints([256], gpu), mask_metadata=md)


@pytest.mark.parametrize("D,G,Sq", [(64, 1, 3), (128, 4, 8), (256, 2, 1)])
def test_values_at_the_end_of_fp16(gpu, D, G, Sq):
    """Values near fp16's largest, among codes that stand for more than it: behind a sequence, and at keys that rows leave out."""
    cache = sa.empty_paged_cache(3, 1, D, page_size=64, device=gpu)
    cache.k.fill_(0x7E), cache.v.fill_(0xFE)  # (+-448 times the block's scale)
    cache.k_scales.fill_(1.0), cache.v_scales.fill_(1.0)
    g = torch.Generator().manual_seed(40)
    k = torch.randn(1, 1, 70, D, generator=g).half().to(gpu)
    v = (6e4 * (2 * torch.rand(1, 1, 70, D, generator=g) - 1)).half().to(gpu)
    v[0, 0, 69], v[0, 0, 68] = 60000.0, -60000.0
    table = ints([[2, 0]], gpu)
    sa.paged_cache_append(cache, k, v, table, ints([0], gpu))
    assert (cache.v_scales[2] == 256.0).all()  # 448 * 256 > 65504
    q = queries(1, G, Sq, D, torch.float16, 41, gpu)
    o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints([70], gpu), return_lse=True)
    check(cache, table, [70], q, o, lse)
    # a token of 2^17, which the first rows do not see
    x = torch.zeros(1, 1, 1, D, dtype=torch.bfloat16, device=gpu)
    x[...] = 2.0 ** 17
    sa.paged_cache_append(cache, x, x, table, ints([70], gpu))
    see = torch.ones(1, 1, Sq, 128, dtype=torch.bool)
    see[:, :, :, 70] = False
    o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints([71], gpu), see.to(gpu), return_lse=True)
    assert torch.isfinite(o).all()
    check(cache, table, [71], q, o, lse, see=see)


def test_wide_scores(gpu):
    """Scores of several hundred either way: weights that vanish, a reference value that rises late."""
    for dtype in (torch.bfloat16, torch.float16):
        lens = [2000, 900]
        cache, table = make(2, 2, 128, 64, lens, dtype, 16, gpu)
        q = queries(2, 4, 2, 128, dtype, 17, gpu, size=8.0)
        o, lse = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), return_lse=True)
        check(cache, table, lens, q, o, lse)


def test_layouts(gpu):
    """q as [B,Sq,H,D] storage, as an unaligned view; tables and lengths with strides; more than one batch element sharing pages."""
    B, H, Sq, D = 3, 4, 2, 128
    lens = [100, 200, 150]
    cache, table = make(B, 2, D, 32, lens, torch.bfloat16, 18, gpu)
    table[2] = table[1]
    base = queries(B, Sq, H, D + 8, torch.bfloat16, 19, gpu)
    wide = torch.zeros(B, 2 * table.shape[1], dtype=torch.int32, device=gpu)
    wide[:, ::2] = table
    held = torch.zeros(B, 2, dtype=torch.int32, device=gpu)
    held[:, 0] = ints(lens, gpu)
    for q in (base[..., :D].transpose(1, 2), base[..., 3:D + 3].transpose(1, 2), base[..., :1, :D].transpose(1, 2).expand(B, H, Sq, D)):
        o = sa.sparse_attention_decode_paged(q, cache, wide[:, ::2], held[:, 0])
        check(cache, table, lens, q, o)


def test_a_serving_loop_with_fork_compaction_and_graph(gpu):
    """Prompts, single tokens, a fork, a compaction, as they are used together; the steps from a captured graph replayed with other
    tokens, each against the same calls made eagerly on a copy of the cache."""
    B, H, G, D, P, width, dtype = 3, 2, 4, 128, 32, 12, torch.bfloat16
    cache = sa.empty_paged_cache(200, H, D, page_size=P, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(20)
    rand = lambda *s: torch.randn(*s, generator=g, device=gpu).to(dtype)  # noqa: E731
    lens = ints([0] * B, gpu)
    free, _ = sa.paged_cache_free_pages(cache, torch.zeros(1, 1, dtype=torch.int32, device=gpu), ints([0], gpu))
    table = free[50:50 + B * width].view(B, width).contiguous()
    counts = ints([77, 1, 64], gpu)
    sa.paged_cache_append(cache, rand(B, H, 77, D), rand(B, H, 77, D), table, lens, counts)
    lens = lens + counts
    # the prompt's own attention, dense, from what the cache holds
    K, V = sa.paged_cache_gather(cache, table, lens, length=128)
    q = rand(B, H * G, 128, D)
    at = torch.arange(128, device=gpu)
    mask = (at[None, :] <= at[:, None])[None, None] & (at < lens[:, None, None, None])
    o = sa.sparse_attention(q, K.repeat_interleave(G, 1), V.repeat_interleave(G, 1), mask.expand(B, H * G, 128, 128), 128, 32)
    tail = sa.sparse_attention_decode_paged(q[:, :, 76:77].contiguous(), cache, table, lens)
    assert float((o[0, :, 76:77].float() - tail[0].float()).abs().max()) < 2e-2  # (the prompt kernels' parity bound)
    parents = ints([0, 0, 2, 1], gpu)
    pages, n_free = sa.paged_cache_free_pages(cache, table, lens)
    table, lens = sa.paged_cache_fork(cache, table, lens, parents, pages[:4])
    # every child's pages to write on are its own: the columns behind its last page
    more = pages[4:4 + 4 * width].view(4, width)
    table = torch.where(torch.arange(width, device=gpu)[None] * P >= lens[:, None], more, table)
    keep = table.clone()
    table, used = sa.paged_cache_compact(cache, table, lens)
    live = torch.arange(width, device=gpu)[None] * P < lens[:, None]
    pages, _ = sa.paged_cache_free_pages(cache, table, lens)
    assert int(used) == len(keep[live].unique()) and int(pages[0]) == int(used)
    table = torch.where(live, table, pages[:4 * width].view(4, width))

    k, v, q = torch.empty(4, H, 1, D, dtype=dtype, device=gpu), torch.empty(4, H, 1, D, dtype=dtype, device=gpu), torch.empty(4, H * G, 1, D, dtype=dtype, device=gpu)
    k.copy_(rand(4, H, 1, D)), v.copy_(rand(4, H, 1, D)), q.copy_(rand(4, H * G, 1, D))
    start = lens.clone()

    def step(cache, lens):
        sa.paged_cache_append(cache, k, v, table, lens)
        lens += 1
        return sa.sparse_attention_decode_paged(q, cache, table, lens, return_lse=True)

    def copy_of(c):
        return sa.PagedCache(c.k.clone(), c.v.clone(), c.k_scales.clone(), c.v_scales.clone(), c.head_dim)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(copy_of(cache), start.clone())
    torch.cuda.current_stream().wait_stream(side)
    eager, eager_lens = copy_of(cache), lens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = step(cache, lens)
    for _ in range(40):
        k.copy_(rand(4, H, 1, D) * 3), v.copy_(rand(4, H, 1, D)), q.copy_(rand(4, H * G, 1, D))
        graph.replay()
        want = step(eager, eager_lens)
        torch.cuda.synchronize()
        assert torch.equal(lens, eager_lens) and torch.equal(o, want[0]) and torch.equal(lse, want[1])
    for a, b in zip((cache.k, cache.v, cache.k_scales, cache.v_scales), (eager.k, eager.v, eager.k_scales, eager.v_scales)):
        assert torch.equal(a, b)
    check(cache, table, lens.tolist(), q, o, lse)


def test_another_stream(gpu):
    lens = [500]
    cache, table = make(1, 2, 128, 64, lens, torch.bfloat16, 21, gpu)
    q = queries(1, 4, 1, 128, torch.bfloat16, 22, gpu)
    n = ints(lens, gpu)
    want = sa.sparse_attention_decode_paged(q, cache, table, n)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = sa.sparse_attention_decode_paged(q, cache, table, n)
    stream.synchronize()
    assert torch.equal(got, want)


def test_calls_side_by_side(gpu):
    """Threads with streams of their own, at the same time over one cache, each of whose calls shares planes between workgroups."""
    import threading

    lens = [3000, 77, 1500]
    cache, table = make(3, 2, 128, 64, lens, torch.bfloat16, 23, gpu)
    n = ints(lens, gpu)
    qs = [queries(3, 8, 1 + t, 128, torch.bfloat16, 24 + t, gpu) for t in range(4)]
    want = [sa.sparse_attention_decode_paged(q, cache, table, n, return_lse=True) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def work(t):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(25):
                o, lse = sa.sparse_attention_decode_paged(qs[t], cache, table, n, return_lse=True)
                stream.synchronize()
                if not (torch.equal(o, want[t][0]) and torch.equal(lse, want[t][1])):
                    wrong.append(t)

    threads = [threading.Thread(target=work, args=(t,)) for t in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_two_graphs_of_one_pool(gpu):
    """Graphs that share their memory, replayed in turn with lengths that change between the replays."""
    lens = [900, 33]
    cache, table = make(2, 2, 64, 32, [1000, 1000], torch.float16, 28, gpu)
    n = ints(lens, gpu)
    qs = [queries(2, 4, 2, 64, torch.float16, 29 + t, gpu) for t in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sa.sparse_attention_decode_paged(qs[0], cache, table, n)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g, q in zip(graphs, qs):
        with torch.cuda.graph(g, pool=graphs[0].pool() if outs else None):
            outs.append(sa.sparse_attention_decode_paged(q, cache, table, n, return_lse=True))
    for step in range(6):
        n.copy_(ints([(0, 1, 900, 1000, 33, 640)[step], (1000, 5, 700, 0, 1, 65)[step]], gpu))
        for g, q, (o, lse) in zip(graphs, qs, outs):
            g.replay()
            want = sa.sparse_attention_decode_paged(q, cache, table, n, return_lse=True)
            torch.cuda.synchronize()
            assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_refusals(gpu):
    cache = sa.empty_paged_cache(4, 2, 64, page_size=32, device=gpu)
    table, lens = ints([[0, 1]], gpu), ints([40], gpu)
    q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device=gpu)
    call = sa.sparse_attention_decode_paged
    for bad in (q[:, :3], q[..., :32], q[0], q.expand(2, 4, 1, 64), q.cpu()):
        with pytest.raises(ValueError):
            call(bad, cache, table, lens)
    with pytest.raises(TypeError):
        call(q.float(), cache, table, lens)
    with pytest.raises(sa._native.SparseAttnError):
        call(q.expand(1, 4, 33, 64), cache, table, lens)
    for window in (0, -1):
        with pytest.raises(ValueError):
            call(q, cache, table, lens, window=window)
    mask = torch.ones(1, 2, 1, 64, dtype=torch.bool, device=gpu)
    with pytest.raises(ValueError):
        call(q, cache, table, lens, mask, window=3)
    for bad in (mask[..., :33], mask.expand(1, 2, 1, 64).repeat(1, 1, 1, 2), mask[0], mask.cpu()):
        with pytest.raises(ValueError):
            call(q, cache, table, lens, bad)
    with pytest.raises((ValueError, RuntimeError)):
        call(q, cache, table, lens, mask.expand(1, 2, 1, 64).repeat(1, 2, 1, 1))  # (query heads: the mask has K/V heads)
    with pytest.raises(AssertionError):
        call(q, cache, table, lens, mask.to(torch.uint8))
    with pytest.raises(ValueError):
        call(q, cache, table, lens, mask_metadata=sa.compute_mask_kernel(mask, 1, 64))  # (not the page size)
    with pytest.raises(ValueError):
        call(q, cache, table, lens, mask_metadata=sa.compute_mask_kernel(mask, 1, 32, pack_partial=False))
    with pytest.raises(ValueError):
        call(q, cache, table, lens, counts=ints([1, 1], gpu))
