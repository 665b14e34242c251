"""sparse_attention_decode_tree against a 64-bit attention over what the cache holds, within the bounds of the attention it shares its kernel with
(paged_reference.tolerances), with the mask written out from the parents one by one."""
import ctypes

import pytest
import torch

import sparseattention_amd as sa
from sparseattention_amd import _native
from test_gpu_paged_decode import check, ints, make, queries

gpu_test = pytest.mark.gpu
FAKE = 0x1000


def tree(kind, B, n, seed):
    g = torch.Generator().manual_seed(seed)
    i = torch.arange(n)
    if kind == "chain":
        return (i - 1).expand(B, n).int().contiguous()
    if kind == "star":  # all of them children of the first
        return torch.where(i > 0, 0, -1).expand(B, n).int().contiguous()
    if kind == "roots":  # one token drafted n times
        return torch.full((B, n), -1).int()
    p = (torch.rand(B, n, generator=g) * i).int()
    if kind == "deep":
        p = torch.maximum(p, (i - 1 - (torch.rand(B, n, generator=g) * 3).int()).int())
    p[:, 0] = -1
    if kind == "odd":  # values that say "none" in any way, among others
        none = torch.tensor([-1, -7, 64, 1 << 30, -(1 << 31)])
        pick = torch.rand(B, n, generator=g) < 0.2
        p = torch.where(pick, none[torch.randint(0, 5, (B, n), generator=g)].int(), p)
        own = torch.rand(B, n, generator=g) < 0.1
        p = torch.where(own, (i + torch.randint(0, 2, (B, n), generator=g)).int(), p)
    return p


def see_of(parents, lens, counts, window, Sk):
    B, n = parents.shape
    see = torch.zeros(B, 1, n, Sk, dtype=torch.bool)
    for b, row in enumerate(parents.tolist()):
        m = min(max(counts[b], 0), n)
        base = min(max(lens[b], 0), Sk) - m
        above = []
        for i in range(m):
            p = row[i]
            above.append((above[p] if 0 <= p < i else []) + [i])
            depth = len(above[i]) - 1
            if base > 0:
                see[b, 0, i, max(0, base + depth - window + 1) if window else 0:base] = True
            for d, a in enumerate(above[i]):
                if base + a >= 0 and (not window or depth - d < window):
                    see[b, 0, i, base + a] = True
    return see


def run(cache, table, lens, q, parents, counts=None, window=None):
    dev = q.device
    o, lse = sa.sparse_attention_decode_tree(q, cache, table, ints(lens, dev), parents.to(dev), counts=None if counts is None else ints(counts, dev), window=window,
                                             return_lse=True)
    see = see_of(parents, lens, counts or [parents.shape[1]] * len(lens), window, table.shape[1] * cache.page_size)
    check(cache, table, lens, q, o, lse, see.expand(-1, cache.num_heads, -1, -1), counts)
    return o


@gpu_test
@pytest.mark.parametrize("kind", ["chain", "star", "roots", "random", "deep", "odd"])
@pytest.mark.parametrize("n,G,D,dtype", [(1, 1, 64, torch.bfloat16), (2, 3, 128, torch.float16), (8, 4, 128, torch.bfloat16), (16, 1, 64, torch.float16),
                                         (17, 1, 128, torch.bfloat16), (33, 2, 64, torch.bfloat16), (64, 1, 256, torch.bfloat16), (64, 4, 128, torch.float16)])
def test_trees(gpu, kind, n, G, D, dtype):
    lens = [n, n + 1, n + 31, 700, 64 + n]
    cache, table = make(5, 2, D, 32, lens, dtype, n, gpu)
    run(cache, table, lens, queries(5, 2 * G, n, D, dtype, 1, gpu), tree(kind, 5, n, n))


@gpu_test
@pytest.mark.parametrize("window", [1, 2, 3, 31, 32, 33, 64, 65, 100, 1 << 40])
@pytest.mark.parametrize("kind", ["chain", "deep", "random"])
@pytest.mark.parametrize("n", [6, 64])
def test_windows(gpu, window, kind, n):
    lens = [n, 500, 129]
    cache, table = make(3, 2, 64, 32, lens, torch.bfloat16, 2, gpu)
    run(cache, table, lens, queries(3, 4, n, 64, torch.bfloat16, 3, gpu), tree(kind, 3, n, window % 97), window=window)


@gpu_test
@pytest.mark.parametrize("window", [None, 5])
def test_padded_batch(gpu, window):
    """Trees of their own sizes; sequences shorter than their trees; padding that holds anything."""
    lens, counts = [300, 70, 5, 20, 33, -3], [0, 40, 17, 20, 64, 4]
    cache, table = make(6, 2, 64, 32, [max(x, 0) for x in lens], torch.bfloat16, 4, gpu)
    q = queries(6, 6, 40, 64, torch.bfloat16, 5, gpu)
    q[1, :, 39], q[2, :, 17:] = float("nan"), float("inf")
    q[1, :, 39] = 1.0
    run(cache, table, lens, q, tree("odd", 6, 40, 6), [0, 40, 17, 20, 40, 4], window)
    q = queries(6, 6, 40, 64, torch.bfloat16, 5, gpu)
    o = sa.sparse_attention_decode_tree(q, cache, table, ints(lens, gpu), tree("deep", 6, 40, 6).to(gpu), counts=ints(counts, gpu))
    want = sa.sparse_attention_decode_tree(q, cache, table, ints(lens, gpu), tree("deep", 6, 40, 6).to(gpu), counts=ints([0, 40, 17, 20, 40, 4], gpu))
    assert torch.equal(o, want)  # (a count beyond the rows is all of them)


@gpu_test
@pytest.mark.parametrize("B,H,G,D,n,length", [(1, 1, 1, 64, 5, 131077), (1, 2, 4, 128, 25, 20011), (2, 1, 8, 64, 64, 9000), (300, 1, 1, 64, 3, 90), (40, 8, 2, 128, 12, 1500),
                                           (40, 8, 1, 64, 30, 4000), (24, 4, 3, 128, 25, 9000), (40, 8, 2, 64, 64, 8500), (9, 8, 4, 256, 25, 7000)])
def test_sizes(gpu, B, H, G, D, n, length):
    lens = [max(n, length - 37 * b % length) for b in range(B)]
    cache, table = make(B, H, D, 64, lens, torch.bfloat16, 7, gpu)
    q, parents = queries(B, H * G, n, D, torch.bfloat16, 8, gpu), tree("deep", B, n, 9)
    o = run(cache, table, lens, q, parents)
    assert torch.equal(sa.sparse_attention_decode_tree(q, cache, table, ints(lens, gpu), parents.to(gpu)), o)


@gpu_test
@pytest.mark.parametrize("n,G,pages,window", [(20, 2, 76, None), (40, 2, 112, None), (40, 2, 112, 30)])
def test_many_short_sequences_of_wide_tables(gpu, n, G, pages, window):
    """More sequences than a wave has lanes for, with planes of 64 and of 128 rows, as the tables have room for much more than the sequences hold."""
    lens = [n + 7 * b % 90 for b in range(300)]
    cache, table = make(300, 1, 64, 64, lens, torch.bfloat16, 21, gpu)
    table = torch.cat([table, torch.full((300, pages - table.shape[1]), -1, dtype=torch.int32, device=gpu)], 1)
    run(cache, table, lens, queries(300, G, n, 64, torch.bfloat16, 22, gpu), tree("deep", 300, n, 23), window=window)


@gpu_test
def test_a_chain_is_causal(gpu):
    """Up to 16 rows of a K/V head, to the bit what sparse_attention_decode_paged gives, windows and padding among them."""
    lens, counts = [40, 999, 32], [5, 0, 9]
    cache, table = make(3, 2, 128, 64, lens, torch.bfloat16, 10, gpu)
    for n, G in ((9, 1), (4, 4), (16, 1)):
        q, parents = queries(3, 2 * G, n, 128, torch.bfloat16, 11, gpu), tree("chain", 3, n, 0).to(gpu)
        for kw in (dict(), dict(counts=ints(counts, gpu)), dict(window=7), dict(window=300)):
            a = sa.sparse_attention_decode_tree(q, cache, table, ints(lens, gpu), parents, return_lse=True, **kw)
            b = sa.sparse_attention_decode_paged(q, cache, table, ints(lens, gpu), return_lse=True, **kw)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@gpu_test
def test_nan_reaches_who_attends_to_it(gpu):
    """A draft whose value is NaN makes its own row and its descendants' NaN and no other; so does a key."""
    parents = torch.tensor([[-1, 0, 0, 1, 2, -1]], dtype=torch.int32)
    for what in (0, 1):
        cache = sa.empty_paged_cache(3, 1, 64, page_size=32)
        table = ints([[2, 0]], gpu)
        g = torch.Generator(device=gpu).manual_seed(12)
        x = [torch.randn(1, 1, 40, 64, generator=g, device=gpu).bfloat16() for _ in range(2)]
        x[what][0, 0, 34 + 2, 7] = float("nan")
        sa.paged_cache_append(cache, *x, table, ints([0], gpu))
        o = sa.sparse_attention_decode_tree(queries(1, 2, 6, 64, torch.bfloat16, 13, gpu), cache, table, ints([40], gpu), parents.to(gpu))
        assert torch.isnan(o).any(-1)[0].tolist() == [[False, False, True, False, True, False]] * 2


@gpu_test
def test_pages_that_are_none(gpu):
    lens = [200, 100]
    cache, table = make(2, 2, 64, 32, lens, torch.bfloat16, 14, gpu)
    table[0, 2], table[1, 3], table[0, 6] = -1, cache.num_pages, -5  # (the second's tree lies there; of the first's, the last eight)
    run(cache, table, lens, queries(2, 4, 20, 64, torch.bfloat16, 15, gpu), tree("random", 2, 20, 16))


@gpu_test
def test_layouts(gpu):
    lens = [90, 33]
    cache, table = make(2, 2, 80, 32, lens, torch.bfloat16, 17, gpu)
    q, parents = queries(2, 4, 7, 80, torch.bfloat16, 18, gpu), tree("random", 2, 7, 19).to(gpu)
    want = sa.sparse_attention_decode_tree(q, cache, table, ints(lens, gpu), parents)
    wide = torch.full((7, 4), -9, dtype=torch.int32, device=gpu)
    wide[:, ::2] = parents.T
    odd = torch.zeros(2, 4, 7, 81, dtype=q.dtype, device=gpu)
    odd[..., 1:] = q
    for qq in (q, q.transpose(1, 2).contiguous().transpose(1, 2), odd[..., 1:]):
        for pp in (parents, wide[:, ::2].T):
            assert torch.equal(sa.sparse_attention_decode_tree(qq, cache, table, ints(lens, gpu), pp), want)
    same = parents[:1].expand(2, 7)
    assert torch.equal(sa.sparse_attention_decode_tree(q, cache, table, ints(lens, gpu), same),
                       sa.sparse_attention_decode_tree(q, cache, table, ints(lens, gpu), same.contiguous()))


@gpu_test
def test_captured_and_replayed(gpu):
    lens = ints([60, 20], gpu)
    cache, table = make(2, 2, 64, 32, [150, 150], torch.bfloat16, 20, gpu)
    q, parents = queries(2, 4, 9, 64, torch.bfloat16, 21, gpu), tree("random", 2, 9, 22).to(gpu)
    step = lambda: sa.sparse_attention_decode_tree(q, cache, table, lens, parents)  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(5):
        q.normal_()
        parents.copy_(tree("odd", 2, 9, 30 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step()), i
        lens += 17


def test_refusals_without_a_gpu():
    lib, S2, S4 = _native.load(), _native.strides((4, 1)), _native.strides((1024, 128, 128, 1))
    pool = ctypes.byref(_native.PagedCacheStruct(FAKE, FAKE, FAKE, FAKE, 8, 2, 64, 128, 128))
    bad, unsupported, workspace = _native.SA_ERR_INVALID_ARGUMENT, _native.SA_ERR_UNSUPPORTED, _native.SA_ERR_WORKSPACE

    def call(q=FAKE, table=FAKE, lens=FAKE, parents=FAKE, ps=S2, o=FAKE, B=1, Hq=4, n=8, window=0, dtype=0, scale=0.1, ws=None, size=0, pages=4):
        return lib.sa_sparse_attention_decode_tree(q, S4, pool, table, S2, lens, parents, ps, None, pages, o, S4, B, Hq, n, window, dtype, scale, ws, size, None, None, None)

    for name in ("q", "table", "lens", "parents", "ps", "o"):
        assert call(**{name: None}) == bad, name
    assert call(n=0) == unsupported and call(n=65) == unsupported and call(Hq=3) == bad and call(window=-1) == bad and call(dtype=2) == unsupported
    assert call(scale=0.0) == bad and call(B=0) == bad and call(pages=0) == bad
    need = lib.sa_decode_tree_workspace_bytes(1, 4, 2, 8, 128, 4, 64)
    assert need > 0 and call() == workspace and call(ws=FAKE, size=need - 1) == workspace and call(ws=FAKE + 8, size=need) == workspace
    assert lib.sa_decode_tree_workspace_bytes(1, 4, 2, 64, 128, 4, 64) > 0 and lib.sa_decode_tree_workspace_bytes(1, 4, 2, 65, 128, 4, 64) == 0
    assert lib.sa_decode_paged_workspace_bytes(1, 4, 2, 33, 128, 4, 64) == 0


@gpu_test
def test_refusals(gpu):
    cache, table = make(2, 2, 64, 32, [40, 40], torch.bfloat16, 23, gpu)
    q, parents, lens = queries(2, 4, 5, 64, torch.bfloat16, 24, gpu), tree("chain", 2, 5, 0).to(gpu), ints([40, 40], gpu)
    call = lambda q=q, parents=parents, **kw: sa.sparse_attention_decode_tree(q, cache, table, kw.pop("lens", lens), parents, **kw)  # noqa: E731
    for bad in (parents[:, :4], parents.long(), parents.cpu(), parents[0], parents[:1]):
        with pytest.raises(ValueError, match="parents"):
            call(parents=bad)
    for bad in (q[:, :3], q[:1], q[..., :32], q[0]):
        with pytest.raises(ValueError, match="q must"):
            call(q=bad)
    for kw in (dict(window=0), dict(window=-3), dict(counts=lens[:1]), dict(counts=lens.long()), dict(lens=lens[:1])):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(TypeError):
        call(q=q.float())
    with pytest.raises(ValueError, match="64 nodes"):
        call(q=q[:, :, :1].expand(2, 4, 65, 64), parents=torch.zeros(2, 65, dtype=torch.int32, device=gpu))
    assert call(q=q[:, :, :0], parents=parents[:, :0]).shape == (2, 4, 0, 64)
