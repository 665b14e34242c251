"""Append with norms and rotation on the GPU.  Queries and the values stored are, to the bit, what rotate_heads and paged_cache_append give.  Keys are
rounded once: what is held is the formula's float64 value rounded at the block's scale, but where float32's error, counted in tests/rotary_reference.py, leads over a
border."""
import math

import pytest
import torch

import rotary_reference as ref
import sparseattention_amd as sa
from paged_reference import EXP_MIN, Sequence, exponent_of, round_e4m3
from sparseattention_amd.rotary import Rotary

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def setup(seed, B, H, Hq, S, D, P, lens, dtype, width=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = width or max(1, -(-(max(lens) + S) // P))
    cache = sa.empty_paged_cache(B * width + 2, H, D, page_size=P)
    table = torch.randperm(B * width + 2, generator=g, device="cuda")[:B * width].int().view(B, width)
    x = [torch.randn(B, h, S, D, generator=g, device="cuda").to(dtype) for h in (Hq, H, H)]
    held = [torch.randn(B, H, max(1, max(lens)), D, generator=g, device="cuda").to(dtype) for _ in range(2)]
    sa.paged_cache_append(cache, *held, table, torch.zeros(B, dtype=torch.int32, device="cuda"), counts=ints(*lens))
    w = [(1.0 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2)]
    return cache, table, x, held, w


def clone(cache):
    return sa.PagedCache(cache.k.clone(), cache.v.clone(), cache.k_scales.clone(), cache.v_scales.clone(), cache.head_dim)


def check(cache, table, x, held, lens, rotary, at, counts=None, **kw):
    """at [B,S] or [axes,B,S]: what the call is to use; kw: how it is told."""
    q, k, v = x
    B, H, S, D = k.shape
    P, before = cache.page_size, clone(cache)
    w = dict(q_weight=kw.get("q_weight"), k_weight=kw.get("k_weight"))
    n = [S] * B if counts is None else counts
    out = sa.paged_cache_append_rotated(cache, q, k, v, table, ints(*lens), rotary, None if counts is None else ints(*counts), **kw)
    # queries, values and their scales to the bit
    want_q, rounded_k = sa.rotate_heads(q, k, at, rotary, **w)
    live = torch.arange(S, device="cuda") < ints(*n)[:, None]
    assert torch.equal(out, torch.where(live[:, None, :, None], want_q, 0)) and out.dtype == q.dtype
    sa.paged_cache_append(before, rounded_k, v, table, ints(*lens), counts=None if counts is None else ints(*counts))
    assert torch.equal(cache.v, before.v) and torch.equal(cache.v_scales, before.v_scales)
    # keys
    t = ref.angles(at.expand(B, S) if at.dim() == 2 else at, rotary.frequencies, rotary.axes)
    y, size = ref.forward(k, t, w["k_weight"], 1e-6, rotary.interleaved)
    err = 2.0 ** -21 * size + 1e-38
    ends = [min(a + b, table.shape[1] * P) for a, b in zip(lens, n)]
    got = sa.paged_cache_gather(cache, table, ints(*ends))[0].double().cpu()
    for b in range(B):
        for h in range(H):
            seq = Sequence(D)
            seq.append(held[0][b, h, :lens[b]])
            new = y[b, h, :ends[b] - lens[b]]
            for lo in range(lens[b] // 32 * 32, ends[b], 32):
                hi, a = min(lo + 32, ends[b]), max(lo, lens[b])
                if a >= hi:
                    continue
                page, sub = int(table[b, lo // P]), lo % P // 32
                if not 0 <= page < cache.num_pages:
                    assert not got[b, h, lo:hi].any()
                    continue
                scale = float(cache.k_scales[page, h, sub])
                e_old = seq.exps[-1] if a > lo else EXP_MIN
                part, slack = new[a - lens[b]:hi - lens[b]], err[b, h, a - lens[b]:hi - lens[b]]
                # the scale: of the largest value, which float32 may have put on the other side of a border
                low, high = (max(e_old, exponent_of(part * (1 + f * 2.0 ** -18))) for f in (-1.0, 1.0))
                e = round(math.log2(scale))
                assert low <= e <= high and 2.0 ** e == scale
                lower, upper = (round_e4m3(((part + f * slack) / scale).clamp(-448, 448)) * scale for f in (-1.0, 1.0))
                value = got[b, h, a:hi]
                assert ((value >= lower) & (value <= upper)).all()
                if a > lo:  # what was there, rounded again where the scale grew
                    old = seq.x[lo:]
                    again = round_e4m3(old / scale) * scale if e > e_old else old
                    assert torch.equal(got[b, h, lo:a], again)
    return out


def positions_of(lens, S):
    return ints(*lens)[:, None] + torch.arange(S, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(8, 8), (64, 64), (64, 16), (72, 72), (80, 40), (128, 128), (136, 128), (256, 256), (256, 8)])
def test_head_dims(gpu, dtype, interleaved, D, R):
    lens = [0, 31, 70]
    cache, table, x, held, w = setup(D, 3, 2, 6, 45, D, 32, lens, TYPES[dtype])
    r = sa.rotary_frequencies(R, interleaved=interleaved)
    check(cache, table, x, held, lens, r, positions_of(lens, 45), q_weight=w[0], k_weight=w[1])
    cache, table, x, held, w = setup(D + 1, 3, 2, 6, 45, D, 32, lens, TYPES[dtype])
    check(cache, table, x, held, lens, r, positions_of(lens, 45))


@pytest.mark.parametrize("P", [32, 64, 256])
@pytest.mark.parametrize("S,lens", [(1, [0]), (1, [31, 32, 33, 500]), (2, [31, 30]), (31, [1, 33]), (32, [0, 32, 5]), (33, [31, 64]), (300, [100, 0])])
def test_lengths(gpu, P, S, lens):
    cache, table, x, held, w = setup(S, len(lens), 3, 5, S, 128, P, lens, torch.bfloat16)
    check(cache, table, x, held, lens, sa.rotary_frequencies(128), positions_of(lens, S), q_weight=w[0])


def test_padded_batch(gpu):
    lens, counts = [40, 0, 31, 7], [0, 50, 1, 33]
    cache, table, x, held, w = setup(1, 4, 2, 4, 50, 64, 32, lens, torch.float16)
    for t in x:
        t[0], t[2, :, 1:], t[3, :, 33:] = math.nan, math.inf, math.nan  # (rows of padding hold anything)
    out = check(cache, table, x, held, lens, sa.rotary_frequencies(64), positions_of(lens, 50), counts, q_weight=w[0], k_weight=w[1])
    assert torch.isfinite(out).all()


def test_pages_that_do_not_exist(gpu):
    """Keys and values are not stored, past the table nor on pages that are none; queries come back all the same."""
    lens = [60, 10]
    cache, table, x, held, w = setup(2, 2, 2, 4, 100, 64, 32, lens, torch.bfloat16, width=4)
    table[1, 2] = -1
    table[0, 3] = cache.num_pages
    used = torch.zeros(cache.num_pages, dtype=torch.bool, device="cuda")
    used[table[(table >= 0) & (table < cache.num_pages)].long()] = True
    spare = cache.k[~used].clone()
    check(cache, table, x, held, lens, sa.rotary_frequencies(64), positions_of(lens, 100))
    assert torch.equal(cache.k[~used], spare)
    lens = ints(-5, 2 ** 31 - 1)  # (a length below 0 is 0; the other's tokens are past the table)
    before = clone(cache)
    r = sa.rotary_frequencies(64)
    out = sa.paged_cache_append_rotated(cache, *x, table, lens, r, ints(3, 100))
    at = torch.tensor([[0], [2 ** 31 - 1]], device="cuda") + torch.arange(100, device="cuda")
    want = sa.rotate_heads(x[0], x[1], at, r)
    assert torch.equal(out[1], want[0][1]) and torch.equal(out[0, :, :3], want[0][0, :, :3]) and not out[0, :, 3:].any()
    first = int(table[0, 0])
    changed = (cache.v != before.v).flatten(1).any(1)
    assert changed[first] and int(changed.sum()) == 1


@pytest.mark.parametrize("B,H,Hq,S", [(1, 1, 1, 1), (1, 8, 64, 1), (1, 8, 1, 3), (70, 1, 3, 1), (5, 16, 16, 2), (2, 1, 130, 40)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_heads(gpu, B, H, Hq, S, D):
    lens = [(37 * b) % 100 for b in range(B)]
    cache, table, x, held, w = setup(3, B, H, Hq, S, D, 64, lens, torch.bfloat16)
    check(cache, table, x, held, lens, sa.rotary_frequencies(D), positions_of(lens, S), q_weight=w[0], k_weight=w[1])


def test_layouts(gpu):
    """q, k and v as parts of one projection's output, with odd addresses, and with strides of sizes of 1."""
    lens = [33, 5]
    cache, table, x, held, w = setup(4, 2, 2, 4, 9, 64, 32, lens, torch.bfloat16)
    r = sa.rotary_frequencies(64)
    whole = torch.cat(x, 1).transpose(1, 2).contiguous().transpose(1, 2)
    parts = whole[:, :4], whole[:, 4:6], whole[:, 6:]
    wide = [torch.zeros(2, t.shape[1], 9, 65, dtype=t.dtype, device="cuda") for t in x]
    for a, t in zip(wide, x):
        a[..., 1:] = t
    ways = [clone(cache) for _ in range(3)]
    outs = [sa.paged_cache_append_rotated(c, *t, table, ints(*lens), r, q_weight=w[0]) for c, t in zip(ways, (x, parts, [a[..., 1:] for a in wide]))]
    for c, o in zip(ways[1:], outs[1:]):
        assert torch.equal(o, outs[0]) and torch.equal(c.k, ways[0].k) and torch.equal(c.v, ways[0].v) and torch.equal(c.k_scales, ways[0].k_scales)


def test_positions(gpu):
    lens = [20, 3]
    r = sa.rotary_frequencies(64, sections=(8, 12, 12))
    at = torch.randint(0, 3000, (3, 2, 12), device="cuda").int()
    cache, table, x, held, w = setup(5, 2, 2, 4, 12, 64, 32, lens, torch.bfloat16)
    check(cache, table, x, held, lens, r, at, positions=at, k_weight=w[1])
    r = sa.rotary_frequencies(64, 500000.0)
    for at in (torch.randint(0, 1 << 30, (2, 12), device="cuda"), torch.arange(12, device="cuda")[None].int()):
        cache, table, x, held, w = setup(6, 2, 2, 4, 12, 64, 32, lens, torch.bfloat16)
        if int(at.max()) < 5000:
            check(cache, table, x, held, lens, r, at, positions=at)
        out = sa.paged_cache_append_rotated(cache, *x, table, ints(*lens), r, positions=at)
        assert torch.equal(out, sa.rotate_heads(x[0], x[1], at, r)[0])


@pytest.mark.parametrize("n", [1, 2, 17, 33, 64])
def test_trees(gpu, n):
    """Positions are the lengths and the depths; parents that are not in front of their node are none."""
    lens, counts = [50, 31, 0], [n, max(1, n // 2), n]
    g = torch.Generator().manual_seed(n)
    parents = torch.stack([(torch.rand(n, generator=g) * torch.arange(n)).int() - (torch.rand(n, generator=g) < 0.1).int() for _ in range(3)])
    parents[:, 0] = torch.tensor([-1, 0, 5])
    if n > 2:
        parents[2, 2] = 40 if n < 40 else 2
    depth = torch.zeros(3, n, dtype=torch.int32)
    for b in range(3):
        for i in range(counts[b]):
            p = int(parents[b, i])
            depth[b, i] = depth[b, p] + 1 if 0 <= p < i else 0
    at = ints(*lens)[:, None] + depth.cuda()
    cache, table, x, held, w = setup(n, 3, 2, 4, n, 64, 32, lens, torch.bfloat16)
    wide = torch.zeros(3, 2 * n, dtype=torch.int32, device="cuda")
    wide[:, ::2] = parents.cuda()
    check(cache, table, x, held, lens, sa.rotary_frequencies(64), at, counts, parents=wide[:, ::2], k_weight=w[1])


def test_values_that_are_not_finite(gpu):
    """Keys that are not finite after norm and rotation are held as NaN and do not count for the scale."""
    lens = [3]
    cache, table, x, held, w = setup(8, 1, 2, 2, 20, 64, 32, lens, torch.bfloat16)
    x[1][0, 0, 4, 7], x[1][0, 1, 9, 60] = math.inf, math.nan
    r = sa.rotary_frequencies(32)
    other = clone(cache)
    sa.paged_cache_append_rotated(cache, *x, table, ints(*lens), r)
    k = sa.paged_cache_gather(cache, table, ints(23))[0]
    bad = torch.zeros_like(k, dtype=torch.bool)
    bad[0, 0, 7, [7, 23]] = bad[0, 1, 12, 60] = True
    assert torch.equal(torch.isnan(k), bad | torch.zeros_like(bad))
    x[1][0, 0, 4, 7] = x[1][0, 0, 4, 23] = x[1][0, 1, 9, 60] = 0.0
    sa.paged_cache_append_rotated(other, *x, table, ints(*lens), r)
    clean = sa.paged_cache_gather(other, table, ints(23))[0]
    assert torch.equal(k[~bad], clean[~bad])
    # with a norm a NaN makes its whole row so; of an infinity, which is the row's root mean square too, the pair that has it is NaN and the rest 0
    cache, table, x, held, w = setup(8, 1, 2, 2, 20, 64, 32, lens, torch.bfloat16)
    x[1][0, 0, 4, 7], x[1][0, 1, 5, 50] = math.inf, math.nan
    sa.paged_cache_append_rotated(cache, *x, table, ints(*lens), r, k_weight=w[1])
    k = sa.paged_cache_gather(cache, table, ints(23))[0]
    bad = torch.zeros_like(k, dtype=torch.bool)
    bad[0, 0, 7, [7, 23]] = bad[0, 1, 8] = True
    assert torch.equal(torch.isnan(k), bad) and not k[0, 0, 7][~bad[0, 0, 7]].any()


def test_large_and_small_keys(gpu):
    """Weights that make keys far larger or smaller than 16 bits of the inputs are: up to the cache's largest, which clamps."""
    for power in (-80, -40, 30, 100):
        lens = [10]
        cache, table, x, held, w = setup(9, 1, 1, 1, 8, 64, 32, lens, torch.bfloat16)
        check(cache, table, x, held, lens, sa.rotary_frequencies(64), positions_of(lens, 8), k_weight=torch.full((64,), 2.0 ** power, device="cuda"),
              q_weight=torch.ones(64, device="cuda"))


def test_refusals(gpu):
    cache, table, x, held, w = setup(10, 2, 2, 4, 5, 64, 32, [0, 0], torch.bfloat16)
    r, lens = sa.rotary_frequencies(64), ints(0, 0)
    call = lambda q=x[0], k=x[1], v=x[2], **kw: sa.paged_cache_append_rotated(cache, q, k, v, table, lens, kw.pop("rotary", r), **kw)  # noqa: E731
    for bad in (dict(q=x[0][:, :, :4]), dict(q=x[0][:1]), dict(k=x[0]), dict(v=x[2][..., :32]), dict(q=x[0][:, :0])):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(q=x[0].half()), dict(v=x[2].half()), dict(q=x[0].float(), k=x[1].float(), v=x[2].float()), dict(q_weight=w[0].half())):
        with pytest.raises(TypeError):
            call(**bad)
    at = torch.zeros(2, 5, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="not both"):
        call(positions=at, parents=at)
    for bad in (at[:, :4], at.long(), at.cpu(), at[0]):
        with pytest.raises(ValueError, match="parents"):
            call(parents=bad)
    with pytest.raises(ValueError, match="positions"):
        call(rotary=sa.rotary_frequencies(64, sections=(16, 16)))
    with pytest.raises(ValueError, match="positions"):
        call(positions=at[:, :3])
    with pytest.raises(ValueError, match="rotary"):
        call(rotary=Rotary(r.frequencies.cpu()))
    cache_odd = sa.empty_paged_cache(4, 2, 60, page_size=32)
    with pytest.raises(ValueError, match="head dims"):
        sa.paged_cache_append_rotated(cache_odd, *(t[..., :60] for t in x), table, lens, sa.rotary_frequencies(32))
    wide = torch.zeros(2, 2, 65, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="64 nodes"):
        call(wide, wide, wide, parents=torch.zeros(2, 65, dtype=torch.int32, device="cuda"))
    assert call(x[0][:, :, :0], x[1][:, :, :0], x[2][:, :, :0]).shape == (2, 4, 0, 64)


def test_captured_and_replayed(gpu):
    lens = [30, 7]
    cache, table, x, held, w = setup(11, 2, 2, 4, 3, 64, 32, lens, torch.bfloat16, width=8)
    r, at = sa.rotary_frequencies(64), ints(*lens)
    step = lambda c: sa.paged_cache_append_rotated(c, *x, table, at, r, q_weight=w[0], k_weight=w[1])  # noqa: E731
    step(clone(cache))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for i in range(5):
        for t in x:
            t.normal_()
        eager = clone(cache)
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager)
        assert torch.equal(out, want) and torch.equal(cache.k, eager.k) and torch.equal(cache.v, eager.v) and torch.equal(cache.k_scales, eager.k_scales), i
        at += 3
