"""The operators as they are used together: steps with drafted tokens over a paged cache, and a training step's rotation and attention."""
import concurrent.futures
import math
import textwrap

import pytest
import torch

import rotary_reference as ref
import sparseattention_amd as sa
from sparseattention_amd import drafts
from test_gpu_paged_decode import check as check_attention
from test_gpu_paged_keep import check as check_keep
from test_gpu_paged_rotated import check as check_append
from test_gpu_paged_tree import see_of, tree
from test_gpu_verify import check as check_verify

pytestmark = pytest.mark.gpu


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def held_rows(cache, table, lens):
    """What a cache holds, as 16-bit rows to compare with."""
    return [t for t in sa.paged_cache_gather(cache, table, ints(*lens), length=max(max(lens), 1))]


def test_steps_each_held_to_its_definition(gpu):
    """Prompts, then steps of a tree each: rotated append, attention, verification and keeping, every one against its reference on what the one before left;
    then a page is compacted away and the sequences go on."""
    g = torch.Generator(device="cuda").manual_seed(0)
    B, H, G, D, P, n, V = 3, 2, 3, 64, 32, 9, 300
    rotary = sa.rotary_frequencies(D)
    qw, kw = ((1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16() for _ in range(2))
    cache = sa.empty_paged_cache(40, H, D, page_size=P)
    table = torch.randperm(40, generator=g, device="cuda")[:B * 9].int().view(B, 9)
    rows = lambda h, s: torch.randn(B, h, s, D, generator=g, device="cuda").bfloat16()  # noqa: E731
    lens, prompts = [0] * B, [70, 31, 1]
    x = [rows(h, 70) for h in (H * G, H, H)]
    check_append(cache, table, x, [torch.zeros(B, H, 1, D, device="cuda")] * 2, lens, rotary, torch.arange(70, device="cuda")[None].expand(B, 70).int(), prompts, q_weight=qw, k_weight=kw)
    lens = list(prompts)
    emitted = 0
    for step in range(6):
        parents = tree("deep", B, n, step)
        parents[:, 0] = -1
        counts = [n, n - step, max(1, n - 2 * step)]
        q = sa.paged_cache_append_rotated(cache, rows(H * G, n), rows(H, n), rows(H, n), table, ints(*lens), rotary, ints(*counts), parents=parents.cuda(), q_weight=qw, k_weight=kw)
        ends = [a + c for a, c in zip(lens, counts)]
        o, lse = sa.sparse_attention_decode_tree(q, cache, table, ints(*ends), parents.cuda(), counts=ints(*counts), return_lse=True)
        see = see_of(parents, ends, counts, None, table.shape[1] * P)
        check_attention(cache, table, ends, q, o, lse, see.expand(-1, H, -1, -1), counts)
        p = torch.softmax(3.0 * torch.randn(B, n, V, generator=g, device="cuda"), -1)
        tokens = torch.argmax(p, -1).gather(1, parents.long().clamp(min=0).cuda())
        u = torch.rand(B, n, generator=g, device="cuda")
        path, accepted, token = check_verify(p, tokens, u, parents.cuda(), None, counts)
        check_keep(cache, table, lens, [row[:m] for row, m in zip(path.tolist(), accepted.tolist())], n)
        lens = [a + m for a, m in zip(lens, accepted.tolist())]
        emitted += int(accepted.sum())
        if step == 3:
            table, used = sa.paged_cache_compact(cache, table, ints(*lens))
            free, count = sa.paged_cache_free_pages(cache, table, ints(*lens))
            table = torch.where(table < 0, 0, table)
            for b in range(B):  # (fresh pages behind what each sequence has)
                first = -(-lens[b] // P)
                table[b, first:first + 3] = free[3 * b:3 * b + 3]
    assert emitted > 6 * B  # (some drafts were accepted, or the test tests little)
    q = rows(H * G, 1)
    o = sa.sparse_attention_decode_paged(q, cache, table, ints(*lens))
    check_attention(cache, table, lens, q, o)


def test_a_step_captured_and_replayed(gpu):
    """One graph of a whole step, replayed over lengths that it moves on itself, against the same step run eagerly on another cache."""
    g = torch.Generator(device="cuda").manual_seed(1)
    B, H, G, D, P, n, V = 4, 2, 4, 128, 64, 12, 5000
    rotary = sa.rotary_frequencies(D)
    table = torch.randperm(80, generator=g, device="cuda")[:B * 10].int().view(B, 10)
    start = ints(200, 3, 64, 90)
    x = [torch.randn(B, h, 200, D, generator=g, device="cuda").bfloat16() for h in (H, H)]
    caches = [sa.empty_paged_cache(80, H, D, page_size=P) for _ in range(2)]
    lens = [start.clone() for _ in range(2)]
    for c in caches:
        sa.paged_cache_append(c, *x, table, torch.zeros_like(start), counts=start)
    qkv = torch.randn(B, n, (G + 2) * H, D, generator=g, device="cuda").bfloat16().transpose(1, 2)
    parents = tree("deep", B, n, 2).cuda()
    out_of = torch.randn(H * G * D, V, generator=g, device="cuda") * 0.2
    tokens, u = torch.randint(V, (B, n), generator=g, device="cuda"), torch.rand(B, n, generator=g, device="cuda")

    def step(cache, lens):
        q = sa.paged_cache_append_rotated(cache, qkv[:, :H * G], qkv[:, H * G:-H], qkv[:, -H:], table, lens, rotary, parents=parents)
        o = sa.sparse_attention_decode_tree(q, cache, table, lens + n, parents)
        p = torch.softmax(o.transpose(1, 2).reshape(B * n, -1).float() @ out_of, -1).view(B, n, V)
        path, accepted, token = sa.verify_drafts(p, tokens, u, parents)
        sa.paged_cache_keep(cache, table, lens, path, accepted)
        lens.add_(accepted)
        return q, o, path, accepted, token

    for _ in range(2):
        scratch = sa.PagedCache(*(t.clone() for t in (caches[0].k, caches[0].v, caches[0].k_scales, caches[0].v_scales)), D)
        step(scratch, start.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(caches[0], lens[0])
    for i in range(6):
        qkv.normal_()
        u.uniform_()
        tokens.random_(0, V)
        parents.copy_(tree("deep", B, n, 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step(caches[1], lens[1])):
            assert torch.equal(a, b), i
        assert torch.equal(lens[0], lens[1])
        for a, b in zip(held_rows(caches[0], table, lens[0].tolist()), held_rows(caches[1], table, lens[1].tolist())):
            assert torch.equal(a, b), i


def test_the_documented_step(gpu):
    """The calls that the module's documentation shows, run as they stand there."""
    block = [line for line in drafts.__doc__.splitlines() if line.startswith("    ")]
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = sa.empty_paged_cache(8, 2, 64, page_size=32)
    table, lens, n = ints(*range(8)).view(2, 4), ints(33, 60), 5
    q, k, v = (torch.randn(2, h, n, 64, generator=g, device="cuda").bfloat16() for h in (4, 2, 2))
    parents, tokens = tree("deep", 2, n, 4).cuda(), torch.randint(20, (2, n), generator=g, device="cuda")
    names = dict(vars(sa), cache=cache, page_table=table, lens=lens, n=n, q=q, k=k, v=v, parents=parents, tokens=tokens, rotary=sa.rotary_frequencies(64),
                 uniforms=torch.zeros(2, n, device="cuda"), probabilities=lambda o: torch.full((2, n, 20), 0.05, device="cuda"))
    exec(textwrap.dedent("\n".join(block)), names)
    # (numbers of 0 accept every draft that has a chance: the first child each time, down to a leaf)
    for b, row in enumerate(parents.tolist()):
        path = [0]
        while path[-1] in row[path[-1] + 1:]:
            path.append(row.index(path[-1], path[-1] + 1))
        assert names["path"][b].tolist() == path + [-1] * (n - len(path)) and int(names["lens"][b] - lens[b]) == len(path)
    assert names["token"].tolist() == [0, 0] and names["o"].shape == q.shape


def test_far_into_a_large_pool(gpu):
    """Pages whose codes lie beyond 2^32 bytes of the pool: the step there is, to the bit, the step in a small one."""
    g = torch.Generator(device="cuda").manual_seed(5)
    H, D, P, n = 8, 128, 64, 9
    pages = (5 << 30) // (H * P * D)  # 5 GiB of K, as much of V
    large, small = sa.empty_paged_cache(pages, H, D, page_size=P), sa.empty_paged_cache(6, H, D, page_size=P)
    far = ints(pages - 1, pages - 5, 3, pages - 2, 0, pages - 7).view(2, 3)
    near, lens = ints(5, 1, 3, 4, 0, 2).view(2, 3), ints(120, 58)
    x = [torch.randn(2, H, 130, D, generator=g, device="cuda").bfloat16() for _ in range(2)]
    qkv = torch.randn(2, 4 * H, n, D, generator=g, device="cuda").bfloat16()
    parents, rotary = tree("deep", 2, n, 6).cuda(), sa.rotary_frequencies(D)
    path, accepted = ints(0, 2, 5, 7, *[-1] * 5)[None].expand(2, n), ints(4, 3)
    outs = []
    for cache, table in ((large, far), (small, near)):
        sa.paged_cache_append(cache, *x, table, torch.zeros_like(lens), counts=lens)
        q = sa.paged_cache_append_rotated(cache, qkv[:, :2 * H], qkv[:, 2 * H:3 * H], qkv[:, 3 * H:], table, lens, rotary, parents=parents)
        o = sa.sparse_attention_decode_tree(q, cache, table, lens + n, parents)
        sa.paged_cache_keep(cache, table, lens, path, accepted)
        outs.append([q, o, *sa.paged_cache_gather(cache, table, lens + accepted)])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_calls_side_by_side(gpu):
    """Threads with a stream each, all operators in all of them."""
    def work(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        with torch.cuda.stream(torch.cuda.Stream()):
            cache = sa.empty_paged_cache(12, 2, 64, page_size=32)
            table, lens, n = ints(*range(12)).view(3, 4), ints(33, 60, 5), 7
            q, k, v = (torch.randn(3, h, n, 64, generator=g, device="cuda").bfloat16() for h in (4, 2, 2))
            parents, rotary = tree("deep", 3, n, seed).cuda(), sa.rotary_frequencies(64)
            p = torch.softmax(3.0 * torch.randn(3, n, 9000, generator=g, device="cuda"), -1)
            tokens, u = torch.argmax(p, -1).gather(1, parents.long().clamp(min=0)), torch.rand(3, n, generator=g, device="cuda")
            w = torch.ones(64, device="cuda")
            results = []
            for _ in range(20):
                y = sa.paged_cache_append_rotated(cache, q, k, v, table, lens, rotary, parents=parents, q_weight=w)
                o = sa.sparse_attention_decode_tree(y, cache, table, lens + n, parents)
                path, accepted, token = sa.verify_drafts(p, tokens, u, parents)
                sa.paged_cache_keep(cache, table, lens, path, accepted)
                grads = sa.rotate_heads_backward(q, k, q, k, lens[:, None].expand(3, n).contiguous(), rotary, w, w)
                results.append([y, o, path, accepted, token, *grads])
            torch.cuda.current_stream().synchronize()
            for r in results[2:]:  # (the first keeping may make scales grow, which stay)
                assert all(torch.equal(a, b) for a, b in zip(r, results[1]))
            return [t.cpu() for t in results[1]]

    alone = [work(s) for s in range(4)]
    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        for a, b in zip(alone, pool.map(work, range(4))):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_training_step(gpu):
    """Rotation and attention of a training step, forward and gradients, against autograd through the same formulas in 64 bits.  The attention's own bounds
    hold for its inputs (2e-2 of each gradient's scale in bf16); the rotation adds one rounding to each input and to each gradient, 2^-8 of them."""
    g = torch.Generator(device="cuda").manual_seed(2)
    B, H, S, D = 1, 2, 256, 64
    q, k, v, do = (torch.randn(B, H, S, D, generator=g, device="cuda").bfloat16() for _ in range(4))
    qw, kw = ((1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16() for _ in range(2))
    mask = torch.ones(S, S, dtype=torch.bool, device="cuda").tril()[None, None]
    rotary, at = sa.rotary_frequencies(D, interleaved=True), torch.arange(S, device="cuda")
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, qw, kw)]
    qr, kr = sa.rotate_heads_trainable(leaves[0], leaves[1], at, rotary, leaves[3], leaves[4])
    o = sa.sparse_attention_trainable(qr, kr, leaves[2], mask, 128, 64)
    got = [o, *torch.autograd.grad(o, leaves, do)]
    exact = [t.detach().double().cpu().requires_grad_() for t in (q, k, v, qw, kw)]
    t = ref.angles(at[None].expand(B, S), rotary.frequencies)
    qe, ke = (ref.turned(ref.normed(a, w, 1e-6), t, True) for a, w in ((exact[0], exact[3]), (exact[1], exact[4])))
    s = (qe @ ke.mT) / math.sqrt(D)
    oe = torch.softmax(s.masked_fill(~mask.cpu(), -math.inf), -1) @ exact[2]
    want = [oe, *torch.autograd.grad(oe, exact, do.double().cpu())]
    for name, a, b in zip(("o", "dq", "dk", "dv", "dq_weight", "dk_weight"), got, want):
        assert (a.detach().double().cpu() - b.detach()).abs().max() <= (2e-2 + 3 * 2.0 ** -8) * b.detach().abs().max(), name
