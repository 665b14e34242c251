"""verify_drafts against its definition in 64 bits, walked one child at a time.  Which nodes are accepted has to agree: the tests compare products and differences of numbers
of at most 32 bits, the same in the same order here.  The next token's running sum has to be the first beyond its goal, but for the rounding of sums of V numbers in another
order: 2^-53 times V of the whole at most."""
import math

import pytest
import torch

import sparseattention_amd as sa

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def clean(x):
    return torch.where((x > 0) & torch.isfinite(x), x, 0.0).double().cpu()


def walk(p, tokens, u, parents, q, n):
    """p [n,V] and q in 64 bits: (path, residual probabilities of the next token)."""
    V = p.shape[1]
    if n == 0:
        return [], None
    path, node = [0], 0
    u = [x if x > 0 else 0.0 for x in u]
    while True:
        rest, rejected, taken = 1.0, [], None
        for c in range(node + 1, n):
            parent = c - 1 if parents is None else parents[c]
            x = tokens[c]
            if not (0 <= parent < c and parent == node and 0 <= x < V):
                continue
            chance = float(p[node, x])
            if q is None:
                chance = 0.0 if x in rejected else chance
                ok = u[c] * rest < chance
            else:
                ok = u[c] * float(q[node, x]) < chance
            if ok:
                taken = c
                break
            rejected.append(x)
            rest -= chance
        if taken is None:
            break
        path.append(taken)
        node = taken
    r = p[node].clone()
    if rejected:
        if q is None:
            r[rejected] = 0.0
        else:
            r = (r - q[node]).clamp(min=0.0)
        if not r.any():
            r = p[node].clone()
    return path, r


def check(p, tokens, u, parents=None, q=None, counts=None):
    B, n, V = p.shape
    path, accepted, token = sa.verify_drafts(p, tokens, u, parents, q, None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda"))
    assert path.dtype == accepted.dtype == torch.int32 and token.dtype == tokens.dtype
    assert path.shape == (B, n) and accepted.shape == token.shape == (B,)
    pc, qc = clean(p), None if q is None else clean(q)
    tl, ul, pl = tokens.tolist(), u.double().cpu().tolist(), None if parents is None else parents.tolist()
    for b in range(B):
        m = n if counts is None else min(max(counts[b], 0), n)
        want, r = walk(pc[b], tl[b], ul[b], pl[b] if pl else None, None if qc is None else qc[b], m)
        assert path[b].tolist() == want + [-1] * (n - len(want)), b
        assert int(accepted[b]) == len(want)
        got = int(token[b])
        if r is None or not r.any():
            assert got == -1
            continue
        sums = torch.cumsum(r, 0)
        whole, slack = float(sums[-1]), float(sums[-1]) * V * 2.0 ** -53
        goal = (ul[b][0] if ul[b][0] > 0 else 0.0) * whole
        assert 0 <= got < V and r[got] > 0
        if goal >= whole - slack:
            assert not r[got + 1:].any() or float(sums[got]) > goal - slack
        else:
            assert float(sums[got]) > goal - slack and float(sums[got] - r[got]) <= goal + slack
    return path, accepted, token


def make(seed, B, n, V, dtype, drawn, sharp=4.0, wide=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = sharp * torch.randn(B, n, V, generator=g, device="cuda")
    p = torch.softmax(logits, -1).to(dtype)
    q = torch.softmax(logits + 0.5 * torch.randn(B, n, V, generator=g, device="cuda"), -1).to(dtype) if drawn else None
    u = torch.rand(B, n, generator=g, device="cuda")
    i = torch.arange(n, device="cuda")
    parents = None if drawn else torch.where(i > 0, i - 1 - (torch.rand(B, n, generator=g, device="cuda") * i.clamp(max=3)).long().clamp(max=2), -1).int()
    after = torch.multinomial((q if drawn else p).float().view(-1, V) + 1e-30, 1, generator=g).view(B, n)
    up = (i - 1).clamp(min=0).expand(B, n) if drawn else parents.long().clamp(min=0)
    tokens = after.gather(1, up)
    if not drawn:
        other = torch.randint(V, (B, n), generator=g, device="cuda")
        tokens = torch.where(torch.rand(B, n, generator=g, device="cuda") < 0.3, other, tokens)
    return p, tokens if wide else tokens.int(), u, parents, q


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("B,n,V", [(1, 1, 1), (3, 2, 1), (5, 4, 3), (7, 9, 100), (4, 64, 1023), (2, 6, 1024), (3, 33, 2049), (9, 5, 32001), (1, 8, 131072), (2, 2, 50257), (300, 3, 4099)])
def test_sizes(gpu, dtype, drawn, B, n, V):
    p, tokens, u, parents, q = make(B + n + V, B, n, V, TYPES[dtype], drawn, wide=V % 2 == 0)
    check(p, tokens, u, parents, q)


def test_largest_vocabulary(gpu):
    p, tokens, u, parents, q = make(1, 1, 2, 1 << 21, torch.float32, True, sharp=1.0)
    check(p, tokens, u, None, q)
    u[:, 1] = 0.999999  # (after a rejection)
    check(p, tokens, u, None, q)
    check(p, tokens, u, torch.tensor([[-1, 0]], dtype=torch.int32, device="cuda"))
    p, tokens, u, parents, q = make(2, 1100, 2, 70001, torch.bfloat16, False, sharp=1.0)  # (more rows than workgroups are wanted: parts as long as they get)
    check(p, tokens, u, parents)


def test_layouts(gpu):
    """Any strides of nodes and sequences, rows that start anywhere, columns apart (copied)."""
    p, tokens, u, parents, q = make(3, 4, 7, 501, torch.float32, False)
    want = check(p, tokens, u, parents)
    wide = torch.zeros(7, 4, 1005, device="cuda")
    wide[..., 3:504] = p.transpose(0, 1)
    apart = torch.zeros(4, 7, 1002, device="cuda")
    apart[..., ::2] = p
    for pp in (wide.transpose(0, 1)[..., 3:504], apart[..., ::2]):
        for tt, uu, rr in ((tokens, u, parents), (tokens.T.contiguous().T, u.T.contiguous().T, parents.T.contiguous().T)):
            assert all(torch.equal(a, b) for a, b in zip(sa.verify_drafts(pp, tt, uu, rr), want))
    for dtype in (torch.bfloat16, torch.float16):
        h = torch.zeros(4, 7, 503, dtype=dtype, device="cuda")
        h[..., 1:502] = p
        check(h[..., 1:502], tokens, u, parents)
    p, tokens, u, _, q = make(4, 4, 7, 501, torch.float32, True)
    want = check(p, tokens, u, None, q)
    assert all(torch.equal(a, b) for a, b in zip(sa.verify_drafts(p, tokens, u, None, q[:, :6]), want))
    one = sa.verify_drafts(p[:1].expand(3, 7, 501), tokens[:1].expand(3, 7), u[:1].expand(3, 7), None, q[:1].expand(3, 7, 501))
    assert all(torch.equal(a, b[:1].expand_as(a)) for a, b in zip(one, want))


@pytest.mark.parametrize("drawn", [False, True])
def test_padded_batch(gpu, drawn):
    """Trees of fewer nodes: rows, tokens and numbers behind them are not looked at."""
    p, tokens, u, parents, q = make(5, 6, 12, 333, torch.float32, drawn)
    counts = [0, 1, 12, 5, -3, 99]
    for b, c in enumerate(counts):
        m = min(max(c, 0), 12)
        p[b, m:], tokens[b, m:], u[b, m:] = math.nan, 1 << 40, math.nan
    check(p, tokens, u, parents, q, counts)


def test_tokens_and_parents_that_are_none(gpu):
    p, tokens, u, parents, _ = make(6, 8, 10, 50, torch.float32, False)
    tokens[:, 0] = -1
    tokens[::2, 3], tokens[1::2, 2], tokens[3, 1], tokens[4, 4] = -1, 50, 1 << 32, -(1 << 40)
    parents[2, 5], parents[3, 6], parents[5, 4], parents[6, 1], parents[7] = 5, 9, -8, 1 << 30, -1
    check(p, tokens, u, parents)
    u.zero_()
    check(p, tokens, u, parents)
    p, tokens, u, _, q = make(7, 8, 10, 50, torch.float32, True)
    tokens[::2, 3] = -1  # (a chain that ends: nothing is rejected there, and the token comes from p)
    u.zero_()
    check(p, tokens, u, None, q)


def test_numbers_at_the_ends(gpu):
    """0 accepts what has any probability and takes the first such token; numbers that are none, and 1 and more, have a meaning too."""
    for drawn in (False, True):
        p, tokens, u, parents, q = make(8, 5, 6, 70, torch.float32, drawn)
        p[:, :, :5] = 0.0
        u.zero_()
        path, accepted, token = check(p, tokens, u, parents, q)
        for value in (1.0 - 2.0 ** -24, 1.0, 7.0, math.inf, -1.0, math.nan):
            u.fill_(value)
            check(p, tokens, u, parents, q) if math.isfinite(value) else sa.verify_drafts(p, tokens, u, parents, q)
        u.fill_(math.nan)
        assert torch.equal(sa.verify_drafts(p, tokens, u, parents, q)[2], token)  # (as 0)


def test_probabilities_that_are_none(gpu):
    p, tokens, u, parents, _ = make(9, 6, 5, 200, torch.float32, False)
    p[0, :, 7], p[1, :, 8], p[2, :, 9], p[3] = math.nan, math.inf, -math.inf, 0.0
    p[4, :, :100] *= -1.0
    p[5] = math.nan
    _, _, token = check(p, tokens, u, parents)
    assert token[3] == -1 and token[5] == -1
    p, tokens, u, _, q = make(10, 3, 5, 200, torch.float32, True)
    q[0, :, 3:50], q[1] = math.nan, math.inf
    check(p, tokens, u, None, q)


def test_rejected_tokens_that_are_all_there_is(gpu):
    """Where nothing is left of p it is taken as it is: a certain token whose number was beyond its probability, p that is q."""
    p = torch.zeros(2, 3, 9000, device="cuda")
    p[:, :, 4321] = 0.5  # (rows need not add up to 1)
    tokens = torch.full((2, 3), 4321, device="cuda")
    u = torch.tensor([[0.3, 0.9, 0.9], [0.0, 0.9, 0.1]], device="cuda")
    parents = torch.tensor([[-1, 0, 0]] * 2, dtype=torch.int32, device="cuda")
    path, accepted, token = check(p, tokens, u, parents)
    assert accepted.tolist() == [1, 1] and token.tolist() == [4321, 4321]
    p = torch.softmax(torch.randn(2, 3, 9000, device="cuda"), -1)
    check(p, tokens, torch.full((2, 3), 1.0, device="cuda"), None, p.clone())


def test_the_same_token_twice(gpu):
    """A sibling with a rejected token has no chance left, and does not count twice."""
    p = torch.zeros(1, 4, 6, device="cuda")
    p[..., 1], p[..., 2], p[..., 5] = 0.5, 0.25, 0.25
    tokens = torch.tensor([[0, 1, 1, 2]], device="cuda")
    parents = torch.tensor([[-1, 0, 0, 0]], dtype=torch.int32, device="cuda")
    path, accepted, token = check(p, tokens, torch.tensor([[0.0, 0.75, 0.0, 0.49]], device="cuda"), parents)
    assert path.tolist() == [[0, 3, -1, -1]] and token.tolist() == [1]
    path, accepted, token = check(p, tokens, torch.tensor([[0.9, 0.75, 0.0, 0.51]], device="cuda"), parents)
    assert path.tolist() == [[0, -1, -1, -1]] and token.tolist() == [5]


@pytest.mark.parametrize("drawn", [False, True])
def test_distribution(gpu, drawn):
    """The first token that comes out is distributed as the target says: counts of 200000 draws within 5 standard deviations of theirs (a chance of 6e-7 each, 12 of them)."""
    B, V, g = 200000, 6, torch.Generator(device="cuda").manual_seed(11)
    p1 = torch.tensor([[0.05, 0.4, 0.1, 0.3, 0.0, 0.15], [0.2, 0.2, 0.2, 0.2, 0.1, 0.1], [1.0, 0, 0, 0, 0, 0], [0.1, 0, 0, 0, 0.9, 0]], device="cuda")
    q1 = torch.tensor([[0.3, 0.2, 0.1, 0.1, 0.1, 0.2]], device="cuda").expand(4, 6)
    p = p1.expand(B, 4, V)
    u = torch.rand(B, 4, generator=g, device="cuda")
    if drawn:
        tokens = torch.multinomial(q1[:1].expand(B, V), 4, replacement=True, generator=g)
        path, accepted, token = sa.verify_drafts(p, tokens, u, None, q1.expand(B, 4, V))
    else:
        tokens = torch.tensor([0, 3, 1, 3], device="cuda").expand(B, 4)
        parents = torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda").expand(B, 4)
        path, accepted, token = sa.verify_drafts(p, tokens, u, parents)
    first = torch.where(accepted > 1, tokens.gather(1, path[:, 1:2].long().clamp(min=0))[:, 0], token)
    count = torch.bincount(first, minlength=V).double().cpu()
    want = p1[0].double().cpu()
    assert ((count - B * want).abs() <= 5 * torch.sqrt(B * want * (1 - want))).all(), count


def test_captured_and_replayed(gpu):
    p, tokens, u, parents, _ = make(12, 5, 8, 40000, torch.float32, False)
    step = lambda: sa.verify_drafts(p, tokens, u, parents)  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(6):
        u.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), i


def test_on_two_streams(gpu):
    cases = [make(20 + i, 6, 8, 60000, torch.float32, False) for i in range(2)]
    want = [sa.verify_drafts(*c[:4]) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(sa.verify_drafts(*c[:4]))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


def test_offsets_beyond_32_bits(gpu):
    """Rows further apart than 2^32 bytes, target and draft."""
    store = torch.zeros((3 << 29) + 200000, device="cuda")  # 6 GiB
    for strides in ((3 << 29, 50000, 1), (50000, 3 << 28, 1)):
        for drawn in (False, True):
            p, tokens, u, parents, q = make(14, 2, 3, 40000, torch.float32, drawn)
            a = store.as_strided((2, 3, 40000) if strides[1] < strides[0] else (1, 3, 40000), strides)
            a.copy_(p[:len(a)])
            got = sa.verify_drafts(a, tokens[:len(a)], u[:len(a)], None if drawn else parents[:len(a)], q[:len(a)] if drawn else None)
            assert all(torch.equal(x, y[:len(a)]) for x, y in zip(got, sa.verify_drafts(p, tokens, u, parents, q)))
            if drawn:
                a.copy_(q[:len(a)])
                got = sa.verify_drafts(p[:len(a)], tokens[:len(a)], u[:len(a)], None, a)
                assert all(torch.equal(x, y[:len(a)]) for x, y in zip(got, sa.verify_drafts(p, tokens, u, parents, q)))


def test_refusals(gpu):
    p, tokens, u, parents, _ = make(13, 2, 4, 30, torch.float32, False)
    for bad in (dict(tokens=tokens[:, :3]), dict(tokens=tokens.float()), dict(uniforms=u.double()), dict(uniforms=u[:1]), dict(parents=parents.long()), dict(tokens=tokens.cpu()),
                dict(parents=parents[:1]), dict(counts=parents[:, 0].long()), dict(counts=parents[0]), dict(draft_probs=p, parents=parents), dict(draft_probs=p[:, :2], parents=None),
                dict(draft_probs=p[..., :20], parents=None)):
        with pytest.raises(ValueError):
            sa.verify_drafts(**{**dict(target_probs=p, tokens=tokens, uniforms=u, parents=parents), **bad})
    with pytest.raises(TypeError):
        sa.verify_drafts(p, tokens, u, None, p.half())
    with pytest.raises(ValueError, match="nodes"):
        sa.verify_drafts(p[:, :1].expand(2, 65, 30), tokens[:, :1].expand(2, 65), u[:, :1].expand(2, 65))
    path, accepted, token = sa.verify_drafts(p[:0], tokens[:0], u[:0])
    assert path.shape == (0, 4) and accepted.shape == token.shape == (0,)
