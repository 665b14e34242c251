"""Norm and rotation of heads and its gradients on the GPU against the formula in 64 bits, within bounds counted from the roundings
(tests/rotary_reference.py)."""
import math

import pytest
import torch

import rotary_reference as ref
import sparseattention_amd as sa

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FAR = 2 * math.pi * 2.0 ** -24  # the angle's own error, at positions of 2^31


def rows(g, B, H, S, D, dtype, layout="bhsd"):
    x = torch.randn(B, H, S, D, generator=g, device="cuda") * torch.exp(torch.randn(B, H, S, 1, generator=g, device="cuda"))
    x = x.to(dtype)
    if layout == "bshd":
        x = x.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "part":  # of a projection's output
        wide = torch.zeros(B, S, H + 3, D, dtype=dtype, device="cuda")
        wide[:, :, 1:H + 1] = x.transpose(1, 2)
        x = wide.transpose(1, 2)[:, 1:H + 1]
    elif layout == "odd":  # rows that are not 16-byte aligned: copied
        wide = torch.zeros(B, H, S, D + 1, dtype=dtype, device="cuda")
        wide[..., 1:] = x
        x = wide[..., 1:]
    return x


def check(q, k, positions, rotary, qw=None, kw=None, eps=1e-6, far=0.0, grad=True):
    t = ref.angles(positions.expand(q.shape[0], -1) if positions.dim() == 2 else positions.expand(q.shape[0], q.shape[2]) if positions.dim() == 1 else
                   positions.expand(-1, q.shape[0], -1), rotary.frequencies, rotary.axes)
    out = sa.rotate_heads(q, k, positions, rotary, qw, kw, eps)
    for name, x, w, y in (("q", q, qw, out[0]), ("k", k, kw, out[1])):
        want, size = ref.forward(x, t, w, eps, rotary.interleaved)
        assert y.dtype == x.dtype
        ref.assert_within(y, want, ref.forward_tolerance(want, size, x.dtype, far), name)
    if not grad:
        return
    g = torch.Generator(device="cuda").manual_seed(17)
    ups = [torch.randn(x.shape, generator=g, device="cuda").to(x.dtype) for x in (q, k)]
    dq, dk, dqw, dkw = sa.rotate_heads_backward(*ups, q, k, positions, rotary, qw, kw, eps)
    for name, up, x, w, dx, dw in (("dq", ups[0], q, qw, dq, dqw), ("dk", ups[1], k, kw, dk, dkw)):
        want, tol, want_w, tol_w = ref.backward(up, x, t, w, eps, rotary.interleaved, x.dtype)
        ref.assert_within(dx, want, tol, name)
        assert (dw is None) == (w is None)
        if w is not None:
            assert dw.dtype == w.dtype
            ref.assert_within(dw, want_w, tol_w, name + "_weight")
    return out, (dq, dk, dqw, dkw)


def weights(g, D, dtype):
    return tuple((1.0 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(8, 8), (24, 16), (64, 64), (64, 32), (72, 72), (80, 80), (128, 128), (128, 64), (136, 8), (200, 200), (256, 256), (256, 64)])
def test_head_dims(gpu, dtype, interleaved, D, R):
    g = torch.Generator(device="cuda").manual_seed(D + R)
    q, k = rows(g, 2, 5, 7, D, TYPES[dtype]), rows(g, 2, 2, 7, D, TYPES[dtype])
    at = torch.randint(0, 5000, (2, 7), generator=g, device="cuda").int()
    check(q, k, at, sa.rotary_frequencies(R, interleaved=interleaved), *weights(g, D, TYPES[dtype]))
    check(q, k, at, sa.rotary_frequencies(R, interleaved=interleaved))


@pytest.mark.parametrize("B,S,Hq,H", [(1, 1, 1, 1), (1, 1, 32, 8), (3, 1, 7, 3), (64, 1, 4, 1), (1, 33, 1, 2), (2, 129, 9, 1), (5, 3, 130, 1), (1, 2049, 3, 3)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_sizes(gpu, B, S, Hq, H, D):
    g = torch.Generator(device="cuda").manual_seed(B * S)
    q, k = rows(g, B, Hq, S, D, torch.bfloat16), rows(g, B, H, S, D, torch.bfloat16)
    check(q, k, torch.arange(S, device="cuda"), sa.rotary_frequencies(D), *weights(g, D, torch.float32))


@pytest.mark.parametrize("layout", ["bshd", "part", "odd"])
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(gpu, layout, dtype):
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k = rows(g, 2, 6, 19, 80, TYPES[dtype], layout), rows(g, 2, 3, 19, 80, TYPES[dtype], layout)
    check(q, k, torch.arange(19, device="cuda").int()[None], sa.rotary_frequencies(80), *weights(g, 80, TYPES[dtype]))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("sections", [(32,), (16, 16), (8, 12, 12), (0, 1, 31)])
def test_axes(gpu, sections, wide):
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k = rows(g, 3, 4, 21, 64, torch.bfloat16), rows(g, 3, 2, 21, 64, torch.bfloat16)
    at = torch.randint(-300, 300, (len(sections), 3, 21), generator=g, device="cuda")
    at = at if wide else at.int()
    r = sa.rotary_frequencies(64, sections=sections)
    check(q, k, at, r)
    check(q, k, at.transpose(1, 2).contiguous().transpose(1, 2)[:, :1], r)
    r.axes[5] = 77  # (taken as the last one there is)
    inside = sa.Rotary(r.frequencies, r.axes.clamp(max=len(sections) - 1))
    for a, b in zip(sa.rotate_heads(q, k, at, r), sa.rotate_heads(q, k, at, inside)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("position", [0, 1, -1, 8191, 1 << 20, (1 << 20) + 1, (1 << 31) - 1, -(1 << 31)])
def test_far_positions(gpu, position):
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k = rows(g, 1, 4, 6, 128, torch.float32), rows(g, 1, 1, 6, 128, torch.float32)
    check(q, k, torch.full((1, 6), position, device="cuda", dtype=torch.int32), sa.rotary_frequencies(128, 500000.0), far=FAR * max(2.0 ** -10, abs(position) / 2 ** 31),
          grad=False)


def test_values_that_are_not_finite(gpu):
    """Without a norm only the pairs that hold such a value have it; with one their whole row; no other row has."""
    g = torch.Generator(device="cuda").manual_seed(8)
    q, k = rows(g, 1, 3, 5, 64, torch.bfloat16), rows(g, 1, 1, 5, 64, torch.bfloat16)
    q[0, 0, 0, 3], q[0, 1, 2, 60], q[0, 2, 4, 5] = math.inf, math.nan, -math.inf
    r = sa.rotary_frequencies(32)
    at = torch.arange(5, device="cuda")
    out = sa.rotate_heads(q, k, at, r)[0]
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[0, 0, 0, [3, 19]] = want[0, 2, 4, [5, 21]] = True
    want[0, 1, 2, 60] = True
    assert torch.equal(bad, want)
    out = sa.rotate_heads(q, k, at, r, *weights(g, 64, torch.bfloat16))[0]
    rows_bad = torch.isnan(out).any(-1)
    assert rows_bad.sum() == 3 and rows_bad[0, 0, 0] and rows_bad[0, 1, 2] and rows_bad[0, 2, 4]


def test_zero_rows_and_eps(gpu):
    q, k = torch.zeros(1, 2, 3, 64, device="cuda"), torch.zeros(1, 1, 3, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    r, at = sa.rotary_frequencies(64), torch.arange(3, device="cuda")
    out = sa.rotate_heads(q, k, at, r, w, w)
    assert not out[0].any() and not out[1].any()
    g = torch.Generator(device="cuda").manual_seed(9)
    q, k = rows(g, 1, 2, 3, 64, torch.float32), rows(g, 1, 1, 3, 64, torch.float32)
    check(q, k, at, r, w, None, eps=0.0)  # (17 of the wave's lanes have no row)
    check(q, k, at, r, None, w, eps=0.5)


def test_nothing_to_do(gpu):
    r = sa.rotary_frequencies(64)
    w = torch.ones(64, device="cuda")
    for B, S in ((0, 3), (2, 0)):
        q, k = torch.zeros(B, 2, S, 64, device="cuda"), torch.zeros(B, 1, S, 64, device="cuda")
        at = torch.zeros(B, S, device="cuda", dtype=torch.int32)
        assert [x.shape for x in sa.rotate_heads(q, k, at, r)] == [q.shape, k.shape]
        dq, dk, dqw, dkw = sa.rotate_heads_backward(q, k, q, k, at, r, w, w)
        assert dq.shape == q.shape and not dqw.any() and not dkw.any()


def test_refusals(gpu):
    q, k = torch.zeros(2, 4, 6, 64, device="cuda"), torch.zeros(2, 2, 6, 64, device="cuda")
    r, at = sa.rotary_frequencies(64), torch.zeros(2, 6, device="cuda", dtype=torch.int32)
    axes = sa.rotary_frequencies(64, sections=(16, 16))
    w = torch.ones(64, device="cuda")
    for a in (at[:, :5], at[:1].expand(3, 6), at.float(), at.cpu(), at[None]):
        with pytest.raises(ValueError, match="positions"):
            sa.rotate_heads(q, k, a, r)
    with pytest.raises(ValueError, match="positions"):
        sa.rotate_heads(q, k, at, axes)
    for bad in (sa.Rotary(r.frequencies.float()), sa.Rotary(r.frequencies[:30]), sa.Rotary(r.frequencies.cpu()), sa.rotary_frequencies(128),
                sa.Rotary(r.frequencies, axes.axes[:5]), sa.Rotary(r.frequencies, axes.axes.long())):
        with pytest.raises(ValueError, match="rotary"):
            sa.rotate_heads(q, k, at[None] if bad.axes is not None else at, bad)
    for bad in (w[:32], w.cpu(), w[None]):
        with pytest.raises(ValueError, match="q_weight"):
            sa.rotate_heads(q, k, at, r, bad)
    for pair in ((w.half(), None), (None, w.double())):
        with pytest.raises(TypeError):
            sa.rotate_heads(q, k, at, r, *pair)
    with pytest.raises(TypeError, match="share"):
        sa.rotate_heads(q.half(), k.half(), at, r, w, w.half())
    for eps in (-1.0, math.nan, math.inf, 1e39):
        with pytest.raises(ValueError, match="eps"):
            sa.rotate_heads(q, k, at, r, w, w, eps)
    with pytest.raises(ValueError, match="head dims"):
        sa.rotate_heads(q[..., :60], k[..., :60], at, sa.rotary_frequencies(32))
    with pytest.raises(ValueError, match="dq"):
        sa.rotate_heads_backward(q[:, :2], k, q, k, at, r)
    with pytest.raises(ValueError, match="k is on"):
        sa.rotate_heads(q, k.cpu(), at, r)


def test_autograd(gpu):
    """The function for autograd gives what the two calls give; outputs that nothing uses count with zeros."""
    g = torch.Generator(device="cuda").manual_seed(10)
    q, k = rows(g, 2, 4, 37, 128, torch.bfloat16, "part"), rows(g, 2, 2, 37, 128, torch.bfloat16, "part")
    qw, kw = weights(g, 128, torch.bfloat16)
    r, at = sa.rotary_frequencies(128), torch.arange(37, device="cuda")
    up = [torch.randn(x.shape, generator=g, device="cuda").to(x.dtype) for x in (q, k)]
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, qw, kw)]
    y = sa.rotate_heads_trainable(leaves[0], leaves[1], at, r, leaves[2], leaves[3])
    for a, b in zip(y, sa.rotate_heads(q, k, at, r, qw, kw)):
        assert torch.equal(a, b) and a.requires_grad and not b.requires_grad
    got = torch.autograd.grad(y, leaves, up)
    for a, b in zip(got, sa.rotate_heads_backward(*up, q, k, at, r, qw, kw)):
        assert torch.equal(a, b)
    y = sa.rotate_heads_trainable(leaves[0], leaves[1], at, r, leaves[2], leaves[3])
    got = torch.autograd.grad(y[0].float().sum(), leaves)  # (a gradient that is one number expanded)
    want = sa.rotate_heads_backward(torch.ones_like(q), torch.zeros_like(k), q, k, at, r, qw, kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not got[1].any()
    y = sa.rotate_heads_trainable(leaves[0], k, at, r, leaves[2])
    assert torch.autograd.grad(y, leaves[0], up, allow_unused=True)[0] is not None
    y = sa.rotate_heads_trainable(leaves[0], leaves[1], at, r)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, leaves[:2], up, create_graph=True)
    y = sa.rotate_heads_trainable(leaves[0], leaves[1], at, r)
    with torch.no_grad():
        leaves[0].zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, leaves[:2], up)


def test_float32_gradients_against_differences(gpu):
    """Differences of the kernel's own float32 outputs, summed in 64 bits, along a direction: with steps of h they are off by h^2 / 6 of the third
    derivative and by the outputs' rounding over h.  Values and weights are around 1: h = 2^-6 leaves 2^-12 of the sum of the terms' magnitudes."""
    g = torch.Generator(device="cuda").manual_seed(11)
    q, k = torch.randn(2, 3, 9, 64, generator=g, device="cuda"), torch.randn(2, 1, 9, 64, generator=g, device="cuda")
    qw, kw = weights(g, 64, torch.float32)
    r, at = sa.rotary_frequencies(64), torch.arange(9, device="cuda")
    up = [torch.randn(x.shape, generator=g, device="cuda") for x in (q, k)]
    grads = sa.rotate_heads_backward(*up, q, k, at, r, qw, kw)

    def f(x):
        y = sa.rotate_heads(*x[:2], at, r, *x[2:])
        return sum((a.double() * b.double()).sum() for a, b in zip(y, up))

    h = 2.0 ** -6
    for i, grad in enumerate(grads):
        x = [q, k, qw, kw]
        v = torch.randn(x[i].shape, generator=g, device="cuda")
        ends = [f(x[:i] + [x[i] + s * h * v] + x[i + 1:]) for s in (1.0, -1.0)]
        want = float((grad.double() * v.double()).sum())
        assert abs(float(ends[0] - ends[1]) / (2 * h) - want) <= 2.0 ** -12 * float((grad.double() * v.double()).abs().sum()) + 2.0 ** -12


def test_captured_and_replayed(gpu):
    g = torch.Generator(device="cuda").manual_seed(12)
    q, k = rows(g, 2, 4, 50, 128, torch.bfloat16), rows(g, 2, 2, 50, 128, torch.bfloat16)
    qw, kw = weights(g, 128, torch.bfloat16)
    r, at = sa.rotary_frequencies(128), torch.arange(50, device="cuda").int()
    up = [torch.randn(x.shape, generator=g, device="cuda").to(x.dtype) for x in (q, k)]
    step = lambda: (*sa.rotate_heads(q, k, at, r, qw, kw), *sa.rotate_heads_backward(*up, q, k, at, r, qw, kw))  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        q.copy_(rows(g, 2, 4, 50, 128, torch.bfloat16))
        at += 1000 * i
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), i


def test_on_another_stream(gpu):
    g = torch.Generator(device="cuda").manual_seed(13)
    q, k = rows(g, 2, 8, 512, 128, torch.bfloat16), rows(g, 2, 2, 512, 128, torch.bfloat16)
    r, at = sa.rotary_frequencies(128), torch.arange(512, device="cuda")
    want = sa.rotate_heads(q, k, at, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = q * 1
        got = sa.rotate_heads(x, k, at, r)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_repeatable(gpu):
    """Sums for the weights do not depend on what runs when."""
    g = torch.Generator(device="cuda").manual_seed(14)
    q, k = rows(g, 4, 16, 1000, 128, torch.bfloat16), rows(g, 4, 4, 1000, 128, torch.bfloat16)
    qw, kw = weights(g, 128, torch.float32)
    r, at = sa.rotary_frequencies(128), torch.arange(1000, device="cuda")
    first = sa.rotate_heads_backward(q, k, q, k, at, r, qw, kw)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(sa.rotate_heads_backward(q, k, q, k, at, r, qw, kw), first))


@pytest.mark.parametrize("interleaved", [False, True])
def test_large_outputs(gpu, interleaved):
    """Outputs that go past the caches are, to the bit, those of parts of them that do not."""
    g = torch.Generator(device="cuda").manual_seed(15)
    B, S, H, D = 4, 2049, 64, 128
    q = torch.randn(B, S, H + 8, D, generator=g, device="cuda").bfloat16().transpose(1, 2)
    q, k = q[:, :H], q[:, H:]
    qw, kw = weights(g, D, torch.bfloat16)
    r, at = sa.rotary_frequencies(D, interleaved=interleaved), torch.arange(S, device="cuda")
    ups = [torch.randn(x.shape, generator=g, device="cuda").bfloat16() for x in (q, k)]
    whole = (*sa.rotate_heads(q, k, at, r, qw, kw), *sa.rotate_heads_backward(*ups, q, k, at, r, qw, kw)[:2])
    parts = [(*sa.rotate_heads(q[b:b + 1], k[b:b + 1], at, r, qw, kw), *sa.rotate_heads_backward(ups[0][b:b + 1], ups[1][b:b + 1], q[b:b + 1], k[b:b + 1], at, r, qw, kw)[:2])
             for b in range(B)]
    assert (q.numel() + k.numel()) * 2 >= 128 << 20 > (q.numel() + k.numel()) // 2
    for a, b in zip(whole, zip(*parts)):
        assert torch.equal(a, torch.cat(b))


def test_backward_captured_and_replayed(gpu):
    """A training step's forward and gradients in a graph; where an eager graph of the same leaves lives, the capture is refused and the process goes on."""
    g = torch.Generator(device="cuda").manual_seed(16)
    q, k = rows(g, 2, 4, 50, 128, torch.bfloat16), rows(g, 2, 2, 50, 128, torch.bfloat16)
    leaves = [x.requires_grad_() for x in (q, k, *weights(g, 128, torch.bfloat16))]
    r, at = sa.rotary_frequencies(128), torch.arange(50, device="cuda")
    ups = [torch.randn(x.shape, generator=g, device="cuda").to(x.dtype) for x in (q, k)]

    def step():
        y = sa.rotate_heads_trainable(leaves[0], leaves[1], at, r, leaves[2], leaves[3])
        return [x.detach() for x in y] + list(torch.autograd.grad(y, leaves, ups))

    step()
    torch.cuda.synchronize()
    alive = sa.rotate_heads_trainable(leaves[0], leaves[1], at, r, leaves[2], leaves[3])
    torch.autograd.grad(alive, leaves, ups, retain_graph=True)
    with pytest.raises(RuntimeError, match="still holds these leaves"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            q.normal_()
            leaves[2].uniform_(0.5, 1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), i


def test_broadcast_inputs(gpu):
    """Rows, weights and gradients that are one tensor expanded: their own gradients are the sums over what they were expanded to."""
    g = torch.Generator(device="cuda").manual_seed(18)
    q, k = rows(g, 1, 4, 9, 64, torch.float32).requires_grad_(), rows(g, 2, 1, 9, 64, torch.float32).requires_grad_()
    w = (1.0 + 0.3 * torch.randn((), generator=g, device="cuda")).requires_grad_()
    r, at = sa.rotary_frequencies(64), torch.arange(9, device="cuda")[None]
    ups = [torch.randn(1, 1, 9, 64, generator=g, device="cuda").expand(2, 4, 9, 64), torch.randn(2, 3, 1, 64, generator=g, device="cuda").expand(2, 3, 9, 64)]
    wide = q.expand(2, 4, 9, 64), k.expand(2, 3, 9, 64), w.expand(64), w.expand(64)
    y = sa.rotate_heads_trainable(wide[0], wide[1], at, r, wide[2], wide[3])
    got = torch.autograd.grad(y, [q, k, w], ups)
    full = [x.detach().contiguous() for x in wide]
    for a, b in zip(y, sa.rotate_heads(full[0], full[1], at, r, full[2], full[3])):
        assert torch.equal(a, b)
    dq, dk, dqw, dkw = sa.rotate_heads_backward(*(u.contiguous() for u in ups), full[0], full[1], at, r, full[2], full[3])
    assert torch.equal(got[0], dq.sum(0, keepdim=True)) and torch.equal(got[1], dk.sum(1, keepdim=True))
    assert torch.allclose(got[2], dqw.sum() + dkw.sum(), rtol=2.0 ** -18, atol=0.0)  # (128 numbers added up in float32, in some order)


def test_offsets_beyond_32_bits(gpu):
    """Sequences, tokens and heads further apart than 2^32 bytes, in and out."""
    g = torch.Generator(device="cuda").manual_seed(19)
    store = torch.zeros((5 << 29) + (1 << 20), dtype=torch.bfloat16, device="cuda")  # 5 GiB
    far = 5 << 28
    r, at = sa.rotary_frequencies(64), torch.arange(2, device="cuda")
    for strides in ((far, 1024, 64, 1), (4096, 1024, far, 1), (256, far, 64, 1)):
        q = store.as_strided((2, 2, 2, 64), strides)
        q.copy_(rows(g, 2, 2, 2, 64, torch.bfloat16))
        w = torch.ones(64, device="cuda")
        want = sa.rotate_heads(q.contiguous(), q.contiguous(), at, r, w, w)
        assert all(torch.equal(a, b) for a, b in zip(sa.rotate_heads(q, q, at, r, w, w), want))
        up = rows(g, 2, 2, 2, 64, torch.bfloat16)
        want = sa.rotate_heads_backward(up, up, q.contiguous(), q.contiguous(), at, r, w, w)
        assert all(torch.equal(a, b) for a, b in zip(sa.rotate_heads_backward(up, up, q, q, at, r, w, w), want))
