"""rotate_heads_trainable under capture beside graphs of the same leaves that are still alive: refused where the backward would come to the default stream, which cannot wait for a
captured one; everything else goes through and replays right."""
import gc

import pytest
import torch

import sparseattention_amd as sa
from test_gpu_rotate import rows, weights

pytestmark = pytest.mark.gpu
HELD = "still holds these leaves"


def setting(seed):
    """Leaves that the rotation does not take as they are: q, k as views of the rows of a projection, weights as products."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, y = (torch.randn(2, 50, h * 128, generator=g, device="cuda").bfloat16().requires_grad_() for h in (4, 2))
    qw, kw = (w.requires_grad_() for w in weights(g, 128, torch.bfloat16))
    r, at = sa.rotary_frequencies(128), torch.arange(50, device="cuda")
    ups = [torch.randn(2, h, 50, 128, generator=g, device="cuda").bfloat16() for h in (4, 2)]

    def forward():
        q, k = (t.view(2, 50, -1, 128).transpose(1, 2) for t in (x, y))
        return sa.rotate_heads_trainable(q, k, at, r, 1 * qw, 1 * kw)

    return [x, y, qw, kw], ups, forward


def replays(graph, out, leaves, step):
    for i in range(4):
        with torch.no_grad():
            leaves[0].normal_()
            leaves[2].uniform_(0.5, 1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), i


@pytest.mark.parametrize("held", range(4))
def test_leaves_behind_views_of_a_living_graph(gpu, held):
    """One of the leaves is held by a graph of the default stream, that of another operator: refused, the process goes on, and without it the capture goes through."""
    leaves, ups, forward = setting(held)

    def step():
        y = forward()
        return [t.detach() for t in y] + list(torch.autograd.grad(y, leaves, ups))

    step()
    torch.cuda.synchronize()
    alive = leaves[held] * 2
    with pytest.raises(RuntimeError, match=HELD):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    del alive
    gc.collect()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    replays(graph, out, leaves, step)


def test_inputs_of_the_default_stream(gpu):
    """q is not a leaf but made by the program's own operations outside of the capture."""
    leaves, ups, _ = setting(4)
    q, k = (t.view(2, 50, -1, 128).transpose(1, 2) for t in leaves[:2])
    r, at = sa.rotary_frequencies(128), torch.arange(50, device="cuda")
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match=HELD):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(sa.rotate_heads_trainable(q, k, at, r), leaves[:2], ups)


def test_warm_up_of_a_side_stream_alive(gpu):
    """A whole step as torch documents its capture: the last warm-up's outputs, of a side stream, are still there.  That stream joins the capture."""
    leaves, ups, forward = setting(5)

    def step():
        y = forward()
        return [t.detach() for t in y] + list(torch.autograd.grad(y, leaves, ups, retain_graph=True)), y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            alive = step()[1]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()[0]
    assert alive[0].grad_fn is not None
    side.synchronize()
    with torch.cuda.stream(side):
        replays(graph, out, leaves, lambda: step()[0])


@pytest.mark.parametrize("no_grad", [True, False])
def test_a_forward_alone(gpu, no_grad):
    """A capture without a backward has no need of the leaves, whatever holds them."""
    leaves, ups, forward = setting(6)
    q, k = (t.detach().view(2, 50, -1, 128).transpose(1, 2) for t in leaves[:2])
    r, at = sa.rotary_frequencies(128), torch.arange(50, device="cuda")
    call = lambda: sa.rotate_heads_trainable(q, k, at, r, *leaves[2:])  # noqa: E731
    alive = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        if no_grad:
            with torch.no_grad():
                out = call()
        else:
            out = [t.detach() for t in call()]
    assert alive[0].grad_fn is not None
    replays(graph, out, leaves, call)


def test_gradients_that_nobody_asks_for(gpu):
    """The weights are held by a graph of the default stream, and only q's and k's gradients are asked for."""
    leaves, ups, forward = setting(7)

    def step():
        y = forward()
        return [t.detach() for t in y] + list(torch.autograd.grad(y, leaves[:2], ups))

    step()
    alive = [w * 2 for w in leaves[2:]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    assert alive[0].grad_fn is not None
    replays(graph, out, leaves, step)
