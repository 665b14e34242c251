"""Norm and rotation of heads: refusals on the host before anything is launched, and the reference's gradients against differences (these
run without a GPU)."""
import ctypes

import pytest
import torch

import rotary_reference as ref
import sparseattention_amd as sa
from sparseattention_amd import _native

FAKE = 0x1000  # never dereferenced: every call below must fail validation first
BAD, UNSUPPORTED, WORKSPACE = _native.SA_ERR_INVALID_ARGUMENT, _native.SA_ERR_UNSUPPORTED, _native.SA_ERR_WORKSPACE
S4 = _native.strides((1024, 128, 128, 1))


def rotation(f=FAKE, axes=None, positions=FAKE, wide=0, n=1, R=128, qw=None, kw=None, wt=0, eps=1e-6):
    return ctypes.byref(_native.RotationStruct(f, axes, positions, (ctypes.c_int64 * 3)(0, 8, 1), wide, n, R, 0, qw, kw, wt, eps))


def forward(q=FAKE, qs=S4, k=FAKE, out=FAKE, r=None, B=1, Hq=2, H=1, S=4, D=128, dtype=0):
    return _native.load().sa_rotate_heads(q, qs, k, S4, out, S4, FAKE, S4, r or rotation(), B, Hq, H, S, D, dtype, None)


def backward(dq=FAKE, q=FAKE, dqw=None, r=None, ws=None, size=0, B=1, Hq=2, H=1, S=4, D=128, dtype=0, **_):
    return _native.load().sa_rotate_heads_bwd(dq, S4, FAKE, S4, q, S4, q, S4, FAKE, S4, FAKE, S4, dqw, None, r or rotation(), ws, size, B, Hq, H, S, D, dtype, None)


@pytest.mark.parametrize("call", [forward, backward])
def test_rotations(call):
    assert call(r=rotation(f=None)) == BAD and call(r=rotation(positions=None)) == BAD and call(r=rotation(n=0)) == BAD
    assert call(r=rotation(R=0)) == UNSUPPORTED and call(r=rotation(R=20)) == UNSUPPORTED and call(r=rotation(R=136)) == UNSUPPORTED
    assert call(r=rotation(eps=-1.0)) == BAD and call(r=rotation(eps=float("nan"))) == BAD and call(r=rotation(eps=float("inf"))) == BAD
    assert call(r=rotation(qw=FAKE, wt=1)) == UNSUPPORTED and call(r=rotation(f=FAKE + 4)) == UNSUPPORTED
    assert call(r=rotation(positions=FAKE + 4, wide=1)) == UNSUPPORTED and call(r=rotation(kw=FAKE + 2, wt=2)) == UNSUPPORTED
    for name in ("B", "Hq", "H", "S"):
        assert call(**{name: 0}) == BAD
    assert call(D=0) == UNSUPPORTED and call(D=100) == UNSUPPORTED and call(D=264) == UNSUPPORTED and call(dtype=3) == UNSUPPORTED
    assert call(B=1 << 16, S=1 << 16) == UNSUPPORTED and call(H=(1 << 20) + 1) == UNSUPPORTED


def test_more_than_a_launch_has():
    assert forward(B=1 << 15, S=1 << 15) == UNSUPPORTED


def test_rows_and_weights():
    assert forward(q=None) == BAD and forward(k=None) == BAD and forward(out=None) == BAD and forward(q=FAKE + 8) == UNSUPPORTED
    assert forward(qs=_native.strides((1024, 128, 124, 1))) == UNSUPPORTED and forward(qs=_native.strides((1024, 128, 128, 2))) == UNSUPPORTED
    assert forward(qs=_native.strides((1024, 128, 130, 1)), dtype=2) == UNSUPPORTED
    assert backward(dq=None) == BAD and backward(dqw=FAKE) == BAD  # (no weight to have a gradient)
    weighted = rotation(qw=FAKE)
    assert backward(q=None, r=weighted) == BAD and backward(dqw=FAKE, r=weighted) == WORKSPACE
    need = _native.load().sa_rotate_heads_bwd_workspace_bytes(1, 2, 1, 4, 128)
    assert need > 0 and backward(dqw=FAKE, r=weighted, ws=FAKE, size=need - 1) == WORKSPACE
    assert _native.load().sa_rotate_heads_bwd_workspace_bytes(0, 2, 1, 4, 128) == 0


def test_python_refuses():
    with pytest.raises(ValueError, match="multiple of 8"):
        sa.rotary_frequencies(20, device="cpu")
    for kw in (dict(base=0.0), dict(base=float("inf")), dict(sections=(3, 4)), dict(sections=()), dict(sections=(-1, 33))):
        with pytest.raises(ValueError):
            sa.rotary_frequencies(64, device="cpu", **kw)
    r = sa.rotary_frequencies(64, sections=(8, 12, 12), device="cpu")
    assert r.axes.tolist() == [0] * 8 + [1] * 12 + [2] * 12 and r.axes.dtype == torch.int32 and r.frequencies[0] == 1.0
    r, at = sa.rotary_frequencies(64, device="cpu"), torch.arange(4)
    q, k = torch.zeros(1, 2, 4, 64), torch.zeros(1, 1, 4, 64)
    for call in (sa.rotate_heads, sa.rotate_heads_trainable, lambda *a: sa.rotate_heads_backward(q, k, *a)):
        with pytest.raises(RuntimeError, match="GPU"):
            call(q, k, at, r)
        for bad in ((q[0], k), (q, k[:, :, :3]), (q[:0], k), (q[..., :32], k)):
            with pytest.raises(ValueError):
                call(*bad, at, r)
        with pytest.raises(TypeError):
            call(q.double(), k.double(), at, r)
        with pytest.raises(TypeError):
            call(q, k.half(), at, r)
        with pytest.raises(TypeError, match="frequencies"):
            call(q, k, at, object())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
def test_the_reference_gradient_against_differences(interleaved, weighted):
    """Central differences of the float64 function with steps h are off by h^2 / 6 of its third derivative (here less than 10^2 of the values) and
    2^-52 / h of the values: 10^-6 with h = 10^-5 holds both."""
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(2, 3, 5, 24, generator=g, dtype=torch.float64) for _ in range(2))
    w = 1.0 + 0.3 * torch.randn(24, generator=g, dtype=torch.float64) if weighted else None
    t = ref.angles(torch.arange(10).view(2, 5), 10.0 ** -torch.arange(8).double(), None)
    dx, _, dw, _ = ref.backward(dy, x, t, w, 1e-3, interleaved, torch.float64)
    f = lambda x, w: (ref.forward(x, t, w, 1e-3, interleaved)[0] * dy).sum()  # noqa: E731
    h = 1e-5
    for _ in range(8):
        v = torch.randn(x.shape, generator=g, dtype=torch.float64)
        assert abs((f(x + h * v, w) - f(x - h * v, w)) / (2 * h) - (dx * v).sum()) <= 1e-6 * (dx.abs() * v.abs()).sum()
        if weighted:
            v = torch.randn(24, generator=g, dtype=torch.float64)
            assert abs((f(x, w + h * v) - f(x, w - h * v)) / (2 * h) - (dw * v).sum()) <= 1e-6 * (dw.abs() * v.abs()).sum()
