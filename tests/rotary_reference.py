"""Norm and rotation of the rows of heads in plain torch, in 64 bits, on the CPU: what the tests hold the kernels against."""
import math

import torch


def pairs(R, interleaved):
    """The columns of the first and of the second members of the pairs."""
    j = torch.arange(R // 2)
    return (2 * j, 2 * j + 1) if interleaved else (j, j + R // 2)


def angles(positions, frequencies, axes=None):
    """[B, S, R/2] of positions [B, S], or [axes, B, S] with axes, reduced to half a turn."""
    p = positions.double().cpu()
    p = p[..., None] if axes is None else p[axes.long().cpu()].permute(1, 2, 0)
    t = p * frequencies.double().cpu()
    return t - 2 * math.pi * torch.round(t / (2 * math.pi))


def normed(x, weight, eps):
    x = x.double()
    if weight is None:
        return x
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()


def turned(y, t, interleaved, back=False):
    """Rows y [B, H, S, D] by t [B, S, R/2]."""
    a, b = pairs(2 * t.shape[-1], interleaved)
    co, si = torch.cos(t)[:, None], torch.sin(t)[:, None] * (-1.0 if back else 1.0)
    out = y.clone()
    out[..., a] = y[..., a] * co - y[..., b] * si
    out[..., b] = y[..., a] * si + y[..., b] * co
    return out


def sizes(y, R, interleaved):
    """For each element the magnitudes of its pair added up (its own where it is not rotated): what errors of sine and cosine are relative to."""
    a, b = pairs(R, interleaved)
    out = y.abs().clone()
    out[..., a] = out[..., b] = y[..., a].abs() + y[..., b].abs()
    return out


def forward(x, t, weight, eps, interleaved):
    y = normed(x.cpu(), weight.cpu() if weight is not None else None, eps)
    return turned(y, t, interleaved), sizes(y, 2 * t.shape[-1], interleaved)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def forward_tolerance(out, size, dtype, far=0.0):
    """One rounding to the output's type.  In front of it, in float32 (half a step: 2^-24): the norm's factor (a sum of squares in 13 steps at
    most, of which the root halves the error, the root itself and two products: 12 * 2^-24), sine and cosine (argument and series: 2^-22 together), two products and a
    sum (3 * 2^-24): less than 2^-21 of the pair's magnitudes.  far: the angle's own error.  fp16 below 2^-14 has steps of 2^-24."""
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    return half_step(dtype) * out.abs() * (1 + 2.0 ** -20) + (2.0 ** -21 + far) * size + tiny


def backward(dy, x, t, weight, eps, interleaved, dtype):
    """(dx, its tolerance, dw, its tolerance)."""
    dy, x = dy.double().cpu(), x.double().cpu()
    R, D = 2 * t.shape[-1], x.shape[-1]
    g, gsize = turned(dy, t, interleaved, back=True), sizes(dy, R, interleaved)
    u, tiny = half_step(dtype), 2.0 ** -25 if dtype == torch.float16 else 1e-38
    if weight is None:
        return g, u * g.abs() * (1 + 2.0 ** -20) + 2.0 ** -21 * gsize + tiny, None, None
    w = weight.double().cpu()
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    dx = r * w * g - x * r ** 3 * (x * w * g).mean(-1, keepdim=True)
    # the same with magnitudes: every factor is off by less than 2^-20 of its own
    size = r * w.abs() * gsize + x.abs() * r ** 3 * (x * w * gsize).abs().mean(-1, keepdim=True)
    terms = (g * x * r)
    rows = terms.shape[0] * terms.shape[1] * terms.shape[2]
    dw, wsize = terms.sum((0, 1, 2)), (gsize * (x * r).abs()).sum((0, 1, 2))
    dwt = half_step(weight.dtype) * dw.abs() * (1 + 2.0 ** -20) + ((rows + 16) * 2.0 ** -24 + 2.0 ** -20) * wsize + 1e-30
    return dx, u * dx.abs() * (1 + 2.0 ** -20) + 2.0 ** -19 * size + tiny, dw, dwt


def assert_within(got, want, tolerance, what=""):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, f"{what}: {got.shape} instead of {want.shape}"
    bad = ~((got - want).abs() <= tolerance) & ~(torch.isnan(got) & torch.isnan(want))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} beyond, by up to {float(((got - want).abs() / tolerance)[bad].max()):.3g} times the tolerance"
