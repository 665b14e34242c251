"""The 8-bit paged K/V cache in plain torch, in 64 bits, on the CPU: what the tests hold its kernels against."""
import math

import torch

BLOCK = 32
EXP_MIN, EXP_MAX = -96, 119


def round_e4m3(y: torch.Tensor) -> torch.Tensor:
    """float64, magnitudes up to 448, to the nearest number of four significant bits from 2^-9 upwards, ties to even."""
    size = y.abs().clamp(min=2.0 ** -6)
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(size).exponent - 4))
    return torch.round(y / step) * step


def exponent_of(x: torch.Tensor) -> int:
    x = x[torch.isfinite(x)].abs()
    top = float(x.max()) if x.numel() else 0.0
    if top == 0.0:
        return EXP_MIN
    m, e = math.frexp(top)
    return min(max(e - 9 if m <= 0.875 else e - 8, EXP_MIN), EXP_MAX)


def held_at(x: torch.Tensor, e: int) -> torch.Tensor:
    y = round_e4m3((x / 2.0 ** e).clamp(-448.0, 448.0)) * 2.0 ** e
    return torch.where(torch.isfinite(x), y, math.nan)


class Sequence:
    """One head's tokens [n, D] as a cache holds them after a row of appends."""

    def __init__(self, D):
        self.x = torch.zeros(0, D, dtype=torch.float64)
        self.exps = []

    def append(self, new: torch.Tensor):
        new = new.double().cpu()
        while len(new):
            at = len(self.x) % BLOCK
            part, new = new[:BLOCK - at], new[BLOCK - at:]
            e = exponent_of(part)
            if at:
                if e > self.exps[-1]:
                    self.x[-at:] = held_at(self.x[-at:], e)
                    self.exps[-1] = e
                e = self.exps[-1]
            else:
                self.exps.append(e)
            self.x = torch.cat([self.x, held_at(part, e)])


def attention(q, k, v, see):
    """q [R,D], k, v [n,D] and see [R,n] in 64 bits: o [R,D], lse [R], and what bounds the kernels' error: the sum of p |v| and the
    largest sum of |q k|, scaled, per row."""
    scale = q.shape[-1] ** -0.5
    s = torch.where(see, (q @ k.nan_to_num(0.0).T) * scale, -math.inf)
    s = torch.where(see & torch.isnan(k).any(-1), math.nan, s)
    lse = torch.logsumexp(s, -1) if k.shape[0] else torch.full((q.shape[0],), -math.inf, dtype=torch.float64)
    p = torch.where(see, torch.exp(s - lse[:, None]), 0.0)
    bad = (see.double() @ torch.isnan(v).double()) > 0
    o = torch.where(bad, math.nan, p @ v.nan_to_num(0.0))
    size = p.nan_to_num(0.0) @ v.nan_to_num(0.0).abs()
    arg = torch.where(see, (q.abs() @ k.nan_to_num(0.0).abs().T) * scale, 0.0).amax(-1) if k.shape[0] else torch.zeros(q.shape[0], dtype=torch.float64)
    return o, lse, size, arg


def tolerances(o, lse, size, arg, n, vmax, D, dtype):
    """How far the kernels may be off.  A weight p is rounded to 16 bits (half a step: u), and half an ulp of fp16's smallest
    numbers where it is below those (the largest weight of a row is at least 1 before the division); the output is rounded
    once more; a score is a float32 sum of D products, exp2 and the sums over keys are float32."""
    u = torch.finfo(dtype).eps / 2
    score = ((D + 8) * 2.0 ** -24) * arg
    tiny = n * 2.0 ** -25 * vmax if dtype == torch.float16 else 0.0
    out = u * o.abs() + (u + 2.0 ** -20 + n * 2.0 ** -24 + 2.2 * score)[:, None] * size * 1.01 + tiny + 1e-30
    return out, 1.1 * score + 2.0 ** -20 * (1.0 + lse.abs()) + n * 2.0 ** -24
