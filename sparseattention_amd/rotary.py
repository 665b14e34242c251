"""Norms of queries and keys for each head and their rotation by position, in front of attention.

The reference's attention takes q and k as they are (sparse_attn_kernel.py:149).  A training step's or a prompt's attention is

    q, k = rotate_heads_trainable(q, k, positions, rotary, q_weight, k_weight)
    o = sparse_attention_trainable(q, k, v, mask, BLOCK_Q, BLOCK_K, ...)

and where keys go to a paged cache :func:`sparseattention_amd.paged_cache_append_rotated` does the same on their way in.  The calls enqueue work
on the current stream of q's device and read no tensor on the host.  Kernels: csrc/rotate.hip."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _native


@dataclass
class Rotary:
    """How positions turn pairs of a head's first R columns: pair ``j`` by ``positions * frequencies[j]`` radians.

    ``frequencies``: float64 [R/2], R a multiple of 8.  ``axes``: None, or int32 [R/2], which row of ``positions`` [axes, B, S] (time, height, width,
    ...) each pair turns by.  Pairs are columns ``(j, j + R/2)`` or, ``interleaved``, ``(2j, 2j + 1)``.  Both tensors on the device of the calls."""

    frequencies: torch.Tensor
    axes: Optional[torch.Tensor] = None
    interleaved: bool = False


def rotary_frequencies(R: int, base: float = 10000.0, *, sections: Optional[Sequence[int]] = None, interleaved: bool = False, device=None) -> Rotary:
    """The usual :class:`Rotary`: ``base ** (-2j / R)``; with ``sections`` (pairs of each axis, R/2 in all) the first ``sections[0]`` pairs turn by
    row 0 of the positions, the next ones by row 1, and so on."""
    if R < 8 or R > 256 or R % 8:
        raise ValueError(f"the rotated columns must be a multiple of 8 up to 256 (got {R})")
    if not 0.0 < base < float("inf"):
        raise ValueError(f"base must be positive and finite (got {base})")
    device = torch.device("cuda") if device is None else torch.device(device)
    j = torch.arange(R // 2, dtype=torch.float64)
    axes = None
    if sections is not None:
        if not sections or min(sections) < 0 or sum(sections) != R // 2:
            raise ValueError(f"sections must add up to the {R // 2} pairs (got {tuple(sections)})")
        axes = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(list(sections))).to(torch.int32).to(device)
    return Rotary((float(base) ** (-2.0 * j / R)).to(device), axes, bool(interleaved))


def rotate_heads(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rotary: Rotary, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """``(q', k')`` like ``q`` [B,Hq,S,D] and ``k`` [B,H,S,D] (bf16, fp16 or float32, any strides; D a multiple of 8 up to 256): each head's row
    over ``sqrt(mean(x^2) + eps)`` times its weight [D] (None: no norm), then rotated.

    ``positions``: int32 or int64, [S] or [B,S] (or [1,S]); [axes,B,S] with ``rotary.axes``, whose entries are taken as the nearest axis there is.
    Angles are exact to 2^-24 of a turn up to positions of 2^31; all else is float32, rounded once.  (Squares of values beyond 1e18 do not fit
    float32, nor, where ``eps`` is below 1e-37, those of rows below 1e-18.)  Weights are of q's type or float32, both the same."""
    return _native.host().rotate_heads(q, k, positions, rotary, q_weight, k_weight, eps)


def rotate_heads_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rotary: Rotary,
                          q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """``(dq, dk, dq_weight, dk_weight)``: the gradients of :func:`rotate_heads` for those of its outputs (``dq``, ``dk`` like them); a weight that
    is None has None.  Sums for the weights are made in a fixed order."""
    return _native.host().rotate_heads_backward(dq, dk, q, k, positions, rotary, q_weight, k_weight, eps)


def rotate_heads_trainable(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rotary: Rotary, q_weight: Optional[torch.Tensor] = None,
                           k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """:func:`rotate_heads` for autograd: gradients for q, k and the weights (once; second derivatives are refused).

    A backward under graph capture is refused where gradients it is asked for go on to something of the default stream, which cannot join a capture: leaves that a graph made
    there before holds as long as its outputs live, or inputs made there."""
    return _native.host().rotate_heads_trainable(q, k, positions, rotary, q_weight, k_weight, eps)
