"""Verification of drafted tokens against the target's probabilities.

The reference decodes nothing.  A step with drafted tokens over a paged cache (paged_cache.py), a tree of n whose root is the last token that the sequence
has, of a model that norms and rotates its heads:

    q = paged_cache_append_rotated(cache, q, k, v, page_table, lens, rotary, parents=parents)
    o = sparse_attention_decode_tree(q, cache, page_table, lens + n, parents)
    path, accepted, token = verify_drafts(probabilities(o), tokens, uniforms, parents)
    paged_cache_keep(cache, page_table, lens, path, accepted)
    lens = lens + accepted

(first, second and fourth line in each layer with its own cache), after which ``token`` is the root of the next tree.  Kernel: csrc/verify.hip."""
from __future__ import annotations

from typing import Optional

import torch

from . import _native


def verify_drafts(target_probs: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor, parents: Optional[torch.Tensor] = None,
                  draft_probs: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None):
    """``(path, accepted, next_token)``: which drafted tokens the target keeps, and the token behind them.

    ``tokens`` [B,n] (int32 or int64, n <= 64): node 0 is the last token that the sequence has (its number is not looked at), node ``i`` was drafted behind
    ``parents[b, i]`` in ``[0, i)`` (int32 [B,n]; any other value: behind none) or, without ``parents``, behind node ``i - 1``.  ``target_probs``
    [B,n,V] (bf16, fp16 or float32, V <= 2^21): row ``i`` has the target's probabilities of the token behind node ``i``, which the tests take to add up to 1.
    ``uniforms`` float32 [B,n]: random numbers in [0, 1).

    From node 0 on the children of the node at hand are tried in their order.  Child ``c`` with token ``x`` is accepted if ``uniforms[b, c] * rest < p(x)``,
    where ``rest`` is 1 less the p of the siblings rejected before it (and p(x) is 0 if x was one of them); then its children are tried.  Where no child is accepted
    the next token is the first whose running sum of p without the rejected tokens is beyond ``uniforms[b, 0]`` times the whole.  What comes out is
    distributed as the target's own tokens are, however the drafts were made.

    ``draft_probs`` [B, n - 1 or more, V] (chains only, target_probs' type): row ``i`` is what the token of node ``i + 1`` was drawn from.  It is accepted if
    ``uniforms[b, i + 1] * q(x) < p(x)``, and after a rejection the next token comes from max(p - q, 0): the target's distribution too, with more accepted.

    ``path`` int32 [B,n]: the accepted nodes, node 0 first, -1 behind; ``accepted`` int32 [B]: how many; ``next_token`` [B] like tokens.  ``counts`` (int32
    [B]): trees of fewer nodes; with none nothing is accepted and the next token is -1, as it is where p has no positive entry.  A node whose
    token is outside [0, V) is not there.  Negative, infinite and NaN probabilities count as 0; if the rejected tokens were all that p has, the next token comes from p.
    Everything is computed in 64 bits.  The call reads nothing on the host and can be captured into a graph."""
    return _native.host().verify_drafts(target_probs, tokens, uniforms, parents, draft_probs, counts)
