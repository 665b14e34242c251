"""Measured calls around the attention of a decoding step with drafted tokens: norms and position rotation of queries and keys
(alone, with their gradients, and on the way into the 8-bit paged K/V cache), attention for a tree of drafts over that cache, their
verification, and keeping the accepted ones in it.

A case is a dict of plain values.  ``prepare`` makes what a program holds before the call, ``run`` is one pass and gives
its outputs, ``work`` the bytes and operations that the pass cannot do without, ``exact`` the outputs in 64 bits.  Where
``own`` is false ``run`` computes the same from elementary torch operations on a cache of natural layout.

The cache holds a block of 32 consecutive tokens of one head as e4m3 codes times 2^e, e the least integer for which the
block's largest magnitude is at most 448 * 2^e.  Tokens that come to a block that holds some never lower its e; where it grows, what the
block held is rounded again.

Rotation: a pair (a, b) of a head's first R columns, (j, j + R/2) or interleaved (2j, 2j + 1), turns by
positions[axis of j] * frequency of j.  Norm: x / sqrt(mean(x^2) + eps) * weight over a head's D columns, before the rotation.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 32  # tokens that share a scale
E_MIN, E_MAX = -96, 119
EPS = 1e-6


def listed() -> list[dict]:
    return [
        # patches of a small batch of images, positions of (time, height, width), no norms: forward only
        dict(name="rotate_images", kind="rotate", B=2, S=1031, Hq=16, H=16, D=80, R=80, axes=3, interleaved=False, norm=False, start=0, grad=False,
             dtype="fp16"),
        # a training step's queries and keys of packed sequences, norms with their weights, and all gradients: the largest of its kind
        dict(name="rotate_train", kind="rotate", B=4, S=4096, Hq=32, H=8, D=128, R=128, axes=1, interleaved=False, norm=True, start=0, grad=True,
             dtype="bf16"),
        # one token for every sequence of a batch under way: latency
        dict(name="append_tokens", kind="append", B=64, H=8, G=4, D=128, R=128, P=64, S=1, held=2048, spread=0.9, ragged=0.0, norm=True,
             interleaved=False, dtype="bf16"),
        # a chunk of a long prompt far behind its start
        dict(name="append_chunk", kind="append", B=1, H=8, G=4, D=128, R=128, P=64, S=4096, held=50001, spread=0.0, ragged=0.0, norm=True,
             interleaved=False, dtype="bf16"),
        # new prompts of a padded batch, half precision, interleaved pairs in half of the columns, no norms: the largest of its kind
        dict(name="append_prompts", kind="append", B=16, H=12, G=1, D=64, R=32, P=32, S=2047, held=0, spread=0.0, ragged=0.8, norm=False,
             interleaved=True, dtype="fp16"),
        # a single conversation with a few drafts: the smallest attention, all latency
        dict(name="tree_one", kind="tree", B=1, H=8, G=4, D=128, P=64, n=8, length=2011, spread=0.0, window=0, dtype="bf16"),
        # a serving batch of very different lengths, a tree of drafts for each, the row statistics kept
        dict(name="tree_batch", kind="tree", B=32, H=8, G=4, D=128, P=64, n=25, length=8192, spread=0.9, window=0, lse=True, dtype="bf16"),
        # wide trees over long contexts, half precision: the largest
        dict(name="tree_long", kind="tree", B=8, H=8, G=4, D=64, P=128, n=64, length=65536, spread=0.3, window=0, dtype="fp16"),
        # chains of a few tokens drawn from a draft model, checked with its probabilities
        dict(name="verify_chains", kind="verify", B=8, n=6, V=32000, drawn=True, dtype="fp32"),
        # trees for a full batch, a large vocabulary
        dict(name="verify_trees", kind="verify", B=64, n=32, V=131072, drawn=False, dtype="fp32"),
        # the accepted path of one conversation's drafts moved up in its cache: latency
        dict(name="keep_one", kind="keep", B=1, H=8, D=128, P=64, n=8, length=2011, spread=0.0, dtype="bf16"),
        # the same for a full batch and wide trees
        dict(name="keep_batch", kind="keep", B=128, H=8, D=128, P=64, n=64, length=1024, spread=0.9, dtype="bf16"),
    ]


def _log_uniform(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["rotate", "rotate", "append", "append", "tree", "tree", "tree", "verify", "verify", "keep"])
    D = rng.choice([64, 80, 128, 128, 256])
    c = dict(kind=kind, D=D, H=rng.choice([1, 2, 4, 8, 8, 12, 16]), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind in ("rotate", "append"):
        c["R"] = rng.choice([D, D, D // 2])
        c["norm"] = rng.random() < 0.6
        c["interleaved"] = rng.random() < 0.4
        c["S"] = 1 if rng.random() < 0.3 else _log_uniform(rng, 2, 8192)
    if kind != "rotate":
        c["P"] = rng.choice([32, 64, 64, 128, 256])
        c["spread"] = round(rng.uniform(0.0, 1.0), 2)
    G = rng.choice([1, 1, 2, 4, 4, 7, 8])
    if kind == "rotate":
        c["Hq"] = c["H"] * G
        c["axes"] = rng.choice([1, 1, 2, 3])
        c["grad"] = rng.random() < 0.6
        c["start"] = rng.choice([0, 0, _log_uniform(rng, 1, 1 << 20)])
        c["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c["B"] = _log_uniform(rng, 1, max(1, min(128, (1 << 25) // ((c["Hq"] + c["H"]) * D * c["S"]))))
    elif kind == "append":
        c["G"] = G
        c["B"] = _log_uniform(rng, 1, max(1, min(128, (1 << 25) // (c["H"] * (G + 2) * D * (c["S"] + 256)))))
        c["held"] = rng.choice([0, 1, 31, 32, _log_uniform(rng, 2, 8192)])
        c["ragged"] = rng.choice([0.0, round(rng.uniform(0.0, 1.0), 2)])
    elif kind == "tree":
        c["G"] = G
        c["n"] = rng.choice([1, 2, 5, 16, 33, 64])
        c["length"] = _log_uniform(rng, c["n"], 65536)
        c["B"] = _log_uniform(rng, 1, max(1, min(128, (1 << 26) // (c["H"] * D * c["length"]))))
        c["window"] = rng.choice([0, 0, _log_uniform(rng, 1, 8192)])
        c["lse"] = rng.random() < 0.3
    elif kind == "verify":
        c = dict(kind=kind, n=rng.choice([1, 2, 5, 16, 33, 64]), V=_log_uniform(rng, 100, 200000), drawn=rng.random() < 0.5,
                 dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))
        c["B"] = _log_uniform(rng, 1, max(1, min(128, (1 << 26) // (c["n"] * c["V"]))))
    else:
        c["n"] = rng.choice([1, 2, 5, 16, 33, 64])
        c["length"] = _log_uniform(rng, c["n"], 8192)
        c["B"] = _log_uniform(rng, 1, max(1, min(128, (1 << 26) // (c["H"] * D * c["length"]))))
    most = max(work(x)["bytes"] for x in listed() if x["kind"] == kind)
    while work(c)["bytes"] > most:  # sequences, then tokens, then heads
        name = next(x for x in ("B", "S", "length", "H", "V") if c.get(x, 1) > (c["n"] if x == "length" else 1))
        c[name] //= 2
        c[name] = max(c[name], c["n"] if name == "length" else 1)
        if name == "H" and "Hq" in c:
            c["Hq"] = c["H"] * G
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _spread(n: int, top: int, spread: float) -> list[int]:
    """n numbers from top * (1 - spread) to top, the first one top, spread evenly in an irregular order."""
    return [max(0, round(top * (1.0 - spread * ((i * 0.6180339887) % 1.0)))) for i in range(n)]


def _lens(c) -> list[int]:
    """Tokens that each sequence holds; of trees the drafts are among them, of kept ones not."""
    if c["kind"] == "append":
        return _spread(c["B"], c["held"], c["spread"])
    return [max(x, c["n"] if c["kind"] == "tree" else 0) for x in _spread(c["B"], c["length"], c["spread"])]


def _counts(c) -> list[int]:
    return _spread(c["B"], c["S"], c["ragged"])


def _pages_of(tokens: int, P: int) -> int:
    return -(-tokens // P)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _uniform(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _tokens(c, n: int, g, keys: bool) -> torch.Tensor:
    """[B, H, n, D] keys (a few channels much larger than the rest, as rotated keys have them) or values."""
    x = _normal(g, c["B"], c["H"], n, c["D"])
    if keys:
        x *= torch.exp(0.7 * _normal(g, 1, c["H"], 1, c["D"]))
    return x.to(DTYPES[c["dtype"]])


def _trees(B: int, n: int, g) -> torch.Tensor:
    """int32 [B, n]: node 0 is the root, every other one's parent one of the four nodes in front of it."""
    i = torch.arange(n, device="cuda")
    back = (_uniform(g, B, n) * i.clamp(max=4)).floor().long().clamp(max=3)
    return torch.where(i > 0, i - 1 - torch.minimum(back, (i - 1).clamp(min=0)), -1).to(torch.int32)


def _paths(parents: torch.Tensor, g):
    """(path int32 [B, n], accepted int32 [B]): the way from the root to a node drawn from each tree, -1 behind."""
    B, n = parents.shape
    at = (_uniform(g, B) * n).long().clamp(max=n - 1)
    on = torch.zeros(B, n, dtype=torch.bool, device="cuda")
    for _ in range(n):
        on.scatter_(1, at[:, None], True)
        at = parents.gather(1, at[:, None])[:, 0].long().clamp(min=0)
    count = on.sum(1)
    order = torch.argsort((~on).int(), dim=1, stable=True)
    path = torch.where(torch.arange(n, device="cuda") < count[:, None], order, -1)
    return path.to(torch.int32), count.to(torch.int32)


def _probabilities(logits: torch.Tensor, dtype) -> torch.Tensor:
    return torch.softmax(logits, -1).to(dtype)


def _drawn(p: torch.Tensor, g) -> torch.Tensor:
    """One token of each row of probabilities, [B, n]."""
    return torch.stack([torch.argmax(r.float() / -torch.log(_uniform(g, *r.shape).clamp(min=1e-30)), -1) for r in p])


def _frequencies(c) -> torch.Tensor:
    j = torch.arange(c["R"] // 2, dtype=torch.float64, device="cuda")
    return 10000.0 ** (-2.0 * j / c["R"])


def _axes(c):
    n = c.get("axes", 1)
    return None if n == 1 else (torch.arange(c["R"] // 2, device="cuda") * n // (c["R"] // 2)).to(torch.int32)


def _qkv(c, g, Hq: int, H: int, with_v: bool):
    """q, k (and v) [B, heads, S, D] as views of one projection's output [B, S, heads * D]."""
    x = _normal(g, c["B"], c["S"], Hq + H * (1 + with_v), c["D"])
    x[:, :, :Hq + H] *= torch.exp(0.7 * _normal(g, Hq + H, c["D"]))
    x = x.to(DTYPES[c["dtype"]]).transpose(1, 2)
    return x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:]


def _weights(c, g):
    if not c["norm"]:
        return None, None
    return tuple((1.0 + 0.3 * _normal(g, c["D"])).to(DTYPES[c["dtype"]]) for _ in range(2))


def _inputs(c, seed: int) -> dict:
    """Everything random or fixed that a case starts from, before any of it is held in 8 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, B = c["kind"], c["B"]
    s = {}
    if kind == "rotate":
        s["q"], s["k"], _ = _qkv(c, g, c["Hq"], c["H"], False)
        s["q_weight"], s["k_weight"] = _weights(c, g)
        at = c["start"] + torch.arange(c["S"], device="cuda").expand(B, c["S"])
        if c["axes"] > 1:  # a frame, and a place in a grid of 32 columns
            at = torch.stack([at // 1024, at % 1024 // 32, at % 32][:c["axes"]])
        s["positions"] = at.to(torch.int32).contiguous()
        if c["grad"]:
            s["dq"], s["dk"] = (_normal(g, B, c["S"], h, c["D"]).to(DTYPES[c["dtype"]]).transpose(1, 2) for h in (c["Hq"], c["H"]))
        return s
    if kind == "verify":
        n, V, dtype = c["n"], c["V"], DTYPES[c["dtype"]]
        logits = 4.0 * _normal(g, B, n, V)
        s["target"] = _probabilities(logits, dtype)
        s["uniforms"] = _uniform(g, B, n)
        if c["drawn"]:
            logits += 0.5 * _normal(g, B, n, V)
            s["draft"] = _probabilities(logits, dtype)
            after = _drawn(s["draft"], g)
            s["parents"] = None
            s["tokens"] = torch.cat([after[:, :1], after[:, :-1]], 1).contiguous()
        else:
            s["draft"] = None
            s["parents"] = _trees(B, n, g)
            after = _drawn(s["target"], g)
            s["tokens"] = after.gather(1, s["parents"].long().clamp(min=0))
            # (siblings other than the first are mostly other tokens)
            other = torch.randint(V, (B, n), generator=g, device="cuda")
            s["tokens"] = torch.where(_uniform(g, B, n) < 0.4, other, s["tokens"]).contiguous()
        return s
    P = c["P"]
    lens = _lens(c)
    counts = _counts(c) if kind == "append" else [c["n"]] * B if kind == "keep" else [0] * B
    ends = [a + b for a, b in zip(lens, counts)]
    # the columns of the table that new or moved tokens touch
    first = [a // P for a in lens]
    cols = max(1, max(_pages_of(e, P) - f for e, f in zip(ends, first)))
    width = max(1, _pages_of(max(ends), P)) + (cols if kind != "tree" else 0)
    used = B * width
    pages = torch.randperm(used + B * cols + 3, generator=g, device="cuda").to(torch.int32)
    s["pool"], s["width"], s["most"] = used + B * cols + 3, width, max(ends)
    s["lens"], s["table"] = _ints(lens), pages[:used].view(B, width).contiguous()
    held = max(1, max(lens) + (c["n"] if kind == "keep" else 0))
    s["held_k"], s["held_v"] = (_tokens(c, held, g, keys) for keys in (True, False))
    at = _ints(first).long()[:, None] + torch.arange(cols, device="cuda")
    s["touched"] = s["table"].gather(1, at.clamp(max=width - 1)).contiguous()
    if kind == "append":
        s["q"], s["k"], s["v"] = _qkv(c, g, c["H"] * c["G"], c["H"], True)
        s["q_weight"], s["k_weight"] = _weights(c, g)
        s["counts"] = _ints(counts)
        s["touched_lens"] = _ints([e - f * P for e, f in zip(ends, first)])
        s["touched_most"] = max(e - f * P for e, f in zip(ends, first))
    elif kind == "tree":
        s["q"] = _normal(g, B, c["H"] * c["G"], c["n"], c["D"]).to(DTYPES[c["dtype"]])
        s["parents"] = _trees(B, c["n"], g)
    else:
        s["path"], s["accepted"] = _paths(_trees(B, c["n"], g), g)
        # the pages that drafts touch are kept as they are, and the path in copies of them
        s["copies"] = pages[used:used + B * cols].view(B, cols).contiguous()
        s["table"] = s["table"].scatter(1, at, s["copies"])
        s["touched_lens"] = s["lens"] - _ints([f * P for f in first]) + s["accepted"]
        s["touched_most"] = cols * P
    return s


def prepare(case, seed: int) -> dict:
    s = dict(_inputs(case, seed), case=case)
    kind = case["kind"]
    if kind in ("rotate", "append"):
        s["frequencies"], s["axes"] = _frequencies(case), _axes(case)
        if own:
            import sparseattention_amd as sa

            s["rotary"] = sa.Rotary(s["frequencies"], s["axes"], case["interleaved"])
    if kind == "rotate" and own and case["grad"]:
        for name in ("q", "k", "q_weight", "k_weight"):
            if s[name] is not None:
                s[name].requires_grad_()
    if kind in ("rotate", "verify"):
        return s
    held_k, held_v = s.pop("held_k"), s.pop("held_v")
    table, lens = s["table"], s["lens"]
    if kind == "keep":  # what the copies are made from
        first = torch.div(lens, case["P"], rounding_mode="floor").long()[:, None] + torch.arange(s["touched"].shape[1], device="cuda")
        table, lens = table.scatter(1, first, s["touched"]), lens + case["n"]
    if own:
        import sparseattention_amd as sa

        s["cache"] = sa.empty_paged_cache(s["pool"], case["H"], case["D"], page_size=case["P"], device="cuda")
        sa.paged_cache_append(s["cache"], held_k, held_v, table, torch.zeros_like(lens), counts=lens)
    else:
        shape = (s["pool"], case["H"], case["P"], case["D"])
        for name, x in (("ck", held_k), ("cv", held_v)):
            s[name] = torch.zeros(shape, dtype=torch.float8_e4m3fn, device="cuda")
            s[name + "_exp"] = torch.full((s["pool"], case["H"], case["P"] // BLOCK), E_MIN, dtype=torch.int32, device="cuda")
            _append_plain(s[name], s[name + "_exp"], x, table, torch.zeros_like(lens), lens)
    return s


# ---- the plain form ---------------------------------------------------------------------------------------------------
def _pairs(x: torch.Tensor, R: int, interleaved: bool):
    if interleaved:
        return x[..., 0:R:2], x[..., 1:R:2]
    return x[..., :R // 2], x[..., R // 2:R]


def _unpaired(a, b, rest, interleaved: bool):
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def _angles_plain(s, positions):
    """cos and sin in 32 bits, [B, 1, S, R/2], of positions [B, S] or [axes, B, S]; the angles in 64, as positions may be far."""
    at = positions.double()[..., None] if s["axes"] is None else positions.double()[s["axes"].long()].permute(1, 2, 0)
    t = (at * s["frequencies"])[:, None]
    return torch.cos(t).float(), torch.sin(t).float()


def _rotate_plain(x, weight, angles, R, interleaved):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.float()
    (a, b), (co, si) = _pairs(y, R, interleaved), angles
    return _unpaired(a * co - b * si, a * si + b * co, y[..., R:], interleaved)


def _rotate_backward_plain(dy, x, weight, angles, R, interleaved):
    dy, (co, si) = dy.float(), angles
    a, b = _pairs(dy, R, interleaved)
    g = _unpaired(a * co + b * si, b * co - a * si, dy[..., R:], interleaved)
    if weight is None:
        return g.to(x.dtype), None
    y = x.float()
    r = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    hat = y * r
    wg = g * weight.float()
    dx = r * (wg - hat * (wg * hat).mean(-1, keepdim=True))
    return dx.to(x.dtype), (g * hat).double().sum((0, 1, 2)).to(weight.dtype)


def _exponent(amax: torch.Tensor) -> torch.Tensor:
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)  # 448 = 0.875 * 2^9
    return torch.where(amax > 0, e.to(torch.int32), E_MIN).clamp(E_MIN, E_MAX)


def _codes(x: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    y = torch.ldexp(x, -e).clamp(-448.0, 448.0)
    return torch.where(torch.isfinite(x), y, math.nan).to(torch.float8_e4m3fn)


def _finite_top(x, chosen):
    return torch.where(chosen & torch.isfinite(x), x.abs(), 0.0).amax((-1, -2))


def _append_plain(codes, exps, x, table, lens, counts) -> None:
    """x [B,H,S,D], the first counts[b] tokens to positions lens[b] ... of sequence b."""
    B, H, S, D = x.shape
    P = codes.shape[2]
    per = P // BLOCK
    blocks = codes.view(-1, H, per, BLOCK, D)
    step = max(1, (1 << 28) // (H * D * (S + 2 * BLOCK)))  # (sequences at a time: the intermediate tensors are 32 bits wide)
    for b0 in range(0, B, step):
        n = min(step, B - b0)
        sl = slice(b0, b0 + n)
        blk = lens[sl].long()[:, None] // BLOCK + torch.arange((S + 2 * BLOCK - 2) // BLOCK, device=x.device)  # [n, nb] blocks of the sequence
        nb = blk.shape[1]
        pos = blk[:, :, None] * BLOCK + torch.arange(BLOCK, device=x.device)  # [n, nb, 32] tokens
        src = pos - lens[sl].long()[:, None, None]
        new = (src >= 0) & (src < counts[sl].long()[:, None, None])
        live = new.any(-1)
        page = table[sl].long().gather(1, (blk // per).clamp(max=table.shape[1] - 1))
        old_codes = blocks[page, :, blk % per]  # [n, nb, H, 32, D]
        old_exp = torch.where((blk * BLOCK < lens[sl].long()[:, None])[..., None], exps[page, :, blk % per], E_MIN)
        rows = src.clamp(0, S - 1).view(n, 1, nb * BLOCK, 1).expand(n, H, nb * BLOCK, D)
        val = x[sl].float().gather(2, rows).view(n, H, nb, BLOCK, D).transpose(1, 2)
        sel = new[:, :, None, :, None]
        e = torch.maximum(old_exp, _exponent(_finite_top(val, sel)))
        again = _codes(torch.ldexp(old_codes.float(), old_exp[..., None, None]), e[..., None, None])
        kept = torch.where((e > old_exp)[..., None, None], again.float(), old_codes.float())
        out = torch.where(sel, _codes(val, e[..., None, None]).float(), kept).to(torch.float8_e4m3fn)
        at = live.nonzero(as_tuple=True)
        blocks.view(torch.uint8)[page[at], :, (blk % per)[at]] = out[at].view(torch.uint8)
        exps[page[at], :, (blk % per)[at]] = e[at]


def _keep_plain(codes, exps, table, lens, path, accepted) -> None:
    """Tokens lens + path[i] become tokens lens + i, i < accepted."""
    H, P, D = codes.shape[1:]
    B, n = path.shape
    per = P // BLOCK
    blocks = codes.view(-1, H, per, BLOCK, D)
    lens = lens.long()
    first = lens // BLOCK  # the block that holds token lens
    nb = (n + 2 * BLOCK - 2) // BLOCK
    blk = first[:, None] + torch.arange(nb, device=lens.device)
    page = table.long().gather(1, (blk // per).clamp(max=table.shape[1] - 1))
    sub = blk % per
    old_exp = exps[page, :, sub]  # [B, nb, H]
    old = torch.ldexp(blocks.view(torch.uint8)[page, :, sub].view(torch.float8_e4m3fn).float(), old_exp[..., None, None])  # [B, nb, H, 32, D]
    values = old.transpose(1, 2).reshape(B, H, nb * BLOCK, D)
    # which token of these blocks comes to which place
    place = torch.arange(nb * BLOCK, device=lens.device).expand(B, -1)
    i = place - (lens - first * BLOCK)[:, None]
    moved = (i >= 0) & (i < accepted.long()[:, None])
    source = torch.where(moved, (lens - first * BLOCK)[:, None] + path.long().gather(1, i.clamp(0, n - 1)), place)
    source = source.clamp(0, nb * BLOCK - 1)
    came = values.gather(2, source[:, None, :, None].expand(B, H, nb * BLOCK, D)).view(B, H, nb, BLOCK, D).transpose(1, 2)
    moved, source = moved.view(B, nb, BLOCK), source.view(B, nb, BLOCK)
    here = source // BLOCK == torch.arange(nb, device=lens.device)[:, None]
    counts = ((moved & here).any(-1) | (blk * BLOCK < lens[:, None]))[..., None]  # the block's own scale does
    e = torch.maximum(torch.where(counts, old_exp, E_MIN), _exponent(_finite_top(came, (moved & ~here)[:, :, None, :, None])))
    out = _codes(came, e[..., None, None])
    at = moved.any(-1).nonzero(as_tuple=True)
    blocks.view(torch.uint8)[page[at], :, sub[at]] = out[at].view(torch.uint8)
    exps[page[at], :, sub[at]] = e[at]


def _dense_plain(codes, exps, table, n: int) -> torch.Tensor:
    """The first n tokens of the sequences of a table [B, pages] in 32 bits, [B, H, n, D]."""
    _, H, P, D = codes.shape
    pages = table[:, :_pages_of(n, P)].long()
    x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()  # [B, pages, H, P, D]
    x = torch.ldexp(x, exps[pages].repeat_interleave(BLOCK, -1)[..., None])
    return x.transpose(1, 2).reshape(len(table), H, -1, D)[:, :, :n]


def _gather_plain(s, table, lens, most: int):
    out = []
    for name in ("ck", "cv"):
        x = _dense_plain(s[name], s[name + "_exp"], table, most)
        live = torch.arange(most, device="cuda") < lens[:, None]
        out.append(torch.where(live[:, None, :, None], x, 0.0).to(DTYPES[s["case"]["dtype"]]))
    return out


def _ancestors_plain(parents: torch.Tensor) -> torch.Tensor:
    """bool [B, n, n]: whether the row's node is the column's or comes from it."""
    B, n = parents.shape
    x = torch.eye(n, device=parents.device).expand(B, n, n).contiguous()
    x.scatter_(2, parents.long().clamp(min=0)[..., None], (parents >= 0).float()[..., None].maximum(x.gather(2, parents.long().clamp(min=0)[..., None])))
    for _ in range(max(1, n.bit_length())):
        x = (x @ x).clamp(max=1.0)
    return x > 0


def _tree_plain(s):
    c = s["case"]
    H, G, n, D, m = c["H"], c["G"], c["n"], c["D"], s["most"]
    above = _ancestors_plain(s["parents"])
    depth = above.sum(-1) - 1  # [B, n]
    outs, sums = [], []
    step = max(1, (1 << 28) // (H * m * max(D, G * n)))
    for b in range(0, c["B"], step):
        sl = slice(b, b + step)
        k, v = (_dense_plain(s[name], s[name + "_exp"], s["table"][sl], m) for name in ("ck", "cv"))
        at = torch.arange(m, device="cuda")
        base = s["lens"][sl].long() - n  # tokens in front of the drafts
        node = at - base[:, None]
        draft = (node >= 0) & (node < n)
        see = above[sl].gather(2, node.clamp(0, n - 1)[:, None].expand(-1, n, -1)) & draft[:, None] | (node < 0)[:, None]
        if c["window"]:
            place = torch.where(draft, base[:, None] + depth[sl].gather(1, node.clamp(0, n - 1)), at)  # positions of the keys
            see = see & (place[:, None] > (base[:, None] + depth[sl])[..., None] - c["window"])
        see = see[:, None, None]
        q = s["q"][sl].float().view(-1, H, G * n, D)
        x = (q @ k.transpose(2, 3).contiguous()).view(-1, H, G, n, m) * D ** -0.5
        x = torch.where(see, x, -math.inf)
        top = x.amax(-1, keepdim=True)
        p = torch.where(see, torch.exp(x - top), 0.0)
        l = p.sum(-1, keepdim=True)
        o = (p.view(-1, H, G * n, m) @ v).view(-1, H, G, n, D) / l
        outs.append(o.view(-1, H * G, n, D).to(DTYPES[c["dtype"]]))
        sums.append((top + torch.log(l)).view(-1, H * G, n))
    o = torch.cat(outs)
    return (o, torch.cat(sums)) if c.get("lse") else o


def _verify_plain(s):
    c = s["case"]
    B, n, V = c["B"], c["n"], c["V"]
    tokens, p, u = s["tokens"], s["target"], s["uniforms"].double()
    parents = s["parents"]
    if parents is None:
        parents = (torch.arange(n, device="cuda") - 1).expand(B, n)
    seq = torch.arange(B, device="cuda")
    cur = torch.zeros(B, dtype=torch.long, device="cuda")
    rest = torch.ones(B, dtype=torch.float64, device="cuda")
    rejected = torch.zeros(B, n, dtype=torch.bool, device="cuda")  # children of the node at hand
    path = torch.full((B, n), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    count = torch.ones(B, dtype=torch.long, device="cuda")
    for i in range(1, n):
        child = parents[:, i] == cur
        x = tokens[:, i]
        at = p[seq, cur, x].double()
        if s["draft"] is not None:
            ok = u[:, i] * s["draft"][seq, cur, x].double() < at
        else:
            at = torch.where((rejected & (tokens == x[:, None])).any(1), 0.0, at)
            ok = u[:, i] * rest < at
        ok = ok & child
        no = child & ~ok
        rest = torch.where(ok, 1.0, torch.where(no, rest - at, rest))
        rejected[:, i] = no
        rejected = rejected & ~ok[:, None]
        cur = torch.where(ok, i, cur)
        path.scatter_(1, count.clamp(max=n - 1)[:, None], torch.where(ok, i, path.gather(1, count.clamp(max=n - 1)[:, None])[:, 0]).to(torch.int32)[:, None])
        count = count + ok.long()
    r = p[seq, cur].double()
    if s["draft"] is not None:
        left = (r - s["draft"][seq, cur].double()).clamp(min=0.0)
        r = torch.where(rejected.any(1, keepdim=True), left, r)
    else:
        out = torch.zeros(B, V, dtype=torch.int32, device="cuda")
        out.scatter_add_(1, tokens, rejected.to(torch.int32))
        r = torch.where(out > 0, 0.0, r)
    up_to = torch.cumsum(r, 1)
    return path, count.to(torch.int32), (up_to <= u[:, :1] * up_to[:, -1:]).sum(1)


def _run_plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "rotate":
        angles = _angles_plain(s, s["positions"])
        out = [_rotate_plain(s[x], s[x + "_weight"], angles, c["R"], c["interleaved"]).to(s[x].dtype) for x in "qk"]
        if c["grad"]:
            grads = [_rotate_backward_plain(s["d" + x], s[x], s[x + "_weight"], angles, c["R"], c["interleaved"]) for x in "qk"]
            out += [g[0] for g in grads] + [g[1] for g in grads if g[1] is not None]
        return out
    if kind == "append":
        angles = _angles_plain(s, s["lens"][:, None] + torch.arange(c["S"], device="cuda"))
        q, k = (_rotate_plain(s[x], s[x + "_weight"], angles, c["R"], c["interleaved"]) for x in "qk")
        for name, x in (("ck", k), ("cv", s["v"])):
            _append_plain(s[name], s[name + "_exp"], x, s["table"], s["lens"], s["counts"])
        live = torch.arange(c["S"], device="cuda") < s["counts"][:, None]
        q = torch.where(live[:, None, :, None], q, 0.0).to(s["q"].dtype)
        return [q, *_gather_plain(s, s["touched"], s["touched_lens"], s["touched_most"])]
    if kind == "tree":
        return _tree_plain(s)
    if kind == "verify":
        return _verify_plain(s)
    src, dst = s["touched"].flatten().long(), s["copies"].flatten().long()
    for name in ("ck", "cv"):
        raw = s[name].view(torch.uint8)
        raw[dst] = raw[src]
        s[name + "_exp"][dst] = s[name + "_exp"][src]
        _keep_plain(s[name], s[name + "_exp"], s["table"], s["lens"], s["path"], s["accepted"])
    return _gather_plain(s, s["copies"], s["touched_lens"], s["touched_most"])


# ---- the framework's calls --------------------------------------------------------------------------------------------
def _run_own(s):
    import sparseattention_amd as sa

    c = s["case"]
    kind = c["kind"]
    if kind == "rotate":
        norm = dict(q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
        if not c["grad"]:
            return list(sa.rotate_heads(s["q"], s["k"], s["positions"], s["rotary"], **norm))
        q, k = sa.rotate_heads_trainable(s["q"], s["k"], s["positions"], s["rotary"], **norm)
        leaves = [s[x] for x in ("q", "k", "q_weight", "k_weight") if s[x] is not None]
        return [q, k, *torch.autograd.grad([q, k], leaves, [s["dq"], s["dk"]])]
    if kind == "append":
        q = sa.paged_cache_append_rotated(s["cache"], s["q"], s["k"], s["v"], s["table"], s["lens"], s["rotary"], counts=s["counts"],
                                          q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
        return [q, *sa.paged_cache_gather(s["cache"], s["touched"], s["touched_lens"], length=s["touched_most"], dtype=DTYPES[c["dtype"]])]
    if kind == "tree":
        return sa.sparse_attention_decode_tree(s["q"], s["cache"], s["table"], s["lens"], s["parents"], window=c["window"] or None,
                                               return_lse=bool(c.get("lse")))
    if kind == "verify":
        return sa.verify_drafts(s["target"], s["tokens"], s["uniforms"], parents=s["parents"], draft_probs=s["draft"])
    sa.paged_cache_copy(s["cache"], s["touched"].view(-1), s["copies"].view(-1))
    sa.paged_cache_keep(s["cache"], s["table"], s["lens"], s["path"], s["accepted"])
    return list(sa.paged_cache_gather(s["cache"], s["copies"], s["touched_lens"], length=s["touched_most"], dtype=DTYPES[c["dtype"]]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- work -------------------------------------------------------------------------------------------------------------
def work(case) -> dict:
    c = case
    kind, B = c["kind"], c["B"]
    size = 4 if c["dtype"] == "fp32" else 2
    if kind == "rotate":
        elements = B * c["S"] * (c["Hq"] + c["H"]) * c["D"]
        return {"bytes": elements * size * (5 if c["grad"] else 2), "flops": elements * (30 if c["grad"] else 10)}
    if kind == "verify":
        return {"bytes": B * c["V"] * size * (2 if c["drawn"] else 1), "flops": B * c["V"]}
    row = 2 * c["H"] * c["D"]  # elements of a token's K and V
    lens, P = _lens(c), c["P"]
    if kind == "append":
        counts = _counts(c)
        tail = [a + b - a // P * P for a, b in zip(lens, counts)]
        # queries read and written, new tokens read and stored; the touched pages read back whole
        data = sum(counts) * (c["H"] * c["G"] * c["D"] * 2 + row + row // 2) + B * c["S"] * c["H"] * c["G"] * c["D"] * 2 + sum(tail) * row
        return {"bytes": data + B * max(tail) * row * 2, "flops": sum(counts) * c["H"] * (c["G"] + 1) * c["D"] * 10}
    if kind == "tree":
        return {"bytes": sum(lens) * row + 4 * B * c["H"] * c["G"] * c["n"] * c["D"], "flops": 2 * sum(lens) * row * c["G"] * c["n"]}
    cols = max(_pages_of(a + c["n"], P) - a // P for a in lens)
    # pages copied, a part of the drafts moved, pages read back
    return {"bytes": B * cols * P * row * (2 + 1 + 2) + B * c["n"] * row, "flops": 0}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _round64(y: torch.Tensor) -> torch.Tensor:
    """Numbers of 64 bits with magnitudes up to 448 to the nearest of four significant bits, from 2^-9 upwards."""
    least = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(least - 3.0)
    return torch.round(y / step) * step


def _scale64(top: torch.Tensor) -> torch.Tensor:
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -200) / 448.0))
    e = torch.where(torch.exp2(e - 1.0) * 448.0 >= top, e - 1.0, e)
    e = torch.where(torch.exp2(e) * 448.0 < top, e + 1.0, e)
    return torch.exp2(e.clamp(E_MIN, E_MAX))


def _top64(x):
    return x.abs().amax((-1, -2), keepdim=True)


def _held64(x: torch.Tensor):
    """[H, n, D] as the cache holds it when stored at once from an empty one, and its blocks' scales [H, blocks, 1, 1]."""
    H, n, D = x.shape
    y = torch.nn.functional.pad(x.double(), (0, 0, 0, -n % BLOCK)).view(H, -1, BLOCK, D)
    out, scale = torch.empty_like(y), _scale64(_top64(y))
    for t in range(0, y.shape[1], 256):
        sl = slice(t, t + 256)
        out[:, sl] = _round64(y[:, sl] / scale[:, sl]) * scale[:, sl]
    return out.view(H, -1, D)[:, :n], scale


def _appended64(held: torch.Tensor, new: torch.Tensor) -> torch.Tensor:
    """[H, n + m, D] after new [H, m, D] has been stored behind held [H, n, D]."""
    n = held.shape[1]
    kept, scales = _held64(held)
    cut = n // BLOCK * BLOCK
    old, rest = kept[:, cut:], new.double()
    room = min(BLOCK - (n - cut), rest.shape[1]) if n > cut else 0
    parts = [kept[:, :cut]]
    if room:
        was = scales[:, -1]
        scale = torch.maximum(was, _scale64(_top64(rest[:, :room])))
        parts += [torch.where(scale > was, _round64(old / scale) * scale, old), _round64(rest[:, :room] / scale) * scale]
    else:
        parts.append(old)
    if rest.shape[1] > room:
        parts.append(_held64(rest[:, room:])[0])
    return torch.cat(parts, 1)


def _kept64(held: torch.Tensor, n: int, path: list[int]) -> torch.Tensor:
    """[H, n + len(path), D]: of held [H, n + drafts, D], stored at once, the first n tokens and the drafts of the path."""
    x, scales = _held64(held)
    rows, out = [n + i for i in path], x.clone()
    for block in range(n // BLOCK, (n + len(path) - 1) // BLOCK + 1):
        lo, hi = block * BLOCK, min(block * BLOCK + BLOCK, n + len(path))
        come = rows[max(lo, n) - n:hi - n]
        same = [r for r in come if r // BLOCK == block]
        others = [r for r in come if r // BLOCK != block]
        scale = torch.full_like(scales[:, 0], 2.0 ** E_MIN)
        if same or lo < n:
            scale = torch.maximum(scale, scales[:, block])
        if others:
            scale = torch.maximum(scale, _scale64(_top64(x[:, others])))
        all_rows = list(range(lo, max(lo, min(n, hi)))) + come
        out[:, lo:hi] = _round64((x[:, all_rows] / scale).clamp(-448.0, 448.0)) * scale
    return out[:, :n + len(path)]


def _padded64(rows: list, most: int) -> torch.Tensor:
    return torch.stack([torch.nn.functional.pad(r[:, :most], (0, 0, 0, most - min(most, r.shape[1]))) for r in rows])


def _turn64(x: torch.Tensor, at: torch.Tensor, R: int, interleaved: bool, back: bool = False) -> torch.Tensor:
    """Pairs of [..., S, D] as complex numbers times exp(i t), t [..., S, R/2]."""
    z = torch.polar(torch.ones_like(at), -at if back else at)
    y = x.double().clone()
    lo, hi = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    turned = torch.complex(y[..., lo].clone(), y[..., hi].clone()) * z
    y[..., lo], y[..., hi] = turned.real, turned.imag
    return y


def _normed64(x, weight):
    if weight is None:
        return x.double()
    y = x.double()
    return y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS) * weight.double()


def _frequencies64(c):
    return torch.tensor([10000.0 ** (-2.0 * j / c["R"]) for j in range(c["R"] // 2)], dtype=torch.float64, device="cuda")


def _exact_rotate(c, s):
    f = _frequencies64(c)
    half, n = c["R"] // 2, c["axes"]
    at = s["positions"].double().view(n, c["B"], 1, c["S"], 1)
    t = torch.cat([at[j * n // half] * f[j] for j in range(half)], -1)
    out, grads, weights = [], [], []
    for name in ("q", "k"):
        x, w = s[name], s[name + "_weight"]
        out.append(_turn64(_normed64(x, w), t, c["R"], c["interleaved"]))
        if not c["grad"]:
            continue
        g = _turn64(s["d" + name], t, c["R"], c["interleaved"], back=True)
        if w is None:
            grads.append(g)
            continue
        y = x.double()
        size = torch.sqrt(y.pow(2).mean(-1, keepdim=True) + EPS)
        weights.append((g * y / size).sum(2).sum((0, 1)))
        g *= w.double()
        along = (g * y).sum(-1, keepdim=True)
        grads.append(g / size - y * along / (c["D"] * size.pow(3)))
    return out + grads + weights


def _exact_append(c, s):
    lens, counts, f = _lens(c), _counts(c), _frequencies64(c)
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    ks, vs = [], []
    for b, (n, m) in enumerate(zip(lens, counts)):
        t = torch.arange(n, n + m, dtype=torch.float64, device="cuda")[:, None] * f
        q[b, :, :m] = _turn64(_normed64(s["q"][b, :, :m], s["q_weight"]), t, c["R"], c["interleaved"])
        k = _turn64(_normed64(s["k"][b, :, :m], s["k_weight"]), t, c["R"], c["interleaved"])
        for to, held, new in ((ks, s["held_k"], k), (vs, s["held_v"], s["v"][b, :, :m])):
            to.append(_appended64(held[b, :, :n], new)[:, n // c["P"] * c["P"]:])
    return [q, _padded64(ks, s["touched_most"]), _padded64(vs, s["touched_most"])]


def _exact_tree(c, s):
    H, G, n, D = c["H"], c["G"], c["n"], c["D"]
    outs, sums = [], []
    for b, length in enumerate(_lens(c)):
        k, v = (_held64(s[x][b, :, :length])[0] for x in ("held_k", "held_v"))
        off = torch.ones(n, length, dtype=torch.bool)
        above = []
        for i, parent in enumerate(s["parents"][b].tolist()):
            above.append((above[parent] if parent >= 0 else []) + [i])
            depth = len(above[i]) - 1
            first = max(0, length - n + depth - c["window"] + 1) if c["window"] else 0
            off[i, first:length - n] = False
            off[i, [length - n + a for d, a in enumerate(above[i]) if not c["window"] or depth - d < c["window"]]] = False
        x = torch.matmul(s["q"][b].double().view(H, G * n, D), k.mT.contiguous()).view(H, G, n, length) / math.sqrt(D)
        x = x.masked_fill(off.cuda(), -math.inf)
        total = torch.logsumexp(x, -1)
        p = torch.exp(x - total[..., None])
        outs.append(torch.matmul(p.view(H, G * n, length), v).view(H * G, n, D))
        sums.append(total.view(H * G, n))
    return (torch.stack(outs), torch.stack(sums)) if c.get("lse") else torch.stack(outs)


def _exact_verify(c, s):
    B, n = c["B"], c["n"]
    tokens, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    parents = [list(range(-1, n - 1))] * B if s["parents"] is None else s["parents"].tolist()
    paths, counts, after = [], [], []
    for b in range(B):
        path, taken = [0], True
        while taken:
            taken, tried, left = False, [], 1.0
            row = s["target"][b, path[-1]].double()
            q = None if s["draft"] is None else s["draft"][b, path[-1]].double()
            children = [i for i in range(n) if parents[b][i] == path[-1]]
            chances = row[[tokens[b][i] for i in children]].tolist()
            offers = [None] * len(children) if q is None else q[[tokens[b][i] for i in children]].tolist()
            for i, chance, offer in zip(children, chances, offers):
                x = tokens[b][i]
                if q is None:
                    chance = 0.0 if x in tried else chance
                    taken = u[b][i] * left < chance
                else:
                    taken = u[b][i] * offer < chance
                if taken:
                    path.append(i)
                    break
                tried.append(x)
                left -= chance
        if tried:
            if q is None:
                row[tried] = 0.0
            else:
                row = torch.relu(row - q)
        sums = row.cumsum(0)
        after.append(int(torch.searchsorted(sums, u[b][0] * sums[-1], right=True)))
        counts.append(len(path))
        paths.append(path + [-1] * (n - len(path)))
    return _ints(paths), _ints(counts), torch.tensor(after, device="cuda")


def exact(case, seed: int):
    c = case
    s = _inputs(c, seed)
    if c["kind"] != "keep":
        return {"rotate": _exact_rotate, "append": _exact_append, "tree": _exact_tree, "verify": _exact_verify}[c["kind"]](c, s)
    out = []
    path, accepted = s["path"].tolist(), s["accepted"].tolist()
    for held in (s["held_k"], s["held_v"]):
        rows = [_kept64(held[b, :, :n + c["n"]], n, path[b][:accepted[b]])[:, n // c["P"] * c["P"]:] for b, n in enumerate(_lens(c))]
        out.append(_padded64(rows, s["touched_most"]))
    return out
