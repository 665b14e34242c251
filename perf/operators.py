"""Measured calls of the 8-bit paged K/V cache: storing tokens, few-rows attention over it, reading it back, and the
operations on its pages.

A case is a dict of plain values.  ``prepare`` makes what a program holds before the call, ``run`` is one pass and gives
its outputs, ``work`` the bytes and operations that the pass cannot do without, ``exact`` the outputs in 64 bits.  Where
``own`` is false ``run`` computes the same from elementary torch operations on a cache of natural layout.

The cache holds a block of 32 consecutive tokens of one head as e4m3 codes times 2^e, e the least integer for which the
block's largest magnitude is at most 448 * 2^e.  Appending to a block that holds tokens never lowers its e; where it grows,
what the block held is rounded again.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 32  # tokens that share a scale
E_MIN, E_MAX = -96, 119


def listed() -> list[dict]:
    return [
        # one token for every sequence of a batch under way: latency, most blocks half full
        dict(name="append_tokens", kind="append", B=64, H=8, D=128, P=64, S=1, held=2048, spread=0.9, ragged=0.0, dtype="bf16"),
        # a chunk of a prompt behind an odd number of tokens already held
        dict(name="append_chunk", kind="append", B=1, H=8, D=128, P=64, S=4096, held=1001, spread=0.0, ragged=0.0, dtype="bf16"),
        # new prompts of a padded batch, half precision, the head dim of the small configurations
        dict(name="append_prompts", kind="append", B=16, H=12, D=64, P=32, S=2047, held=0, spread=0.0, ragged=0.8, dtype="fp16"),
        # a single conversation's next token: the smallest attention, all latency
        dict(name="attend_one", kind="attend", B=1, H=8, G=4, D=128, P=64, Sq=1, length=2011, spread=0.0, mask="causal", dtype="bf16"),
        # a serving batch of very different lengths
        dict(name="attend_batch", kind="attend", B=64, H=8, G=4, D=128, P=64, Sq=1, length=8192, spread=0.95, mask="causal", dtype="bf16"),
        # four tokens checked at once with a sliding window, half precision, the row statistics kept
        dict(name="attend_window", kind="attend", B=16, H=4, G=8, D=64, P=32, Sq=4, length=16384, spread=0.5, mask="window",
             window=4096, dtype="fp16"),
        # a long context of which each head reads a quarter of the pages, lists kept by the program
        dict(name="attend_pages", kind="attend", B=2, H=8, G=4, D=128, P=64, Sq=1, length=131072, spread=0.1, mask="pages", p=0.75,
             dtype="bf16"),
        # long contexts of a full batch: the largest
        dict(name="attend_long", kind="attend", B=32, H=8, G=8, D=128, P=128, Sq=1, length=32768, spread=0.3, mask="causal", dtype="bf16"),
        # a long prompt's cache read back for its next chunk
        dict(name="gather_prompt", kind="gather", B=1, H=8, D=128, P=64, length=16391, spread=0.0, dtype="bf16"),
        # the same for a ragged batch in half precision
        dict(name="gather_batch", kind="gather", B=16, H=12, D=64, P=32, length=4096, spread=0.9, dtype="fp16"),
        # every sequence of a batch continued four ways
        dict(name="fork_batch", kind="fork", B=64, H=8, D=128, P=64, n=256, length=2048, spread=0.8, dtype="bf16"),
        # half a pool freed: what lives moves to its front
        dict(name="compact_pool", kind="compact", B=24, H=8, D=128, P=64, length=8192, spread=0.7, dtype="bf16"),
    ]


def _log_uniform(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "gather", "fork", "compact"])
    c = dict(kind=kind, D=rng.choice([64, 80, 128, 128, 256]), P=rng.choice([32, 64, 64, 128, 256]), H=rng.choice([1, 2, 4, 8, 8, 12, 16]),
             dtype=rng.choice(["bf16", "bf16", "fp16"]), spread=round(rng.uniform(0.0, 1.0), 2))
    heads = c["H"] * c["D"]
    if kind == "append":
        c["S"] = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 8192)
        c["B"] = _log_uniform(rng, 1, max(1, min(128, (1 << 26) // (heads * (c["S"] + 256)))))
        c["held"] = rng.choice([0, 1, 31, 32, _log_uniform(rng, 2, 8192)])
        c["ragged"] = rng.choice([0.0, round(rng.uniform(0.0, 1.0), 2)])
    elif kind == "attend":
        c["length"] = _log_uniform(rng, 1, 65536)
        c["B"] = _log_uniform(rng, 1, max(1, min(128, (1 << 29) // (heads * c["length"]))))
        c["G"] = rng.choice([1, 1, 2, 4, 7, 8])
        c["Sq"] = rng.choice([1, 1, 1, 2, 5, 16, 32])
        c["mask"] = rng.choice(["causal", "causal", "window", "pages"])
        if c["mask"] == "window":
            c["window"] = _log_uniform(rng, 1, 8192)
        if c["mask"] == "pages":
            c["p"] = round(rng.uniform(0.1, 0.9), 2)
    else:
        c["length"] = _log_uniform(rng, 1, 16384)
        c["B"] = _log_uniform(rng, 1, max(1, min(64, (1 << 27) // (heads * c["length"]))))
        if kind == "fork":
            c["n"] = _log_uniform(rng, 1, 256)
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _spread(n: int, top: int, spread: float) -> list[int]:
    """n numbers from top * (1 - spread) to top, the first one top, spread evenly in an irregular order."""
    return [max(0, round(top * (1.0 - spread * ((i * 0.6180339887) % 1.0)))) for i in range(n)]


def _lens(c) -> list[int]:
    return _spread(c["B"], c["held"] if c["kind"] == "append" else c["length"], c["spread"])


def _counts(c) -> list[int]:
    return _spread(c["B"], c["S"], c["ragged"])


def _pages_of(tokens: int, P: int) -> int:
    return -(-tokens // P)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tokens(c, n: int, g: torch.Generator, keys: bool) -> torch.Tensor:
    """[B, H, n, D] keys (a few channels much larger than the rest, as rotated keys have them) or values."""
    x = torch.randn(c["B"], c["H"], n, c["D"], generator=g, device="cuda")
    if keys:
        x *= torch.exp(0.7 * torch.randn(1, c["H"], 1, c["D"], generator=g, device="cuda"))
    return x.to(DTYPES[c["dtype"]])


def _inputs(c, seed: int) -> dict:
    """Everything random or fixed that a case starts from, before any of it is held in 8 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, B, P = c["kind"], c["B"], c["P"]
    lens = _lens(c)
    counts = _counts(c) if kind == "append" else [0] * B
    most = max(a + b for a, b in zip(lens, counts))
    width = max(1, _pages_of(most, P))
    used = B * width
    pool = 2 * used + 3 if kind == "compact" else used + (c["n"] if kind == "fork" else 0) + 3
    pages = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    s = dict(lens=_ints(lens), table=pages[:used].view(B, width).contiguous(), pool=pool, most=most, width=width)
    s["held_k"], s["held_v"] = (_tokens(c, max(1, max(lens)), g, keys) for keys in (True, False))
    if kind == "append":
        s["new_k"], s["new_v"] = (_tokens(c, c["S"], g, keys) for keys in (True, False))
        s["counts"] = _ints(counts)
        # the columns of the table that the new tokens touch, and how many tokens those pages hold afterwards
        first = [a // P for a in lens]
        cols = max(1, max(_pages_of(a + b, P) - f for a, b, f in zip(lens, counts, first)))
        at = (_ints(first).long()[:, None] + torch.arange(cols, device="cuda")).clamp(max=width - 1)
        s["touched"] = s["table"].gather(1, at).contiguous()
        s["touched_lens"] = _ints([a + b - f * P for a, b, f in zip(lens, counts, first)])
        s["touched_most"] = max(a + b - f * P for a, b, f in zip(lens, counts, first))
    elif kind == "attend":
        s["q"] = torch.randn(B, c["H"] * c["G"], c["Sq"], c["D"], generator=g, device="cuda").to(DTYPES[c["dtype"]])
        if c["mask"] == "pages":
            keep = torch.rand(B, c["H"], 1, width, generator=g, device="cuda") >= c["p"]
            keep[..., 0] = keep[..., -1] = True
            mask = keep.repeat_interleave(P, -1).expand(B, c["H"], c["Sq"], width * P).contiguous()
            # the last page's keys behind the rows, as a causal mask has them
            at = torch.arange(width * P, device="cuda")
            ends = (s["lens"].long() - c["Sq"])[:, None] + torch.arange(c["Sq"], device="cuda")
            s["mask"] = mask & (at <= ends[:, None, :, None])
    elif kind == "fork":
        s["parents"] = torch.randint(B, (c["n"],), generator=g, device="cuda").to(torch.int32)
        s["new_pages"] = pages[used:used + c["n"]].contiguous()
        s["tail_lens"] = (s["lens"][s["parents"].long()] % P).to(torch.int32)
    return s


def prepare(case, seed: int) -> dict:
    s = dict(_inputs(case, seed), case=case)
    held_k, held_v = s.pop("held_k"), s.pop("held_v")
    if own:
        import sparseattention_amd as sa

        s["cache"] = sa.empty_paged_cache(s["pool"], case["H"], case["D"], page_size=case["P"], device="cuda")
        sa.paged_cache_append(s["cache"], held_k, held_v, s["table"], torch.zeros_like(s["lens"]), counts=s["lens"])
        if "mask" in s:
            s["metadata"] = sa.compute_mask_kernel(s.pop("mask"), case["Sq"], case["P"])
    else:
        shape = (s["pool"], case["H"], case["P"], case["D"])
        for name, x in (("k", held_k), ("v", held_v)):
            s[name] = torch.zeros(shape, dtype=torch.float8_e4m3fn, device="cuda")
            s[name + "_exp"] = torch.full((s["pool"], case["H"], case["P"] // BLOCK), E_MIN, dtype=torch.int32, device="cuda")
            _append_plain(s[name], s[name + "_exp"], x, s["table"], torch.zeros_like(s["lens"]), s["lens"])
    return s


# ---- the plain form ---------------------------------------------------------------------------------------------------
def _exponent(amax: torch.Tensor) -> torch.Tensor:
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)  # 448 = 0.875 * 2^9
    return torch.where(amax > 0, e.to(torch.int32), E_MIN).clamp(E_MIN, E_MAX)


def _codes(x: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    y = torch.ldexp(x, -e).clamp(-448.0, 448.0)
    return torch.where(torch.isfinite(x), y, math.nan).to(torch.float8_e4m3fn)


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
        first = lens[sl].long() // BLOCK
        nb = (S + 2 * BLOCK - 2) // BLOCK
        blk = first[:, None] + torch.arange(nb, device=x.device)  # [n, nb] blocks of the sequence
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
        size = torch.where(sel & torch.isfinite(val), val.abs(), 0.0)
        e = torch.maximum(old_exp, _exponent(size.amax((-1, -2))))
        again = _codes(torch.ldexp(old_codes.float(), old_exp[..., None, None]), e[..., None, None])
        kept = torch.where((e > old_exp)[..., None, None], again.float(), old_codes.float())
        out = torch.where(sel, _codes(val, e[..., None, None]).float(), kept).to(torch.float8_e4m3fn)
        at = live.nonzero(as_tuple=True)
        blocks.view(torch.uint8)[page[at], :, (blk % per)[at]] = out[at].view(torch.uint8)
        exps[page[at], :, (blk % per)[at]] = e[at]


def _dense_plain(codes, exps, table, n: int) -> torch.Tensor:
    """The first n tokens of the sequences of a table [B, pages] in 32 bits, [B, H, n, D]; tokens of pages that do not exist are
    zero."""
    _, H, P, D = codes.shape
    pages = table[:, :_pages_of(n, P)].long()
    ok = (pages >= 0) & (pages < codes.shape[0])
    pages = torch.where(ok, pages, 0)
    x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()  # [B, pages, H, P, D]
    x = torch.ldexp(x, exps[pages].repeat_interleave(BLOCK, -1)[..., None])
    x = torch.where(ok[:, :, None, None, None], x, 0.0)
    return x.transpose(1, 2).reshape(len(table), H, -1, D)[:, :, :n]


def _gather_plain(s, table, lens, most: int):
    out = []
    _, H, P, D = s["k"].shape
    step = max(1, (1 << 28) // (H * D * max(most, P)))  # (sequences at a time: the intermediate tensors are 32 bits wide)
    for name in ("k", "v"):
        parts = []
        for b in range(0, len(table), step):
            x = _dense_plain(s[name], s[name + "_exp"], table[b:b + step], most)
            live = torch.arange(most, device="cuda") < lens[b:b + step, None]
            parts.append(torch.where(live[:, None, :, None], x, 0.0).to(DTYPES[s["case"]["dtype"]]))
        out.append(torch.cat(parts))
    return out


def _attend_plain(s):
    c = s["case"]
    H, G, Sq, D, n = c["H"], c["G"], c["Sq"], c["D"], s["most"]
    outs, sums = [], []
    step = max(1, (1 << 29) // (H * n * max(D, G * Sq)))
    for b in range(0, c["B"], step):
        sl = slice(b, b + step)
        k, v = (_dense_plain(s[name], s[name + "_exp"], s["table"][sl], n) for name in ("k", "v"))
        at = torch.arange(n, device="cuda")
        lens = s["lens"][sl, None, None, None, None]
        row = lens - Sq + torch.arange(Sq, device="cuda")[:, None]
        if c["mask"] == "pages":
            see = s["mask"][sl, :, None, :, :n] & (at < lens)
        else:
            see = at <= row
            if c["mask"] == "window":
                see = see & (at > row - c["window"])
        q = s["q"][sl].float().view(-1, H, G * Sq, D)
        x = (q @ k.transpose(2, 3).contiguous()).view(-1, H, G, Sq, n) * D ** -0.5
        x = torch.where(see, x, -math.inf)
        top = x.amax(-1, keepdim=True)
        p = torch.where(see, torch.exp(x - torch.where(top == -math.inf, 0.0, top)), 0.0)
        l = p.sum(-1, keepdim=True)
        o = (p.view(-1, H, G * Sq, n) @ v).view(-1, H, G, Sq, D) / torch.where(l > 0, l, 1.0)
        outs.append(o.view(-1, H * G, Sq, D).to(DTYPES[c["dtype"]]))
        sums.append((top + torch.log(l)).view(-1, H * G, Sq))
    o = torch.cat(outs)
    return (o, torch.cat(sums)) if c["mask"] == "window" else o


def _copy_plain(s, src, dst) -> None:
    src, dst = src.long(), dst.long()
    for name in ("k", "v"):
        raw = s[name].view(torch.uint8)
        raw[dst] = raw[src]
        s[name + "_exp"][dst] = s[name + "_exp"][src]


def _fork_plain(s):
    P, width = s["case"]["P"], s["width"]
    parents = s["parents"].long()
    lens = s["lens"][parents]
    table = s["table"][parents]
    full = (lens // P).long()
    tail = lens % P != 0
    at = torch.arange(width, device="cuda") == full[:, None]
    last = table.gather(1, full.clamp(max=width - 1)[:, None])[:, 0]
    _copy_plain(s, last[tail], s["new_pages"][tail])
    used = torch.arange(width, device="cuda") < ((lens + P - 1) // P)[:, None]
    table = torch.where(at & tail[:, None], s["new_pages"][:, None], table)
    return torch.where(used, table, -1), lens


def _compact_plain(s):
    P, pool = s["case"]["P"], s["pool"]
    used = torch.arange(s["width"], device="cuda") < ((s["lens"] + P - 1) // P)[:, None]
    live = torch.zeros(pool, dtype=torch.bool, device="cuda")
    live[s["table"][used].long()] = True
    count = live.sum()
    at = torch.arange(pool, device="cuda")
    holes, movers = at[~live & (at < count)], at[live & (at >= count)]
    _copy_plain(s, movers, holes)
    to = at.clone()
    to[movers] = holes
    return torch.where(used, to[s["table"].long()].to(torch.int32), -1), count.to(torch.int32).view(1)


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "append":
        for name in ("k", "v"):
            _append_plain(s[name], s[name + "_exp"], s["new_" + name], s["table"], s["lens"], s["counts"])
        return _gather_plain(s, s["touched"], s["touched_lens"], s["touched_most"])
    if kind == "attend":
        return _attend_plain(s)
    if kind == "gather":
        return _gather_plain(s, s["table"], s["lens"], s["most"])
    if kind == "fork":
        table, lens = _fork_plain(s)
        return [table, lens, *_gather_plain(s, s["new_pages"][:, None], s["tail_lens"], s["case"]["P"])]
    table, count = _compact_plain(s)
    return [table, count, *_gather_plain(s, table, s["lens"], s["most"])]


# ---- the framework's calls --------------------------------------------------------------------------------------------
def _run_own(s):
    import sparseattention_amd as sa

    c, cache = s["case"], s["cache"]
    kind, dtype = c["kind"], DTYPES[c["dtype"]]
    if kind == "append":
        sa.paged_cache_append(cache, s["new_k"], s["new_v"], s["table"], s["lens"], counts=s["counts"])
        return list(sa.paged_cache_gather(cache, s["touched"], s["touched_lens"], length=s["touched_most"], dtype=dtype))
    if kind == "attend":
        if c["mask"] == "pages":
            return sa.sparse_attention_decode_paged(s["q"], cache, s["table"], s["lens"], mask_metadata=s["metadata"])
        if c["mask"] == "window":
            return sa.sparse_attention_decode_paged(s["q"], cache, s["table"], s["lens"], window=c["window"], return_lse=True)
        return sa.sparse_attention_decode_paged(s["q"], cache, s["table"], s["lens"])
    if kind == "gather":
        return list(sa.paged_cache_gather(cache, s["table"], s["lens"], length=s["most"], dtype=dtype))
    if kind == "fork":
        table, lens = sa.paged_cache_fork(cache, s["table"], s["lens"], s["parents"], s["new_pages"])
        return [table, lens, *sa.paged_cache_gather(cache, s["new_pages"][:, None], s["tail_lens"], length=c["P"], dtype=dtype)]
    table, count = sa.paged_cache_compact(cache, s["table"], s["lens"])
    return [table, count, *sa.paged_cache_gather(cache, table, s["lens"], length=s["most"], dtype=dtype)]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- work -------------------------------------------------------------------------------------------------------------
def work(case) -> dict:
    c = case
    kind, B, P = c["kind"], c["B"], c["P"]
    lens = _lens(c)
    row = 2 * c["H"] * c["D"]  # elements of a token's K and V
    flops = 0
    if kind == "append":
        counts = _counts(c)
        most = max(a + b - a // P * P for a, b in zip(lens, counts))
        # new tokens read and stored; the touched pages read back whole
        data = sum(counts) * row * 3 + sum(a + b - a // P * P for a, b in zip(lens, counts)) * row + B * most * row * 2
    elif kind == "attend":
        q = B * c["H"] * c["G"] * c["Sq"] * c["D"]
        keys = lens
        if c["mask"] == "window":
            keys = [min(n, c["window"] + c["Sq"] - 1) for n in lens]
        if c["mask"] == "pages":
            keys = [min(n, round(n * (1.0 - c["p"])) + P) for n in lens]
        data = sum(keys) * row + 4 * q
        flops = 2 * sum(keys) * row * c["G"] * c["Sq"]
    elif kind == "gather":
        data = sum(lens) * row + B * max(1, max(lens)) * row * 2
    elif kind == "fork":
        tails = [n % P for n in lens]
        share = sum(tails) / len(tails)
        data = round(c["n"] * (2 * share * row + share * row + P * row * 2)) + c["n"] * _pages_of(max(lens), P) * 8
    else:
        pages = sum(_pages_of(n, P) for n in lens)
        pool = 2 * B * max(1, _pages_of(max(lens), P)) + 3
        data = round(pages * (1.0 - pages / pool) * P * row * 2) + sum(lens) * row + B * max(1, max(lens)) * row * 2
    return {"bytes": int(data), "flops": int(flops)}


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


def _held64(x: torch.Tensor) -> torch.Tensor:
    """[H, n, D] as the cache holds it when stored at once from an empty one."""
    out = torch.empty_like(x, dtype=torch.float64)
    for t in range(0, x.shape[1], 8192):
        y = x[:, t:t + 8192].double()
        n = y.shape[1]
        y = torch.nn.functional.pad(y, (0, 0, 0, -n % BLOCK)).view(x.shape[0], -1, BLOCK, x.shape[2])
        scale = _scale64(y.abs().amax((-1, -2), keepdim=True))
        out[:, t:t + 8192] = (_round64(y / scale) * scale).view(x.shape[0], -1, x.shape[2])[:, :n]
    return out


def _appended64(held: torch.Tensor, new: torch.Tensor) -> torch.Tensor:
    """[H, n + m, D] after new [H, m, D] has been stored behind held [H, n, D]."""
    n = held.shape[1]
    kept = _held64(held)
    cut = n // BLOCK * BLOCK
    old, rest = kept[:, cut:], new.double()
    room = min(BLOCK - (n - cut), rest.shape[1]) if n > cut else 0
    parts = [kept[:, :cut]]
    if room:
        tops = [t.abs().amax((-1, -2), keepdim=True) for t in (held[:, cut:].double(), rest[:, :room])]
        was, scale = _scale64(tops[0]), _scale64(torch.maximum(*tops))
        parts += [torch.where(scale > was, _round64(old / scale) * scale, old), _round64(rest[:, :room] / scale) * scale]
    else:
        parts.append(old)
    if rest.shape[1] > room:
        parts.append(_held64(rest[:, room:]))
    return torch.cat(parts, 1)


def _padded64(rows: list, most: int) -> torch.Tensor:
    return torch.stack([torch.nn.functional.pad(r[:, :most], (0, 0, 0, most - min(most, r.shape[1]))) for r in rows])


def exact(case, seed: int):
    c = case
    kind, B, P = c["kind"], c["B"], c["P"]
    s = _inputs(c, seed)
    lens = _lens(c)
    held = (s["held_k"], s["held_v"])
    if kind == "append":
        counts = _counts(c)
        out = []
        for old, new in zip(held, (s["new_k"], s["new_v"])):
            rows = [_appended64(old[b, :, :n], new[b, :, :m])[:, n // P * P:] for b, (n, m) in enumerate(zip(lens, counts))]
            out.append(_padded64(rows, s["touched_most"]))
        return out
    if kind == "attend":
        H, G, Sq, D = c["H"], c["G"], c["Sq"], c["D"]
        outs, sums = [], []
        for b, n in enumerate(lens):
            k, v = (_held64(x[b, :, :n]) for x in held)
            at = torch.arange(n, device="cuda")
            rows = n - Sq + torch.arange(Sq, device="cuda")[:, None]
            if c["mask"] == "pages":
                off = ~s["mask"][b, :, None, :, :n]
            else:
                off = (at > rows) | ((rows - at >= c["window"]) if c["mask"] == "window" else False)
            x = torch.matmul(s["q"][b].double().view(H, G * Sq, D), k.mT.contiguous()).view(H, G, Sq, n) / math.sqrt(D)
            x = x.masked_fill(off, -math.inf)
            total = torch.logsumexp(x, -1) if n else torch.full((H, G, Sq), -math.inf, dtype=torch.float64, device="cuda")
            p = torch.exp(x - total[..., None]).nan_to_num(0.0)
            outs.append(torch.matmul(p.view(H, G * Sq, n), v).view(H * G, Sq, D))
            sums.append(total.view(H * G, Sq))
        return (torch.stack(outs), torch.stack(sums)) if c["mask"] == "window" else torch.stack(outs)
    rows = [[_held64(x[b, :, :n]) for b, n in enumerate(lens)] for x in held]
    if kind == "gather":
        return [_padded64(r, s["most"]) for r in rows]
    if kind == "fork":
        parents = s["parents"].tolist()
        new, table, old = s["new_pages"].tolist(), [], s["table"].tolist()
        for i, b in enumerate(parents):
            keep = old[b][:lens[b] // P] + ([new[i]] if lens[b] % P else [])
            table.append(keep + [-1] * (s["width"] - len(keep)))
        tails = [[r[b][:, lens[b] // P * P:] for b in parents] for r in rows]
        return [_ints(table), _ints([lens[b] for b in parents]), *(_padded64(t, P) for t in tails)]
    table = [row[:_pages_of(n, P)] for row, n in zip(s["table"].tolist(), lens)]
    live = sorted({page for row in table for page in row})
    count = len(live)
    free = sorted(set(range(count)) - set(live))
    to = {page: page for page in live}
    to.update(zip([page for page in live if page >= count], free))
    table = [[to[page] for page in row] + [-1] * (s["width"] - len(row)) for row in table]
    return [_ints(table), _ints([count]), *(_padded64(r, s["most"]) for r in rows)]
