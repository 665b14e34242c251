"""Refusals of the verification of drafts and of keeping them, on the host before anything is launched (so these run without a GPU)."""
import ctypes

import pytest
import torch

import sparseattention_amd as sa
from sparseattention_amd import _native

FAKE = 0x1000  # never dereferenced: every call below must fail validation first
BAD, UNSUPPORTED, WORKSPACE = _native.SA_ERR_INVALID_ARGUMENT, _native.SA_ERR_UNSUPPORTED, _native.SA_ERR_WORKSPACE
S2, S3 = _native.strides((8, 1)), _native.strides((800, 100, 1))


def verify(p=FAKE, ps=S3, q=None, qs=S3, tokens=FAKE, wide=0, u=FAKE, parents=None, rs=S2, path=FAKE, accepted=FAKE, token=FAKE, B=2, n=8, V=100, dtype=2, ws=None, size=0):
    return _native.load().sa_verify_drafts(p, ps, q, qs, tokens, S2, wide, u, S2, parents, rs, None, path, accepted, token, B, n, V, dtype, ws, size, None)


def test_verify():
    for name in ("p", "ps", "tokens", "u", "path", "accepted", "token"):
        assert verify(**{name: None}) == BAD, name
    assert verify(q=FAKE, qs=None) == BAD and verify(parents=FAKE, rs=None) == BAD and verify(q=FAKE, parents=FAKE) == BAD
    for name in ("B", "n", "V"):
        assert verify(**{name: 0}) == BAD, name
    assert verify(n=65) == UNSUPPORTED and verify(V=(1 << 21) + 1) == UNSUPPORTED and verify(dtype=3) == UNSUPPORTED
    assert verify(ps=_native.strides((1600, 200, 2))) == UNSUPPORTED and verify(q=FAKE, qs=_native.strides((1600, 200, 2))) == UNSUPPORTED
    assert verify(p=FAKE + 2) == UNSUPPORTED and verify(p=FAKE + 1, dtype=0) == UNSUPPORTED and verify(tokens=FAKE + 4, wide=1) == UNSUPPORTED
    assert verify(token=FAKE + 4, wide=1) == UNSUPPORTED
    need = _native.load().sa_verify_drafts_workspace_bytes(2, 8, 100)
    assert need > 0 and verify() == WORKSPACE and verify(ws=FAKE, size=need - 1) == WORKSPACE and verify(ws=FAKE + 4, size=need) == WORKSPACE
    for sizes in ((0, 8, 100), (2, 0, 100), (2, 65, 100), (2, 8, 0), (2, 8, (1 << 21) + 1)):
        assert _native.load().sa_verify_drafts_workspace_bytes(*sizes) == 0
    assert verify(B=1 << 30, V=1 << 21, ws=FAKE, size=1 << 60) == UNSUPPORTED  # (more workgroups than a grid has)


def test_keep():
    pool = ctypes.byref(_native.PagedCacheStruct(FAKE, FAKE, FAKE, FAKE, 8, 2, 64, 128, 128))
    keep = lambda c=pool, table=FAKE, lens=FAKE, path=FAKE, ps=S2, accepted=FAKE, B=1, n=8, pages=4: _native.load().sa_paged_cache_keep(  # noqa: E731
        c, table, S2, lens, path, ps, accepted, B, n, pages, None)
    for name in ("c", "table", "lens", "path", "ps", "accepted"):
        assert keep(**{name: None}) == BAD, name
    assert keep(B=0) == BAD and keep(pages=0) == BAD and keep(n=0) == UNSUPPORTED and keep(n=65) == UNSUPPORTED
    assert keep(B=1 << 22) == UNSUPPORTED  # (more workgroups than a launch has)
    assert keep(c=ctypes.byref(_native.PagedCacheStruct(FAKE, FAKE, FAKE, FAKE, 8, 2, 48, 128, 128))) == UNSUPPORTED


def test_python_refuses_without_a_gpu():
    p, x, u = torch.zeros(2, 3, 10), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    with pytest.raises(RuntimeError, match="GPU"):
        sa.verify_drafts(p, x, u)
    with pytest.raises(ValueError, match="target_probs"):
        sa.verify_drafts(p[0], x, u)
    with pytest.raises(TypeError):
        sa.verify_drafts(p.double(), x, u)
    cache = sa.PagedCache(torch.zeros(4, 2, 2, 2048, dtype=torch.uint8), torch.zeros(4, 2, 2, 2048, dtype=torch.uint8), torch.zeros(4, 2, 2), torch.zeros(4, 2, 2), 64)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        sa.paged_cache_keep(cache, table, lens, table, lens)


def test_not_recorded_by_a_trace():
    """torch.jit.trace would keep the outputs as they were allocated, without the call."""
    p, x, u = torch.zeros(2, 3, 10), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    cache = sa.PagedCache(torch.zeros(4, 2, 2, 2048, dtype=torch.uint8), torch.zeros(4, 2, 2, 2048, dtype=torch.uint8), torch.zeros(4, 2, 2), torch.zeros(4, 2, 2), 64)
    table, lens, r = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), sa.rotary_frequencies(64, device="cpu")
    q, k, at = torch.zeros(1, 2, 2, 64), torch.zeros(1, 2, 2, 64), torch.arange(2)
    for name, call in (("rotate_heads ", lambda q: sa.rotate_heads(q, k, at, r)), ("rotate_heads_trainable", lambda q: sa.rotate_heads_trainable(q, k, at, r)),
                       ("rotate_heads_backward", lambda q: sa.rotate_heads_backward(q, k, q, k, at, r)),
                       ("paged_cache_append_rotated", lambda q: sa.paged_cache_append_rotated(cache, q, k, k, table, lens, r)),
                       ("sparse_attention_decode_tree", lambda q: sa.sparse_attention_decode_tree(q, cache, table, lens, table)),
                       ("paged_cache_keep", lambda q: sa.paged_cache_keep(cache, table, lens, table, lens) or q)):
        with pytest.raises(RuntimeError, match=name + ".*cannot be recorded" if name[-1] != " " else "rotate_heads cannot be recorded"):
            torch.jit.trace(call, (q,))
    with pytest.raises(RuntimeError, match="verify_drafts cannot be recorded"):
        torch.jit.trace(lambda p: sa.verify_drafts(p, x, u), (p,))
