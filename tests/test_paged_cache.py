"""Refusals of the paged K/V cache's entry points, on the host before anything is launched (so these run without a GPU)."""
import ctypes

import pytest
import torch

import sparseattention_amd as sa
from sparseattention_amd import _native

FAKE = 0x1000  # never dereferenced: every call below must fail validation first
BAD, UNSUPPORTED, WORKSPACE = _native.SA_ERR_INVALID_ARGUMENT, _native.SA_ERR_UNSUPPORTED, _native.SA_ERR_WORKSPACE
S2 = _native.strides((4, 1))
S3 = _native.strides((8, 8, 1))
S4 = _native.strides((1024, 128, 128, 1))


def pool(k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, pages=8, H=2, page=64, D=128, cols=128):
    return ctypes.byref(_native.PagedCacheStruct(k, v, ks, vs, pages, H, page, D, cols))


def append(c=None, k=FAKE, ks=S4, table=FAKE, lens=FAKE, B=1, S=4, pages=4, dtype=0):
    return _native.load().sa_paged_cache_append(c or pool(), k, ks, FAKE, S4, table, S2, lens, None, B, S, pages, dtype, None)


def gather(c=None, k=FAKE, length=64, B=1, pages=4, dtype=0):
    return _native.load().sa_paged_cache_gather(c or pool(), k, S4, FAKE, S4, FAKE, S2, FAKE, B, length, pages, dtype, None)


def decode(c=None, q=FAKE, qs=S4, Hq=4, Sq=1, window=0, scale=0.1, lists=False, packed=FAKE, tiles=4, dtype=0, B=1):
    ids = (FAKE, S4, FAKE, S3, FAKE, S4, FAKE, S3, packed, S2) if lists else (None,) * 10
    return _native.load().sa_sparse_attention_decode_paged(q, qs, c or pool(), FAKE, S2, FAKE, None, 4, FAKE, S4, *ids, tiles, B, Hq, Sq,
                                                           window, dtype, scale, None, 0, None, None, None)


@pytest.mark.parametrize("call", [append, gather, decode])
def test_pools(call):
    assert call(pool(k=None)) == BAD and call(pool(vs=None)) == BAD
    assert call(pool(pages=0)) == BAD and call(pool(pages=(1 << 20) + 1)) == BAD and call(pool(H=0)) == BAD
    assert call(pool(page=16)) == UNSUPPORTED and call(pool(page=48)) == UNSUPPORTED and call(pool(page=512)) == UNSUPPORTED
    assert call(pool(cols=0)) == UNSUPPORTED and call(pool(cols=132)) == UNSUPPORTED and call(pool(cols=60)) == UNSUPPORTED
    assert call(pool(D=80)) == UNSUPPORTED and call(pool(k=FAKE + 8)) == UNSUPPORTED
    assert call(pool(pages=1 << 20, H=1024, page=256)) == UNSUPPORTED
    assert call(B=0) == BAD and call(dtype=2) == UNSUPPORTED


def test_append_and_gather():
    assert append(k=None) == BAD and append(table=None) == BAD and append(lens=None) == BAD
    assert append(S=0) == BAD and append(pages=0) == BAD and append(pages=1 << 25) == UNSUPPORTED
    assert append(k=FAKE + 2) == UNSUPPORTED and append(ks=_native.strides((1024, 128, 132, 1))) == UNSUPPORTED
    assert append(ks=_native.strides((1024, 128, 128, 2))) == UNSUPPORTED
    assert append(S=1 << 30, B=1 << 10) == UNSUPPORTED  # (more workgroups than a grid has)
    assert gather(k=None) == BAD and gather(length=0) == BAD and gather(k=FAKE + 4) == UNSUPPORTED


def test_pages():
    lib = _native.load()
    assert lib.sa_paged_cache_copy(pool(), None, FAKE, 1, None) == BAD and lib.sa_paged_cache_copy(pool(), FAKE, FAKE, 0, None) == BAD
    fork = lambda n=1, parents=FAKE: lib.sa_paged_cache_fork(pool(), FAKE, S2, FAKE, 1, 4, parents, FAKE, n, FAKE, FAKE, None)  # noqa: E731
    assert fork(n=0) == BAD and fork(parents=None) == BAD
    need = lib.sa_paged_cache_compact_workspace_bytes(8)
    assert need > 0 and lib.sa_paged_cache_compact_workspace_bytes(0) == 0 and lib.sa_paged_cache_compact_workspace_bytes((1 << 20) + 1) == 0
    compact = lambda ws=FAKE, size=need, out=FAKE: lib.sa_paged_cache_compact(pool(), FAKE, S2, FAKE, 1, 4, out, FAKE, ws, size, None)  # noqa: E731
    assert compact(out=None) == BAD and compact(ws=None) == WORKSPACE and compact(size=need - 1) == WORKSPACE
    free = lambda pages=8, page=64, out=FAKE: lib.sa_paged_cache_free_pages(FAKE, S2, FAKE, 1, 4, pages, page, out, FAKE, None)  # noqa: E731
    assert free(pages=0) == BAD and free(page=65) == UNSUPPORTED and free(out=None) == BAD


def test_decode():
    assert decode(q=None) == BAD and decode(qs=_native.strides((1024, 128, 129, 1))) == UNSUPPORTED
    assert decode(Sq=0) == UNSUPPORTED and decode(Sq=33) == UNSUPPORTED
    assert decode(Hq=3) == BAD and decode(Hq=0) == BAD
    assert decode(scale=0.0) == BAD and decode(scale=float("nan")) == BAD and decode(scale=float("inf")) == BAD
    assert decode(window=-1) == BAD and decode(lists=True, window=3) == BAD
    assert decode(lists=True, packed=None) == BAD and decode(lists=True, tiles=5) == BAD and decode(lists=True, tiles=0) == BAD
    assert decode(lists=True, packed=FAKE + 2) == UNSUPPORTED


def test_python_refuses_without_a_gpu():
    with pytest.raises(ValueError, match="page_size"):
        sa.empty_paged_cache(4, 2, 64, page_size=48, device="cuda")
    for bad in ((0, 2, 64), ((1 << 20) + 1, 2, 64), (4, 0, 64), (4, 2, 0), (4, 2, 257)):
        with pytest.raises(ValueError):
            sa.empty_paged_cache(*bad, device="cuda")
    with pytest.raises(RuntimeError, match="GPU"):
        sa.empty_paged_cache(4, 2, 64, device="cpu")
    cache = sa.PagedCache(torch.zeros(4, 2, 2, 2048, dtype=torch.uint8), torch.zeros(4, 2, 2, 2048, dtype=torch.uint8),
                          torch.zeros(4, 2, 2), torch.zeros(4, 2, 2), 64)
    table, lens, x = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: sa.paged_cache_append(cache, x, x, table, lens), lambda: sa.paged_cache_gather(cache, table, lens),
                 lambda: sa.paged_cache_copy(cache, lens, lens), lambda: sa.paged_cache_fork(cache, table, lens, lens, lens),
                 lambda: sa.paged_cache_compact(cache, table, lens), lambda: sa.paged_cache_free_pages(cache, table, lens),
                 lambda: sa.sparse_attention_decode_paged(x, cache, table, lens)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        sa.paged_cache_gather(object(), table, lens)
