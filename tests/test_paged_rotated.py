"""Refusals of the append with norms and rotation, on the host before anything is launched (so these run without a GPU)."""
import ctypes

import pytest
import torch

import sparseattention_amd as sa
from sparseattention_amd import _native

FAKE = 0x1000  # never dereferenced: every call below must fail validation first
BAD, UNSUPPORTED = _native.SA_ERR_INVALID_ARGUMENT, _native.SA_ERR_UNSUPPORTED
S2 = _native.strides((4, 1))
S4 = _native.strides((1024, 128, 128, 1))


def pool(k=FAKE, pages=8, H=2, page=64, D=128, cols=128):
    return ctypes.byref(_native.PagedCacheStruct(k, FAKE, FAKE, FAKE, pages, H, page, D, cols))


def rotation(f=FAKE, axes=None, positions=None, R=128, eps=1e-6, n=1):
    return ctypes.byref(_native.RotationStruct(f, axes, positions, (ctypes.c_int64 * 3)(0, 8, 1), 0, n, R, 0, None, None, 0, eps))


def append(c=None, q=FAKE, qs=S4, out=FAKE, k=FAKE, v=FAKE, table=FAKE, lens=FAKE, parents=None, ps=S2, r=None, B=1, Hq=4, S=4, pages=4, dtype=0):
    return _native.load().sa_paged_cache_append_rotated(c or pool(), q, qs, out, S4, k, S4, v, S4, table, S2, lens, None, parents, ps, r or rotation(), B, Hq, S, pages,
                                                        dtype, None)


def test_arguments():
    assert append(pool(k=None)) == BAD and append(pool(page=48)) == UNSUPPORTED and append(pool(cols=132)) == UNSUPPORTED
    for name in ("q", "out", "k", "v", "table", "lens"):
        assert append(**{name: None}) == BAD, name
    assert append(q=FAKE + 8) == UNSUPPORTED and append(qs=_native.strides((1024, 128, 132, 1))) == UNSUPPORTED
    assert append(B=0) == BAD and append(S=0) == BAD and append(Hq=0) == BAD and append(pages=0) == BAD and append(dtype=2) == UNSUPPORTED
    assert append(r=rotation(f=None)) == BAD and append(r=rotation(R=136)) == UNSUPPORTED and append(r=rotation(eps=-1.0)) == BAD
    assert append(pool(cols=64), r=rotation(R=72)) == UNSUPPORTED
    assert append(r=rotation(axes=FAKE)) == BAD  # (no positions to choose from)
    assert append(parents=FAKE, ps=None) == BAD and append(parents=FAKE, S=65) == UNSUPPORTED
    assert append(parents=FAKE, r=rotation(positions=FAKE)) == BAD
    assert append(S=1 << 30, B=1 << 10) == UNSUPPORTED  # (more workgroups than a grid has)


def test_python_refuses_without_a_gpu():
    cache = sa.PagedCache(torch.zeros(4, 2, 2, 2048, dtype=torch.uint8), torch.zeros(4, 2, 2, 2048, dtype=torch.uint8), torch.zeros(4, 2, 2), torch.zeros(4, 2, 2), 64)
    table, lens, x = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        sa.paged_cache_append_rotated(cache, x, x, x, table, lens, sa.rotary_frequencies(64, device="cpu"))
