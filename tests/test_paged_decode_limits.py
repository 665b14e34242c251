"""Attentions over the paged cache with more planes of rows than a launch has, refused on the host with the sizes that they have (so these run without a GPU)."""
import ctypes

import pytest

from sparseattention_amd import _native

FAKE = 0x1000  # never dereferenced
S2, S3, S4 = _native.strides((4, 1)), _native.strides((64, 8, 1)), _native.strides((1024, 128, 128, 1))


def tree(B, H, Hq, n, pages, page_size=64):
    pool = ctypes.byref(_native.PagedCacheStruct(FAKE, FAKE, FAKE, FAKE, 1, H, page_size, 128, 128))
    lib = _native.load()
    rc = lib.sa_sparse_attention_decode_tree(FAKE, S4, pool, FAKE, S2, FAKE, FAKE, S2, None, pages, FAKE, S4, B, Hq, n, 0, 0, 0.1, None, 0, None, None, None)
    return rc, lib.sa_last_error().decode()


@pytest.mark.parametrize("B,H,G,n,pages,planes,rows,chunks", [
    (1 << 23, 4, 1, 8, 4, 1 << 25, 16, 8),            # too many sequences' heads
    (1 << 20, 8, 1, 64, 4, 1 << 23, 64, 8),           # (planes that a launch has)
    (1 << 20, 8, 4, 64, 4, 1 << 24, 128, 8),
    (1 << 20, 8, 4, 64, 64, 1 << 24, 128, 128),       # too many chunks of them
    (1 << 21, 8, 4, 64, 4, 1 << 25, 128, 8),
    (64, 1, 1, 64, 1 << 22, 64, 64, 1 << 23),         # few planes of a long table
    (1, 1, 256, 64, 1 << 17, 512, 32, 1 << 18),       # one head's rows, in planes of 32
])
def test_tree_says_what_it_refuses(B, H, G, n, pages, planes, rows, chunks):
    rc, message = tree(B, H, G * H, n, pages)
    if planes <= 1 << 24 and planes * chunks <= 1 << 30:
        assert rc == _native.SA_ERR_WORKSPACE
    else:
        assert rc == _native.SA_ERR_UNSUPPORTED and f"{planes} planes of {rows} rows and {chunks} chunks" in message, message


def test_paged_says_what_it_refuses():
    pool = ctypes.byref(_native.PagedCacheStruct(FAKE, FAKE, FAKE, FAKE, 1, 4, 64, 128, 128))
    lib, none = _native.load(), None
    rc = lib.sa_sparse_attention_decode_paged(FAKE, S4, pool, FAKE, S2, FAKE, none, 4, FAKE, S4, none, none, none, none, none, none, none, none, none, none, 0, 1 << 23, 4, 1, 0, 0, 0.1,
                                              none, 0, none, none, none)
    message = lib.sa_last_error().decode()
    assert rc == _native.SA_ERR_UNSUPPORTED and f"{1 << 25} planes of 16 rows and 8 chunks" in message, message
