"""What page copies refuse, without a GPU: the checks of the C entry (addresses are never
dereferenced) and of the pool's method."""
import ctypes
from array import array

import numpy as np
import pytest
import torch

from llm_infer_rust_amd import _native, kv_cache
from llm_infer_rust_amd.kv_cache import KVCacheLayout, KVCachePool

A = 0x10000


def copy(src, dst, tokens=None, planes=2, pages=8, page_tokens=16, token_bytes=256, pool=A,
         pairs=None):
    n = len(src) if pairs is None else pairs
    arr = lambda v: (ctypes.c_int32 * max(len(v), 1))(*v)  # noqa: E731
    return _native.lib().mi355x_copy_pages(pool, planes, pages, page_tokens, token_bytes, arr(src),
                                           arr(dst), None if tokens is None else arr(tokens), n,
                                           None)


@pytest.mark.parametrize("kwargs,what", [
    (dict(src=[8], dst=[1]), b"outside the pool"),
    (dict(src=[-1], dst=[1]), b"outside the pool"),
    (dict(src=[1], dst=[8]), b"outside the pool"),
    (dict(src=[1, 2], dst=[3, -2]), b"outside the pool"),
    (dict(src=[1, 2], dst=[3, 3]), b"destination"),
    (dict(src=[1, 2], dst=[2, 3]), b"destination"),
    (dict(src=[1], dst=[1]), b"destination"),
    (dict(src=[1, 2], dst=[3, 1]), b"destination"),
    (dict(src=[1], dst=[2], tokens=[17]), b"token count"),
    (dict(src=[1], dst=[2], tokens=[-1]), b"token count"),
    (dict(src=[1], dst=[2], planes=0), b"geometry"),
    (dict(src=[1], dst=[2], planes=70000), b"geometry"),
    (dict(src=[1], dst=[2], pages=0), b"geometry"),
    (dict(src=[1], dst=[2], page_tokens=0), b"geometry"),
    (dict(src=[1], dst=[2], token_bytes=3), b"geometry"),
    (dict(src=[1], dst=[2], pairs=-1), b"geometry"),
    (dict(src=[1], dst=[2], planes=65535, page_tokens=1 << 20, token_bytes=2), b"page too large"),
    (dict(src=[1], dst=[2], pool=None), b"null"),
    (dict(src=[1], dst=[2], pool=0x10001), b"misaligned"),
])
def test_refused(kwargs, what):
    err = copy(**kwargs)
    assert err is not None and what in err


def test_a_refused_call_leaves_no_marks():
    """Marks of one call's pages do not stay for the next (of the same thread)."""
    assert b"destination" in copy([1, 2], [3, 3])
    assert b"destination" in copy([4], [4])
    # nothing to copy: no launch, so no GPU is needed, but the pairs are checked
    assert copy([1, 2], [3, 4], [0, 0]) is None
    assert copy([3, 4], [1, 2], [0, 0]) is None
    assert copy([], []) is None


def test_method_refuses():
    pool = KVCachePool(KVCacheLayout(2, 4, 16, 2, 8), torch.bfloat16, "cpu")
    with pytest.raises(_native.NativeError):
        pool.copy_pages([1], [2])


def test_host_ids():
    want = [3, 0, 2 ** 31 - 1, -2 ** 31]
    for values in (want, tuple(want), np.array(want), np.array(want, np.int32), torch.tensor(want),
                   [np.int64(w) for w in want], array("q", want)):
        assert list(kv_cache._host_ids(values)) == want
    assert list(kv_cache._host_ids(range(5, 8))) == [5, 6, 7]
    assert list(kv_cache._host_ids(np.arange(8)[::2])) == [0, 2, 4, 6]
    for values in ([1.5], [[1]], [2 ** 31], [-2 ** 31 - 1], np.array([2 ** 31]), np.array([1.0]),
                   np.array([[1]]), b"abcd", "1234", ["1"], [None]):
        with pytest.raises(kv_cache.ModelError):
            kv_cache._host_ids(values)
