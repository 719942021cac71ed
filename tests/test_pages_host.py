"""Pages with several holders, completions' places and what the plan is told of them (CPU)."""
import types

import numpy as np
import pytest

from llm_infer_rust_amd.backend import ModelError, SharedPrefix, shared_arrays
from llm_infer_rust_amd.engine import Engine, PageAllocator, Request
from llm_infer_rust_amd.sampling import SamplingParams


def test_pages_are_free_after_their_last_holder():
    pages = PageAllocator(8)
    a = pages.alloc(4)
    pages.share(a[:3])
    pages.share(a[:2])
    b = pages.alloc(1)
    pages.release(a)
    assert sorted(pages.free) == sorted([a[3]] + [p for p in range(1, 9) if p not in a + b])
    pages.release(a[:2] + b)
    assert a[0] not in pages.free and b[0] in pages.free
    pages.release(a[:3])
    assert sorted(pages.free) == list(range(1, 9)) and not pages.more_holders


def test_release_keeps_its_order_without_shared_pages():
    plain, shared = PageAllocator(8), PageAllocator(8)
    x, y = plain.alloc(3), shared.alloc(3)
    shared.share([8])  # one page elsewhere has two holders
    plain.release(x)
    shared.release(y)
    assert plain.free == shared.free


def request(uid, size, group=None):
    r = Request(uid, np.arange(size), SamplingParams())
    r.completions = group if group is not None else [r]
    if group is not None:
        group.append(r)
    return r


def test_neighbours_of_one_prompt():
    first, second = [], []
    a = [request(i, 100, first) for i in range(3)]
    b = [request(3, 70)]
    c = [request(4 + i, 50, second) for i in range(2)]
    self = types.SimpleNamespace(cfg=types.SimpleNamespace(share_prefixes=True))
    got = Engine._shared(self, a + b + c)
    assert got == SharedPrefix([3, 1, 2], [100, 0, 50])
    assert Engine._shared(self, a[:1] + b + c[:1], 8) == SharedPrefix([1, 1, 1, 5], [0, 0, 0, 0])
    assert Engine._shared(self, [], 4) == SharedPrefix([4], [0])
    self.cfg.share_prefixes = False
    assert Engine._shared(self, a) is None


def test_slots_before_and_after_the_fork():
    group = []
    a, b = request(0, 10, group), request(1, 10, group)
    assert a.slots == 2 and b.slots == 1
    a.output.append(3)
    assert a.slots == 1
    assert request(2, 10).slots == 1


def test_parameters():
    p = SamplingParams(n=0).normalized()
    assert p.n == 1 and p.logprobs is None


@pytest.mark.parametrize("rows,lens", [([4], [-1]), ([3], [1]), ([5], [1]), ([2, 2], [1]), ([], []),
                                       ([0, 4], [1, 1]), ([4.0], [1]), ([4], [2 ** 31]),
                                       ([-1, 5], [1, 1]), ([[4]], [[1]])])
def test_groups_that_do_not_fit_the_batch(rows, lens):
    with pytest.raises(ModelError):
        shared_arrays(SharedPrefix(rows, lens), 4)


def test_groups_as_arrays():
    rows, lens = shared_arrays(SharedPrefix(rows=(1, 3), lens=np.array([5, 0])), 4)
    assert rows.dtype == lens.dtype == np.int32
    assert rows.tolist() == [1, 3] and lens.tolist() == [5, 0]
