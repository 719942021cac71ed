"""Page copies over all layers, bit for bit."""
import numpy as np
import pytest
import torch

from llm_infer_rust_amd._native import NativeError
from llm_infer_rust_amd.kv_cache import KVCacheLayout, KVCachePool, ModelError

pytestmark = pytest.mark.gpu


def make(layers, pages, page, heads, width, dtype=torch.bfloat16):
    pool = KVCachePool(KVCacheLayout(layers, pages, page, heads, width), dtype, "cuda")
    g = torch.Generator(device="cuda").manual_seed(layers + pages)
    pool.buffer[:, :, 1:].normal_(generator=g)
    return pool


def expect(pool, src, dst, tokens=None):
    want = pool.buffer.clone()
    for i, (s, d) in enumerate(zip(src, dst)):
        n = pool.layout.page_size if tokens is None else tokens[i]
        want[:, :, d, :n] = pool.buffer[:, :, s, :n]
    return want


def bits(t):
    return t.view(torch.int16 if t.element_size() == 2 else torch.int32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layers,page,heads,width", [
    (1, 1, 1, 8), (2, 16, 8, 128), (3, 13, 5, 128), (2, 24, 1, 128), (1, 7, 3, 5), (4, 64, 2, 64),
    (1, 1024, 8, 128)])
@pytest.mark.parametrize("partial", [False, True])
def test_copies(gpu, dtype, layers, page, heads, width, partial):
    rng = np.random.default_rng(page)
    pool = make(layers, 40, page, heads, width, dtype)
    ids = rng.permutation(40) + 1
    src, dst = [int(ids[i % 5]) for i in range(30)], [int(i) for i in ids[5:35]]
    tokens = [int(rng.integers(0, page + 1)) for _ in src] if partial else None
    want = expect(pool, src, dst, tokens)
    pool.copy_pages(src, dst, tokens)
    assert torch.equal(bits(pool.buffer), bits(want))


def test_more_pairs_than_a_launch_holds(gpu):
    pool = make(2, 1500, 4, 2, 16)
    rng = np.random.default_rng(0)
    ids = rng.permutation(1500) + 1
    for n in (240, 320, 321, 480, 481, 700):
        src, dst = ids[:n], ids[n:2 * n]
        tokens = rng.integers(0, 5, n)
        want = expect(pool, src.tolist(), dst.tolist(), tokens.tolist())
        pool.copy_pages(src, dst, tokens)
        assert torch.equal(bits(pool.buffer), bits(want)), n


def test_nan_payloads_and_the_page_behind(gpu):
    """Bits are copied, not values, and what is behind the last token stays."""
    pool = make(2, 4, 16, 2, 128)
    bits(pool.buffer)[:, :, 1] = 0x7f81
    want = expect(pool, [1], [2], [5])
    pool.copy_pages([1], [2], [5])
    assert torch.equal(bits(pool.buffer), bits(want))
    assert bool((pool.buffer[:, :, 0] == 0).all())


def test_offsets_past_4_gib(gpu):
    """Two planes of 5 GiB each: page and plane offsets pass 32 bits."""
    layout = KVCacheLayout(1, 5 * 1024, 1024, 4, 128)
    pool = KVCachePool(layout, torch.bfloat16, "cuda")
    src, dst = [5119, 1, 2500], [5118, 5120, 2]
    for s in src + dst:
        pool.buffer[:, :, s].normal_()
    want = [pool.buffer[:, :, s].clone() for s in src]
    pool.copy_pages(src, dst)
    for w, d in zip(want, dst):
        assert torch.equal(pool.buffer[:, :, d], w)


def test_streams_and_graphs(gpu):
    pool = make(2, 20, 16, 8, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = expect(pool, [1, 1], [2, 3])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pool.copy_pages([1, 1], [2, 3])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(pool.buffer, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.copy_pages([4, 5], [6, 7], [9, 16])
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        pool.buffer[:, :, 1:].normal_(generator=g)
        want = expect(pool, [4, 5], [6, 7], [9, 16])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool.buffer, want)


def test_refusals(gpu):
    pool = make(1, 8, 4, 1, 8)
    before = pool.buffer.clone()
    for args in (([1], [0]), ([1], [-1]), ([1, 2], [3]), ([1], [2], [1, 2]), ([1.5], [2]),
                 ([[1]], [[2]]), ([1], [2 ** 33])):
        with pytest.raises(ModelError):
            pool.copy_pages(*args)
    for args in (([9], [1]), ([1], [9]), ([1, 2], [2, 3]), ([1, 2], [3, 3]), ([1], [2], [5])):
        with pytest.raises(NativeError):
            pool.copy_pages(*args)
    pool.copy_pages([], [])
    pool.copy_pages([1], [2], [0])
    assert torch.equal(pool.buffer, before)
