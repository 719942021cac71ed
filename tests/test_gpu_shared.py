"""Attention over prefixes that rows of a batch share, decode and several new tokens a row."""
import gc

import numpy as np
import pytest
import torch

from llm_infer_rust_amd.backend import (AttentionMetadata, BatchPhase, DecodeHostMetadata,
                                        ModelError, SharedPrefix)
from shared_helpers import Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def shared_however_little_it_saves(monkeypatch):
    monkeypatch.setenv("MI355X_SHARED_FROM", "0")


BF16, FP16 = torch.bfloat16, torch.float16


def own_lengths(rows, low, high, seed=0):
    return np.random.default_rng(seed).integers(low, high + 1, rows).tolist()


DECODE = [
    # groups (rows, shared), longest own part, heads, kv heads, page, type
    ([(4, 1100)], 150, 32, 8, 16, BF16),
    ([(2, 64)], 1, 16, 8, 16, BF16),
    ([(2, 65)], 1, 16, 8, 1, FP16),
    ([(3, 63)], 70, 16, 8, 16, BF16),
    ([(1, 500), (2, 128), (1, 9), (5, 700)], 90, 16, 8, 13, BF16),
    ([(40, 1000)], 300, 32, 8, 16, FP16),
    ([(70, 640)], 40, 64, 8, 64, BF16),
    ([(33, 333), (17, 777), (3, 2000)], 100, 8, 8, 24, BF16),
    ([(9, 4000)], 60, 8, 1, 16, BF16),
    ([(9, 900)], 60, 6, 3, 8, FP16),
    ([(20, 512)], 200, 16, 4, 128, BF16),
    ([(130, 256)], 20, 4, 2, 16, BF16),
    ([(65, 1500)], 33, 16, 16, 16, FP16),
    ([(50, 300), (4, 200)], 33, 24, 12, 16, BF16),
    ([(30, 300), (4, 200)], 33, 20, 5, 16, BF16),
    ([(256, 192)], 5, 32, 8, 16, BF16),
    ([(6, 300)] * 12, 64, 32, 4, 16, BF16),
]


@pytest.mark.parametrize("groups,own,heads,kv_heads,page,dtype", DECODE)
@pytest.mark.parametrize("copies", [False, True])
def test_decode(gpu, groups, own, heads, kv_heads, page, dtype, copies):
    rows = sum(r for r, _ in groups)
    b = Batch(groups, own_lengths(rows, 1, own), None, heads, kv_heads, page, dtype,
              seed=rows + own, copies=copies)
    got, info = b.run(b.decode_meta())
    print(f"[shared] {info} worst {b.check(got):.2f} of the limit", flush=True)
    plain, none = b.run(b.decode_meta(shared=False))
    assert none["items"] == 0
    b.check(plain)


@pytest.mark.parametrize("groups,own,heads,kv_heads,page,dtype", DECODE)
def test_decode_shares_every_group(gpu, groups, own, heads, kv_heads, page, dtype):
    rows = sum(r for r, _ in groups)
    b = Batch(groups, own_lengths(rows, 1, own), None, heads, kv_heads, page, dtype)
    _, info = b.run(b.decode_meta())
    shared = [n for r, n in groups if r > 1 and n >= 64]
    assert info["groups"] == len(shared) and info["tokens"] == sum(n // 64 * 64 for n in shared)


EXTEND = [
    ([(5, 700)], 0, 40, 32, 8, 16, BF16),
    ([(48, 1024)], 0, 40, 32, 8, 16, BF16),
    ([(7, 300), (1, 100), (4, 64), (3, 63)], 90, 7, 16, 8, 16, FP16),
    ([(2, 128)], 5, 1, 16, 8, 1, BF16),
    ([(3, 1000)], 300, 260, 32, 8, 13, BF16),
    ([(20, 640)], 70, 5, 64, 8, 64, BF16),
    ([(9, 500)], 20, 33, 8, 8, 24, BF16),
    ([(4, 200)], 10, 70, 8, 1, 8, FP16),
    ([(6, 333)] * 5, 64, 9, 6, 3, 128, BF16),
]


@pytest.mark.parametrize("groups,own,new,heads,kv_heads,page,dtype", EXTEND)
def test_extend(gpu, groups, own, new, heads, kv_heads, page, dtype):
    rows = sum(r for r, _ in groups)
    fresh = own_lengths(rows, 1, new, seed=1)
    cached = own_lengths(rows, 0, own, seed=2)
    b = Batch(groups, [t + c for t, c in zip(fresh, cached)], fresh, heads, kv_heads, page, dtype,
              seed=rows + new)
    got, info = b.run(b.extend_meta())
    print(f"[shared] {info} worst {b.check(got):.2f} of the limit", flush=True)
    assert info["groups"] == sum(r > 1 and n >= 64 for r, n in groups)
    plain, none = b.run(b.extend_meta(shared=False))
    assert none["items"] == 0
    b.check(plain)


def test_what_saves_little_is_left_to_the_plain_kernels(gpu, monkeypatch):
    """By default 8 MiB of K and V a layer are saved, by prefixes of at least 128 tokens, or nothing
    is shared; with fewer kv heads than a slice holds it always is."""
    monkeypatch.delenv("MI355X_SHARED_FROM")
    for groups, kv_heads, used in (([(2, 1024)], 8, False), ([(4, 1024)], 8, True),
                                   ([(256, 127)], 8, False), ([(40, 128), (3, 64)], 8, True),
                                   ([(2, 128)], 1, True), ([(1, 5000)], 1, False)):
        b = Batch(groups, [3] * sum(r for r, _ in groups), heads=4 * kv_heads, kv_heads=kv_heads)
        got, info = b.run(b.decode_meta())
        assert (info["items"] > 0) == used, (groups, info)
        b.check(got)
        assert info["tokens"] == (sum(n for r, n in groups if r > 1 and n >= 128) if used else 0)


def test_four_kv_heads_share_where_the_prefix_is_long(gpu, monkeypatch):
    """One slice of four heads streams rows' own keys slower than the plain kernel: the prefix saves 16
    MiB and a third of what the rows read of their own, or it is not shared."""
    monkeypatch.delenv("MI355X_SHARED_FROM")
    for groups, own, used in (([(48, 256)], 3000, False), ([(48, 2000)], 1000, True),
                              ([(12, 512)], 64, False), ([(48, 256)], 64, True),
                              ([(12, 1024)], 3000, False), ([(20, 900), (28, 128)], 2500, False)):
        b = Batch(groups, [own] * sum(r for r, _ in groups), heads=16, kv_heads=4)
        got, info = b.run(b.decode_meta())
        assert (info["items"] > 0) == used, (groups, own, info)
        b.check(got)


@pytest.mark.parametrize("rows,new,prefix,heads,kv_heads,used", [
    # us, plain and shared: where the plain kernel's columns are full, sharing is the slower one
    (48, 128, 512, 32, 8, False),    # 84, 202
    (16, 512, 2048, 32, 8, False),   # 333, 464
    (48, 64, 512, 64, 8, False),     # 83, 191
    (4, 1024, 2048, 32, 8, False),   # 186, 274
    (48, 16, 2048, 32, 8, True),     # 100, 62
    (16, 2, 8192, 16, 8, True),      # 154, 21
    (48, 64, 8192, 16, 8, True),     # 326, 257
    (2, 16, 512, 8, 1, True),        # 21.3, 16.7
])
def test_extends_share_where_that_is_quicker(gpu, monkeypatch, rows, new, prefix, heads, kv_heads,
                                             used):
    monkeypatch.delenv("MI355X_SHARED_FROM")
    table = torch.arange(1, (prefix + new) // 16 + 2, dtype=torch.int32, device=gpu).repeat(rows, 1)
    starts = [i * new for i in range(rows + 1)]
    meta = AttentionMetadata(
        BatchPhase.PREFILL, block_table=table,
        cu_seqlens_q=torch.tensor(starts, dtype=torch.int32, device=gpu),
        prefix_lens=torch.full((rows,), prefix, dtype=torch.int32, device=gpu),
        host_cu_seqlens_q=starts, host_prefix_lens=[prefix] * rows,
        shared_prefix=SharedPrefix([rows], [prefix]))
    attention = Batch([(2, 64)], [1, 1], heads=heads, kv_heads=kv_heads).attention()
    batch = attention.prepare(meta, starts[-1])
    assert (batch.plan.plan.shared_info()["items"] > 0) == used


def test_partials_of_no_use_are_left_to_the_plain_kernels(gpu, monkeypatch):
    """A batch whose partial outputs pass the limit runs plain, on the same plan as ones that share."""
    d = Batch([(40, 600)], own_lengths(40, 1, 50), heads=16, kv_heads=8)
    e = Batch([(9, 500)], [30] * 9, [30] * 9, heads=16, kv_heads=8)
    attention = d.attention()
    for most in (None, 100_000, None, 0, 1 << 40):
        if most is None:
            monkeypatch.delenv("MI355X_SHARED_MOST", raising=False)
        else:
            monkeypatch.setenv("MI355X_SHARED_MOST", str(most))
        for b, meta in ((d, d.decode_meta()), (e, e.extend_meta())):
            got, info = b.run(meta, attention)
            assert (info["items"] > 0) == (most is None or most > 100_000)
            b.check(got)


def test_partials_have_a_limit(gpu):
    """4 GiB by default: 516 bytes a token, q head and part, at least two parts. Planned, not run."""
    rows, prefix = 1100, 4096
    table = torch.arange(1, prefix // 16 + 6, dtype=torch.int32, device=gpu).repeat(rows, 1)
    attention = Batch([(2, 64)], [1, 1], heads=64).attention()
    for new in (8, 64):  # 0.54 GiB and 4.3 GiB at the least
        starts = [i * new for i in range(rows + 1)]
        meta = AttentionMetadata(
            BatchPhase.PREFILL, block_table=table,
            cu_seqlens_q=torch.tensor(starts, dtype=torch.int32, device=gpu),
            prefix_lens=torch.full((rows,), prefix, dtype=torch.int32, device=gpu),
            host_cu_seqlens_q=starts, host_prefix_lens=[prefix] * rows,
            shared_prefix=SharedPrefix([rows], [prefix]))
        batch = attention.prepare(meta, starts[-1])
        assert (batch.plan.plan.shared_info()["items"] > 0) == (new == 8)
        del batch


def test_whole_request_is_shared(gpu):
    """A group's lens may cover every token: the last ones are then each row's own."""
    b = Batch([(3, 128), (2, 64), (2, 40)], [0] * 7, [1] * 7)
    got, info = b.run(b.decode_meta())
    b.check(got)
    assert info["tokens"] in (0, 64)  # 127 and 63 tokens that may be shared


def test_strided_queries_and_output(gpu):
    b = Batch([(6, 400)], own_lengths(6, 1, 50), heads=16, kv_heads=8)
    packed = torch.randn(6, 32 * 128, device="cuda").to(BF16)
    packed[:, :16 * 128] = b.q.view(6, -1)
    attention, q = b.attention(), packed[:, :16 * 128].view(6, 16, 128)
    batch = attention.prepare(b.decode_meta(), 6)
    assert batch.plan.plan.shared_info()["items"]
    out = torch.full((7, 16 * 128), 7.0, dtype=BF16, device="cuda")
    batch.forward_into(q, None, None, b.cache(), out[:6])
    b.check(out[:6].view(6, 16, 128))
    assert bool((out[6] == 7).all())  # rows behind the last are left as they were


def test_sharp_scores(gpu):
    """Scores far apart: one key of the prefix or of the own part takes all the weight."""
    for scale in (8.0, 60.0):
        b = Batch([(5, 300), (2, 700)], own_lengths(7, 1, 90), heads=32, kv_heads=8, q_scale=scale)
        want, mass = b.reference()
        for meta in (b.decode_meta(), b.decode_meta(shared=False)):
            got, _ = b.run(meta)
            assert bool(torch.isfinite(got).all())
            # sum |q k| / sqrt(128) is at most 200 * scale: its fp32 rounding moves a score by 128 *
            # 2^-24 of that at the very most, and the output by as much of 2 |v|, |v| below 6
            limit = 2 ** -7 * mass + 2 ** -8 * want.abs() + 200 * scale * 128 * 2 ** -24 * 12
            assert bool(((got.double() - want).abs() <= limit).all())


def ascending(rows=40, keys=4096, heads=32, kv_heads=8, dtype=BF16):
    """Queries along the first axis and one key in 64 that they like, each a little more than the one
    before; only the last of them has a value. Its weight is the largest there is, and the output is
    that weight times the value, whatever the others' weights are rounded to."""
    b = Batch([(rows, keys)], [1] * rows, None, heads, kv_heads, 16, dtype)
    g = torch.Generator().manual_seed(1)
    b.q.zero_()
    b.q[:, :, 0] = (8 + 40 * torch.rand(rows, heads, generator=g)).to(dtype).cuda()
    k, v = b.k.view(-1, kv_heads, 128), b.v.view(-1, kv_heads, 128)
    k.zero_()
    k[:, :, 0] = -64
    last = v[b.slots[0][keys - 7]].clone()
    v.zero_()
    for i in range(keys // 64):
        k[b.slots[0][64 * i + 57], :, 0] = i / 8
    v[b.slots[0][keys - 7]] = last
    return b


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_the_largest_weight_is_exact(gpu, dtype):
    """Decode rows keep the largest probability at 1, with shared prefixes too: the output is rounded
    once (half a step). Beside that, the sum's fp32 weights: scores of up to 2^7 in log2 units and
    their references are off by 2^-24 of that each, and the weights by ln 2 times both: 2e-5."""
    b = ascending(dtype=dtype)
    want, _ = b.reference()
    limit = (torch.finfo(dtype).eps / 2 + 2e-5) * want.abs() + 1e-7
    for meta in (b.decode_meta(shared=False), b.decode_meta()):
        got, info = b.run(meta)
        print(f"[shared] {info}", flush=True)
        worst = float(((got.double() - want).abs() / limit).max())
        assert worst <= 1.0, worst
    assert info["products"] and info["items"] <= 8 * 64 // 2  # parts of two tiles and more


def test_a_first_tile_without_weight(gpu):
    """Scores of -inf in the first tiles, and all others far below 0: what has weight there counts."""
    b = ascending(keys=2048)
    k = b.k.view(-1, 8, 128)
    for slots in b.slots:
        k[slots, :, 0] = -64  # from -65 to -391 in log2 units
        k[slots[-1], :, 0] = -66
    for tile in range(0, 32, 2):  # the first tile of every part of an even number of them
        k[b.slots[0][64 * tile:64 * tile + 64], :, 0] = -float("inf")
    b.v.copy_(torch.randn(b.v.shape, generator=torch.Generator().manual_seed(2)).to(BF16).cuda())
    got, info = b.run(b.decode_meta())
    assert info["products"]
    b.check(got)


def test_nan_of_one_row_stays_there(gpu):
    """A NaN among a row's own keys reaches that row only; one in the prefix all of its group."""
    b = Batch([(4, 256), (3, 128)], [20] * 7, heads=16, kv_heads=8)
    flat = b.k.view(-1, 8, 128)
    flat[b.slots[2][270]] = float("nan")
    got, info = b.run(b.decode_meta())
    assert info["items"]
    bad = torch.isnan(got.float()).flatten(1).any(1).tolist()
    assert bad == [False, False, True, False, False, False, False]
    flat[b.slots[4][100]] = float("nan")
    got, _ = b.run(b.decode_meta())
    assert torch.isnan(got.float()).flatten(1).any(1).tolist() == [False, False, True, False, True,
                                                                   True, True]


def test_same_bits_every_time(gpu):
    b = Batch([(40, 1000), (3, 500)], own_lengths(43, 1, 300), heads=32, kv_heads=8)
    attention = b.attention()
    first, _ = b.run(b.decode_meta(), attention)
    for _ in range(4):
        again, _ = b.run(b.decode_meta(), attention)
        assert torch.equal(first, again)


def test_offsets_past_4_gib(gpu):
    """Pages whose slots lie past 2^31 elements of the cache."""
    b = Batch([(4, 300)], [30] * 4, heads=32, kv_heads=8)
    far = (2 ** 32 // (16 * 8 * 128)) + 5
    pages = b.k.size(0)
    for name in ("k", "v"):
        big = torch.zeros(far + pages, 16, 8, 128, dtype=BF16, device="cuda")
        big[far:] = getattr(b, name)
        setattr(b, name, big)
    b.table[b.table >= 0] += far
    b.slots = [s + far * 16 for s in b.slots]
    got, info = b.run(b.decode_meta())
    assert info["items"]
    b.check(got)


def test_one_plan_with_and_without_groups(gpu):
    """An eager backend re-plans the same handle; what an earlier batch shared is forgotten."""
    shapes = [([(40, 600)], 50), ([(2, 900)], 20), ([(1, 70), (1, 30)], 9), ([(130, 128)], 3)]
    batches = [Batch(g, own_lengths(sum(r for r, _ in g), 1, own), heads=16, kv_heads=8, seed=i)
               for i, (g, own) in enumerate(shapes)]
    attention = batches[0].attention()
    for b in batches + batches[::-1]:
        for shared in (True, False):
            got, _ = b.run(b.decode_meta(shared), attention)
            b.check(got)
            got, _ = b.run(b.extend_meta(shared), attention)
            b.check(got)


def test_streams(gpu):
    b = Batch([(12, 700)], own_lengths(12, 1, 90), heads=32, kv_heads=8)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got, _ = b.run(b.decode_meta())
    torch.cuda.current_stream().wait_stream(side)
    b.check(got)


@pytest.mark.parametrize("rows,heads,kv_heads", [(6, 32, 8), (64, 32, 8), (64, 32, 4), (64, 8, 1),
                                                 (40, 16, 2), (200, 8, 8), (64, 24, 12)])
def test_graph(gpu, rows, heads, kv_heads):
    """One captured launch serves any groups, also none; replays are checked one by one."""
    cols = 80
    table = torch.zeros(rows, cols, dtype=torch.int32, device="cuda")
    lens = torch.ones(rows, dtype=torch.int32, device="cuda")
    kinds = [[(rows, 500)], [(1, 100)] * rows, [(rows // 2, 640), (rows - rows // 2, 64)],
             [(2, 300)] * (rows // 2), [(rows, 0)], [(rows - 2, 1000), (2, 100)]]
    batches = [Batch(g, own_lengths(rows, 1, 60, seed=i), heads=heads, kv_heads=kv_heads, seed=i)
               for i, g in enumerate(kinds)]
    pages = max(b.k.size(0) for b in batches)
    k, v = (torch.zeros(pages, 16, kv_heads, 128, dtype=BF16, device="cuda") for _ in range(2))
    q = torch.zeros(rows, heads, 128, dtype=BF16, device="cuda")
    attention, cache = batches[0].attention(), batches[0].cache()
    cache.bind_kv_cache(k, v)
    meta = AttentionMetadata(BatchPhase.DECODE, block_table=table, cache_seqlens=lens,
                             shared_prefix=SharedPrefix([rows], [0]))
    state = attention.prepare_decode_graph(meta)
    batch = attention.prepare(meta, rows)
    out = torch.zeros(rows, heads * 128, dtype=BF16, device="cuda")
    batch.forward_into(q, None, None, cache, out)
    torch.cuda.synchronize()
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch.forward_into(q, None, None, cache, out)
    for b in batches + batches[::-1]:
        k[:b.k.size(0)] = b.k
        v[:b.v.size(0)] = b.v
        q.copy_(b.q)
        table.fill_(-1)
        table[:, :b.table.size(1)] = b.table
        lens.copy_(b.lens)
        state.prepare_replay(DecodeHostMetadata(b.keys), b.shared())
        graph.replay()
        torch.cuda.synchronize()
        b.check(out.view(rows, heads, 128))
        state.prepare_replay(DecodeHostMetadata(b.keys))  # and without its groups
        graph.replay()
        torch.cuda.synchronize()
        b.check(out.view(rows, heads, 128))


def test_graph_prepared_without_groups_ignores_them(gpu):
    b = Batch([(4, 200)], [10] * 4)
    attention = b.attention()
    meta = b.decode_meta(shared=False)
    state = attention.prepare_decode_graph(meta)
    batch = attention.prepare(meta, 4)
    state.prepare_replay(DecodeHostMetadata(b.keys), b.shared())
    assert state.plan.shared_info()["items"] == 0
    b.check(batch.forward(b.q, None, None, b.cache()).view(b.q.shape))


def test_refusals(gpu):
    b = Batch([(4, 200)], [10] * 4)
    attention = b.attention()
    for rows, lens in (([4], [211]), ([3], [200]), ([5], [200]), ([4], [-1]), ([2, 2], [200]),
                       ([0, 4], [0, 1]), ([], []), ([4.0], [200]), ([4], [2 ** 40])):
        for meta in (b.decode_meta(), b.extend_meta()):
            meta.shared_prefix = SharedPrefix(rows, lens)
            with pytest.raises(ModelError):
                attention.prepare(meta, 4)
                pytest.fail(f"{rows} {lens} {meta.forward_mode}")
    meta = b.extend_meta()
    meta.shared_prefix = SharedPrefix([4], [210])  # of the 209 cached tokens
    with pytest.raises(ModelError):
        attention.prepare(meta, 4)
    got, _ = b.run(b.decode_meta(), attention)  # the backend is still usable
    b.check(got)
