"""Token log probabilities, entropy and alternatives against their definition in 64 bits."""
import math

import pytest
import torch

from llm_infer_rust_amd import sampling
from llm_infer_rust_amd._native import NativeError, device_cus, lib

pytestmark = pytest.mark.gpu
INF = float("inf")


def reference(x, tokens, top):
    """Everything in float64 on the CPU; alternatives by value, equal ones by the lower id."""
    d = x.detach().cpu().double()
    lp = torch.log_softmax(d, 1)
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, torch.where(p.isnan(), p, torch.zeros_like(p))).sum(1)
    ok = (tokens.cpu() >= 0) & (tokens.cpu() < x.size(1))
    given = lp.gather(1, tokens.cpu().clamp(0, x.size(1) - 1)[:, None])[:, 0]
    given = torch.where(ok, given, torch.full_like(given, float("nan")))
    key = torch.where(d.isnan(), torch.full_like(d, INF), d)
    # NaN above +inf: two stable sorts, the finer key first
    first = torch.sort(key, dim=1, descending=True, stable=True).indices
    nan = torch.sort(d.isnan().gather(1, first).to(torch.int8), dim=1, descending=True,
                     stable=True).indices
    ids = first.gather(1, nan)[:, :top]
    return given, entropy, ids, lp.gather(1, ids)


def tolerance(x):
    """A thread's chain of fp32 additions holds at most 1,024 terms (a segment of 262,144 logits
    over 256 threads) with the trees above it, each off by 2^-24 of the sum; a term's own
    exponent is off by 2^-24 of its distance R to the row's maximum, in log2 units, and so is the
    result's. Eight for the exp2, log2 and the products around them."""
    d = x.detach().cpu().double()
    d = torch.where(d.isfinite(), d, torch.zeros_like(d))
    reach = float((d.amax(1) - d.amin(1)).max()) / math.log(2)
    return (1024 + 64 + 8 * min(reach, 1e4)) * 2.0 ** -24


def check(x, tokens, top):
    got = sampling.token_logprobs(x, tokens, top=top)
    given, entropy, ids, values = reference(x, tokens, top)
    tol = tolerance(x)
    assert got.logprobs.dtype == got.entropy.dtype == got.top_logprobs.dtype == torch.float32
    assert got.top_ids.dtype == torch.int64
    assert torch.equal(got.top_ids.cpu(), ids)
    far = 2.0 ** -22  # results far from 0 are rounded relative to their size
    torch.testing.assert_close(got.logprobs.cpu().double(), given, rtol=far, atol=tol,
                               equal_nan=True)
    torch.testing.assert_close(got.top_logprobs.cpu().double(), values, rtol=far, atol=tol,
                               equal_nan=True)
    # w / s is a mean of log2 units, up to 20 of them where it counts
    torch.testing.assert_close(got.entropy.cpu().double(), entropy, rtol=far, atol=24 * tol,
                               equal_nan=True)
    return got


def make(rows, vocab, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * scale).to(dtype)
    return x.cuda(), torch.randint(vocab, (rows,), generator=g).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (3, 2, 0), (5, 7, 7), (2, 50, 5), (9, 63, 63), (4, 64, 64), (700, 513, 20),
    (3, 1000, 64), (300, 2049, 8), (2, 8192, 20), (600, 8193, 5), (1, 16385, 64), (5, 32000, 20),
    (700, 32003, 3), (17, 50257, 20), (1, 151936, 5), (3, 151936, 20), (600, 20000, 0),
    (2, 300001, 10)])
def test_against_definition(gpu, dtype, rows, vocab, top):
    x, tokens = make(rows, vocab, dtype, seed=rows + vocab)
    check(x, tokens, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(3, 5000), (2, 40000), (600, 9000)])
def test_rows_that_order_hardly(gpu, dtype, rows, vocab):
    top = 20
    _, tokens = make(rows, vocab, dtype)
    lowest = torch.finfo(dtype).min
    ramp = torch.linspace(-30, 30, vocab).to(dtype)
    cases = {
        "equal": torch.zeros(vocab),
        "ascending": ramp,
        "descending": ramp.flip(0),
        "two values": (torch.arange(vocab) % 2).float(),
        "lowest": torch.full((vocab,), lowest),
        "lowest but three": torch.full((vocab,), lowest).index_fill(
            0, torch.tensor([0, vocab // 2, vocab - 1]), 2.5),
        "-inf but three": torch.full((vocab,), -INF).index_fill(
            0, torch.tensor([1, vocab // 3, vocab - 2]), -4.0),
        "-inf but one": torch.full((vocab,), -INF).index_fill(0, torch.tensor([vocab - 1]), 1.0),
        "-inf": torch.full((vocab,), -INF),
        "a NaN": ramp.float().index_fill(0, torch.tensor([vocab // 2]), float("nan")),
        "NaN": torch.full((vocab,), float("nan")),
        "+inf": ramp.float().index_fill(0, torch.tensor([7, vocab - 5]), INF),
        "zeros of both signs": torch.where(torch.arange(vocab) % 3 == 0, -0.0, 0.0),
        "one far above": torch.zeros(vocab).index_fill(0, torch.tensor([vocab // 2]), 300.0),
        "crowded": torch.where(torch.arange(vocab) % 512 < 16, 5.0 + ramp.float() / 64, -ramp),
    }
    for name, row in cases.items():
        print(f"[logprobs] {name}", flush=True)
        check(row.to(dtype).cuda().expand(rows, vocab).contiguous(), tokens, top)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 100.0, 6e4, 3e37, 3.3e38])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_far_values(gpu, dtype, scale):
    g = torch.Generator().manual_seed(3)
    x = ((torch.rand(5, 20000, generator=g) * 2 - 1) * scale).to(dtype).cuda()
    tokens = x.float().argmax(1)
    got = check(x, tokens, 4)
    assert bool(torch.isfinite(got.logprobs).all())
    check(-x.abs(), tokens, 4)
    check(x - x.amax(1, keepdim=True), tokens, 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_strides_and_alignment(gpu, dtype):
    base, _ = make(40, 9001, dtype, seed=5)
    for off in range(0, 9):
        for vocab in (8990, 4001, 300):
            x = base[:, off:off + vocab]
            tokens = torch.arange(40, device=gpu) % vocab
            check(x, tokens, 5)
    one = base[3:4, 1:2000]
    check(one, torch.tensor([7], device=gpu), 3)
    check(base[:, :2000][::2], torch.arange(20, device=gpu), 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(2, 40000), (1, 151936), (600, 9000)])
def test_a_nan_beside_masked_logits(gpu, dtype, rows, vocab):
    """One NaN makes every probability of its row NaN, those of masked tokens too, in any split of
    the row."""
    lowest = torch.finfo(dtype).min
    for masked in (-INF, lowest):
        x, _ = make(rows, vocab, dtype, seed=8)
        x[:, ::3] = masked
        x[:, vocab // 2 + 1 - (vocab // 2) % 3] = float("nan")
        for token in (0, 1, vocab // 3 * 3 - 3):
            got = check(x, torch.full((rows,), token, device=gpu), 4)
            assert bool(got.logprobs.isnan().all()) and bool(got.top_logprobs.isnan().all())


@pytest.mark.parametrize("rows,vocab", [(2, 40000), (1, 151936), (600, 9000), (700, 5000)])
@pytest.mark.parametrize("offset", [3e3, 6e4, 9e5, 1e6, -9e5])
def test_rows_far_from_zero(gpu, rows, vocab, offset):
    """fp32 logits some units apart around a far offset: only their differences count."""
    x, tokens = make(rows, vocab, torch.float32, seed=rows, scale=4.0)
    check(x + offset, tokens, 5)
    ramp = torch.linspace(-20, 20, vocab, device=gpu)  # every thread's reference moves all along
    check((ramp + offset).expand(rows, vocab).contiguous(), tokens, 5)


def test_rows_do_not_depend_on_their_number(gpu):
    """The alternatives of a row are the same in any batch; its sums as far as rounding goes."""
    x, tokens = make(700, 30000, torch.bfloat16, seed=9)
    whole = sampling.token_logprobs(x, tokens, top=20)
    for rows in (1, 2, 17, 300):
        part = sampling.token_logprobs(x[:rows], tokens[:rows], top=20)
        assert torch.equal(part.top_ids, whole.top_ids[:rows])
        torch.testing.assert_close(part.logprobs, whole.logprobs[:rows], rtol=0,
                                   atol=2 * tolerance(x[:rows]))


def test_same_bits_every_time(gpu):
    for rows, vocab in ((2, 151936), (600, 20000)):
        x, tokens = make(rows, vocab, torch.bfloat16, seed=2)
        first = sampling.token_logprobs(x, tokens, top=20)
        for _ in range(5):
            for a, b in zip(first, sampling.token_logprobs(x, tokens, top=20)):
                assert torch.equal(a, b)


def test_tokens_outside_the_vocabulary(gpu):
    x, _ = make(4, 3000, torch.float32)
    tokens = torch.tensor([-1, 3000, 5, 2 ** 40], device=gpu)
    got = check(x, tokens, 2)
    assert got.logprobs.isnan().tolist() == [True, True, False, True]
    assert bool(torch.isfinite(got.entropy).all())


def test_long_rows_past_4_gib(gpu):
    """Rows whose offsets pass 32 bits."""
    rows, vocab = 4, 40000
    base = torch.zeros(3 * 800_000_000 + vocab, dtype=torch.bfloat16, device=gpu)
    x = torch.as_strided(base, (rows, vocab), (800_000_000, 1))
    values, tokens = make(rows, vocab, torch.bfloat16, seed=4)
    x.copy_(values)
    check(x, tokens, 10)


def test_streams_and_graphs(gpu):
    for rows in (3, 600):
        x, tokens = make(rows, 20000, torch.bfloat16, seed=6)
        want = sampling.token_logprobs(x, tokens, top=8)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = sampling.token_logprobs(x, tokens, top=8)
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = sampling.token_logprobs(x, tokens, top=8)
        for seed in range(4):
            fresh, _ = make(rows, 20000, torch.bfloat16, seed=seed)
            x.copy_(fresh)
            graph.replay()
            want = sampling.token_logprobs(x, tokens, top=8)
            torch.cuda.synchronize()
            for a, b in zip(held, want):
                assert torch.equal(a, b)


def test_no_rows(gpu):
    got = sampling.token_logprobs(torch.empty(0, 100, device=gpu),
                                  torch.empty(0, dtype=torch.int64, device=gpu), top=3)
    assert got.logprobs.shape == (0,) and got.top_ids.shape == (0, 3)


def test_refusals(gpu):
    x, tokens = make(4, 100, torch.float32)
    bad = [
        lambda: sampling.token_logprobs(x.cpu(), tokens.cpu()),
        lambda: sampling.token_logprobs(x.double(), tokens),
        lambda: sampling.token_logprobs(x[0], tokens),
        lambda: sampling.token_logprobs(x.t(), tokens),
        lambda: sampling.token_logprobs(x[:, :0], tokens),
        lambda: sampling.token_logprobs(x.as_strided((4, 100), (50, 1)), tokens),
        lambda: sampling.token_logprobs(x, tokens.int()),
        lambda: sampling.token_logprobs(x, tokens[:3]),
        lambda: sampling.token_logprobs(x, tokens.cpu()),
        lambda: sampling.token_logprobs(x, tokens, top=-1),
        lambda: sampling.token_logprobs(x, tokens, top=65),
        lambda: sampling.token_logprobs(x[:, :5], tokens, top=6),
        lambda: sampling.token_logprobs(x.clone().requires_grad_(), tokens),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(NativeError):
            call()
            pytest.fail(str(i))
    native, cus = lib(), device_cus(gpu)
    assert native.mi355x_token_logprobs_workspace_bytes(1, 151936, 5, cus) > 0
    out = torch.empty(64, device=gpu)
    wide, one = make(1, 151936, torch.float32)
    err = native.mi355x_token_logprobs(wide.data_ptr(), 1, 151936, 151936, 2, one.data_ptr(), 0,
                                       out.data_ptr(), out.data_ptr(), None, None, None, 0, cus, 0)
    assert b"workspace" in err
