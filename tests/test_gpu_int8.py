"""Row quantisation and 8-bit projections (mi355x_quantize_rows, mi355x_linear_int8).

The quantised values are compared bit for bit with the 64-bit definition: with 16-bit rows the
quotient 127 x / max is never closer to a half than fp32 resolves. The int32 sums are exact, so a
product is off by three fp32 roundings (the sum's conversion, two scales: 3 x 2^-24) and one to the
output type (eps / 2); silu(y) u adds the exponential's and the quotient's, below 2^-20, times the
sensitivity of silu to y (|g silu'(g) / silu(g)| <= 1 + |g|).
"""
import pytest
import torch

from llm_infer_rust_amd import int8
from llm_infer_rust_amd._native import NativeError

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rows64(x):
    xd = x.double()
    top = xd.abs().amax(1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * xd / top), torch.zeros_like(xd)), top / 127


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t,k", [(1, 1), (3, 15), (7, 16), (5, 17), (130, 1000), (9, 1024),
                                 (4, 1040), (33, 4096), (2, 5001), (3, 12288), (2, 20000)])
def test_quantize_rows(gpu, dtype, t, k):
    x = (torch.randn(t, k, generator=gen(k)) * 3).to(dtype)
    values, scales = int8.quantize_rows(x.to(gpu))
    want, s = rows64(x)
    assert values.shape == (t, k) and values.dtype == torch.int8
    if dtype == torch.float32:  # 127 x is rounded: a step where the quotient is within that of a half
        frac = (127 * x.double() / x.double().abs().amax(1, keepdim=True)).abs() % 1
        clear = (frac - 0.5).abs() > 1e-4
        assert torch.equal(values.cpu()[clear].double(), want[clear])
        assert int((values.cpu().double() - want).abs().max()) <= 1
    else:
        assert torch.equal(values.cpu().double(), want)
    assert torch.allclose(scales.cpu().double(), s[:, 0], rtol=2.0 ** -23, atol=0)
    padded = values.as_strided((t, values.stride(0)), (values.stride(0), 1)) if t > 1 else values
    assert bool((padded[:, k:] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_quotient_of_a_16_bit_type(gpu, dtype):
    """Rows of one maximum and every smaller magnitude of its upper 16 binades: all ties."""
    bits = torch.arange(0, 2 ** 15, dtype=torch.int32).to(torch.int16)
    every = bits.view(dtype)
    every = every[every.isfinite()]
    rows = []
    for top in (1.0, 1.984375, 127.0, 254.0, 3.0, 96.0, 65280.0, 2.0 ** -14):
        m = torch.tensor(top).to(dtype)
        r = torch.where(every <= m, every, torch.zeros_like(every)).clone()
        r[0] = m
        rows.append(r)
    x = torch.stack(rows)
    x[:, 1::2] *= -1
    values, _ = int8.quantize_rows(x.to(gpu))
    assert torch.equal(values.cpu().double(), rows64(x)[0])


def test_rows_at_the_ends_of_the_range(gpu):
    big = torch.finfo(torch.bfloat16).max
    x = torch.zeros(7, 40, dtype=torch.bfloat16)
    x[1, 3], x[1, 4] = big, -big / 2
    x[2, 5], x[2, 6] = 2.0 ** -133, 0.0           # the smallest subnormal
    x[3, 0], x[3, 1] = 2.0 ** -126, 2.0 ** -127
    x[4, 9] = float("nan")
    x[5, 9], x[5, 10] = float("inf"), 1.0
    x[6] = -1.0
    values, scales = (a.cpu() for a in int8.quantize_rows(x.to(gpu)))
    assert values[0].count_nonzero() == 0 and scales[0] == 0
    assert values[1, 3] == 127 and values[1, 4] == -64 and scales[1] == big / 127
    assert values[2, 5] == 127 and values[2].count_nonzero() == 1 and scales[2] > 0
    assert values[3, 0] == 127 and values[3, 1] == 64
    assert bool(scales[4:6].isnan().all()) and values[4:6].count_nonzero() == 0
    assert bool((values[6] == -127).all())


def check(got, x, weight, silu):
    q, s = rows64(x.to(got.device))
    w, ws = weight.values.double(), weight.scales.double()
    y = q @ w.T * s * ws
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-38
    if silu:
        g, u = y.chunk(2, 1)
        want = g * torch.sigmoid(g) * u
        bound = want.abs() * (half + (3 * 2.0 ** -24) * (2 + g.abs()) + 2.0 ** -20) * 1.01 + tiny
        bound += (u.abs() + 1e-30) * 1e-36
    else:
        want = y
        bound = want.abs() * (half + 4 * 2.0 ** -24) * 1.01 + tiny
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


SHAPES = [(1, 6144, 4096), (1, 17, 33), (2, 64, 16), (3, 130, 100), (5, 1001, 1203), (16, 96, 512),
          (17, 64, 128), (24, 512, 4096), (63, 130, 200), (64, 64, 64), (65, 129, 1000),
          (200, 300, 136), (256, 4096, 128), (257, 260, 144), (300, 513, 129), (700, 1028, 1024),
          (1030, 258, 2064)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n,k", SHAPES)
@pytest.mark.parametrize("silu", [False, True])
def test_linear_int8(gpu, dtype, t, n, k, silu):
    n += n % 2 if silu else 0
    g = gen(t + n + k)
    x = torch.randn(t, k, generator=g).to(dtype)
    weight = int8.Int8Weight.quantize((torch.randn(n, k, generator=g) * k ** -0.5).to(gpu))
    check(int8.linear_int8(x.to(gpu), weight, silu_mul=silu), x, weight, silu)


# Every tile and split that is chosen by size: 64 x 64 in two and four parts of K, 128 x 128 whole, in
# parts and two a compute unit, 256 x 128, 256 x 256 (with a row tile of half the rows and with one of
# more), ragged in every dimension.
LARGE = [(1040, 258, 4110), (64, 4100, 4110), (1030, 2050, 65), (130, 8198, 4110), (1290, 6146, 65),
         (4100, 1028, 65), (1550, 6146, 65), (1630, 6146, 129), (2500, 4098, 640)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n,k", LARGE)
@pytest.mark.parametrize("silu", [False, True])
def test_linear_int8_of_many_rows(gpu, dtype, t, n, k, silu):
    g = torch.Generator(device=gpu).manual_seed(t + n + k)
    x = torch.randn(t, k, generator=g, device=gpu).to(dtype)
    weight = int8.Int8Weight.quantize(torch.randn(n, k, generator=g, device=gpu) * k ** -0.5)
    out = torch.full((t + 1, n), 7.0, dtype=dtype, device=gpu)
    width = n // 2 if silu else n
    got = int8.linear_int8(x, weight, out=out[:t, :width], silu_mul=silu)
    check(got, x, weight, silu)
    assert bool((out[t] == 7).all()) and bool((out[:, width:] == 7).all())


@pytest.mark.parametrize("t", [1, 40, 300])
def test_extreme_values_do_not_overflow(gpu, t):
    """K at the longest that is taken, every product 127 * 127: the int32 sum is 2,114,076,672."""
    k = int8.MAX_K
    x = torch.ones(t, k, dtype=torch.bfloat16, device=gpu)
    weight = int8.Int8Weight(torch.full((32, k), 127, dtype=torch.int8, device=gpu),
                             torch.full((32,), 2.0 ** -10, device=gpu))
    out = int8.linear_int8(x, weight)
    want = torch.tensor(127 * 2.0 ** -10 * k).to(torch.bfloat16)
    assert bool((out == want.to(gpu)).all())
    weight.values.fill_(-128)
    out = int8.linear_int8(x, weight)
    want = torch.tensor(-128 * 2.0 ** -10 * k).to(torch.bfloat16)
    assert bool((out == want.to(gpu)).all())


def test_strides_alignment_and_given_output(gpu):
    g = gen(5)
    for t in (3, 50, 400):
        wide = torch.randn(t, 300, generator=g).to(torch.float16).to(gpu)
        x = wide[:, 7:256]  # rows of 249 elements, 14 bytes off, stride 600 bytes
        values = torch.randint(-128, 128, (70, 300), generator=g, dtype=torch.int8).to(gpu)[:, 3:252]
        weight = int8.Int8Weight(values, torch.rand(70, generator=g).to(gpu))
        out = torch.full((t + 2, 75), 7.0, dtype=torch.float16, device=gpu)
        got = int8.linear_int8(x, weight, out=out[1:t + 1, 1:71])
        check(got, x, weight, False)
        assert bool((out[0] == 7).all()) and bool((out[-1] == 7).all())
        assert bool((out[:, 0] == 7).all()) and bool((out[:, 71:] == 7).all())
        assert torch.equal(got, int8.linear_int8(x.contiguous(), weight))


def test_non_finite_rows_stay_alone(gpu):
    g = gen(6)
    weight = int8.Int8Weight.quantize(torch.randn(96, 256, generator=g).to(gpu))
    for t in (6, 70, 500):
        x = torch.randn(t, 256, generator=g).to(torch.bfloat16)
        clean = int8.linear_int8(x.to(gpu), weight)
        x[1, 7], x[4, 200] = float("nan"), float("-inf")
        got = int8.linear_int8(x.to(gpu), weight)
        assert bool(got[1].isnan().all()) and bool(got[4].isnan().all())
        rest = [r for r in range(t) if r not in (1, 4)]
        assert torch.equal(got[rest], clean[rest])


def test_weights(gpu):
    w = torch.randn(3, 10, 37, generator=gen(1)).to(torch.bfloat16)
    weight = int8.Int8Weight.quantize(w.to(gpu))
    q, s = rows64(w.view(30, 37))
    assert torch.equal(weight.values.cpu().double().view(30, 37), q)
    assert weight.shape == (3, 10, 37) and weight.scales.shape == (3, 10)
    again = int8.Int8Weight(weight.values.contiguous(), weight.scales)
    assert torch.equal(again.values, weight.values) and again.row_stride == 128
    assert torch.allclose(weight.dequantize().cpu().double().view(30, 37), q * s, rtol=1e-6)


def test_weight_rows_of_whole_16_byte_words(gpu):
    """The C entry takes rows that end inside a 128-byte step too: K = 150 in rows of 160 bytes, the
    padding of any value."""
    from llm_infer_rust_amd._native import check as ok, lib
    g = gen(9)
    for t, n in ((2, 200), (9, 200), (70, 200), (600, 200), (1290, 6146), (1550, 6146)):
        x = torch.randn(t, 150, generator=g).to(torch.bfloat16).to(gpu)
        padded = torch.randint(-128, 128, (n, 160), generator=g, dtype=torch.int8).to(gpu)
        scales = torch.rand(n, generator=g).to(gpu)
        want = int8.linear_int8(x, int8.Int8Weight(padded[:, :150], scales))
        out = torch.empty_like(want)
        need = lib().mi355x_linear_int8_workspace_bytes(t, n, 150, 256)
        ws = torch.empty(need + 16, dtype=torch.uint8, device=gpu)
        ok(lib().mi355x_linear_int8(x.data_ptr(), 150, padded.data_ptr(), 160, scales.data_ptr(),
                                    out.data_ptr(), n, t, n, 150, False, ws.data_ptr(), need,
                                    256, 0, torch.cuda.current_stream().cuda_stream), "linear")
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_empty_batch_and_refusals(gpu):
    weight = int8.Int8Weight.quantize(torch.randn(8, 32, device=gpu))
    x = torch.randn(4, 32, device=gpu).to(torch.bfloat16)
    assert int8.linear_int8(x[:0], weight).shape == (0, 8)
    stack = int8.Int8Weight.quantize(torch.randn(2, 8, 32, device=gpu))
    odd = int8.Int8Weight.quantize(torch.randn(7, 32, device=gpu))
    for bad in (lambda: int8.linear_int8(x.float(), weight), lambda: int8.linear_int8(x.cpu(), weight),
                lambda: int8.linear_int8(x[:, :31], weight), lambda: int8.linear_int8(x, stack),
                lambda: int8.linear_int8(x, odd, silu_mul=True),
                lambda: int8.linear_int8(x.t().contiguous().t(), weight),
                lambda: int8.linear_int8(x, weight, out=torch.empty(4, 9, dtype=x.dtype, device=gpu)),
                lambda: int8.linear_int8(x, weight, out=x[:, :8]),
                lambda: int8.linear_int8(x, weight.values), lambda: int8.linear_int8(x[0], weight),
                lambda: int8.linear_int8(x.clone().requires_grad_(), weight),
                lambda: int8.quantize_rows(x.double()), lambda: int8.quantize_rows(x[:, :0]),
                lambda: int8.Int8Weight(weight.values, weight.scales[:7]),
                lambda: int8.Int8Weight(weight.values.cpu(), weight.scales.cpu()),
                lambda: int8.Int8Weight(torch.zeros(1, int8.MAX_K + 1, dtype=torch.int8, device=gpu),
                                        torch.ones(1, device=gpu))):
        with pytest.raises(NativeError):
            bad()


def test_rows_gigabytes_apart(gpu):
    wide = torch.empty((2 << 30) + 4096, dtype=torch.bfloat16, device=gpu)
    rows = wide.as_strided((3, 250), ((1 << 30) + 5, 1))
    rows.copy_(torch.randn(3, 250, generator=gen(3)))
    weight = int8.Int8Weight.quantize(torch.randn(66, 250, generator=gen(4)).to(gpu))
    assert torch.equal(int8.linear_int8(rows, weight), int8.linear_int8(rows.contiguous(), weight))
    values, scales = int8.quantize_rows(rows)
    want, want_scales = int8.quantize_rows(rows.contiguous())
    assert torch.equal(values, want) and torch.equal(scales, want_scales)


def test_given_output_of_no_rows_and_one(gpu):
    weight = int8.Int8Weight.quantize(torch.randn(8, 32, generator=gen(1)).to(gpu))
    x = torch.randn(1, 32, generator=gen(2)).to(torch.float16).to(gpu)
    out = torch.empty(0, 8, dtype=x.dtype, device=gpu)
    assert int8.linear_int8(x[:0], weight, out=out).shape == (0, 8)
    out = torch.full((1, 11), 7.0, dtype=x.dtype, device=gpu)
    assert torch.equal(int8.linear_int8(x, weight, out=out[:, 2:10]), int8.linear_int8(x, weight))
    assert out[0, :2].tolist() == [7.0] * 2 and float(out[0, 10]) == 7.0


def test_two_streams_at_once(gpu):
    """Calls with and without a split K, each stream's results as if it ran alone."""
    jobs = []
    for t, n, k in ((64, 4100, 4110), (1, 512, 1000), (40, 258, 300), (1550, 6146, 65)):
        x = torch.randn(t, k, generator=gen(t)).to(torch.bfloat16).to(gpu)
        weight = int8.Int8Weight.quantize(torch.randn(n, k, generator=gen(n)).to(gpu))
        jobs.append((x, weight, int8.linear_int8(x, weight)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for _ in range(10):
        for (x, weight, _), stream, mine in zip(jobs, streams, got):
            with torch.cuda.stream(stream):
                mine.append(int8.linear_int8(x, weight))
    torch.cuda.synchronize()
    for (_, _, want), mine in zip(jobs, got):
        assert all(torch.equal(want, out) for out in mine)


def test_captured_replays(gpu):
    calls = []
    for t in (1, 48, 300):
        weight = int8.Int8Weight.quantize(torch.randn(128, 96, generator=gen(t)).to(gpu))
        x = torch.randn(t, 96, generator=gen(t)).to(torch.bfloat16).to(gpu)
        int8.linear_int8(x, weight)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = int8.linear_int8(x, weight)
        calls.append((x, weight, graph, out))
    for r in range(3):
        for x, weight, graph, out in calls:
            x.copy_(torch.randn(x.shape, generator=gen(100 + r)).to(x.dtype))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, int8.linear_int8(x, weight))


def test_captured_replays_of_a_split_product(gpu):
    calls = []
    for seed in (1, 2):  # two graphs with workspaces of their own
        weight = int8.Int8Weight.quantize(torch.randn(4100, 4110, generator=gen(seed)).to(gpu))
        x = torch.randn(64, 4110, generator=gen(seed + 2)).to(torch.bfloat16).to(gpu)
        int8.linear_int8(x, weight, silu_mul=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = int8.linear_int8(x, weight, silu_mul=True)
        calls.append((x, weight, graph, out))
    for r in range(3):
        for x, _, graph, _ in calls:
            x.copy_(torch.randn(x.shape, generator=gen(r)).to(x.dtype))
            graph.replay()
        torch.cuda.synchronize()
        for x, weight, _, out in calls:
            assert torch.equal(out, int8.linear_int8(x, weight, silu_mul=True))
