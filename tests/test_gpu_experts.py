"""Routing and expert MLPs (mi355x_route_experts, mi355x_expert_mlp) against 64-bit formulas.

Bounds. Routing: ids are exact (selection is on the logits themselves); the weights are two fp32
exponentials and a quotient, 2^-20 relative. 16-bit experts: the products sum in fp32 (K 2^-24 of the
sum of magnitudes), silu(g) u is rounded to x's type (half a step, eps / 2 of every term of the
second product), and the sum over the slots (eps / 2). The weighted slot outputs are fp32; the bounds
leave room for 16-bit mantissas under a power of two for every 32 columns (``block_errors``: half a
unit, 2^-15 of the largest of the 32, or a unit for a value within half a unit of the top). Bounds of
every column's own are in test_gpu_experts_columns.py. 8-bit experts: integer sums are exact;
silu(g) u differs by fp32 rounding from the 64-bit value and may fall on the other side of a rounding
border, a step of its scale for one element a row.
"""
import pytest
import torch

from llm_infer_rust_amd import experts, int8
from llm_infer_rust_amd._native import NativeError

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ routing
def route64(logits, top_k, normalize):
    z = logits.double()
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top_k]
    p = torch.softmax(z, 1)
    w = p.gather(1, order)
    return (w / w.sum(1, keepdim=True) if normalize else w), order


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t,e,k", [(1, 8, 2), (5, 1, 1), (3, 64, 64), (130, 65, 6), (257, 128, 8),
                                   (9, 1000, 12), (2, 1024, 64), (4, 300, 7)])
@pytest.mark.parametrize("normalize", [False, True])
def test_route(gpu, dtype, t, e, k, normalize):
    logits = (torch.randn(t, e, generator=gen(t + e)) * 2).to(dtype)
    w, ids = experts.route_experts(logits.to(gpu), k, normalize=normalize)
    want_w, want_ids = route64(logits, k, normalize)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(ids.cpu().long(), want_ids)  # ties of 16-bit logits included
    assert torch.allclose(w.double().cpu(), want_w, rtol=2.0 ** -20, atol=1e-30)


def test_route_ties_and_strides(gpu):
    wide = torch.zeros(6, 40, dtype=torch.bfloat16, device=gpu)
    wide[:, 3] = 1.0
    wide[2, 20] = 1.0
    wide[4, :] = -0.0
    wide[4, 7] = 0.0  # equal to -0
    w, ids = experts.route_experts(wide[:, 2:30], 3)
    assert ids[0].tolist() == [1, 0, 2] and ids[2].tolist() == [1, 18, 0]
    assert ids[4].tolist() == [0, 1, 2]
    assert torch.allclose(w.sum(1), torch.ones(6, device=gpu))


def test_route_masked_rows(gpu):
    lowest = torch.finfo(torch.float32).min
    logits = torch.randn(6, 16, generator=gen(3))
    logits[0] = float("-inf")                       # nothing left
    logits[1, 2:] = float("-inf")                   # fewer left than top_k
    logits[2, 4:] = lowest                          # masked with the type's lowest value
    logits[3, 5] = float("nan")
    logits[4, 9] = float("inf")
    w, ids = (a.cpu() for a in experts.route_experts(logits.to(gpu), 4))
    assert ids[0].tolist() == [0, 1, 2, 3] and w[0].tolist() == [0.0] * 4
    assert set(ids[1, :2].tolist()) == {0, 1} and ids[1, 2:].tolist() == [2, 3]
    assert w[1, 2:].tolist() == [0.0, 0.0] and abs(float(w[1].sum()) - 1) < 1e-6
    assert sorted(ids[2].tolist()) == [0, 1, 2, 3]
    assert ids[3, 0] == 5 and bool(w[3].isnan().all())
    assert ids[4, 0] == 9 and bool(w[4].isnan().all())
    want, order = route64(logits[5:], 4, True)
    assert torch.equal(ids[5:].long(), order)
    allmin = torch.full((1, 8), lowest, device=gpu)
    w, ids = experts.route_experts(allmin, 2)
    assert ids.tolist() == [[0, 1]] and w.tolist() == [[0.5, 0.5]]


def test_route_refusals(gpu):
    x = torch.zeros(2, 8, device=gpu)
    assert experts.route_experts(x[:0], 2)[0].shape == (0, 2)
    for bad in (lambda: experts.route_experts(x, 0), lambda: experts.route_experts(x, 9),
                lambda: experts.route_experts(x.double(), 2),
                lambda: experts.route_experts(x.t(), 2),
                lambda: experts.route_experts(x.cpu(), 2),
                lambda: experts.route_experts(torch.zeros(1, 1025, device=gpu), 2),
                lambda: experts.route_experts(x.clone().requires_grad_(), 2)):
        with pytest.raises(NativeError):
            bad()


# ------------------------------------------------------------------ expert MLPs
def problem(t, e, k, h, i, dtype, seed, skew=1.0):
    g = gen(seed)
    x = torch.randn(t, h, generator=g).to(dtype)
    logits = torch.randn(t, e, generator=g) + skew * torch.randn(e, generator=g)
    w, ids = route64(logits, k, True)
    gu = (torch.randn(e, 2 * i, h, generator=g) * h ** -0.5).to(dtype)
    dn = (torch.randn(e, h, i, generator=g) * i ** -0.5).to(dtype)
    return x, ids.to(torch.int32), w.float(), gu, dn


def glu(y):
    g, u = y.chunk(2, -1)
    return g * torch.sigmoid(g) * u


def block_errors(y):
    """What holding rows of slot outputs in 16 bits under a scale for 32 columns costs at most: half a
    unit, 2^-15 of a block's largest; a unit where a value is within half a unit of the top."""
    n, h = y.shape
    padded = torch.nn.functional.pad(y.abs(), (0, -h % 32)).view(n, -1, 32)
    top = padded.amax(2, keepdim=True)
    units = torch.where(padded >= top * (1 - 2.0 ** -14), 2.0 ** -14, 2.0 ** -15) * top
    return units.view(n, -1)[:, :h] * 1.01


def reference(x, ids, weights, gu, dn, gpu):
    """The 64-bit result and the bound of the rounding errors of the 16-bit path (see the top)."""
    x, weights, gu, dn = (a.to(gpu).double() for a in (x, weights, gu, dn))
    ids = ids.to(gpu)
    out, terms, first, blocks = (torch.zeros_like(x) for _ in range(4))
    for e in range(gu.size(0)):
        t, s = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        act = glu(x[t] @ gu[e].T)
        # sums of fp32 products: g and u each off by K 2^-24 of the sum of magnitudes
        mag = x[t].abs() @ gu[e].abs().T * (x.size(1) * 2.0 ** -24)
        g, u = (x[t] @ gu[e].T).chunk(2, -1)
        mg, mu = mag.chunk(2, -1)
        off = mg * 1.1 * u.abs() + mu * (g.abs()) + act.abs() * 2.0 ** -21
        w = weights[t, s, None]
        y = act @ dn[e].T * w
        out.index_put_((t,), y, accumulate=True)
        blocks.index_put_((t,), block_errors(y), accumulate=True)
        terms.index_put_((t,), (act.abs() @ dn[e].abs().T) * w.abs(), accumulate=True)
        first.index_put_((t,), (off @ dn[e].abs().T) * w.abs(), accumulate=True)
    return out, terms, first + blocks


def check16(got, x, ids, weights, gu, dn, gpu):
    out, terms, first = reference(x, ids, weights, gu, dn, gpu)
    half = torch.finfo(got.dtype).eps / 2
    inter = dn.size(2)
    # act's rounding and the second sum on every term, the slots' codes, the last rounding, subnormal
    # fp16 steps; the fp32 sum over the slots is far below the codes
    bound = (terms * (half * 1.01 + (inter + 8) * 2.0 ** -24) + out.abs() * half * 1.01
             + first * 1.01 + 2.0 ** -24)
    err = (got.double() - out).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    # and closer on the whole: two independent roundings, each half / sqrt(3) of a value at most
    assert float(err.norm() / (out.norm() + 1e-30)) < 1.5 * half


SHAPES = [
    (1, 8, 2, 64, 64), (1, 4, 4, 8, 8), (2, 16, 8, 136, 72), (3, 5, 1, 1000, 24),
    (16, 8, 2, 256, 128), (17, 128, 8, 128, 64), (40, 3, 2, 512, 200), (77, 8, 2, 264, 520),
    (200, 4, 2, 192, 320), (300, 7, 3, 328, 264), (1200, 5, 2, 136, 136),
    (40, 6, 2, 104, 2056), (90, 2, 2, 72, 4104),  # down cut along K, in four parts (8 bits: two and four)
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k,h,i", SHAPES)
def test_expert_mlp(gpu, dtype, t, e, k, h, i):
    p = problem(t, e, k, h, i, dtype, t * 7 + e)
    got = experts.expert_mlp(*(a.to(gpu) for a in p))
    check16(got, *p, gpu)


# The larger tiles, chosen by size (test_gpu_product_forms.py says which): 128 x 128 for both products,
# 256 x 256 (groups of rows that end in a half tile and in a whole one) for either, with K in whole
# 128-byte steps and not; the most slots a token, one expert, and more experts than slots.
LARGE = [(1200, 2, 2, 72, 1032), (1200, 2, 2, 2056, 72), (600, 16, 2, 72, 1032), (600, 16, 2, 2056, 72),
         (2500, 6, 2, 1032, 520), (3000, 3, 2, 512, 1024), (1, 64, 64, 64, 64), (5, 64, 64, 72, 40),
         (33, 1, 1, 128, 64), (700, 1, 1, 128, 64), (50, 1024, 3, 64, 32),
         (2100, 5, 2, 2056, 72), (2100, 5, 2, 72, 1032), (4100, 5, 2, 1032, 520),
         (3000, 3, 2, 2056, 128), (1000, 8, 1, 72, 1544)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k,h,i", LARGE)
def test_expert_mlp_of_many_rows(gpu, dtype, t, e, k, h, i):
    p = problem(t, e, k, h, i, dtype, t * 7 + e)
    out = torch.full((t + 1, h + 8), 7.0, dtype=dtype, device=gpu)
    got = experts.expert_mlp(*(a.to(gpu) for a in p), out=out[:t, :h])
    check16(got, *p, gpu)
    assert bool((out[t] == 7).all()) and bool((out[:, h:] == 7).all())


@pytest.mark.parametrize("t,e,k", [(6, 12, 4), (300, 16, 4), (3000, 8, 4)])
def test_ids_outside_add_nothing(gpu, t, e, k):
    x, ids, w, gu, dn = problem(t, e, k, 128, 64, torch.bfloat16, t)
    ids[:, 1] = -1
    ids[::3, :] = e + 5             # nothing left of these rows
    ids[1, 2] = 2 ** 31 - 1
    w[::3, :] = float("nan")        # weights of slots that take no part are never read
    got = experts.expert_mlp(*(a.to(gpu) for a in (x, ids, w, gu, dn)))
    assert bool((got[::3] == 0).all())
    check16(got, x, ids, torch.where((ids >= 0) & (ids < e), w, torch.zeros_like(w)), gu, dn, gpu)


def test_one_expert_takes_all_and_repeats(gpu):
    for t in (9, 700):
        x, ids, w, gu, dn = problem(t, 6, 2, 128, 64, torch.float16, t)
        ids[:] = 4                  # the same expert twice in every row
        got = experts.expert_mlp(*(a.to(gpu) for a in (x, ids, w, gu, dn)))
        check16(got, x, ids, w, gu, dn, gpu)


def test_non_finite_rows_stay_alone(gpu):
    for t in (5, 90, 900):
        x, ids, w, gu, dn = problem(t, 4, 2, 128, 64, torch.bfloat16, t)
        clean = experts.expert_mlp(*(a.to(gpu) for a in (x, ids, w, gu, dn)))
        x[3, 5] = float("nan")
        x[1, 0] = float("inf")
        for i8 in (False, True):
            mats = (gu.to(gpu), dn.to(gpu))
            if i8:
                mats = tuple(int8.Int8Weight.quantize(m) for m in mats)
            got = experts.expert_mlp(x.to(gpu), ids.to(gpu), w.to(gpu), *mats)
            assert bool(got[3].isnan().all()) and not bool(got[1].isfinite().any())
            rest = [r for r in range(t) if r not in (1, 3)]
            assert bool(got[rest].isfinite().all())
            if not i8:
                assert torch.equal(got[rest], clean[rest])


def test_strided_rows_and_given_output(gpu):
    for t in (7, 150):
        x, ids, w, gu, dn = (a.to(gpu) for a in problem(t, 6, 2, 128, 64, torch.bfloat16, t))
        want = experts.expert_mlp(x, ids, w, gu, dn)
        wide = torch.zeros(t, 200, dtype=x.dtype, device=gpu)
        wide[:, 16:144] = x
        out = torch.full((t + 2, 131), 7.0, dtype=x.dtype, device=gpu)
        got = experts.expert_mlp(wide[:, 16:144], ids, w, gu, dn, out=out[1:t + 1, 1:129])
        assert torch.equal(got, want) and got.data_ptr() == out[1:, 1:].data_ptr()
        assert bool((out[0] == 7).all()) and bool((out[-1] == 7).all())
        assert bool((out[:, 0] == 7).all()) and bool((out[:, 129:] == 7).all())


def quantized(rows):
    top = rows.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * rows / top), torch.zeros_like(rows)), top / 127


def check8(got, x, ids, weights, gu, dn, gpu):
    """gu, dn: Int8Weight. 64-bit integers throughout but for the two quantisations."""
    xd, wd = x.to(gpu).double(), weights.to(gpu).double()
    ids = ids.to(gpu)
    q, s = quantized(xd)
    out, step, mag = (torch.zeros_like(xd) for _ in range(3))
    for e in range(gu.size(0)):
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        act = glu(q[t] @ gu.values[e].double().T * s[t] * gu.scales[e].double())
        qa, sa = quantized(act)
        w = wd[t, slot, None]
        y = qa @ dn.values[e].double().T * sa * dn.scales[e].double()
        out.index_put_((t,), y * w, accumulate=True)
        mag.index_put_((t,), (y * w).abs(), accumulate=True)
        step.index_put_((t,), block_errors(y * w), accumulate=True)
        # one element of a slot's row on the other side of a rounding border
        one = sa * (dn.values[e].double().abs().amax(1) * dn.scales[e].double())[None, :]
        step.index_put_((t,), one * w.abs(), accumulate=True)
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - out).abs()
    bound = step + out.abs() * half * 1.01 + mag * 2.0 ** -18 + 2.0 ** -24
    assert bool((err <= bound).all()), float((err / bound).max())
    assert float(err.norm() / (out.norm() + 1e-30)) < 2 * half


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k,h,i", SHAPES + [(1, 4, 2, 33, 17), (19, 5, 2, 131, 77),
                                                (90, 3, 2, 200, 1), (700, 6, 2, 257, 99)])
def test_expert_mlp_int8(gpu, dtype, t, e, k, h, i):
    x, ids, w, gu, dn = problem(t, e, k, h, i, dtype, t * 5 + e)
    gu8, dn8 = (int8.Int8Weight.quantize(m.to(gpu)) for m in (gu, dn))
    got = experts.expert_mlp(x.to(gpu), ids.to(gpu), w.to(gpu), gu8, dn8)
    check8(got, x, ids, w, gu8, dn8, gpu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k,h,i", LARGE + [(1200, 2, 2, 2055, 67), (600, 16, 2, 71, 1033),
                                                (600, 16, 2, 2055, 131), (2100, 5, 2, 2055, 67),
                                                (2100, 5, 2, 71, 1033)])
def test_expert_mlp_int8_of_many_rows(gpu, dtype, t, e, k, h, i):
    x, ids, w, gu, dn = problem(t, e, k, h, i, dtype, t * 5 + e)
    gu8, dn8 = (int8.Int8Weight.quantize(m.to(gpu)) for m in (gu, dn))
    out = torch.full((t + 1, h + 8), 7.0, dtype=dtype, device=gpu)
    got = experts.expert_mlp(x.to(gpu), ids.to(gpu), w.to(gpu), gu8, dn8, out=out[:t, :h])
    check8(got, x, ids, w, gu8, dn8, gpu)
    assert bool((out[t] == 7).all()) and bool((out[:, h:] == 7).all())


@pytest.mark.parametrize("t", [1, 40, 600])
def test_weights_of_more_than_four_gib(gpu, t):
    """Experts 0 and 19 of 20 whose matrices start up to 5 GB behind the first."""
    h, i = 8192, 8192
    gu = torch.zeros(20, 2 * i, h, dtype=torch.bfloat16, device=gpu)
    dn = torch.zeros(20, h, i, dtype=torch.bfloat16, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(t)
    for e in (0, 19):
        gu[e].normal_(0, h ** -0.5, generator=g)
        dn[e].normal_(0, i ** -0.5, generator=g)
    x = torch.randn(t, h, generator=g, device=gpu).to(torch.bfloat16)
    ids = torch.randint(0, 2, (t, 2), generator=g, device=gpu, dtype=torch.int32)
    w = torch.rand(t, 2, generator=g, device=gpu)
    got = experts.expert_mlp(x, ids * 19, w, gu, dn)
    check16(got, x, ids, w, gu[::19], dn[::19], gpu)


@pytest.mark.parametrize("h,i", [(64, 17408), (17408, 64)])
@pytest.mark.parametrize("i8", [False, True])
def test_slots_of_more_than_four_gib(gpu, h, i, i8):
    """65,536 tokens of two slots: 131,072 rows of 34 KB between the products, or behind them. The
    tokens that are checked have their slots at both ends of the grouped order."""
    t = 65536
    g = torch.Generator(device=gpu).manual_seed(h)
    x = torch.randn(t, h, generator=g, device=gpu).to(torch.bfloat16)
    gu = (torch.randn(2, 2 * i, h, generator=g, device=gpu) * h ** -0.5).to(torch.bfloat16)
    dn = (torch.randn(2, h, i, generator=g, device=gpu) * i ** -0.5).to(torch.bfloat16)
    ids = torch.tensor([0, 1], dtype=torch.int32, device=gpu).repeat(t, 1)
    w = torch.rand(t, 2, generator=g, device=gpu)
    if i8:
        gu, dn = int8.Int8Weight.quantize(gu), int8.Int8Weight.quantize(dn)
    got = experts.expert_mlp(x, ids, w, gu, dn)
    some = torch.tensor([0, 1, 777, t // 2, t - 300, t - 2, t - 1], device=gpu)
    (check8 if i8 else check16)(got[some], x[some], ids[some], w[some], gu, dn, gpu)


@pytest.mark.parametrize("k", [2, 20])
def test_rows_gigabytes_apart(gpu, k):
    x, ids, w, gu, dn = (a.to(gpu) for a in problem(3, 32, k, 128, 64, torch.bfloat16, k))
    wide = torch.empty((2 << 30) + 4096, dtype=torch.bfloat16, device=gpu)
    rows = wide.as_strided((3, 128), ((1 << 30) + 8, 1))
    rows.copy_(x)
    check16(experts.expert_mlp(rows, ids, w, gu, dn), x, ids, w, gu, dn, gpu)
    gu8, dn8 = int8.Int8Weight.quantize(gu), int8.Int8Weight.quantize(dn)
    check8(experts.expert_mlp(rows, ids, w, gu8, dn8), x, ids, w, gu8, dn8, gpu)
    weights, chosen = experts.route_experts(rows, 5)
    want, want_ids = experts.route_experts(x, 5)
    assert torch.equal(weights, want) and torch.equal(chosen, want_ids)


@pytest.mark.parametrize("t", [3, 60, 1200, 3100])
def test_infinite_weights(gpu, t):
    """An infinity in `down` reaches its column and no other; the 32 columns that share its scale are
    then held in bf16, half a step of 2^-9 for each slot of the expert."""
    x, ids, w, gu, dn = problem(t, 2, 2, 2056, 72, torch.bfloat16, t)
    dn[1, 40, 3] = float("inf")
    got = experts.expert_mlp(*(a.to(gpu) for a in (x, ids, w, gu, dn)))
    assert not bool(got[:, 40].isfinite().any())
    rest = [c for c in range(2056) if c != 40]
    assert bool(got[:, rest].isfinite().all())
    dn[1, 40, 3] = 0.0
    out, terms, first = reference(x, ids, w, gu, dn, gpu)
    half = 2.0 ** -8
    bound = terms * (half * 1.01 + 80 * 2.0 ** -24) + out.abs() * half * 1.01 + first * 1.01
    bound[:, 32:64] += terms[:, 32:64] * 2.0 ** -8
    err = (got.double() - out).abs()[:, rest]
    assert bool((err <= bound[:, rest]).all()), float((err / bound[:, rest]).max())


def test_two_streams_at_once(gpu):
    jobs = []
    for t, h, i, i8 in ((2, 128, 64, False), (40, 104, 2056, False), (90, 128, 64, True),
                        (600, 2056, 72, False), (1200, 72, 1032, True),
                        (4100, 1032, 520, False), (3001, 2056, 72, True)):
        x, ids, w, gu, dn = (a.to(gpu) for a in problem(t, 4, 2, h, i, torch.bfloat16, t))
        if i8:
            gu, dn = int8.Int8Weight.quantize(gu), int8.Int8Weight.quantize(dn)
        args = (x, ids, w, gu, dn)
        jobs.append((args, experts.expert_mlp(*args)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for _ in range(10):
        for (args, _), stream, mine in zip(jobs, streams, got):
            with torch.cuda.stream(stream):
                mine.append(experts.expert_mlp(*args))
    torch.cuda.synchronize()
    for (_, want), mine in zip(jobs, got):
        assert all(torch.equal(want, out) for out in mine)


def test_more_slots_than_a_pass_takes(gpu):
    t, k = 9000, 16  # 144,000 slots: two passes
    x, ids, w, gu, dn = problem(t, 32, k, 64, 64, torch.bfloat16, 1)
    got = experts.expert_mlp(*(a.to(gpu) for a in (x, ids, w, gu, dn)))
    check16(got, x, ids, w, gu, dn, gpu)


def test_empty_batch_and_refusals(gpu):
    x, ids, w, gu, dn = (a.to(gpu) for a in problem(8, 4, 2, 64, 32, torch.bfloat16, 0))
    assert experts.expert_mlp(x[:0], ids[:0], w[:0], gu, dn).shape == (0, 64)
    gu8 = int8.Int8Weight.quantize(gu)
    wide = torch.zeros(8, 100, dtype=x.dtype, device=gpu)
    for args in ((x, ids.long(), w, gu, dn), (x, ids, w.half(), gu, dn), (x, ids[:4], w, gu, dn),
                 (x.float(), ids, w, gu, dn), (x, ids, w, gu.half(), dn), (x, ids, w, gu, gu),
                 (x, ids, w, gu8, dn), (x.cpu(), ids, w, gu, dn), (x, ids.cpu(), w, gu, dn),
                 (wide[:, 1:65], ids, w, gu, dn), (wide[:, :64].t().contiguous().t(), ids, w, gu, dn),
                 (x[:, :60], ids, w, gu[:, :, :60].contiguous(), dn[:, :60].contiguous()),
                 (x, ids[:, :0], w[:, :0], gu, dn), (x.clone().requires_grad_(), ids, w, gu, dn)):
        with pytest.raises(NativeError):
            experts.expert_mlp(*args)
    none = torch.empty(0, 64, dtype=x.dtype, device=gpu)
    assert experts.expert_mlp(x[:0], ids[:0], w[:0], gu, dn, out=none).shape == (0, 64)
    with pytest.raises(NativeError):
        experts.expert_mlp(x, ids, w, gu, dn, out=x)
    with pytest.raises(NativeError):
        experts.expert_mlp(x, ids, w, gu, dn, out=torch.empty(8, 63, dtype=x.dtype, device=gpu))


def test_captured_replays_and_streams(gpu):
    """Two graphs of different batches replayed in turn, with eager calls of other sizes between."""
    calls = []
    for t, i8 in ((3, False), (64, True), (500, False)):
        x, ids, w, gu, dn = (a.to(gpu) for a in problem(t, 8, 2, 128, 64, torch.bfloat16, t))
        if i8:
            gu, dn = int8.Int8Weight.quantize(gu), int8.Int8Weight.quantize(dn)
        logits = torch.randn(t, 8, generator=gen(t)).to(gpu)

        def layer(x=x, logits=logits, gu=gu, dn=dn):
            weights, chosen = experts.route_experts(logits, 2)
            return experts.expert_mlp(x, chosen, weights, gu, dn)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            warm = layer()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(warm, layer())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer()
        calls.append((x, logits, layer, graph, out))
    for r in range(3):
        for x, logits, layer, graph, out in calls:
            x.copy_(torch.randn(x.shape, generator=gen(r)).to(x.dtype))
            logits.copy_(torch.randn(logits.shape, generator=gen(r + 9)))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, layer())
