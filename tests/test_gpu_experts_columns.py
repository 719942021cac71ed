"""Expert MLPs whose output columns differ widely in size (an outlier channel of the down projection).

Slot outputs are fp32 until the one rounding at the end, so a small column is as exact beside a large
one as alone. The bound is each column's own, from the terms of its own sums. 16 bits: g and u are
fp32 sums of K products (K 2^-24 of the sum of magnitudes each), silu adds 2^-21 of its value,
silu(g) u is rounded to x's type (half = eps / 2 of every term of the second product), that product
and the sum over the slots are fp32 ((I + k + 8) 2^-24 of the sum of magnitudes), the result is
rounded once (half). 8 bits: the integer sums are exact, the scales and weights are fp32
(2^-18 of the slots' magnitudes is four times their roundings), and silu(g) u may fall on the other
side of a rounding border, a step of its scale for one element a row.
"""
import pytest
import torch

from llm_infer_rust_amd import experts, int8

pytestmark = pytest.mark.gpu


def glu(y):
    g, u = y.chunk(2, -1)
    return g * torch.sigmoid(g) * u


def quantized(rows):
    top = rows.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * rows / top), torch.zeros_like(rows)), top / 127


def problem(t, e, k, h, i, dtype, gpu):
    g = torch.Generator(device=gpu).manual_seed(t + h + i)
    x = torch.randn(t, h, generator=g, device=gpu).to(dtype)
    ids = torch.rand(t, e, generator=g, device=gpu).argsort(1)[:, :k].to(torch.int32).contiguous()
    w = torch.rand(t, k, generator=g, device=gpu)
    gu = (torch.randn(e, 2 * i, h, generator=g, device=gpu) * h ** -0.5).to(dtype)
    dn = torch.randn(e, h, i, generator=g, device=gpu) * i ** -0.5
    dn[:, 5::32] *= 3000.0
    return x, ids, w, gu, dn.to(dtype)


def bounds16(x, ids, w, gu, dn):
    half = torch.finfo(x.dtype).eps / 2
    x, w = x.double(), w.double()
    out, bound = torch.zeros_like(x), torch.zeros_like(x)
    inter = dn.size(2)
    for e in range(gu.size(0)):
        t, s = torch.nonzero(ids == e, as_tuple=True)
        a, b, ws = gu[e].double(), dn[e].double(), w[t, s, None]
        y = x[t] @ a.T
        act = glu(y)
        g, u = y.chunk(2, -1)
        mg, mu = (x[t].abs() @ a.abs().T * (x.size(1) * 2.0 ** -24)).chunk(2, -1)
        off = mg * 1.1 * u.abs() + mu * g.abs() + act.abs() * 2.0 ** -21
        terms = (act.abs() @ b.abs().T) * ws
        out.index_put_((t,), act @ b.T * ws, accumulate=True)
        bound.index_put_((t,), terms * (half * 1.01 + (inter + ids.size(1) + 8) * 2.0 ** -24)
                         + (off @ b.abs().T) * ws * 1.01, accumulate=True)
    return out, bound + out.abs() * half * 1.01 + 2.0 ** -24


def bounds8(x, ids, w, gu, dn):
    half = torch.finfo(x.dtype).eps / 2
    x, w = x.double(), w.double()
    q, s = quantized(x)
    out, bound = torch.zeros_like(x), torch.zeros_like(x)
    for e in range(gu.size(0)):
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        a, b = gu.values[e].double(), dn.values[e].double()
        qa, sa = quantized(glu(q[t] @ a.T * s[t] * gu.scales[e].double()))
        y = qa @ b.T * sa * dn.scales[e].double() * w[t, slot, None]
        one = sa * (b.abs().amax(1) * dn.scales[e].double())[None, :] * w[t, slot, None]
        out.index_put_((t,), y, accumulate=True)
        bound.index_put_((t,), y.abs() * 2.0 ** -18 + one, accumulate=True)
    return out, bound + out.abs() * half * 1.01 + 2.0 ** -24


# One by one; grouped in every tile of the down product, whole and in parts of K.
SHAPES = [(2, 8, 2, 264, 520), (40, 6, 2, 104, 2056), (90, 2, 2, 72, 4104), (77, 8, 2, 264, 520),
          (300, 7, 3, 328, 264), (1200, 2, 2, 2056, 72), (2100, 5, 2, 2056, 72),
          (3000, 3, 2, 2056, 128), (4100, 5, 2, 1032, 520)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k,h,i", SHAPES)
def test_small_columns_beside_large_ones(gpu, dtype, t, e, k, h, i):
    p = problem(t, e, k, h, i, dtype, gpu)
    out, bound = bounds16(*p)
    err = (experts.expert_mlp(*p).double() - out).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("t,e,k,h,i", SHAPES)
def test_small_columns_beside_large_ones_int8(gpu, t, e, k, h, i):
    x, ids, w, gu, dn = problem(t, e, k, h, i, torch.bfloat16, gpu)
    gu, dn = int8.Int8Weight.quantize(gu), int8.Int8Weight.quantize(dn)
    out, bound = bounds8(x, ids, w, gu, dn)
    err = (experts.expert_mlp(x, ids, w, gu, dn).double() - out).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


def test_fp16_activations_past_the_range(gpu):
    """Grouped, silu(g) u above 65,504 is inf in fp16 and its token's result not finite, and no other
    token's; alone the token keeps it in fp32."""
    x, ids, w, gu, _ = problem(40, 4, 2, 128, 64, torch.float16, gpu)
    dn = torch.full((4, 128, 64), 2.0 ** -6, dtype=torch.float16, device=gpu)
    clean = experts.expert_mlp(x, ids, w, gu, dn)
    x[7] *= 400.0
    act = glu(x[7].double() @ gu[int(ids[7, 0])].double().T)
    assert float(act.abs().max()) > 70000.0
    got = experts.expert_mlp(x, ids, w, gu, dn)
    rest = [t for t in range(40) if t != 7]
    assert not bool(got[7].isfinite().any()) and torch.equal(got[rest], clean[rest])
    one = (x[7:8], ids[7:8].contiguous(), w[7:8].contiguous(), gu, dn)
    out, bound = bounds16(*one)
    assert float(out.abs().max()) < 65504.0
    err = (experts.expert_mlp(*one).double() - out).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
