"""8-bit products of rows near the ends of bf16's range: right wherever the result is in range.

The integer sum times the weight row's scale is of ordinary size, and the row's scale is multiplied
last, so nothing on the way leaves fp32's range before the result does. Bounds as for ordinary rows:
three fp32 roundings (4 x 2^-24) and one to bf16 (2^-8); the scale of a row is within 2^-23 of its
value, or half of fp32's smallest step where it is subnormal.
"""
import pytest
import torch

from llm_infer_rust_amd import experts, int8

pytestmark = pytest.mark.gpu


def rows64(x):
    top = x.abs().amax(-1, keepdim=True)
    return torch.round(127 * x / top), top / 127


def glu(y):
    g, u = y.chunk(2, -1)
    return g * torch.sigmoid(g) * u


# Vector math (1, 2 rows), the rows kernel, tiles of 64 x 64 whole and in parts of K, of 128 x 128 and
# of 256 x 256.
SHAPES = [(1, 64, 256), (2, 66, 1000), (9, 96, 512), (200, 300, 136), (64, 4100, 4110),
          (700, 1028, 1024), (1550, 6146, 65)]


@pytest.mark.parametrize("t,n,k", SHAPES)
@pytest.mark.parametrize("size,scale", [(2.0 ** 119, 2.0 ** -100), (2.0 ** -110, 2.0 ** 20)])
@pytest.mark.parametrize("silu", [False, True])
def test_linear_int8(gpu, t, n, k, size, scale, silu):
    g = torch.Generator(device=gpu).manual_seed(t + n + k)
    x = (torch.randn(t, k, generator=g, device=gpu) * size).to(torch.bfloat16)
    values = torch.randint(-127, 128, (n, k), generator=g, device=gpu, dtype=torch.int8)
    scales = torch.rand(n, generator=g, device=gpu) * scale + scale
    if silu:  # gates and ups of ordinary size
        scales *= 1.0 / (size * scale * 127 * k ** 0.5)
    weight = int8.Int8Weight(values, scales)
    got = int8.linear_int8(x, weight, silu_mul=silu).double()
    q, s = rows64(x.double())
    y = q @ values.double().T * scales.double() * s
    if silu:
        gate, u = y.chunk(2, 1)
        want = glu(y)
        rel = 2.0 ** -8 + 5 * 2.0 ** -24 * (2 + gate.abs()) + 2.0 ** -20
    else:
        want, rel = y, 2.0 ** -8 + 5 * 2.0 ** -24
    assert bool(want.isfinite().all())
    bound = want.abs() * rel * 1.01 + 1e-38
    err = (got - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("t,e,k", [(1, 4, 2), (40, 4, 2), (300, 4, 2), (3000, 3, 2)])
def test_expert_mlp(gpu, t, e, k):
    """Rows of 2^119 against gate_up scales of 2^-126: what rows of 2^19 against scales of 2^-26 give,
    bit for bit, as every number on the way is the same up to a power of two."""
    g = torch.Generator(device=gpu).manual_seed(t)
    h, i = 256, 136
    x = (torch.randn(t, h, generator=g, device=gpu) * 2.0 ** 119).to(torch.bfloat16)
    ids = torch.rand(t, e, generator=g, device=gpu).argsort(1)[:, :k].to(torch.int32).contiguous()
    w = torch.rand(t, k, generator=g, device=gpu)
    gv = torch.randint(-127, 128, (e, 2 * i, h), generator=g, device=gpu, dtype=torch.int8)
    gs = (torch.rand(e, 2 * i, generator=g, device=gpu) + 1.0) * 2.0 ** -126
    dn = int8.Int8Weight.quantize(torch.randn(e, h, i, generator=g, device=gpu))
    got = experts.expert_mlp(x, ids, w, int8.Int8Weight(gv, gs), dn)
    small = int8.Int8Weight(gv, gs * 2.0 ** 100)
    want = experts.expert_mlp((x.float() * 2.0 ** -100).to(torch.bfloat16), ids, w, small, dn)
    assert bool(got.isfinite().all()) and bool((got != 0).any())
    assert torch.equal(got, want)
