"""The 8-bit and expert operators record no gradient: a call whose derivative would be wanted is
refused, whatever operand wants it."""
import pytest
import torch

from llm_infer_rust_amd import experts, int8
from llm_infer_rust_amd._native import NativeError

pytestmark = pytest.mark.gpu


def operands(gpu):
    g = torch.Generator(device=gpu).manual_seed(0)
    x = torch.randn(4, 64, generator=g, device=gpu).to(torch.bfloat16)
    logits = torch.randn(4, 3, generator=g, device=gpu)
    gu = (torch.randn(3, 64, 64, generator=g, device=gpu) * 0.1).to(torch.bfloat16)
    dn = (torch.randn(3, 64, 32, generator=g, device=gpu) * 0.1).to(torch.bfloat16)
    return x, logits, gu, dn


def calls(gpu, wants):
    """Every call with one operand passed through ``wants``, by name."""
    x, logits, gu, dn = operands(gpu)
    w, ids = experts.route_experts(logits, 2)
    gu8, dn8 = int8.Int8Weight.quantize(gu), int8.Int8Weight.quantize(dn)
    one = int8.Int8Weight.quantize(gu[0])

    def scaled(weight):
        return int8.Int8Weight(weight.values, wants(weight.scales))
    out = torch.empty_like(x)
    yield "quantize_rows", lambda: int8.quantize_rows(wants(x))
    yield "linear x", lambda: int8.linear_int8(wants(x), one)
    yield "linear scales", lambda: int8.linear_int8(x, scaled(one))
    yield "linear out", lambda: int8.linear_int8(x, one, out=wants(out))
    yield "logits", lambda: experts.route_experts(wants(logits), 2)
    yield "experts x", lambda: experts.expert_mlp(wants(x), ids, w, gu, dn)
    yield "experts weights", lambda: experts.expert_mlp(x, ids, wants(w), gu, dn)
    yield "experts gate_up", lambda: experts.expert_mlp(x, ids, w, wants(gu), dn)
    yield "experts down", lambda: experts.expert_mlp(x, ids, w, gu, wants(dn))
    yield "experts gate_up scales", lambda: experts.expert_mlp(x, ids, w, scaled(gu8), dn8)
    yield "experts down scales", lambda: experts.expert_mlp(x, ids, w, gu8, scaled(dn8))
    yield "experts out", lambda: experts.expert_mlp(x, ids, w, gu, dn, out=wants(out))


def test_gradients(gpu):
    for name, call in calls(gpu, lambda t: t.detach().clone().requires_grad_()):
        with pytest.raises(NativeError):
            call()
            pytest.fail(name)
        with torch.no_grad():
            call()
