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


def test_tangents(gpu):
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        for name, call in calls(gpu, lambda t: fwad.make_dual(t, torch.ones_like(t))):
            with pytest.raises(NativeError):
                call()
                pytest.fail(name)
        for _, call in calls(gpu, lambda t: t):  # no operand carries one
            call()


def test_transforms(gpu):
    x, logits, gu, dn = operands(gpu)
    w, ids = experts.route_experts(logits, 2)
    one = int8.Int8Weight.quantize(gu[0])
    for f, arg in ((lambda t: int8.linear_int8(t, one), x), (lambda t: int8.quantize_rows(t)[1], x),
                   (lambda t: experts.route_experts(t, 2)[0], logits),
                   (lambda t: experts.expert_mlp(t, ids, w, gu, dn), x)):
        for transformed in (lambda a: torch.vmap(f)(torch.stack([a, a])),
                            lambda a: torch.func.jvp(f, (a,), (torch.ones_like(a),)),
                            lambda a: torch.func.vjp(f, a)):
            with pytest.raises(NativeError):
                transformed(arg)
        # operands that the transform does not touch
        got = torch.vmap(lambda s: s * f(arg).float())(torch.ones(2, device=gpu))
        assert torch.equal(got[1], f(arg).float())


def test_tracing(gpu):
    x, logits, gu, _ = operands(gpu)
    one = int8.Int8Weight.quantize(gu[0])
    for f, arg in ((lambda t: int8.linear_int8(t, one), x),
                   (lambda t: experts.route_experts(t, 2)[0], logits)):
        with pytest.raises(NativeError):
            torch.jit.trace(f, (arg,), check_trace=False)
