"""Captured calls of the 8-bit and expert products in the forms that many rows take: slots counted in
several chunks, several passes, the largest tiles, parts of K. Every replay equals the eager call on
the same inputs, with eager calls of other sizes between the replays."""
import pytest
import torch

from llm_infer_rust_amd import experts, int8

pytestmark = pytest.mark.gpu


def replays(gpu, x, call):
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    g = torch.Generator(device=gpu).manual_seed(5)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device=gpu).to(x.dtype))
        graph.replay()
        torch.cuda.synchronize()
        yield out, call()


# (tokens, experts, experts a token, hidden, inter): several chunks of slots and large tiles, two
# passes, parts of K, one by one.
@pytest.mark.parametrize("t,e,k,h,i", [(4100, 5, 2, 1032, 520), (9000, 32, 16, 64, 64),
                                       (90, 2, 2, 72, 4104), (2, 8, 2, 264, 520)])
@pytest.mark.parametrize("i8", [False, True])
def test_experts(gpu, t, e, k, h, i, i8):
    g = torch.Generator(device=gpu).manual_seed(t)
    x = torch.randn(t, h, generator=g, device=gpu).to(torch.bfloat16)
    router = torch.randn(e, h, generator=g, device=gpu).to(torch.bfloat16)
    gu = (torch.randn(e, 2 * i, h, generator=g, device=gpu) * h ** -0.5).to(torch.bfloat16)
    dn = (torch.randn(e, h, i, generator=g, device=gpu) * i ** -0.5).to(torch.bfloat16)
    if i8:
        gu, dn = int8.Int8Weight.quantize(gu), int8.Int8Weight.quantize(dn)
    other = torch.randn(33, h, generator=g, device=gpu).to(torch.bfloat16)

    def layer(rows=x):
        # the logits by elementary steps: the router's own product is not what is captured here
        logits = (rows[:, None, :8].float() * router[None, :, :8].float()).sum(2)
        weights, ids = experts.route_experts(logits, k)
        return experts.expert_mlp(rows, ids, weights, gu, dn)
    for out, eager in replays(gpu, x, layer):
        layer(other)
        assert torch.equal(out, eager) and bool(eager.isfinite().all())


@pytest.mark.parametrize("t,n,k", [(1, 130, 12288), (9, 8200, 5003), (24, 512, 4096),
                                   (1030, 2050, 65), (1550, 6146, 65)])
@pytest.mark.parametrize("silu", [False, True])
def test_linear_int8(gpu, t, n, k, silu):
    g = torch.Generator(device=gpu).manual_seed(t)
    x = torch.randn(t, k, generator=g, device=gpu).to(torch.float16)
    weight = int8.Int8Weight.quantize(torch.randn(n, k, generator=g, device=gpu) * k ** -0.5)
    other = torch.randn(33, k, generator=g, device=gpu).to(torch.float16)
    for out, eager in replays(gpu, x, lambda: int8.linear_int8(x, weight, silu_mul=silu)):
        int8.linear_int8(other, weight, silu_mul=silu)
        assert torch.equal(out, eager)
