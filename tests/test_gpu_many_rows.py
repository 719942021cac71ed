"""Row passes over more rows than one grid has threads for: every row as in a call of its own."""
import pytest
import torch

from llm_infer_rust_amd import experts, int8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,width", [((1 << 24) + 5, 1040), ((1 << 26) + 5, 20)])
def test_quantize_rows(gpu, rows, width):
    free, _ = torch.cuda.mem_get_info(gpu)
    if free < 80 << 30:
        pytest.skip("needs 80 GB")
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=gpu)
    ends = [slice(0, 9), slice((1 << 23) - 4, (1 << 23) + 4), slice((1 << 24) - 4, (1 << 24) + 4),
            slice(rows - 9, rows)]
    g = torch.Generator(device=gpu).manual_seed(0)
    for s in ends:
        x[s] = torch.randn(x[s].shape, generator=g, device=gpu).to(x.dtype)
    values, scales = int8.quantize_rows(x)
    for s in ends:
        want, want_scales = int8.quantize_rows(x[s])
        assert torch.equal(values[s], want) and torch.equal(scales[s], want_scales)
        assert bool((want_scales > 0).all())
    assert scales[(1 << 22):(1 << 22) + 1000].count_nonzero() == 0


def test_route_experts(gpu):
    tokens = (1 << 26) + 5
    logits = torch.zeros(tokens, 4, dtype=torch.bfloat16, device=gpu)
    ends = [slice(0, 9), slice((1 << 23) - 4, (1 << 23) + 4), slice(tokens - 9, tokens)]
    g = torch.Generator(device=gpu).manual_seed(0)
    for s in ends:
        logits[s] = torch.randn(logits[s].shape, generator=g, device=gpu).to(logits.dtype)
    weights, ids = experts.route_experts(logits, 2)
    for s in ends:
        want, want_ids = experts.route_experts(logits[s], 2)
        assert torch.equal(weights[s], want) and torch.equal(ids[s], want_ids)
    middle = slice(1 << 22, (1 << 22) + 1000)
    assert bool((weights[middle] == 0.5).all()) and ids[middle].tolist() == [[0, 1]] * 1000
