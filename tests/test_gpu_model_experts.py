"""Models with layers of experts and with 8-bit matrices, and the serving engine over them.

The reference forward is plain torch in 64 bits over the whole sequence. It takes the experts that
the model chose (a bf16 router logit may order two experts otherwise than the exact one) with its
own weights for them, and checks that every choice is among the largest logits within bf16's error.

Bounds: bf16 activations are rounded about ten times a layer, each 2^-9 relative and independent, so
two layers' logits are off by some sqrt(20) 2^-9 = 0.9% of their norm; 3% is refused. In 8 bits every
product's rows are rounded to steps of max / 127, about 0.9% of the row's norm where max is four
standard deviations: eight products, sqrt(8) 0.9% = 2.5% and the bf16 error on top; 8% is refused,
against the same dequantised matrices.
"""
import numpy as np
import pytest
import torch

from engine_helpers import RecordingEngine
from llm_infer_rust_amd import experts, int8, ops
from llm_infer_rust_amd.engine import Engine, EngineConfig
from llm_infer_rust_amd.kv_cache import ModelError
from llm_infer_rust_amd.model import Qwen3Config, Qwen3Model
from llm_infer_rust_amd.sampling import SamplingParams

pytestmark = pytest.mark.gpu

EXPERTS = Qwen3Config(hidden_size=512, num_layers=2, num_attention_heads=8, num_kv_heads=2,
                      intermediate_size=1024, vocab_size=512, head_dim=128,
                      max_position_embeddings=512, rope_theta=1_000_000.0, num_experts=12,
                      num_experts_per_tok=3, moe_intermediate_size=136)
DENSE = Qwen3Config(hidden_size=512, num_layers=2, num_attention_heads=8, num_kv_heads=2,
                    intermediate_size=1000, vocab_size=512, head_dim=128,
                    max_position_embeddings=512, rope_theta=1_000_000.0)


def build(cfg, gpu, seed=0):
    model = Qwen3Model(cfg, torch.bfloat16, gpu).init_random(seed, std=0.05)
    return model


def matrix(w):
    return (w.dequantize() if isinstance(w, int8.Int8Weight) else w).double()


def rms64(x, w, eps):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()


def forward64(model, ids, chosen):
    """Logits of every position of one prompt; ``chosen``: expert ids of every layer."""
    cfg = model.cfg
    t, d = ids.numel(), cfg.head_dim
    hq, hkv, eps = cfg.num_attention_heads, cfg.num_kv_heads, cfg.rms_norm_eps
    cos, sin = (a[:t].double()[:, None] for a in (model.rope.cos, model.rope.sin))

    def rope(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    mask = torch.ones(t, t, dtype=torch.bool, device=ids.device).tril()
    h = model.embed_tokens[ids].double()
    for i, layer in enumerate(model.layers):
        x = rms64(h, layer.input_layernorm, eps)
        q, k, v = (x @ matrix(layer.qkv_proj).T).split([hq * d, hkv * d, hkv * d], 1)
        q = rope(rms64(q.view(t, hq, d), layer.q_norm, eps))
        k = rope(rms64(k.view(t, hkv, d), layer.k_norm, eps)).repeat_interleave(hq // hkv, 1)
        v = v.view(t, hkv, d).repeat_interleave(hq // hkv, 1)
        s = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) / d ** 0.5
        p = torch.softmax(s.masked_fill(~mask, float("-inf")), -1)
        a = torch.matmul(p, v.transpose(0, 1).contiguous()).transpose(0, 1).reshape(t, hq * d)
        h = h + a @ matrix(layer.o_proj).T
        x = rms64(h, layer.post_attention_layernorm, eps)
        gu, dn = matrix(layer.gate_up_proj), matrix(layer.down_proj)
        if layer.router is None:
            g, u = (x @ gu.T).chunk(2, 1)
            h = h + (g * torch.sigmoid(g) * u) @ dn.T
            continue
        logits = x @ layer.router.double().T
        took = chosen[i].long()
        least = logits.gather(1, took).min(1).values
        best_left = logits.scatter(1, took, float("-inf")).max(1).values
        # a choice may lose to one left out by no more than the logits' own error
        assert bool((least >= best_left - 0.08 * logits.abs().max()).all())
        p = torch.softmax(logits, 1).gather(1, took)
        if cfg.norm_topk_prob:
            p = p / p.sum(1, keepdim=True)
        y = torch.zeros_like(h)
        for s in range(took.size(1)):
            for e in range(cfg.num_experts):
                r = torch.nonzero(took[:, s] == e)[:, 0]
                if r.numel():
                    g, u = (x[r] @ gu[e].T).chunk(2, 1)
                    y[r] += (g * torch.sigmoid(g) * u) @ dn[e].T * p[r, s, None]
        h = h + y
    return rms64(h, model.norm, eps) @ model.lm_head.double().T


def record(monkeypatch):
    chosen = []
    plain = experts.route_experts

    def route(*a, **k):
        weights, ids = plain(*a, **k)
        chosen.append(ids.clone())
        return weights, ids
    monkeypatch.setattr(experts, "route_experts", route)
    return chosen


@pytest.mark.parametrize("cfg", [EXPERTS, DENSE], ids=["experts", "dense"])
@pytest.mark.parametrize("quantized", [False, True])
def test_prefill_and_decode_logits(gpu, monkeypatch, cfg, quantized):
    model = build(cfg, gpu)
    if quantized:
        model.quantize_int8()
    chosen = record(monkeypatch)
    eng = RecordingEngine(model, EngineConfig(max_running_req=2, max_seq_len=128,
                                              use_graphs=False))
    prompt = np.random.default_rng(1).integers(0, cfg.vocab_size, 60)
    req = eng.add_request(prompt, SamplingParams(max_tokens=5))
    eng.run_until_complete()
    ids = torch.tensor(np.concatenate([prompt, req.output[:-1]]), device=gpu)
    layers = ([torch.cat(chosen[i::cfg.num_layers]) for i in range(cfg.num_layers)]
              if cfg.num_experts else [None] * cfg.num_layers)
    want = forward64(model, ids, layers)[len(prompt) - 1:]
    got = torch.cat([r[1] for r in eng.records]).double().to(gpu)
    assert got.shape == want.shape == (5, cfg.vocab_size)
    err = ((got - want).norm(dim=1) / want.norm(dim=1)).max()
    assert float(err) < (0.08 if quantized else 0.03), float(err)


@pytest.mark.parametrize("quantized", [False, True])
def test_graph_decode_matches_eager(gpu, quantized):
    """Continuous batching over captured decode graphs (three rows in a bucket of four, the pad row
    routed like any other) against eager steps of the three rows: the same tokens, and logits within
    the bound of the top."""
    model = build(EXPERTS, gpu, 3)
    if quantized:
        model.quantize_int8()
    runs = []
    for graphs in (True, False):
        eng = RecordingEngine(model, EngineConfig(max_running_req=4, max_seq_len=128,
                                                  use_graphs=graphs, graph_batch_sizes=(4,)))
        rng = np.random.default_rng(4)
        for n in (7, 33, 20):
            eng.add_request(rng.integers(0, EXPERTS.vocab_size, n), SamplingParams(max_tokens=8))
        eng.run_until_complete()
        assert (eng.stats["graph_steps"] > 0) == graphs
        runs.append(eng.records)
        del eng
        torch.cuda.synchronize()
    assert len(runs[0]) == len(runs[1])
    for (ug, lg, pg), (ue, le, pe) in zip(*runs):
        assert ug == ue and pg == pe
        assert float((lg - le).norm() / le.norm()) < (0.08 if quantized else 0.03)


def test_ops_take_8_bit_weights(gpu):
    """Every projection entry with an 8-bit weight: the 8-bit product and the step behind it."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(9, 256, generator=g).to(torch.bfloat16).to(gpu)
    w = int8.Int8Weight.quantize(torch.randn(512, 256, generator=g).to(gpu) * 0.06)
    y = int8.linear_int8(x, w)
    assert torch.equal(ops.linear(x, w), y)
    assert torch.equal(ops.linear_silu_mul(x, w), int8.linear_int8(x, w, silu_mul=True))
    residual = torch.randn(9, 512, generator=g).to(torch.bfloat16).to(gpu)
    gamma = torch.rand(512, generator=g).to(torch.bfloat16).to(gpu)
    want = ops.add_rms_norm(y.clone(), residual.clone(), gamma, 1e-6)
    got = ops.linear_add_rms_norm(x, w, residual, gamma, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    out = torch.empty_like(y)
    assert torch.equal(ops.head_linear(x, w), y) and torch.equal(ops.head_linear(x, w, out=out), y)
    for entry in (ops.decode_linear, ops.decode_linear_silu_mul):  # the 16-bit kernels themselves
        with pytest.raises(ops.NativeError):
            entry(x, w)


def test_quantized_weights_are_not_loaded_over(gpu):
    model = build(DENSE, gpu)
    params = {k: v.clone() for k, v in model.named_parameters().items()}
    model.quantize_int8()
    first = model.layers[0].qkv_proj
    assert model.quantize_int8().layers[0].qkv_proj is first  # once
    with pytest.raises(ModelError):
        model.load_weights(params)
    with pytest.raises(ModelError):
        model.init_random(3)


def test_expert_model_loads_its_weights(gpu):
    a, b = build(EXPERTS, gpu, 1), build(EXPERTS, gpu, 2)
    assert b.load_weights(a.named_parameters()) == len(a.named_parameters())
    eng = Engine(b, EngineConfig(max_running_req=2, max_seq_len=64, use_graphs=False))
    req = eng.add_request(np.arange(9), SamplingParams(max_tokens=4))
    eng.run_until_complete()
    eng = Engine(a, EngineConfig(max_running_req=2, max_seq_len=64, use_graphs=False))
    other = eng.add_request(np.arange(9), SamplingParams(max_tokens=4))
    eng.run_until_complete()
    assert req.output == other.output
