"""``Qwen3Model.quantize_int8`` replaces the matrices that a captured graph reads: it is refused while
such a graph may be replayed. No graph is replayed after a refusal here."""
import gc

import pytest
import torch

from llm_infer_rust_amd import model as model_module
from llm_infer_rust_amd.kv_cache import ModelError
from llm_infer_rust_amd.model import Qwen3Config, Qwen3Model

CFG = Qwen3Config(hidden_size=256, num_layers=1, num_attention_heads=2, num_kv_heads=1,
                  intermediate_size=256, vocab_size=128, head_dim=128,
                  max_position_embeddings=64)


class Holder:
    pass


@pytest.fixture
def cpu_model(monkeypatch):
    """A model whose matrices stay on the CPU, and the names that quantising replaces."""
    class NoAttention:
        @staticmethod
        def new(*_):
            return None

    class Quantised:
        @staticmethod
        def quantize(weight):
            return Quantised()
    monkeypatch.setattr(model_module, "Attention", NoAttention)
    monkeypatch.setattr(model_module, "AttentionSpec", lambda *_: None)
    monkeypatch.setattr(model_module, "Int8Weight", Quantised)
    return Qwen3Model(CFG, torch.bfloat16, "cpu"), Quantised


def test_refused_while_a_holder_of_graphs_lives(cpu_model):
    model, quantised = cpu_model
    holder = Holder()
    holder.itself = holder  # found by the collector only
    with model.captured_for(holder):
        pass
    with pytest.raises(ModelError):
        model.quantize_int8()
    assert isinstance(model.layers[0].qkv_proj, torch.Tensor)  # nothing was replaced
    del holder
    assert isinstance(model.quantize_int8().layers[0].qkv_proj, quantised)


@pytest.mark.gpu
def test_engine_graphs(gpu):
    from llm_infer_rust_amd.engine import Engine, EngineConfig
    from llm_infer_rust_amd.int8 import Int8Weight
    model = Qwen3Model(CFG, torch.bfloat16, gpu).init_random(0)
    eng = Engine(model, EngineConfig(max_running_req=2, max_seq_len=64, graph_batch_sizes=(2,)))
    with pytest.raises(ModelError):
        model.quantize_int8()
    torch.cuda.synchronize()
    del eng
    gc.collect()
    eager = Engine(model, EngineConfig(max_running_req=2, max_seq_len=64, use_graphs=False))
    model.quantize_int8()  # no graph reads the 16-bit matrices any more
    assert isinstance(model.layers[0].qkv_proj, Int8Weight) and not eager.graphs


@pytest.mark.gpu
def test_graphs_of_the_caller(gpu):
    """Captures of ``forward`` whose graphs the model knows nothing of."""
    from llm_infer_rust_amd.engine import Engine, EngineConfig
    model = Qwen3Model(CFG, torch.bfloat16, gpu).init_random(0)
    eng = Engine(model, EngineConfig(max_running_req=1, max_seq_len=64, use_graphs=False))
    eng._capture_buckets()
    with pytest.raises(ModelError):
        model.quantize_int8()
    torch.cuda.synchronize()
    del eng
    gc.collect()
    with pytest.raises(ModelError):
        model.quantize_int8()
