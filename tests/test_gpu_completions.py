"""Several completions of one prompt through the engine: prefilled once, forked, their prompt's
attention computed once where asked for, log probabilities with every token."""
from dataclasses import replace

import numpy as np
import pytest
import torch

from engine_helpers import RecordingEngine
from llm_infer_rust_amd.engine import Engine, EngineConfig, ModelError
from llm_infer_rust_amd.sampling import SamplingParams
from test_gpu_model import TINY, build

pytestmark = pytest.mark.gpu


def engine(model, **kw):
    base = dict(page_size=16, max_running_req=8, max_prefill_tokens_per_batch=96, max_seq_len=256,
                graph_batch_sizes=(1, 4, 8), seed=5)
    return RecordingEngine(model, EngineConfig(**{**base, **kw}))


def check_rows(eng, oracle, reqs, vocab):
    """Every recorded row of logits against the oracle's for that completion's own tokens, and the
    details of its tokens against the row."""
    rows = {r.uid: [] for r in reqs}
    for uids, logits, tokens in eng.records:
        for i, uid in enumerate(uids):
            rows[uid].append((logits[i], tokens[i]))
    for req in reqs:
        assert [t for _, t in rows[req.uid]] == req.output
        oracle.reset()
        want = oracle.forward(req.prompt, 0)[-1]
        pos = len(req.prompt)
        for step, (got, token) in enumerate(rows[req.uid]):
            a, b = got.double().numpy(), np.asarray(want, np.float64)
            cos = float(a @ b / np.linalg.norm(a) / np.linalg.norm(b))
            assert cos > 0.999, (req.uid, step, cos)
            if req.params.logprobs is not None:
                lp = torch.log_softmax(got.double(), 0)
                d = req.details[step]
                assert abs(d.logprob - float(lp[token])) < 1e-4
                assert abs(d.entropy + float((lp.exp() * lp).sum())) < 1e-3
                order = torch.sort(got, descending=True, stable=True).indices
                assert [t for t, _ in d.top] == order[:req.params.logprobs].tolist()
                for t, v in d.top:
                    assert abs(v - float(lp[t])) < 1e-4
            want = oracle.forward(np.array([token]), pos)[-1]
            pos += 1
        assert len(req.details) == (0 if req.params.logprobs is None else len(req.output))


@pytest.mark.parametrize("use_graphs", [True, False])
@pytest.mark.parametrize("share", [True, False])
def test_completions_match_oracle(gpu, use_graphs, share, monkeypatch):
    monkeypatch.setenv("MI355X_SHARED_FROM", "0")
    model, oracle = build(TINY, 1, gpu)
    eng = engine(model, use_graphs=use_graphs, share_prefixes=share)
    rng = np.random.default_rng(7)
    warm = dict(temperature=1.0, max_tokens=6)
    # prompts that end inside a page, at its end, in chunks, and past several tiles
    asked = [(5, 3, None), (32, 2, 4), (150, 4, 0), (70, 1, 2), (131, 5, None), (100, 8, 20)]
    reqs = [r for n, count, lp in asked
            for r in eng.add_request(rng.integers(0, TINY.vocab_size, n),
                                     SamplingParams(n=count, logprobs=lp, **warm)).completions]
    assert len(reqs) == 23
    eng.run_until_complete()
    assert len(eng.finished) == 23 and all(len(r.output) == 6 for r in reqs)
    assert eng.stats["forks"] == 17
    assert len(eng.pages.free) == eng.pool.layout.num_pages and not eng.pages.more_holders
    assert len(set(eng.pages.free)) == len(eng.pages.free)
    check_rows(eng, oracle, reqs, TINY.vocab_size)
    for n, count, _ in asked:  # draws of one prompt differ
        group = [tuple(r.output) for r in reqs if len(r.prompt) == n]
        assert len(group) == count and (count == 1 or len(set(group)) > 1)


def test_completions_of_different_lengths(gpu, monkeypatch):
    """Completions that end early leave the others of their group, and their pages, alone."""
    monkeypatch.setenv("MI355X_SHARED_FROM", "0")
    model, oracle = build(TINY, 2, gpu)
    for share in (True, False):
        eng = engine(model, share_prefixes=share)
        prompt = np.random.default_rng(1).integers(0, TINY.vocab_size, 130)
        eos = 17  # of 512 tokens drawn nearly evenly: rare, but not absent
        reqs = eng.add_request(prompt, SamplingParams(temperature=50.0, n=8, max_tokens=90,
                                                      logprobs=1), eos_token_id=eos).completions
        eng.run_until_complete()
        lengths = [len(r.output) for r in reqs]
        assert all(r.output[-1] == eos or n == 90 for r, n in zip(reqs, lengths))
        assert all(eos not in r.output[:-1] for r in reqs)
        assert len(eng.pages.free) == eng.pool.layout.num_pages and not eng.pages.more_holders
        check_rows(eng, oracle, reqs, TINY.vocab_size)


def test_shared_prompt_is_used(gpu, monkeypatch):
    """Eager steps plan the common prompt as a shared prefix, graph steps too."""
    monkeypatch.setenv("MI355X_SHARED_FROM", "0")
    model, _ = build(TINY, 3, gpu)
    for graphs in (True, False):
        eng = engine(model, use_graphs=graphs, share_prefixes=True)
        eng.add_request(np.arange(200) % 512, SamplingParams(n=8, temperature=1.0, max_tokens=5))
        eng.step()
        eng.step()
        eng.step()
        plan = eng.graphs[8].state.plan if graphs else model.attention.backend._decode_plan
        assert plan.shared_info()["tokens"] in (128, 192)
        eng.run_until_complete()


def test_admission_counts_completions(gpu):
    model, _ = build(TINY, 4, gpu)
    eng = Engine(model, EngineConfig(max_running_req=4, max_seq_len=128, use_graphs=False))
    a = eng.add_request([1, 2, 3], SamplingParams(n=3, max_tokens=4))
    b = eng.add_request([4, 5], SamplingParams(n=2, max_tokens=4))
    eng.step()
    assert len(eng.running) == 3 and eng.waiting == [b]
    eng.run_until_complete()
    assert len(a.completions) == 3 and len(b.completions) == 2
    assert len(eng.finished) == 5
    for params in (SamplingParams(n=5), SamplingParams(logprobs=65), SamplingParams(logprobs=-1)):
        with pytest.raises(ModelError):
            eng.add_request([1], params)


def test_greedy_completions_agree(gpu):
    model, _ = build(TINY, 6, gpu)
    eng = engine(model, share_prefixes=True)
    reqs = eng.add_request(np.arange(90), SamplingParams(n=4, max_tokens=20)).completions
    eng.run_until_complete()
    assert len({tuple(r.output) for r in reqs}) == 1


def test_many_completions_in_one_graph(gpu, monkeypatch):
    """Enough rows and heads for a decode graph whose products and copies each have whole CUs."""
    monkeypatch.setenv("MI355X_SHARED_FROM", "0")
    cfg = replace(TINY, num_attention_heads=32, num_kv_heads=8)
    model, oracle = build(cfg, 7, gpu)
    eng = engine(model, max_running_req=64, graph_batch_sizes=(64,), share_prefixes=True)
    rng = np.random.default_rng(3)
    reqs = [r for n, count in ((150, 36), (70, 20))
            for r in eng.add_request(rng.integers(0, cfg.vocab_size, n), SamplingParams(
                temperature=1.0, n=count, max_tokens=4, logprobs=2)).completions]
    eng.run_until_complete()
    assert eng.stats["forks"] == 54 and eng.stats["graph_steps"] > 0
    assert len(eng.pages.free) == eng.pool.layout.num_pages
    check_rows(eng, oracle, reqs, cfg.vocab_size)
