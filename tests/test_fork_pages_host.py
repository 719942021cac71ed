"""A prompt whose completions find no page for its last tokens can be tried again (CPU)."""
import numpy as np
import pytest
import torch

from llm_infer_rust_amd.batch import BatchContext
from llm_infer_rust_amd.engine import Engine, EngineConfig, ModelError, PageAllocator
from llm_infer_rust_amd.sampling import SamplingParams


class Model:
    """Counts its forwards; logits with a row for every prompt that ends."""

    def __init__(self):
        self.attention, self.forwards = self, 0

    def prepare(self, meta, tokens):
        return None

    def forward(self, ids, positions, batch, loc, last):
        self.forwards += 1
        return torch.zeros(last.numel(), 8)


class Copies(list):
    def copy_pages(self, src, dst, tokens):
        self.append((list(src), list(dst), list(tokens)))


class HostEngine(Engine):
    """An engine without its GPU parts: every draw is token 1."""

    def __init__(self, num_pages, **kw):
        self.cfg = EngineConfig(**{**dict(page_size=16, max_running_req=8, max_seq_len=1280), **kw})
        self.page_size = self.cfg.page_size
        self.pages = PageAllocator(num_pages)
        self.batches = BatchContext(self.cfg.max_running_req, self.cfg.max_seq_len, self.page_size)
        self.waiting, self.running, self.finished = [], [], []
        self.model, self.pool = Model(), Copies()
        self.stats = {"prefill_batches": 0, "forks": 0}
        self._next_uid, self._inflight = 0, None

    def _upload(self, *arrays):
        return [torch.from_numpy(np.ascontiguousarray(a)) for a in arrays]

    def _sample_and_commit(self, logits, rows):
        assert logits.size(0) == len(rows)
        for r in rows:
            r.output.append(1)

    def prefill(self):
        picked = self._select_prefill()
        if picked:
            self._run_prefill(picked)
        return picked


def held(engine):
    return [p for r in engine.running for p in r.pages + r.fork_pages]


def test_a_fork_without_pages_is_tried_again():
    engine = HostEngine(num_pages=8)
    taken = engine.pages.alloc(5)  # other sequences'
    leader = engine.add_request(range(20), SamplingParams(n=4))
    alone = engine.add_request(range(9), SamplingParams())
    for _ in range(2):
        with pytest.raises(ModelError, match="out of KV-cache pages"):
            engine.prefill()  # two pages of the prompt's, one of three for the completions'
        assert engine.model.forwards == 0 and not engine.pool
        assert leader.cursor == 0 and not leader.output and not alone.output
        assert {r for r, _ in engine._select_prefill()} == {leader, alone}
    engine.pages.release(taken)
    assert [r for r, _ in engine.prefill()] == [leader, alone]
    assert engine.running[:4] == leader.completions and engine.running[4] is alone
    assert all(r.output == [1] and r.cursor == r.prompt.size for r in engine.running)
    assert engine.pool == [([leader.pages[1]] * 3, [r.pages[1] for r in leader.completions[1:]],
                            [4] * 3)]
    assert len({r.pages[1] for r in leader.completions}) == 4
    for r in list(engine.running):
        engine.pages.release(r.pages)
    assert sorted(engine.pages.free) == list(range(1, 9)) and not engine.pages.more_holders


def test_an_earlier_fork_waits_for_a_later_one():
    """All prompts of a batch have their pages before any of them runs."""
    engine = HostEngine(num_pages=7)
    first = engine.add_request(range(5), SamplingParams(n=3))
    second = engine.add_request(range(30), SamplingParams(n=4))
    with pytest.raises(ModelError):
        engine.prefill()  # three, then two and three: one too many
    assert engine.running == [first, second] and not engine.stats["forks"]
    assert len(set(held(engine))) == len(held(engine))
    assert sorted(held(engine) + engine.pages.free) == list(range(1, 8))
    engine.pages.free.append(8)
    engine.prefill()
    assert engine.stats["forks"] == 5 and len(engine.running) == 7 and not engine.pages.free
    assert sorted(set(held(engine))) == list(range(1, 9))


def test_chunks_reserve_with_the_last_one():
    engine = HostEngine(num_pages=12, max_prefill_tokens_per_batch=32)
    leader = engine.add_request(range(70), SamplingParams(n=3))
    left = []
    while not leader.output:
        engine.prefill()
        left.append(len(engine.pages.free))
    assert left == [10, 8, 5] and engine.stats["forks"] == 2  # the last: a page and two copies


def test_prompts_that_end_a_page_need_none():
    engine = HostEngine(num_pages=2)
    leader = engine.add_request(range(32), SamplingParams(n=8))
    engine.prefill()
    assert len(engine.running) == 8 and not engine.pool and not engine.pages.free
    assert all(r.pages == leader.pages and not r.fork_pages for r in engine.running)
