"""Inputs and the definition in 64 bits for attention over shared prefixes."""
import math

import numpy as np
import torch

from llm_infer_rust_amd.backend import (Attention, AttentionMetadata, AttentionSpec, BatchPhase,
                                        DecodeHostMetadata, SharedPrefix)
from llm_infer_rust_amd.kv_cache import BaseAttention


class Batch:
    """Groups ``(rows, shared tokens)``; ``own`` tokens of every row behind them, the last ``new`` of
    which are queries. Slots of the cache that belong to no row hold NaN."""

    def __init__(self, groups, own, new=None, heads=16, kv_heads=8, page=16, dtype=torch.bfloat16,
                 seed=0, copies=False, q_scale=1.0):
        rng = np.random.default_rng(seed)
        self.groups, self.page, self.dtype = groups, page, dtype
        self.heads, self.kv_heads = heads, kv_heads
        shared = [n for rows, n in groups for _ in range(rows)]
        self.keys = [s + o for s, o in zip(shared, own)]
        self.new = [1] * len(own) if new is None else list(new)
        assert len(own) == len(shared) and all(0 < t <= n for t, n in zip(self.new, self.keys))
        cols = max(-(-n // page) for n in self.keys)
        pages_needed, rows, twins = 1, [], []
        row = 0
        for count, n in groups:
            whole = 0 if copies else n // page
            common = list(range(pages_needed, pages_needed + whole))
            pages_needed += whole
            first = row
            for _ in range(count):
                rest = -(-self.keys[row] // page) - whole
                rows.append(common + list(range(pages_needed, pages_needed + rest)))
                pages_needed += rest
                if row != first:
                    twins.append((first, row, whole * page, n))
                row += 1
        place = np.concatenate([[0], rng.permutation(pages_needed - 1) + 1])
        table = np.full((len(rows), cols + 2), -1, np.int32)
        for i, p in enumerate(rows):
            table[i, :len(p)] = place[p]
        g = torch.Generator().manual_seed(seed)
        shape = (pages_needed, page, kv_heads, 128)
        kv = [torch.randn(shape, generator=g).to(dtype) for _ in range(2)]
        self.slots = [torch.from_numpy(table[r, np.arange(n) // page].astype(np.int64) * page
                                       + np.arange(n) % page) for r, n in enumerate(self.keys)]
        used = torch.zeros(pages_needed * page, dtype=torch.bool)
        for s in self.slots:
            used[s] = True
        for c in kv:
            flat = c.view(-1, kv_heads, 128)
            for a, b, lo, hi in twins:
                flat[self.slots[b][lo:hi]] = flat[self.slots[a][lo:hi]]
            flat[~used] = float("nan")
        self.k, self.v = (c.cuda() for c in kv)
        self.table = torch.from_numpy(table).cuda()
        self.q = (torch.randn(sum(self.new), heads, 128, generator=g) * q_scale).to(dtype).cuda()
        self.starts = np.concatenate([[0], np.cumsum(self.new)]).tolist()
        self.lens = torch.tensor(self.keys, dtype=torch.int32, device="cuda")

    def attention(self):
        a = Attention.new("mi355x", AttentionSpec(self.heads, self.kv_heads, 128, self.dtype,
                                                  torch.device("cuda", 0)))
        a.bind_cache_layout(self.page)
        return a

    def cache(self):
        c = BaseAttention()
        c.bind_kv_cache(self.k, self.v)
        return c

    def shared(self):
        return SharedPrefix([r for r, _ in self.groups], [n for _, n in self.groups])

    def decode_meta(self, shared=True):
        return AttentionMetadata(BatchPhase.DECODE, decode_host=DecodeHostMetadata(self.keys),
                                 block_table=self.table, cache_seqlens=self.lens,
                                 shared_prefix=self.shared() if shared else None)

    def extend_meta(self, shared=True):
        cached = [n - t for n, t in zip(self.keys, self.new)]
        return AttentionMetadata(
            BatchPhase.PREFILL, block_table=self.table,
            cu_seqlens_q=torch.tensor(self.starts, dtype=torch.int32, device="cuda"),
            prefix_lens=torch.tensor(cached, dtype=torch.int32, device="cuda"),
            host_cu_seqlens_q=self.starts, host_prefix_lens=cached,
            shared_prefix=self.shared() if shared else None)

    def run(self, meta, attention=None):
        """The output and what the plan made of the groups."""
        attention = attention or self.attention()
        batch = attention.prepare(meta, self.q.size(0))
        out = batch.forward(self.q, None, None, self.cache())
        return out.view(self.q.shape), batch.plan.plan.shared_info()

    def reference(self):
        """The output in float64 and, for every element, sum_j p_j |v_j|."""
        q, k, v = (t.double() for t in (self.q, self.k.view(-1, self.kv_heads, 128),
                                        self.v.view(-1, self.kv_heads, 128)))
        per = self.heads // self.kv_heads
        out, mass = torch.empty_like(q), torch.empty_like(q)
        for r, n in enumerate(self.keys):
            a, b = self.starts[r], self.starts[r + 1]
            slots = self.slots[r].cuda()
            kr = k[slots].repeat_interleave(per, 1).permute(1, 2, 0).contiguous()
            vr = v[slots].repeat_interleave(per, 1).permute(1, 0, 2).contiguous()
            s = torch.matmul(q[a:b].permute(1, 0, 2).contiguous(), kr) / math.sqrt(128)
            late = torch.ones(b - a, n, device="cuda").triu(n - (b - a) + 1).bool()
            p = torch.softmax(s.masked_fill(late, -math.inf), 2)
            out[a:b] = torch.matmul(p, vr).permute(1, 0, 2)
            mass[a:b] = torch.matmul(p, vr.abs()).permute(1, 0, 2)
        return out, mass

    def check(self, got):
        """Probabilities are rounded to the cache's type before the product with V (half a step of
        each: at most eps / 2 of sum p |v|), and the output once; scores are fp32 sums of 128
        products, whose own rounding (128 * 2^-24 of sum |q k| / sqrt(128), below 200 here) moves
        every p by less than 2e-3 of itself, and far less as the sums' roundings cancel: 5e-4."""
        want, mass = self.reference()
        half = torch.finfo(self.dtype).eps / 2
        limit = (half + 5e-4) * mass + half * want.abs() + 1e-6
        err = (got.double() - want).abs()
        assert bool(torch.isfinite(got).all())
        worst = float((err / limit).max())
        assert worst <= 1.0, worst
        return worst
