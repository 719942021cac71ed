"""Operators behind many completions of one prompt, as cases that can be timed and checked.

* ``decode``: attention of one new token a row over a paged cache in which groups of rows share a
  long prefix, a model step's layers one after another on one plan;
* ``extend``: the same for several new tokens a row, causal among themselves;
* ``copy``: copies of cache pages over all layers, the first tokens of a page (a sequence that is
  forked inside a page) or whole pages (pages that move);
* ``logprobs``: log probabilities of given tokens, with the distribution's entropy and the most
  likely alternatives.

Where ``own`` is false everything is computed from elementary torch operations in 32 bits; where
it is true the calls are the library's. Lengths, groups and pages to copy belong to a case and are
the same for every seed; values and the pages' places are drawn from the seed.
"""
from __future__ import annotations

import functools
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
HEAD = 128


def _attention(name, kind, groups, rows, prefix, own_tokens, new, heads, kv_heads, page, layers,
               dtype="bf16"):
    c = dict(kind=kind, groups=groups, rows=rows, prefix=prefix, own_tokens=own_tokens, new=new,
             heads=heads, kv_heads=kv_heads, page=page, layers=layers, dtype=dtype)
    return dict(c, name=name) if name else c


def _copy(name, pairs, layers, kv_heads, page, partial, dtype="bf16"):
    c = dict(kind="copy", pairs=pairs, layers=layers, kv_heads=kv_heads, page=page,
             partial=partial, dtype=dtype)
    return dict(c, name=name) if name else c


def _logprobs(name, rows, vocab, top, dtype="bf16"):
    c = dict(kind="logprobs", rows=rows, vocab=vocab, top=top, dtype=dtype)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One user's four completions of a prompt of 1,100 tokens.
        _attention("decode_four", "decode", 1, 4, 1100, 150, 1, 32, 8, 16, 8),
        # A server whose 64 requests open with the same instructions.
        _attention("decode_instructions", "decode", 1, 64, 2048, 700, 1, 32, 8, 16, 4),
        # Several prompts, each with some completions: odd lengths, pages and group sizes, fp16.
        _attention("decode_groups", "decode", 23, 131, 1703, 333, 1, 16, 8, 24, 4, "fp16"),
        # A full batch over one long document.
        _attention("decode_document", "decode", 1, 256, 8192, 1024, 1, 32, 8, 16, 4),
        # Short questions behind the same instructions, prefilled together.
        _attention("extend_questions", "extend", 1, 48, 4096, 0, 40, 32, 8, 16, 2),
        # Candidates of some tokens each, scored for every row of a batch.
        _attention("extend_candidates", "extend", 5, 61, 2900, 500, 7, 16, 8, 16, 4),
        # A prompt inside a page, forked to four rows in an 8B model's cache.
        _copy("copy_fork_four", 3, 36, 8, 16, True),
        # The same for a full batch in a small model's cache.
        _copy("copy_fork_batch", 255, 28, 8, 16, True),
        # Pages that move to other places, whole: odd page size and number of heads.
        _copy("copy_moves", 333, 11, 5, 13, False, "fp16"),
        # One row of a vocabulary, five alternatives.
        _logprobs("logprobs_one_row", 1, 151936, 5),
        # A decode step of a full batch, twenty alternatives.
        _logprobs("logprobs_step", 256, 151936, 20),
        # The tokens of a long prompt scored.
        _logprobs("logprobs_prompt", 4096, 151936, 5),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def _within(case) -> bool:
    """At most the full batch's work over one long document."""
    w = work(case)
    return w["flops"] <= 140e9 and w["bytes"] <= 2.2e9


def draw(rng: random.Random):
    kind = rng.choice(["decode", "decode", "decode", "extend", "extend", "copy", "logprobs",
                       "logprobs"])
    dtype = "bf16" if rng.random() < 0.7 else "fp16"
    if kind in ("decode", "extend"):
        kv_heads = rng.choice([1, 2, 4, 8, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 4, 8])
        rows = _log_int(rng, 2, min(256, 8192 // heads))
        groups = _log_int(rng, 1, max(1, rows // 2))
        prefix = _log_int(rng, 100, 8192)
        new = 1 if kind == "decode" else _log_int(rng, 2, max(2, min(256, 2048 // rows)))
        case = _attention(None, kind, groups, rows, prefix, _log_int(rng, 1, 1024), new, heads,
                          kv_heads, rng.choice([1, 8, 13, 16, 16, 24, 64]),
                          1 if new > 8 else rng.randint(1, 4), dtype)
        while case["layers"] > 1 and not _within(case):
            case["layers"] -= 1
        while not _within(case):
            case["own_tokens"] = max(1, case["own_tokens"] // 2)
            case["prefix"] = max(100, case["prefix"] // 2)
        return case
    if kind == "copy":
        layers, kv_heads = rng.randint(2, 36), rng.choice([1, 2, 5, 8])
        page = rng.choice([1, 8, 13, 16, 16, 24, 64])
        # at most the full batch's bytes
        room = 255 * 28 * 8 * 16 // (layers * kv_heads * page)
        return _copy(None, _log_int(rng, 1, max(1, min(2000, room))), layers, kv_heads, page,
                     page > 1 and rng.random() < 0.5, dtype)
    vocab = _log_int(rng, 50, 200000)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    rows = _log_int(rng, 1, max(1, min(8192, 4096 * 151936 // (vocab * SIZE[dtype] // 2))))
    return _logprobs(None, rows, vocab, rng.randint(0, min(vocab, 24)), dtype)


# ------------------------------------------------------------------ inputs
def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    t = torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=g)
    return t if scale == 1.0 else t.mul_(scale)


@functools.lru_cache(maxsize=64)
def _lengths(groups, rows, prefix, own_tokens, new, decode):
    """Rows and prefix of every group, keys and new tokens of every row."""
    r = random.Random(f"{groups} {rows} {prefix} {own_tokens} {new} {decode}")
    # every group has a row, the rest falls where it falls: groups of one up to many
    sizes = [1] * groups
    for _ in range(rows - groups):
        sizes[min(int(groups * r.random() ** 1.5), groups - 1)] += 1
    prefixes = [prefix if groups == 1 else r.randint(max(1, prefix // 4), prefix)
                for _ in range(groups)]
    keys, fresh = [], []
    for n, p in zip(sizes, prefixes):
        for _ in range(n):
            t = 1 if decode else r.randint(1, new)
            fresh.append(t)
            # a decode row's own tokens hold the new one
            keys.append(p + (r.randint(1, own_tokens) if decode
                             else t + (r.randint(0, own_tokens) if own_tokens else 0)))
    return tuple(sizes), tuple(prefixes), tuple(keys), tuple(fresh)


def _case_lengths(case):
    return _lengths(case["groups"], case["rows"], case["prefix"], case["own_tokens"], case["new"],
                    case["kind"] == "decode")


def _tables(case, seed):
    """The block table (rows of a group hold the same whole pages of their prefix), the number of
    pages, and for rows whose prefix ends inside a page the pages that hold the same tokens."""
    sizes, prefixes, keys, _ = _case_lengths(case)
    page = case["page"]
    cols = max(-(-n // page) for n in keys)
    rows, twins, row, used = [], [], 0, 1
    for n, p in zip(sizes, prefixes):
        whole = p // page
        shared = list(range(used, used + whole))
        used += whole
        first = used
        for _ in range(n):
            rest = -(-keys[row] // page) - whole
            rows.append(shared + list(range(used, used + rest)))
            if p % page and used != first:
                twins.append((first, used, p % page))
            used += rest
            row += 1
    place = np.concatenate([[0], np.random.default_rng(seed).permutation(used - 1) + 1])
    table = np.full((len(rows), cols), -1, np.int32)
    for i, pages in enumerate(rows):
        table[i, :len(pages)] = place[pages]
    return table, used, [(int(place[a]), int(place[b]), n) for a, b, n in twins]


def _attention_inputs(case, seed):
    g, dtype = _gen(seed), DTYPES[case["dtype"]]
    _, _, keys, fresh = _case_lengths(case)
    table, pages, twins = _tables(case, seed)
    caches = []
    for _ in range(case["layers"]):
        k, v = (_randn(g, pages, case["page"], case["kv_heads"], HEAD, dtype=dtype)
                for _ in range(2))
        for a, b, n in twins:
            k[b, :n] = k[a, :n]
            v[b, :n] = v[a, :n]
        caches.append((k, v))
    # queries twice as long as a norm leaves them: scores that favour some keys
    q = [_randn(g, sum(fresh), case["heads"], HEAD, dtype=dtype, scale=2.0)
         for _ in range(case["layers"])]
    return q, caches, torch.from_numpy(table).cuda()


@functools.lru_cache(maxsize=64)
def _pairs(pairs, page, partial):
    """Pages to copy from and to, and how many of their tokens."""
    r = random.Random(f"{pairs} {page} {partial}")
    sources = r.randint(1, max(1, pairs // 8)) if partial else pairs
    ids = list(range(1, sources + pairs + 1))
    r.shuffle(ids)
    # a forked page goes to several rows, a moved one to one place
    src = [ids[i % sources] for i in range(pairs)]
    valid = {s: r.randint(1, page - 1) if partial else page for s in src}
    return tuple(src), tuple(ids[sources:]), tuple(valid[s] for s in src), sources + pairs


def _case_pairs(case):
    return _pairs(case["pairs"], case["page"], case["partial"])


def _logits(case, seed):
    """Rows as a trained head leaves them: a broad bulk and a few tokens far above it; the given
    token is mostly one of those."""
    g, (rows, vocab) = _gen(seed), (case["rows"], case["vocab"])
    x = _randn(g, rows, vocab, dtype=DTYPES[case["dtype"]], scale=2.0)
    likely = torch.randint(vocab, (rows, 6), generator=g, device="cuda")
    x.scatter_(1, likely, (8.0 + 3.0 * _randn(g, rows, 6)).to(x.dtype))
    other = torch.randint(vocab, (rows,), generator=g, device="cuda")
    pick = torch.rand(rows, generator=g, device="cuda") < 0.8
    return x, torch.where(pick, likely[:, 0], other)


def prepare(case, seed):
    state = dict(case=case, kind=case["kind"])
    if case["kind"] == "logprobs":
        state["inputs"] = _logits(case, seed)
        if own:
            from llm_infer_rust_amd import sampling
            state["call"] = sampling.token_logprobs
        return state
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "copy":
        src, dst, valid, pages = _case_pairs(case)
        shape = (2, case["layers"], pages + 1, case["page"], case["kv_heads"], HEAD)
        state["inputs"] = (list(src), list(dst), list(valid) if case["partial"] else None)
        if own:
            from llm_infer_rust_amd.kv_cache import KVCacheLayout, KVCachePool
            state["pool"] = KVCachePool(KVCacheLayout(case["layers"], pages, case["page"],
                                                      case["kv_heads"], HEAD), dtype, "cuda")
            state["buffer"] = state["pool"].buffer
        else:
            state["buffer"] = torch.empty(shape, dtype=dtype, device="cuda")
        state["buffer"].normal_(0.0, 1.0, generator=_gen(seed))
        state["buffer"][:, :, 0].zero_()
        return state
    q, caches, table = _attention_inputs(case, seed)
    _, _, keys, fresh = _case_lengths(case)
    starts = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
    state.update(q=q, caches=caches, table=table, keys=list(keys), fresh=list(fresh),
                 starts=starts.tolist())
    if own:
        from llm_infer_rust_amd import backend
        from llm_infer_rust_amd.kv_cache import BaseAttention
        attention = backend.Attention.new("mi355x", backend.AttentionSpec(
            case["heads"], case["kv_heads"], HEAD, dtype, torch.device("cuda", 0)))
        attention.bind_cache_layout(case["page"])
        bound = []
        for k, v in caches:
            bound.append(BaseAttention())
            bound[-1].bind_kv_cache(k, v)
        state.update(backend=backend, attention=attention, bound=bound,
                     lens_gpu=torch.tensor(keys, dtype=torch.int32, device="cuda"),
                     starts_gpu=torch.from_numpy(starts).cuda(),
                     cached=[n - t for n, t in zip(keys, fresh)],
                     cached_gpu=torch.tensor([n - t for n, t in zip(keys, fresh)],
                                             dtype=torch.int32, device="cuda"))
    return state


# ------------------------------------------------------------------ the plain forms
def _attention_plain(state):
    case, outs = state["case"], []
    page, kv_heads, group = case["page"], case["kv_heads"], case["heads"] // case["kv_heads"]
    slots = []
    for r, n in enumerate(state["keys"]):
        pos = torch.arange(n, device="cuda")
        slots.append(state["table"][r, pos // page].long() * page + pos % page)
    for q, (k, v) in zip(state["q"], state["caches"]):
        out = torch.empty_like(q)
        kf, vf = k.view(-1, kv_heads, HEAD), v.view(-1, kv_heads, HEAD)
        for r, n in enumerate(state["keys"]):
            a, b = state["starts"][r], state["starts"][r + 1]
            t = b - a
            qr = q[a:b].float().view(t, kv_heads, group, HEAD).permute(1, 0, 2, 3)
            kr = kf[slots[r]].float().permute(1, 2, 0).contiguous()
            vr = vf[slots[r]].float().permute(1, 0, 2).contiguous()
            s = torch.matmul(qr.reshape(kv_heads, t * group, HEAD), kr) * HEAD ** -0.5
            if t > 1:
                s = s.view(kv_heads, t, group, n)
                key = torch.arange(n, device="cuda")
                last = torch.arange(n - t, n, device="cuda")
                s = torch.where((key <= last[:, None])[None, :, None], s, float("-inf"))
                s = s.view(kv_heads, t * group, n)
            p = torch.exp(s - s.amax(2, keepdim=True))
            o = torch.matmul(p, vr) / p.sum(2, keepdim=True)
            out[a:b] = o.view(kv_heads, t, group, HEAD).permute(1, 0, 2, 3).reshape(
                t, kv_heads * group, HEAD).to(q.dtype)
        outs.append(out.view(out.size(0), -1))
    return outs


def _copy_plain(buffer, src, dst, valid):
    page = buffer.size(3)
    src, dst = (torch.tensor(x, device="cuda") for x in (src, dst))
    at = torch.arange(page, device="cuda")
    n = torch.full_like(src, page) if valid is None else torch.tensor(valid, device="cuda")
    keep = (at < n[:, None]).view(-1)
    flat = buffer.view(*buffer.shape[:2], -1, *buffer.shape[4:])
    a = (src[:, None] * page + at).view(-1)[keep]
    b = (dst[:, None] * page + at).view(-1)[keep]
    flat[:, :, b] = flat[:, :, a]
    return buffer


def _logprobs_plain(x, tokens, top):
    parts = []
    step = max(1, (1 << 26) // x.size(1))
    for i in range(0, x.size(0), step):
        f = x[i:i + step].float()
        m = f.amax(1, keepdim=True)
        e = torch.exp(f - m)
        z = e.sum(1, keepdim=True)
        lse = m + torch.log(z)
        given = f.gather(1, tokens[i:i + step, None]) - lse
        entropy = lse - (e * f).sum(1, keepdim=True) / z
        if top:  # a stable sort keeps equal logits in the order of their index
            value, ids = torch.sort(f, dim=1, descending=True, stable=True)
            parts.append((given[:, 0], entropy[:, 0], ids[:, :top], value[:, :top] - lse))
        else:
            parts.append((given[:, 0], entropy[:, 0],
                          torch.empty(f.size(0), 0, dtype=torch.int64, device="cuda"),
                          torch.empty(f.size(0), 0, device="cuda")))
    return tuple(torch.cat(p) for p in zip(*parts))


def run(state):
    case = state["case"]
    if state["kind"] == "logprobs":
        x, tokens = state["inputs"]
        if own:
            r = state["call"](x, tokens, top=case["top"])
            return r.logprobs, r.entropy, r.top_ids, r.top_logprobs
        return _logprobs_plain(x, tokens, case["top"])
    if state["kind"] == "copy":
        if own:
            state["pool"].copy_pages(*state["inputs"])
            return state["buffer"]
        return _copy_plain(state["buffer"], *state["inputs"])
    if not own:
        return _attention_plain(state)
    b = state["backend"]
    sizes, prefixes, _, _ = _case_lengths(case)
    shared = b.SharedPrefix(rows=sizes, lens=prefixes)
    if state["kind"] == "decode":
        meta = b.AttentionMetadata(
            b.BatchPhase.DECODE, decode_host=b.DecodeHostMetadata(state["keys"]),
            block_table=state["table"], cache_seqlens=state["lens_gpu"], shared_prefix=shared)
    else:
        meta = b.AttentionMetadata(
            b.BatchPhase.PREFILL, cu_seqlens_q=state["starts_gpu"],
            prefix_lens=state["cached_gpu"], block_table=state["table"],
            host_cu_seqlens_q=state["starts"], host_prefix_lens=state["cached"],
            shared_prefix=shared)
    batch = state["attention"].prepare(meta, state["starts"][-1])
    return [batch.forward(q, None, None, cache) for q, cache in zip(state["q"], state["bound"])]


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_attention(case, seed):
    q, caches, table = _attention_inputs(case, seed)
    _, _, keys, fresh = _case_lengths(case)
    per, outs = case["heads"] // case["kv_heads"], []
    for x, (k, v) in zip(q, caches):
        done, out = 0, []
        for r, n in enumerate(keys):
            pages = table[r, :-(-n // case["page"])].long()
            kr = k[pages].flatten(0, 1)[:n].double()
            vr = v[pages].flatten(0, 1)[:n].double()
            xr = x[done:done + fresh[r]].double()
            done += fresh[r]
            heads = []
            for h in range(case["heads"]):
                s = xr[:, h] @ kr[:, h // per].T / math.sqrt(HEAD)
                # query i is the key n - fresh + i: later ones are not seen
                s = s.masked_fill(torch.ones_like(s).triu(n - fresh[r] + 1).bool(), -math.inf)
                heads.append(torch.softmax(s, 1) @ vr[:, h // per])
            out.append(torch.cat(heads, 1))
        outs.append(torch.cat(out))
    return outs


def _exact_copy(case, seed):
    src, dst, valid, pages = _case_pairs(case)
    b = torch.empty(2, case["layers"], pages + 1, case["page"], case["kv_heads"], HEAD,
                    dtype=DTYPES[case["dtype"]], device="cuda")
    b.normal_(0.0, 1.0, generator=_gen(seed))
    b[:, :, 0] = 0
    for s, d, n in zip(src, dst, valid):
        b[:, :, d].narrow(2, 0, n).copy_(b[:, :, s].narrow(2, 0, n))
    return b.double()


def _exact_logprobs(case, seed):
    x, tokens = _logits(case, seed)
    top, given, entropy, ids, values = case["top"], [], [], [], []
    step = max(1, (1 << 25) // case["vocab"])
    for i in range(0, case["rows"], step):
        d = x[i:i + step].double()
        lp = torch.log_softmax(d, 1)
        given.append(lp[torch.arange(len(d), device="cuda"), tokens[i:i + step]])
        entropy.append(-(lp.exp() * lp).sum(1))
        if not top:
            continue
        edge = torch.topk(d, top, 1).values[:, -1:]
        row, col = (t.cpu().numpy() for t in torch.nonzero(d >= edge, as_tuple=True))
        val = d[torch.from_numpy(row).cuda(), torch.from_numpy(col).cuda()].cpu().numpy()
        order = np.lexsort((col, -val, row))
        first = np.searchsorted(row[order], np.arange(len(d)))
        chosen = col[order][first[:, None] + np.arange(top)]
        ids.append(torch.from_numpy(chosen).cuda())
        values.append(lp.gather(1, ids[-1]))
    empty = torch.empty(case["rows"], 0, dtype=torch.int64, device="cuda")
    return (torch.cat(given), torch.cat(entropy), torch.cat(ids) if top else empty,
            torch.cat(values) if top else empty.double())


def exact(case, seed):
    if case["kind"] in ("decode", "extend"):
        return _exact_attention(case, seed)
    return (_exact_copy if case["kind"] == "copy" else _exact_logprobs)(case, seed)


def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    if case["kind"] == "copy":
        token = 2 * case["layers"] * case["kv_heads"] * HEAD * size
        return {"bytes": 2 * token * sum(_case_pairs(case)[2]), "flops": 0}
    sizes, prefixes, keys, fresh = _case_lengths(case)
    held = sum(prefixes) + sum(keys) - sum(n * p for n, p in zip(sizes, prefixes))
    seen = sum(t * (n - t) + t * (t + 1) // 2 for n, t in zip(keys, fresh))
    return {"bytes": case["layers"] * size * HEAD * (2 * case["kv_heads"] * held
                                                     + 2 * case["heads"] * sum(fresh)),
            "flops": case["layers"] * 4 * HEAD * case["heads"] * seen}
