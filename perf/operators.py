"""The expert-layer and 8-bit operators as cases that can be timed and checked.

Three operators, each over the sizes that serving meets:

* ``linear_int8``: a projection in 8-bit integers. The 16-bit rows are quantised within the call
  (one scale a token), the weight is held in 8 bits (one scale an output channel), alone or with
  the SiLU x mul that follows a gate_up projection;
* ``route_experts``: softmax and top-k over a router's logits;
* ``expert_mlp``: the gate_up, SiLU x mul and down products of the experts that each token was
  routed to, summed with the router's weights, for 16-bit and for 8-bit weights.

Where ``own`` is false everything is computed from elementary torch operations in 32 bits; where
it is true the calls are the library's. Routing is skewed the way trained routers are: every
expert has a popularity of its own (the same for every seed of a case) and every token its noise.
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


def _linear(name, rows, n, k, silu, dtype="bf16"):
    c = dict(kind="linear_int8", rows=rows, n=n, k=k, silu=silu, dtype=dtype)
    return dict(c, name=name) if name else c


def _route(name, tokens, experts, top_k, normalize, dtype="bf16"):
    c = dict(kind="route_experts", tokens=tokens, experts=experts, top_k=top_k,
             normalize=normalize, dtype=dtype)
    return dict(c, name=name) if name else c


def _experts(name, tokens, experts, top_k, hidden, inter, int8, dtype="bf16"):
    c = dict(kind="expert_mlp", tokens=tokens, experts=experts, top_k=top_k, hidden=hidden,
             inter=inter, int8=int8, dtype=dtype)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One interactive user: the packed QKV projection of one token, latency and weight reads.
        _linear("int8_qkv_one_row", 1, 6144, 4096, False),
        # A moderately loaded server's gate_up with its SiLU x mul.
        _linear("int8_gate_up_decode", 24, 24576, 4096, True),
        # Odd sizes in every dimension, fp16: a row that ends inside a 16-byte word.
        _linear("int8_odd", 333, 1001, 1203, False, "fp16"),
        # A full prefill chunk's down projection.
        _linear("int8_down_prefill", 8192, 4096, 12288, False),
        # The router of one decode row, and of a full prefill chunk in fp32.
        _route("route_one_row", 1, 128, 8, True),
        _route("route_prefill", 8192, 128, 8, True, "fp32"),
        # One interactive user through a layer of many small experts.
        _experts("experts_one_row", 1, 128, 8, 2048, 768, False),
        # A full serving batch through the same layer: every expert touched, few rows each.
        _experts("experts_serving", 256, 128, 8, 2048, 768, False),
        # Few, larger experts and an odd number of tokens, fp16.
        _experts("experts_few", 77, 8, 2, 1024, 2816, False, "fp16"),
        # A full prefill chunk: hundreds of rows an expert, ragged.
        _experts("experts_prefill", 8192, 128, 8, 2048, 768, False),
        # 8-bit experts behind a middling decode batch ...
        _experts("experts_int8_decode", 40, 128, 8, 2048, 768, True),
        # ... and behind half a prefill chunk.
        _experts("experts_int8_prefill", 4096, 128, 8, 2048, 768, True),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng: random.Random):
    kind = rng.choice(["linear_int8", "linear_int8", "route_experts", "expert_mlp", "expert_mlp",
                       "expert_mlp"])
    dtype = "bf16" if rng.random() < 0.7 else "fp16"
    if kind == "linear_int8":
        n = _log_int(rng, 17, 24576)
        k = _log_int(rng, 33, 12288)
        # at most the full prefill chunk's products
        rows = _log_int(rng, 1, max(1, min(8192, 8192 * 4096 * 12288 // (n * k))))
        silu = rng.random() < 0.4
        return _linear(None, rows, n + n % 2 if silu else n, k, silu, dtype)
    if kind == "route_experts":
        experts = _log_int(rng, 4, 512)
        return _route(None, _log_int(rng, 1, 8192 * 128 // max(experts, 128)), experts,
                      rng.randint(1, min(experts, 12)), rng.random() < 0.7,
                      rng.choice(["bf16", "fp16", "fp32"]))
    experts = _log_int(rng, 4, 160)
    top_k = rng.randint(1, min(experts, 8))
    int8 = rng.random() < 0.4
    # 16-bit rows are whole 16-byte words, 8-bit ones any length
    step = 1 if int8 else 8
    hidden = step * _log_int(rng, 128 // step, 4096 // step)
    # at most the listed layer's weights and the full chunk's products
    inter = step * _log_int(rng, 64 // step,
                            max(64, min(4096, 128 * 2048 * 768 // (experts * hidden))) // step)
    tokens = _log_int(rng, 1, max(1, min(8192, 8192 * 8 * 2048 * 768
                                         // (top_k * hidden * inter))))
    return _experts(None, tokens, experts, top_k, hidden, inter, int8, dtype)


# ------------------------------------------------------------------ inputs
def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    t = torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=g)
    return t if scale == 1.0 else t.mul_(scale)


def _rows(g, rows, width, dtype):
    """Activations as a norm leaves them: unit rows whose channels differ in scale, a few of them
    several times the others (the outliers that a scale a token has to cover)."""
    channel = torch.exp(0.5 * _randn(g, width))
    return (_randn(g, rows, width) * channel).to(dtype)


def _int8_weight(g, *shape):
    """A checkpoint's 8-bit weight: values and one scale an output channel."""
    values = torch.empty(*shape, dtype=torch.int8, device="cuda")
    scales = torch.empty(*shape[:-1], dtype=torch.float32, device="cuda")
    flat, flat_scales = values.view(-1, shape[-1]), scales.view(-1)
    std = shape[-1] ** -0.5
    step = max(1, (1 << 27) // shape[-1])
    for i in range(0, flat.size(0), step):
        w = _randn(g, min(step, flat.size(0) - i), shape[-1], scale=std)
        s = w.abs().amax(1) / 127.0
        flat[i:i + step] = torch.round(w / s[:, None]).to(torch.int8)
        flat_scales[i:i + step] = s
    return values, scales


def _popularity(case) -> torch.Tensor:
    r = random.Random(case["experts"] * 1000 + case["top_k"])
    return torch.tensor([r.gauss(0.0, 0.7) for _ in range(case["experts"])])


def _logits(g, case):
    bias = _popularity(case).cuda()
    noise = _randn(g, case["tokens"], case["experts"], scale=1.5)
    return (noise + bias).to(DTYPES[case["dtype"]])


def _inputs(case, seed):
    g, dtype = _gen(seed), DTYPES[case["dtype"]]
    if case["kind"] == "linear_int8":
        return (_rows(g, case["rows"], case["k"], dtype),
                *_int8_weight(g, case["n"], case["k"]))
    if case["kind"] == "route_experts":
        return (_logits(g, case),)
    e, h, i = case["experts"], case["hidden"], case["inter"]
    x = _rows(g, case["tokens"], h, dtype)
    weights, ids = _route_plain(_logits(g, case).float(), case["top_k"], True)
    if case["int8"]:
        return x, ids, weights, *_int8_weight(g, e, 2 * i, h), *_int8_weight(g, e, h, i)
    return (x, ids, weights, _randn(g, e, 2 * i, h, dtype=dtype, scale=h ** -0.5),
            _randn(g, e, h, i, dtype=dtype, scale=i ** -0.5))


def prepare(case, seed):
    inputs = _inputs(case, seed)
    state = dict(kind=case["kind"], case=case)
    if not own:
        return dict(state, inputs=inputs)
    from llm_infer_rust_amd import experts, int8
    state["experts"], state["int8"] = experts, int8
    if case["kind"] == "linear_int8":
        x, values, scales = inputs
        return dict(state, inputs=(x, int8.Int8Weight(values, scales)))
    if case["kind"] == "expert_mlp" and case["int8"]:
        x, ids, weights, gv, gs, dv, ds = inputs
        return dict(state, inputs=(x, ids, weights, int8.Int8Weight(gv, gs),
                                   int8.Int8Weight(dv, ds)))
    return dict(state, inputs=inputs)


# ------------------------------------------------------------------ the plain forms
def _quantize_plain(x):
    top = x.abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(x * 127.0 / top), torch.zeros_like(x))
    return q, top / 127.0


def _silu_mul_plain(y):
    half = y.size(1) // 2
    g, u = y[:, :half], y[:, half:]
    return g / (1.0 + torch.exp(-g)) * u


def _linear_int8_plain(x, values, scales, silu):
    q, sx = _quantize_plain(x.float())
    y = q @ values.float().t() * sx * scales
    return (_silu_mul_plain(y) if silu else y).to(x.dtype)


def _route_plain(logits, top_k, normalize):
    p = torch.exp(logits.float() - logits.float().amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    # a stable sort keeps equal logits in the order of their index
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top_k]
    w = p.gather(1, ids)
    if normalize:
        w = w / w.sum(1, keepdim=True)
    return w, ids.to(torch.int32)


def _expert_mlp_plain(x, ids, weights, *mats):
    xf = x.float()
    int8 = len(mats) == 4
    if int8:
        gate_up, gate_up_scales, down, down_scales = mats
        xq, xs = _quantize_plain(xf)
    else:
        gate_up, down = mats
    out = torch.zeros_like(xf)
    flat = ids.reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat, minlength=gate_up.size(0)).tolist()
    row = 0
    for e, n in enumerate(counts):
        if n == 0:
            continue
        slots = order[row:row + n]
        row += n
        t = slots // ids.size(1)
        if int8:
            act = _silu_mul_plain(xq[t] @ gate_up[e].float().t() * xs[t] * gate_up_scales[e])
            q, s = _quantize_plain(act)
            y = q @ down[e].float().t() * s * down_scales[e]
        else:
            y = _silu_mul_plain(xf[t] @ gate_up[e].float().t()) @ down[e].float().t()
        out.index_add_(0, t, y * weights.reshape(-1)[slots, None])
    return out.to(x.dtype)


def run(state):
    case, inputs = state["case"], state["inputs"]
    if state["kind"] == "linear_int8":
        if own:
            return state["int8"].linear_int8(*inputs, silu_mul=case["silu"])
        return _linear_int8_plain(*inputs, case["silu"])
    if state["kind"] == "route_experts":
        if own:
            return state["experts"].route_experts(inputs[0], case["top_k"],
                                                  normalize=case["normalize"])
        return _route_plain(*inputs, case["top_k"], case["normalize"])
    if own:
        return state["experts"].expert_mlp(*inputs)
    return _expert_mlp_plain(*inputs)


# ------------------------------------------------------------------ the definitions in 64 bits
def _int8_rows64(x):
    """Values and scale of every row's 8-bit form; a row of zeros has the scale 0."""
    biggest = x.abs().max(dim=1).values
    safe = torch.where(biggest == 0, torch.ones_like(biggest), biggest)
    return torch.round(127 * x / safe.unsqueeze(1)), biggest / 127


def _glu64(v):
    gate, up = torch.chunk(v, 2, dim=-1)
    return gate * torch.sigmoid(gate) * up


def _exact_linear(case, seed):
    x, values, scales = _inputs(case, seed)
    q, s = _int8_rows64(x.double())
    y = torch.matmul(q, values.double().transpose(0, 1)) * torch.outer(s, scales.double())
    return _glu64(y) if case["silu"] else y


def _exact_route(case, seed):
    (logits,) = _inputs(case, seed)
    scores = logits.double().cpu().numpy()
    ids = np.argsort(-scores, axis=1, kind="stable")[:, :case["top_k"]]
    z = np.exp(scores - scores.max(axis=1, keepdims=True))
    w = np.take_along_axis(z, ids, axis=1)
    w = w / (w if case["normalize"] else z).sum(axis=1, keepdims=True)
    return (torch.from_numpy(w).cuda(),
            torch.from_numpy(np.ascontiguousarray(ids)).to(torch.int32).cuda())


def _exact_experts(case, seed):
    x, ids, weights, *mats = _inputs(case, seed)
    xd, w = x.double(), weights.double()
    out = torch.zeros_like(xd)
    if case["int8"]:
        gate_up, gate_up_scales, down, down_scales = mats
        q, s = _int8_rows64(xd)
    else:
        gate_up, down = mats
    for e in range(case["experts"]):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        if token.numel() == 0:
            continue
        wg, wd = gate_up[e].double(), down[e].double()
        if case["int8"]:
            wg, wd = wg * gate_up_scales[e, :, None].double(), wd * down_scales[e, :, None].double()
            qa, sa = _int8_rows64(_glu64((q[token] * s[token, None]) @ wg.T))
            y = (qa * sa[:, None]) @ wd.T
        else:
            y = _glu64(xd[token] @ wg.T) @ wd.T
        out.index_put_((token,), y * w[token, slot, None], accumulate=True)
    return out


def exact(case, seed):
    return {"linear_int8": _exact_linear, "route_experts": _exact_route,
            "expert_mlp": _exact_experts}[case["kind"]](case, seed)


@functools.lru_cache(maxsize=None)
def _touched(tokens: int, experts: int, top_k: int) -> int:
    """Experts that at least one token of a batch is routed to (the weights a pass reads), from
    one batch drawn from the same distribution as the inputs."""
    bias = _popularity(dict(experts=experts, top_k=top_k)).numpy()
    scores = np.random.default_rng(0).normal(0.0, 1.5, (tokens, experts)) + bias
    return len(np.unique(np.argpartition(-scores, top_k - 1, axis=1)[:, :top_k]))


def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "linear_int8":
        m, n, k = case["rows"], case["n"], case["k"]
        out = n // 2 if case["silu"] else n
        return {"bytes": m * k * size + n * k + 4 * n + m * out * size, "flops": 2 * m * n * k}
    t, e, top_k = case["tokens"], case["experts"], case["top_k"]
    if case["kind"] == "route_experts":
        return {"bytes": t * e * size + 8 * t * top_k, "flops": 5 * t * e}
    h, i = case["hidden"], case["inter"]
    one = 3 * h * i * (1 if case["int8"] else size) + (4 * (2 * i + h) if case["int8"] else 0)
    return {"bytes": _touched(t, e, top_k) * one + 2 * t * h * size + 8 * t * top_k,
            "flops": 6 * t * top_k * h * i}
