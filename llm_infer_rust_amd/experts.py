"""Layers of experts on the gfx950 kernels.

* ``route_experts(logits, top_k)``: the experts of every token and their weights (softmax, top-k);
* ``expert_mlp(x, ids, weights, gate_up, down)``: the gate_up, SiLU x mul and down products of the
  experts that each token was routed to, summed with the router's weights.

In place of the dense MLP of ``src/models/qwen3/model.rs:478-534``; the reference has no layers of
experts. Nothing is read back to the host, so both can be captured in a HIP graph. Inference only:
a call whose derivative would be wanted is refused.
"""
from __future__ import annotations

import torch

from ._native import NativeError, check, device_cus, lib, on_device, stream_of
from .int8 import _ROW_DTYPES, Int8Weight, _output, _refuse_grad, _rows

MAX_EXPERTS = 1024
MAX_TOP_K = 64


def route_experts(logits: torch.Tensor, top_k: int,
                  normalize: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """``(weights fp32 [T, top_k], ids int32 [T, top_k])`` of router logits ``[T, E]`` (bf16, fp16
    or fp32): the ``top_k`` largest probabilities of ``softmax(logits)``, largest first, equal ones
    by the lower index; with ``normalize`` divided by their sum. A row of only -inf gets the
    weights 0, a row with a NaN or a +inf the weights NaN."""
    t, e, ld = _rows(logits, "route_experts")
    dt = _ROW_DTYPES.get(logits.dtype)
    if dt is None:
        raise NativeError(
            f"route_experts: expected bfloat16, float16 or float32, got {logits.dtype}")
    top_k = int(top_k)
    if not 0 < e <= MAX_EXPERTS or not 0 < top_k <= min(e, MAX_TOP_K):
        raise NativeError(f"route_experts: expected 1 to {MAX_EXPERTS} experts and top_k of 1 to "
                          f"min(experts, {MAX_TOP_K})")
    _refuse_grad("route_experts", logits)
    device = logits.device
    weights = torch.empty(t, top_k, dtype=torch.float32, device=device)
    ids = torch.empty(t, top_k, dtype=torch.int32, device=device)
    with on_device(device):
        check(lib().mi355x_route_experts(logits.data_ptr(), ld, weights.data_ptr(),
                                         ids.data_ptr(), t, e, top_k, bool(normalize), dt,
                                         stream_of(logits)), "route_experts")
    return weights, ids


def expert_mlp(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor,
               gate_up: torch.Tensor | Int8Weight, down: torch.Tensor | Int8Weight,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[t] = sum_s weights[t, s] * down[e] @ (silu(g) * u)``, ``(g, u) = gate_up[e] @ x[t]``,
    ``e = ids[t, s]``.

    ``x`` ``[T, H]`` bf16 or fp16; ``ids`` int32 and ``weights`` fp32 ``[T, top_k]`` as
    ``route_experts`` gives them (an id outside ``[0, E)`` adds nothing: pad rows, experts held
    elsewhere); ``gate_up`` ``[E, 2 I, H]`` (gate rows, then up rows) and ``down`` ``[E, H, I]``,
    both of x's type (H, I and x's row stride multiples of 8, 16-byte aligned) or both
    ``Int8Weight`` (any sizes): then x is quantised a token and ``silu(g) * u`` a slot. Sums are fp32.
    With 16-bit weights ``silu(g) * u`` is rounded to x's type between the products, as in a dense
    MLP (in fp16 inf above 65,504); a few slots, which run one by one, keep it in fp32. ``out`` may
    be given; it must not share memory with ``x``."""
    t, h, ldx = _rows(x, "expert_mlp")
    dtype, device = x.dtype, x.device
    dt = _ROW_DTYPES.get(dtype)
    if dt is None or dt == 2:
        raise NativeError(f"expert_mlp: expected bfloat16 or float16 tensor, got {dtype}")
    index = device.index
    if (ids.dtype != torch.int32 or weights.dtype != torch.float32 or ids.dim() != 2
            or ids.size(0) != t or ids.shape != weights.shape or ids.get_device() != index
            or weights.get_device() != index or not ids.is_contiguous()
            or not weights.is_contiguous()):
        raise NativeError("expert_mlp: expected contiguous int32 ids and fp32 weights [T, top_k]")
    top_k = ids.size(1)
    if not 0 < top_k <= MAX_TOP_K:
        raise NativeError(f"expert_mlp: expected top_k of 1 to {MAX_TOP_K}")
    int8 = isinstance(gate_up, Int8Weight)
    if int8 != isinstance(down, Int8Weight):
        raise NativeError("expert_mlp: gate_up and down must be of one kind")
    gu, dn = (gate_up.values, down.values) if int8 else (gate_up, down)
    _refuse_grad("expert_mlp", x, weights, *((gate_up.scales, down.scales) if int8 else (gu, dn)),
                 out)
    if (gu.dim() != 3 or dn.dim() != 3 or gu.get_device() != index or dn.get_device() != index
            or (not int8 and (gu.dtype != dtype or dn.dtype != dtype
                              or not gu.is_contiguous() or not dn.is_contiguous()))):
        raise NativeError("expert_mlp: expected gate_up [E, 2 I, H] and down [E, H, I] of x's type "
                          "on its device")
    e, _, inter = dn.shape
    if gu.shape != (e, 2 * inter, h) or dn.size(1) != h:
        raise NativeError(f"expert_mlp: expected gate_up [E, 2 I, {h}] and down [E, {h}, I], got "
                          f"{tuple(gu.shape)} and {tuple(dn.shape)}")
    if not e or not h or not inter or e > MAX_EXPERTS:
        raise NativeError(f"expert_mlp: expected 1 to {MAX_EXPERTS} experts of no empty dimension")
    xp, gp, dp = x.data_ptr(), gu.data_ptr(), dn.data_ptr()
    if not int8 and ((h | inter | ldx) % 8 or (xp | gp | dp) % 16):
        raise NativeError("expert_mlp: 16-bit weights need H, I and x's row stride to be multiples "
                          "of 8 and 16-byte aligned rows")
    out, ldo = _output(out, x, h, "expert_mlp")
    cus = device_cus(device)
    native = lib()
    need = native.mi355x_expert_mlp_workspace_bytes(t, top_k, e, h, inter, ldx, int8, cus)
    if need < 0:
        raise NativeError("expert_mlp: invalid shape")
    ws = torch.empty(need or 16, dtype=torch.uint8, device=device)
    ldg, ldd, gs, ds = h, inter, None, None
    if int8:
        ldg, ldd = gate_up.row_stride, down.row_stride
        gs, ds = gate_up.scales.data_ptr(), down.scales.data_ptr()
    with on_device(device):
        check(native.mi355x_expert_mlp(
            xp, ldx, ids.data_ptr(), weights.data_ptr(), gp, ldg, gs, dp, ldd, ds, out.data_ptr(),
            ldo, t, top_k, e, h, inter, ws.data_ptr(), need, cus, dt, stream_of(x)), "expert_mlp")
    return out


__all__ = ["route_experts", "expert_mlp", "NativeError"]
