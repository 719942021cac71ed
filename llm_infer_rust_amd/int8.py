"""Projections in 8-bit integers on the gfx950 kernels.

* ``quantize_rows(x)``: int8 rows with one fp32 scale each (``max |x| / 127``);
* ``Int8Weight``: an int8 weight with one fp32 scale an output channel, of one matrix ``[N, K]`` or
  of a stack of experts' matrices ``[E, N, K]``;
* ``linear_int8(x, weight)``: ``x @ weight.T`` with the 16-bit rows of ``x`` quantised in the call,
  exact int32 sums and one rounding, optionally with the SiLU x mul of a gate_up projection.

The counterpart of ``src/layers/linear.rs:5-7`` for weights held in 8 bits; the reference itself
has 16-bit weights only. Inference only: a call whose derivative would be wanted is refused.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from ._native import NativeError, check, device_cus, lib, on_device, stream_of

_ROW_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_K = 131072  # 127 * 127 * K stays inside int32
_STEP = 128     # bytes of K a product takes at once

# Looked up once: every call asks (0.1 us of 8).
_transform_level = torch._C._functorch.maybe_current_level
_of_transform = torch._C._functorch.is_functorch_wrapped_tensor
_is_tracing = torch._C._is_tracing
_is_grad_enabled = torch.is_grad_enabled


def _padded(k: int, to: int) -> int:
    return (k + to - 1) // to * to


def _refuse_grad(what: str, *tensors: torch.Tensor | None) -> None:
    """Refuse a call that torch would have to record: operands that want a gradient or carry a
    tangent, operands of a function transform (vmap, grad, jvp), tracing."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NativeError(f"{what}: no tangent is carried")
    if _transform_level() is not None:
        for t in tensors:
            if t is not None and _of_transform(t):
                raise NativeError(f"{what}: not for torch.func's transforms")
    if _is_tracing():
        raise NativeError(f"{what}: a trace would not hold the call")
    if not _is_grad_enabled():
        return
    for t in tensors:
        if t is not None and t.requires_grad:
            raise NativeError(f"{what}: no gradient is recorded; call it under torch.no_grad()")


def _rows(x: torch.Tensor, what: str) -> tuple[int, int, int]:
    """Rows, columns and row stride of a 2-D GPU tensor of unit column stride whose rows do not
    overlap. A single row's stride is never used and may be anything: its length stands for it."""
    if not x.is_cuda:
        raise NativeError(f"{what}: expected a GPU tensor")
    if x.dim() != 2:
        raise NativeError(f"{what}: expected rows [T, K]")
    (t, k), (stride, unit) = x.shape, x.stride()
    if k > 1 and unit != 1:
        raise NativeError(f"{what}: expected rows [T, K] of unit column stride")
    if t <= 1:
        return t, k, k
    if stride < k:
        raise NativeError(f"{what}: rows must not overlap")
    return t, k, stride


def _output(out: torch.Tensor | None, x: torch.Tensor, width: int,
            what: str) -> tuple[torch.Tensor, int]:
    """The output rows ``[T, width]`` of x's type, given or new, and their stride."""
    t = x.size(0)
    if out is None:
        return torch.empty(t, width, dtype=x.dtype, device=x.device), width
    if out.shape != (t, width) or out.dtype != x.dtype or out.device != x.device:
        raise NativeError(f"{what}: invalid output")
    if t and out.untyped_storage().data_ptr() == x.untyped_storage().data_ptr():
        raise NativeError(f"{what}: out must not share memory with x")
    return out, _rows(out, what)[2]


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(values int8 [T, K], scales fp32 [T])`` of ``x`` ``[T, K]`` in bf16, fp16 or fp32:
    ``scales = max |x| / 127`` and ``values = rint(127 x / max |x|)`` a row (half to even). ``values``
    is a view of rows padded with zeros to 16 columns. A row with an inf or a NaN gets the scale
    NaN, a row of zeros the scale 0."""
    t, k, ldx = _rows(x, "quantize_rows")
    if x.dtype not in _ROW_DTYPES:
        raise NativeError(f"quantize_rows: expected bfloat16, float16 or float32, got {x.dtype}")
    if k == 0:
        raise NativeError("quantize_rows: rows must not be empty")
    _refuse_grad("quantize_rows", x)
    with on_device(x.device):
        values = torch.empty((t, _padded(k, 16)), dtype=torch.int8, device=x.device)
        scales = torch.empty(t, dtype=torch.float32, device=x.device)
        check(lib().mi355x_quantize_rows(x.data_ptr(), ldx, values.data_ptr(),
                                         values.size(1), scales.data_ptr(), t, k,
                                         _ROW_DTYPES[x.dtype], stream_of(x)), "quantize_rows")
    return values[:, :k], scales


class Int8Weight:
    """int8 ``values`` ``[N, K]`` (or ``[E, N, K]`` for experts) and fp32 ``scales`` ``[N]``
    (``[E, N]``): the weight ``values * scales[..., None]``. Rows whose length is no multiple of 128
    are laid out once with a stride that is, so that every row is whole steps of a product."""

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if (values.dtype != torch.int8 or values.dim() not in (2, 3)
                or scales.dtype != torch.float32 or scales.shape != values.shape[:-1]
                or scales.device != values.device):
            raise NativeError("int8 weight: expected int8 values [N, K] or [E, N, K] and one fp32 "
                              "scale a row")
        if not values.is_cuda:
            raise NativeError("int8 weight: expected GPU tensors")
        if 0 in values.shape or values.size(-1) > MAX_K:
            raise NativeError(f"int8 weight: expected 1 to {MAX_K} columns and no empty dimension")
        k = values.size(-1)
        if k % _STEP or not values.is_contiguous() or values.data_ptr() % 16:
            padded = torch.zeros((*values.shape[:-1], _padded(k, _STEP)), dtype=torch.int8,
                                 device=values.device)
            padded[..., :k] = values
            values = padded[..., :k]
        self.values = values
        self.scales = scales.contiguous()

    @staticmethod
    def quantize(weight: torch.Tensor) -> "Int8Weight":
        """The 8-bit form of a bf16, fp16 or fp32 weight: every row by ``quantize_rows``."""
        if weight.dim() not in (2, 3):
            raise NativeError("int8 weight: expected [N, K] or [E, N, K]")
        values, scales = quantize_rows(weight.detach().reshape(-1, weight.size(-1)))
        return Int8Weight(values.view(weight.shape) if values.is_contiguous()
                          else values.reshape(weight.shape), scales.view(weight.shape[:-1]))

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    @property
    def row_stride(self) -> int:
        """Bytes between rows, a multiple of 128."""
        return _padded(self.values.size(-1), _STEP)

    def size(self, dim: int) -> int:
        return self.values.size(dim)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return (self.values.float() * self.scales[..., None]).to(dtype)


@functools.lru_cache(maxsize=4096)
def _linear_workspace(t: int, n: int, k: int, cus: int) -> int:
    """Workspace bytes of a product, -1 for an invalid shape: a function of the sizes alone, kept as
    the question costs 0.6 us of a one-row call's 8."""
    return lib().mi355x_linear_int8_workspace_bytes(t, n, k, cus)


def linear_int8(x: torch.Tensor, weight: Int8Weight, out: torch.Tensor | None = None,
                silu_mul: bool = False) -> torch.Tensor:
    """``x @ weight.T`` in 8-bit integers: ``x`` ``[T, K]`` bf16 or fp16 is quantised a row, the int32
    sums are exact, ``out`` ``[T, N]`` is rounded once. ``silu_mul``: ``weight`` is a gate_up
    projection (gate rows, then up rows) and the result is ``silu(gate) * up`` ``[T, N / 2]``,
    rounded once. Rows that do not overlap may have any stride and alignment; ``out`` may be
    given and must not share memory with ``x``. A row with an inf or a NaN comes out NaN."""
    t, k, ldx = _rows(x, "linear_int8")
    dt = _ROW_DTYPES.get(x.dtype)
    if dt is None or dt == 2:
        raise NativeError(f"linear_int8: expected bfloat16 or float16 tensor, got {x.dtype}")
    if not isinstance(weight, Int8Weight) or weight.values.dim() != 2:
        raise NativeError("linear_int8: expected an Int8Weight [N, K]")
    values, scales = weight.values, weight.scales
    n = values.size(0)
    device = x.device
    if k != values.size(1) or values.get_device() != device.index:
        raise NativeError("linear_int8: expected x [T, K] and a weight [N, K] on one device")
    if silu_mul and n % 2:
        raise NativeError("linear_int8: a gate_up weight has an even number of rows")
    _refuse_grad("linear_int8", x, scales, out)
    out, ldo = _output(out, x, n // 2 if silu_mul else n, "linear_int8")
    cus = device_cus(device)
    need = _linear_workspace(t, n, k, cus)
    if need < 0:
        raise NativeError("linear_int8: invalid shape")
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    with on_device(device):
        check(lib().mi355x_linear_int8(
            x.data_ptr(), ldx, values.data_ptr(), _padded(k, _STEP), scales.data_ptr(),
            out.data_ptr(), ldo, t, n, k, silu_mul, None if ws is None else ws.data_ptr(), need,
            cus, dt, stream_of(x)), "linear_int8")
    return out


__all__ = ["Int8Weight", "linear_int8", "quantize_rows", "NativeError"]
