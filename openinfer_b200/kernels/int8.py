"""8-bit integer layers: rows of numbers held as 8-bit integers with one float32 scale a row, and their product with weights
held the same way (one scale for each output channel).

    rows = rmsnorm_int8(x, norm_weight, eps, delta=branch)       # or quantize_int8(x), silu_mul_int8(gate_up)
    weight = Int8Weight.quantize(w)                              # once, when weights are loaded
    y = linear_int8(rows, weight)

A row y with m = max |y| is held as q = round(y * (127 / m)) (ties to even) and scale = m / 127, so -127..127 are used and the
numbers lie within half a step of y. A row of zeros has scale 0; a row that holds an infinity or a NaN is held as zeros with
the scale NaN, and whatever is made of it is NaN. A product's sums are exact: its result does not depend on which kernel
takes it, on the batch around a row, or on how a long sum is cut.

Every function launches on the current stream of its tensors' device. Results that are not given are allocated; rows start on
16-byte borders (``Int8Rows`` of an odd width are a view into wider rows). Results must not lie in the memory of operands.
"""
from __future__ import annotations

from contextlib import nullcontext
from typing import NamedTuple, Optional

import torch

from . import lib as _lib
from .lib import KernelError
from .ops import act_code

ALIGN = 16                 # bytes that the rows of 8-bit operands start on
MAX_WIDTH = 131071         # the longest sum of products of two 8-bit integers that a 32-bit integer holds: 128 * 128 * 131071 < 2^31

_DT = {torch.float32: 0, torch.bfloat16: 1}


class Int8Rows(NamedTuple):
    """``values`` int8 [rows, width] (rows on 16-byte borders), ``scales`` float32 [rows]: the numbers are values * scales."""
    values: torch.Tensor
    scales: torch.Tensor


def _float_rows(t: torch.Tensor, what: str) -> int:
    """The dtype code of a matrix of floating rows (any row stride, neighbours next to each other)."""
    code = _DT.get(t.dtype)
    if code is None:
        raise KernelError(f"{what}: dtype {t.dtype} is not supported (float32 or bfloat16)")
    if t.dim() != 2 or t.shape[1] < 1 or (t.stride(1) != 1 and t.shape[1] > 1):
        raise KernelError(f"{what}: expected rows of at least one number, neighbours next to each other: shape {tuple(t.shape)}, strides {t.stride()}")
    return code


def _cuda(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise KernelError(f"{what}: the tensor is not on a CUDA device; this package has no CPU path")


def _stride(t: torch.Tensor) -> int:
    """The row stride; where there is one row, its width rounded up to what 8-bit rows start on (the stride then means nothing)."""
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // ALIGN) * ALIGN


def _check_rows(values: torch.Tensor, scales: torch.Tensor, what: str) -> None:
    if values.dtype != torch.int8 or scales.dtype != torch.float32:
        raise KernelError(f"{what}: 8-bit rows are int8 with float32 scales: {values.dtype}, {scales.dtype}")
    if values.dim() != 2 or values.shape[1] < 1 or (values.stride(1) != 1 and values.shape[1] > 1):
        raise KernelError(f"{what}: expected rows of at least one integer, neighbours next to each other: shape {tuple(values.shape)}, strides {values.stride()}")
    rows, width = values.shape
    if values.data_ptr() % ALIGN or (rows > 1 and (values.stride(0) % ALIGN or values.stride(0) < width)):
        raise KernelError(f"{what}: 8-bit rows must start on {ALIGN}-byte borders and not overlap (row stride {values.stride(0)}, width {width})")
    if scales.shape != (rows,) or not scales.is_contiguous():
        raise KernelError(f"{what}: expected {rows} scales in a row: shape {tuple(scales.shape)}")
    if values.device != scales.device:
        raise KernelError(f"{what}: values and scales must be on one device: {values.device}, {scales.device}")


def empty_rows(rows: int, width: int, device) -> Int8Rows:
    """Room for rows of 8-bit integers."""
    room = -(-width // ALIGN) * ALIGN
    values = torch.empty((rows, room), dtype=torch.int8, device=device)
    return Int8Rows(values if room == width else values[:, :width], torch.empty(rows, dtype=torch.float32, device=device))


def _room(out: Optional[Int8Rows], x: torch.Tensor, width: int, what: str) -> Int8Rows:
    if out is None:
        return empty_rows(x.shape[0], width, x.device)
    _check_rows(*out, what)
    if out.values.shape != (x.shape[0], width) or out.values.device != x.device:
        raise KernelError(f"{what}: room for {tuple(out.values.shape)} on {out.values.device}, needed {(x.shape[0], width)} on {x.device}")
    return out


def _on(device: torch.device):
    """The tensors' own device for the launch, whatever the calling thread's current one is."""
    return _HERE if _lib.current_device() == device.index else torch.cuda.device(device)


_HERE = nullcontext()


def _done(L, out: Optional[Int8Rows]) -> None:
    """Rows written into given memory may be those of a weight, which products fetch ahead: the next launch starts behind this one."""
    if out is not None:
        L.oi_launch_fence()


def quantize_int8(x: torch.Tensor, out: Optional[Int8Rows] = None) -> Int8Rows:
    """The rows of ``x`` [rows, width] (float32 or bfloat16, row stride free) as 8-bit integers."""
    code = _float_rows(x, "quantize_int8")
    rows, width = x.shape
    _cuda(x, "quantize_int8")
    held = _room(out, x, width, "quantize_int8")
    if rows:
        with _on(x.device):
            L = _lib.load()
            _lib.check(L.oi_quantize_int8(held.values.data_ptr(), _stride(held.values), held.scales.data_ptr(), x.data_ptr(), code,
                                          x.stride(0), rows, width, _lib.current_stream()), "quantize_int8")
            _done(L, out)
    return held


def rmsnorm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float, *, delta: Optional[torch.Tensor] = None,
                 weight_offset: float = 0.0, out: Optional[Int8Rows] = None) -> Int8Rows:
    """x * rsqrt(mean(x^2) + eps) * (weight_offset + weight), row by row, as 8-bit integers.

    ``delta``: x <- x + delta first (rounded, stored in x), the norm is of the sum as it is stored."""
    code = _float_rows(x, "rmsnorm_int8")
    rows, width = x.shape
    w_code = _DT.get(weight.dtype)
    if w_code is None or weight.shape != (width,) or not weight.is_contiguous() or weight.device != x.device:
        raise KernelError(f"rmsnorm_int8: expected a float32 or bfloat16 weight of {width} numbers on {x.device}: {weight.dtype} {tuple(weight.shape)} on {weight.device}")
    if delta is not None:
        _float_rows(delta, "rmsnorm_int8 delta")
        if delta.dtype != x.dtype or delta.shape != x.shape or delta.device != x.device:
            raise KernelError(f"rmsnorm_int8: x and delta must share a dtype, a shape and a device: {x.dtype} {tuple(x.shape)}, {delta.dtype} {tuple(delta.shape)}")
        if rows > 1 and x.stride(0) < width:
            raise KernelError(f"rmsnorm_int8: rows that overlap (row stride {x.stride(0)}, width {width}) cannot take a sum")
        if (delta.data_ptr(), delta.stride(0)) != (x.data_ptr(), x.stride(0)) and _overlap(x, delta):
            raise KernelError("rmsnorm_int8: x and delta must be the same rows or not overlap")
    _cuda(x, "rmsnorm_int8")
    held = _room(out, x, width, "rmsnorm_int8")
    if rows:
        with _on(x.device):
            L = _lib.load()
            _lib.check(L.oi_rmsnorm_int8(held.values.data_ptr(), _stride(held.values), held.scales.data_ptr(), x.data_ptr(), x.stride(0),
                                         0 if delta is None else delta.data_ptr(), 0 if delta is None else delta.stride(0), code,
                                         weight.data_ptr(), w_code, rows, width, float(eps), float(weight_offset),
                                         _lib.current_stream()), "rmsnorm_int8")
            _done(L, out)
    return held


def silu_mul_int8(gate_up: torch.Tensor, block: Optional[int] = None, act: str = "silu", out: Optional[Int8Rows] = None) -> Int8Rows:
    """act(gate_i) * up_i of a fused gate|up buffer [rows, 2 * inter] as 8-bit integers [rows, inter]; the buffer is laid out in
    blocks of ``block`` gate values followed by their up values (default: all gates, then all ups)."""
    code = _float_rows(gate_up, "silu_mul_int8")
    rows, both = gate_up.shape
    inter = both // 2
    block = inter if block is None else int(block)
    if both % 2 or block < 1 or inter % block:
        raise KernelError(f"silu_mul_int8: gate_up of {both} numbers in blocks of {block} gates and {block} ups")
    act_c = act_code(act)
    _cuda(gate_up, "silu_mul_int8")
    held = _room(out, gate_up, inter, "silu_mul_int8")
    if rows:
        with _on(gate_up.device):
            L = _lib.load()
            _lib.check(L.oi_silu_mul_int8(held.values.data_ptr(), _stride(held.values), held.scales.data_ptr(), gate_up.data_ptr(), code,
                                          gate_up.stride(0), rows, inter, block, act_c, _lib.current_stream()), "silu_mul_int8")
            _done(L, out)
    return held


def dequantize_int8(rows: Int8Rows, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The numbers that 8-bit rows stand for, rounded once to ``dtype`` (float32 or bfloat16)."""
    values, scales = rows
    _check_rows(values, scales, "dequantize_int8")
    if out is None:
        if dtype not in _DT:
            raise KernelError(f"dequantize_int8: dtype {dtype} is not supported (float32 or bfloat16)")
        out = torch.empty(values.shape, dtype=dtype, device=values.device)
    else:
        _check_out(out, values.shape[0], values.shape[1], values.device, "dequantize_int8")
    _cuda(values, "dequantize_int8")
    if values.shape[0]:
        with _on(values.device):
            L = _lib.load()
            _lib.check(L.oi_dequantize_int8(out.data_ptr(), _DT[out.dtype], out.stride(0), values.data_ptr(), _stride(values),
                                            scales.data_ptr(), values.shape[0], values.shape[1], _lib.current_stream()), "dequantize_int8")
    return out


class Int8Weight:
    """A weight [channels, width] for ``linear_int8``: int8 values with a float32 scale for each output channel, laid out once.

    Values whose rows do not start on 16-byte borders are copied into rows that do; others are kept as they are. A product
    fetches its weight while the kernel ahead of it on the stream still runs, but for the first one on each stream. Later
    changes of the weight's tensors (by torch, or through ``out`` of the functions above) are ordered by the stream as ever."""

    __slots__ = ("values", "scales", "channels", "width", "device", "stream")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor) -> None:
        if values.dim() != 2 or values.dtype != torch.int8 or scales.shape != values.shape[:1]:
            raise KernelError(f"Int8Weight: expected int8 [channels, width] and a scale for each channel: {values.dtype} {tuple(values.shape)}, {tuple(scales.shape)}")
        if not 1 <= values.shape[1] <= MAX_WIDTH:
            raise KernelError(f"Int8Weight: sums of {values.shape[1]} products (1 to {MAX_WIDTH} are exact in 32 bits)")
        if values.shape[1] > 1 and values.stride(1) != 1 or values.data_ptr() % ALIGN or values.shape[0] > 1 and (
                values.stride(0) % ALIGN or values.stride(0) < values.shape[1]):
            held = empty_rows(*values.shape, values.device).values
            held.copy_(values)
            values = held
        if not scales.is_contiguous():
            scales = scales.contiguous()
        _check_rows(values, scales, "Int8Weight")
        self.values, self.scales, self.device = values, scales, values.device
        self.channels, self.width = values.shape
        self.stream = None          # the stream of the last product: what wrote the weight is known to be done there

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "Int8Weight":
        """The weight ``w`` [channels, width] (float32 or bfloat16) as 8-bit integers, a scale for each output channel."""
        return cls(*quantize_int8(w))


def linear_int8(x: Int8Rows, weight: Int8Weight, bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [rows, width] times the weight [channels, width], transposed: sums of 8-bit products exact in 32-bit integers, then
    float32(sum) * x's scale * the channel's scale (+ the channel's ``bias``, float32) and one rounding to ``out_dtype``
    (float32 or bfloat16, or that of ``out`` [rows, channels], whose row stride is free)."""
    values, scales = x
    _check_rows(values, scales, "linear_int8")
    rows, width = values.shape
    if width != weight.width or values.device != weight.device:
        raise KernelError(f"linear_int8: rows of {width} on {values.device} and a weight of {weight.channels} x {weight.width} on {weight.device}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (weight.channels,) or not bias.is_contiguous() or bias.device != values.device):
        raise KernelError(f"linear_int8: expected {weight.channels} float32 numbers of bias on {values.device}: {bias.dtype} {tuple(bias.shape)} on {bias.device}")
    if out is None:
        if out_dtype not in _DT:
            raise KernelError(f"linear_int8: output dtype {out_dtype} is not supported (float32 or bfloat16)")
        out = torch.empty((rows, weight.channels), dtype=out_dtype, device=values.device)
    else:
        _check_out(out, rows, weight.channels, values.device, "linear_int8")
    _cuda(values, "linear_int8")
    if rows and weight.channels:
        with _on(values.device):
            L, stream = _lib.load(), _lib.current_stream()
            if weight.stream != stream:
                L.oi_launch_fence()          # the first product on a stream starts when all that is ahead of it has finished
                weight.stream = stream
            _lib.check(L.oi_linear_int8(out.data_ptr(), _DT[out.dtype], out.stride(0), values.data_ptr(), _stride(values), scales.data_ptr(),
                                        weight.values.data_ptr(), _stride(weight.values), weight.scales.data_ptr(),
                                        0 if bias is None else bias.data_ptr(), rows, weight.channels, width, stream), "linear_int8")
    return out


def status() -> int:
    """0, or which bounded wait of a product ran out since the last call (synchronises the device)."""
    from ctypes import byref, c_int
    v = c_int(0)
    _lib.check(_lib.load().oi_linear_int8_status(byref(v)), "linear_int8_status")
    return v.value


def _check_out(out: torch.Tensor, rows: int, width: int, device: torch.device, what: str) -> None:
    if out.dtype not in _DT or out.shape != (rows, width) or out.device != device:
        raise KernelError(f"{what}: expected float32 or bfloat16 results [{rows}, {width}] on {device}: {out.dtype} {tuple(out.shape)} on {out.device}")
    if (width > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < width):
        raise KernelError(f"{what}: result rows must not overlap, neighbours next to each other: strides {out.stride()}")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices of rows share bytes (or may)."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size()
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1
