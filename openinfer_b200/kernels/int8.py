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

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from . import lib as _lib
from .lib import KernelError
from .ops import act_code

MOST = 1 << 30             # rows, and numbers of a row
ALIGN = 16                 # bytes that the rows of 8-bit operands start on
# Rows that are allocated here are a multiple of so many bytes apart: 128 bytes of a row then lie in as few lines of the caches as they
# can (rows 16 bytes off: 2538 x 7746 x 11239 186 us, 149 so; 264 x 4096 x 12200 27.9 and 19.7; 1 x 6144 x 4100 7.6 and 7.3).
APART = 64
MAX_WIDTH = 131071         # the longest sum of products of two 8-bit integers that a 32-bit integer holds: 128 * 128 * 131071 < 2^31

_DT = {torch.float32: 0, torch.bfloat16: 1}


class Int8Rows(NamedTuple):
    """``values`` int8 [rows, width] (rows on 16-byte borders), ``scales`` float32 [rows]: the numbers are values * scales."""
    values: torch.Tensor
    scales: torch.Tensor


_new_rows = tuple.__new__


# At a few rows a call's time is the host's. So a tensor is asked for each thing once, one test covers all that may be wrong, and what
# exactly it was is found out behind it.

def _float_rows(t: torch.Tensor, what: str) -> Tuple[int, int, int, int]:
    """(dtype code, rows, width, row stride) of a matrix of floating rows (any row stride, neighbours next to each other)."""
    code, shape, strides = _DT.get(t.dtype), t.shape, t.stride()
    if code is not None and len(shape) == 2:
        rows, width = shape
        if (strides[1] == 1 and 0 < width <= MOST or width == 1) and rows <= MOST:
            return code, rows, width, strides[0]
    if code is None:
        raise KernelError(f"{what}: dtype {t.dtype} is not supported (float32 or bfloat16)")
    raise KernelError(f"{what}: expected rows of at least one number, neighbours next to each other (at most {MOST} of either): shape {tuple(shape)}, strides {strides}")


def _int8_rows(values: torch.Tensor, scales: torch.Tensor, what: str) -> Tuple[int, int, int, int, int, int]:
    """(address, row stride, rows, width, address of the scales, device index) of 8-bit rows. The stride of one row is its width
    rounded up to what rows start on (it means nothing then)."""
    if values.dtype != torch.int8 or scales.dtype != torch.float32:
        raise KernelError(f"{what}: 8-bit rows are int8 with float32 scales: {values.dtype}, {scales.dtype}")
    shape, strides = values.shape, values.stride()
    if len(shape) != 2 or not 0 < shape[1] <= MOST or (strides[1] != 1 and shape[1] > 1) or shape[0] > MOST:
        raise KernelError(f"{what}: expected rows of at least one integer, neighbours next to each other (at most {MOST} of either): shape {tuple(shape)}, strides {strides}")
    rows, width = shape
    address, stride = values.data_ptr(), strides[0] if rows > 1 else -(-width // ALIGN) * ALIGN
    if address % ALIGN or stride % ALIGN or stride < width:
        raise KernelError(f"{what}: 8-bit rows must start on {ALIGN}-byte borders and not overlap (row stride {stride}, width {width})")
    if scales.shape != (rows,) or not scales.is_contiguous():
        raise KernelError(f"{what}: expected {rows} scales in a row: shape {tuple(scales.shape)}")
    device = values.get_device()
    if device != scales.get_device():
        raise KernelError(f"{what}: values and scales must be on one device: {values.device}, {scales.device}")
    return address, stride, rows, width, scales.data_ptr(), device


def _cuda(device: int, what: str) -> None:
    if device < 0:
        raise KernelError(f"{what}: the tensor is not on a CUDA device; this package has no CPU path")


def _elsewhere(device: int) -> bool:
    """Whether tensors are on another CUDA device than the calling thread's current one: the call is then made again on theirs."""
    return device >= 0 and device != _lib.current_device()


def empty_rows(rows: int, width: int, device) -> Int8Rows:
    """Room for rows of 8-bit integers."""
    values = (torch.empty_strided((rows, width), (-(-width // APART) * APART, 1), dtype=torch.int8, device=device) if width % APART
              else torch.empty(rows, width, dtype=torch.int8, device=device))
    return _new_rows(Int8Rows, (values, torch.empty(rows, dtype=torch.float32, device=device)))


def _room(out: Optional[Int8Rows], x: torch.Tensor, rows: int, width: int, device: int, what: str):
    """(8-bit rows, their address, row stride, address of the scales)"""
    if device < 0:
        _cuda(device, what)
    if out is None:
        out = values, scales = empty_rows(rows, width, x.device)
        return out, values.data_ptr(), -(-width // APART) * APART, scales.data_ptr()
    address, stride, has_rows, has_width, scales, on = _int8_rows(*out, what)
    if (has_rows, has_width, on) != (rows, width, device):
        raise KernelError(f"{what}: room for {(has_rows, has_width)} on {out[0].device}, needed {(rows, width)} on {x.device}")
    return out, address, stride, scales


def _written(L, held: Int8Rows) -> None:
    """Given rows have been written. They may be those of a weight, which products fetch ahead: a product by it sees the change, on
    whatever stream it is, and this thread's next launch starts behind this one."""
    L.oi_launch_fence()
    if not held[0].is_inference():
        increment_version(held[0])


def quantize_int8(x: torch.Tensor, out: Optional[Int8Rows] = None) -> Int8Rows:
    """The rows of ``x`` [rows, width] (float32 or bfloat16, row stride free) as 8-bit integers."""
    code, rows, width, stride = _float_rows(x, "quantize_int8")
    device = x.get_device()
    if _elsewhere(device):
        with torch.cuda.device(device):
            return quantize_int8(x, out)
    held, q, ldq, scales = _room(out, x, rows, width, device, "quantize_int8")
    if rows:
        L = _lib.load()
        failed = L.oi_quantize_int8(q, ldq, scales, x.data_ptr(), code, stride, rows, width, out is None, _lib.current_stream())
        if failed:
            _lib.check(failed, "quantize_int8")
        if out is not None:
            _written(L, held)
    return held


def rmsnorm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float, *, delta: Optional[torch.Tensor] = None,
                 weight_offset: float = 0.0, out: Optional[Int8Rows] = None) -> Int8Rows:
    """x * rsqrt(mean(x^2) + eps) * (weight_offset + weight), row by row, as 8-bit integers. A row's integers are made of x * (weight_offset
    + weight), its root mean square goes into the scale: a number within float32's rounding of a half may become either neighbour.

    ``delta``: x <- x + delta first (rounded, stored in x), the norm is of the sum as it is stored."""
    code, rows, width, stride = _float_rows(x, "rmsnorm_int8")
    device, address, w_code = x.get_device(), x.data_ptr(), _DT.get(weight.dtype)
    if w_code is None or weight.shape != (width,) or not weight.is_contiguous() or weight.get_device() != device:
        raise KernelError(f"rmsnorm_int8: expected a float32 or bfloat16 weight of {width} numbers on {x.device}: {weight.dtype} {tuple(weight.shape)} on {weight.device}")
    d_address = d_stride = 0
    if delta is not None:
        if delta.dtype != x.dtype or delta.shape != x.shape or delta.get_device() != device:
            raise KernelError(f"rmsnorm_int8: x and delta must share a dtype, a shape and a device: {x.dtype} {tuple(x.shape)} on {x.device}, {delta.dtype} {tuple(delta.shape)} on {delta.device}")
        d_stride, d_address = _float_rows(delta, "rmsnorm_int8 delta")[3], delta.data_ptr()
        if rows > 1 and stride < width:
            raise KernelError(f"rmsnorm_int8: rows that overlap (row stride {stride}, width {width}) cannot take a sum")
        size = 2 if code else 4
        if (d_address < address + ((rows - 1) * stride + width) * size and address < d_address + ((rows - 1) * d_stride + width) * size
                and rows and (d_address, d_stride if rows > 1 else stride) != (address, stride)      # one row's stride means nothing
                and not (d_stride == stride > 0 and width <= (d_address - address) // size % stride <= stride - width)):    # rows in turn
            raise KernelError("rmsnorm_int8: x and delta must be the same rows or not overlap")
    if _elsewhere(device):
        with torch.cuda.device(device):
            return rmsnorm_int8(x, weight, eps, delta=delta, weight_offset=weight_offset, out=out)
    held, q, ldq, scales = _room(out, x, rows, width, device, "rmsnorm_int8")
    if rows:
        L = _lib.load()
        failed = L.oi_rmsnorm_int8(q, ldq, scales, address, stride, d_address, d_stride, code, weight.data_ptr(), w_code, rows, width, eps,
                                   weight_offset, out is None, _lib.current_stream())
        if failed:
            _lib.check(failed, "rmsnorm_int8")
        if out is not None:
            _written(L, held)
    return held


def silu_mul_int8(gate_up: torch.Tensor, block: Optional[int] = None, act: str = "silu", out: Optional[Int8Rows] = None) -> Int8Rows:
    """act(gate_i) * up_i of a fused gate|up buffer [rows, 2 * inter] as 8-bit integers [rows, inter]; the buffer is laid out in
    blocks of ``block`` gate values followed by their up values (default: all gates, then all ups). ``act``: "silu" or "gelu_tanh"."""
    code, rows, both, stride = _float_rows(gate_up, "silu_mul_int8")
    inter = both // 2
    block = inter if block is None else int(block)
    if both % 2 or block < 1 or inter % block:
        raise KernelError(f"silu_mul_int8: gate_up of {both} numbers in blocks of {block} gates and {block} ups")
    act_c = act_code(act)
    device = gate_up.get_device()
    if _elsewhere(device):
        with torch.cuda.device(device):
            return silu_mul_int8(gate_up, block, act, out)
    held, q, ldq, scales = _room(out, gate_up, rows, inter, device, "silu_mul_int8")
    if rows:
        L = _lib.load()
        failed = L.oi_silu_mul_int8(q, ldq, scales, gate_up.data_ptr(), code, stride, rows, inter, block, act_c, out is None, _lib.current_stream())
        if failed:
            _lib.check(failed, "silu_mul_int8")
        if out is not None:
            _written(L, held)
    return held


def _results(out: Optional[torch.Tensor], dtype: torch.dtype, rows: int, width: int, like: torch.Tensor, device: int, what: str):
    """(results [rows, width], their dtype code, row stride)"""
    if out is None:
        code = _DT.get(dtype)
        if code is None:
            raise KernelError(f"{what}: output dtype {dtype} is not supported (float32 or bfloat16)")
        _cuda(device, what)
        return torch.empty(rows, width, dtype=dtype, device=like.device), code, width
    code, shape, strides = _DT.get(out.dtype), out.shape, out.stride()
    if code is None or shape != (rows, width) or out.get_device() != device:
        raise KernelError(f"{what}: expected float32 or bfloat16 results [{rows}, {width}] on {like.device}: {out.dtype} {tuple(shape)} on {out.device}")
    if (width > 1 and strides[1] != 1) or (rows > 1 and strides[0] < width):
        raise KernelError(f"{what}: result rows must not overlap, neighbours next to each other: strides {strides}")
    _cuda(device, what)
    return out, code, strides[0]


def dequantize_int8(rows: Int8Rows, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The numbers that 8-bit rows stand for, rounded once to ``dtype`` (float32 or bfloat16) or to that of ``out`` (row stride free).
    They may be a weight, which a product fetches ahead: the next kernel on the stream starts when they are written."""
    q, ldq, count, width, scales, device = _int8_rows(*rows, "dequantize_int8")
    if _elsewhere(device):
        with torch.cuda.device(device):
            return dequantize_int8(rows, dtype, out)
    out, code, stride = _results(out, dtype, count, width, rows[0], device, "dequantize_int8")
    if count:
        failed = _lib.load().oi_dequantize_int8(out.data_ptr(), code, stride, q, ldq, scales, count, width, _lib.current_stream())
        if failed:
            _lib.check(failed, "dequantize_int8")
    return out


class Int8Weight:
    """A weight [channels, width] for ``linear_int8``: int8 values with a float32 scale for each output channel, laid out once.

    Values whose rows do not start on 16-byte borders, or are wider than 64 and not a multiple of 64 bytes apart, are copied into rows
    that are; others are kept as they are. A product fetches its weight's values while the kernel ahead of it on the stream still
    runs, but for the first one on each stream and the first one after a change of the weight's tensors, by torch or through ``out``
    of the functions above. Of a change that torch does not count (through ``.data``, or of tensors made in inference mode) tell
    with ``changed()``."""

    __slots__ = ("values", "scales", "stream", "_seen", "_operands")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor) -> None:
        if values.dim() != 2 or values.dtype != torch.int8 or scales.shape != values.shape[:1]:
            raise KernelError(f"Int8Weight: expected int8 [channels, width] and a scale for each channel: {values.dtype} {tuple(values.shape)}, {tuple(scales.shape)}")
        rows, width = values.shape
        if not 1 <= width <= MAX_WIDTH:
            raise KernelError(f"Int8Weight: sums of {width} products (1 to {MAX_WIDTH} are exact in 32 bits)")
        strides = values.stride()
        if (width > 1 and strides[1] != 1) or values.data_ptr() % ALIGN or (rows > 1 and (
                strides[0] % (APART if width > APART else ALIGN) or strides[0] < width)):
            held = empty_rows(rows, width, values.device).values
            held.copy_(values)
            values = held
        self.values, self.scales = values, scales.contiguous()
        self.stream = None          # of the last product: what wrote the weight is known to be done there
        self.operands()

    def __setattr__(self, name: str, value) -> None:
        object.__setattr__(self, name, value)
        if name in ("values", "scales"):
            object.__setattr__(self, "stream", None)      # other tensors: as after a change, and looked at before the next product
            object.__setattr__(self, "_seen", None)

    @property
    def channels(self) -> int:
        return self.values.shape[0]

    @property
    def width(self) -> int:
        return self.values.shape[1]

    @property
    def device(self) -> torch.device:
        return self.values.device

    def changed(self) -> None:
        """The weight's tensors hold new values: the next product waits for what is ahead of it."""
        self.stream = None

    def operands(self):
        """What ``_int8_rows`` says of the weight; asked again when its tensors have been given other memory or values."""
        values, scales = self.values, self.scales
        seen = (values.data_ptr(), scales.data_ptr(), values.shape, values.stride(), values.dtype, scales.shape, scales.stride(), scales.dtype,
                None if values.is_inference() else values._version)
        if seen != self._seen:
            self._operands = _int8_rows(values, scales, "Int8Weight")
            self._seen, self.stream = seen, None
        return self._operands

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "Int8Weight":
        """The weight ``w`` [channels, width] (float32 or bfloat16) as 8-bit integers, a scale for each output channel."""
        return cls(*quantize_int8(w))


def linear_int8(x: Int8Rows, weight: Int8Weight, bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [rows, width] times the weight [channels, width], transposed: sums of 8-bit products exact in 32-bit integers, then
    float32(sum) * x's scale * the channel's scale (+ the channel's ``bias``, float32) and one rounding to ``out_dtype``
    (float32 or bfloat16, or that of ``out`` [rows, channels], whose row stride is free)."""
    q, ldq, rows, width, scales, device = _int8_rows(*x, "linear_int8")
    w, ldw, channels, w_width, w_scales, w_device = weight.operands()
    if width != w_width or device != w_device:
        raise KernelError(f"linear_int8: rows of {width} on {x[0].device} and a weight of {channels} x {w_width} on {weight.device}")
    if _elsewhere(device):
        with torch.cuda.device(device):
            return linear_int8(x, weight, bias, out_dtype, out)
    b = 0
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (channels,) or not bias.is_contiguous() or bias.get_device() != device:
            raise KernelError(f"linear_int8: expected {channels} float32 numbers of bias on {x[0].device}: {bias.dtype} {tuple(bias.shape)} on {bias.device}")
        b = bias.data_ptr()
    out, code, out_stride = _results(out, out_dtype, rows, channels, x[0], device, "linear_int8")
    if rows and channels:
        L, stream = _lib.load(), _lib.current_stream()
        if weight.stream != stream:
            L.oi_launch_fence()          # the first product on a stream starts when all that is ahead of it has finished
        failed = L.oi_linear_int8(out.data_ptr(), code, out_stride, q, ldq, scales, w, ldw, w_scales, b, rows, channels, width, stream)
        if failed:
            weight.stream = None
            _lib.check(failed, "linear_int8")
        if weight.stream != stream:
            weight.stream = stream
    return out


def status() -> int:
    """0, or which bounded wait of a product ran out since the last call: what it would have made is NaN (synchronises the device)."""
    from ctypes import byref, c_int
    v = c_int(0)
    _lib.check(_lib.load().oi_linear_int8_status(byref(v)), "linear_int8_status")
    return v.value
