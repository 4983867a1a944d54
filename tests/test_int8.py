"""8-bit rows and products: what is refused, without a GPU."""
import ctypes

import pytest
import torch

from openinfer_b200.kernels import int8
from openinfer_b200.kernels import lib as klib
from openinfer_b200.kernels.lib import KernelError

ROWS = torch.zeros(3, 32, dtype=torch.int8)
SCALES = torch.ones(3)
X = torch.zeros(3, 32)


def refused(words, call, *args, **kw):
    with pytest.raises(KernelError, match=words):
        call(*args, **kw)


def test_rows_that_are_not_rows_of_8_bit_integers():
    def held(values, scales=SCALES):
        refused(words, int8.dequantize_int8, int8.Int8Rows(values, scales))
    words = "int8 with float32 scales"
    held(ROWS.to(torch.uint8))
    held(ROWS, SCALES.double())
    words = "at least one integer"
    held(ROWS[0])
    held(ROWS[:, :0])
    held(torch.zeros(32, 3, dtype=torch.int8).t())
    words = "16-byte borders"
    held(torch.zeros(3, 33, dtype=torch.int8))
    held(torch.zeros(3, 48, dtype=torch.int8)[:, 1:33])
    held(torch.zeros(1, 32, dtype=torch.int8).expand(3, 32))
    words = "3 scales"
    held(ROWS, torch.ones(2))
    held(ROWS, torch.ones(6)[::2])
    words = "not on a CUDA device"
    held(ROWS)
    held(torch.zeros(3, 48, dtype=torch.int8)[:, :33])       # an odd width in rows of 48


def test_floating_rows():
    for call in (int8.quantize_int8, int8.silu_mul_int8, lambda x: int8.rmsnorm_int8(x, torch.ones(32), 1e-6)):
        refused("float16 is not supported", call, X.half())
        refused("neighbours next to each other", call, torch.zeros(32, 3).t())
        refused("neighbours next to each other", call, torch.zeros(32))
        refused("at least one number", call, X[:, :0])
        refused("not on a CUDA device", call, X)


def test_more_rows_than_an_entry_point_counts():
    many = torch.zeros(1, 1).expand(2 ** 31 + 5, 1)
    refused("at most 1073741824", int8.quantize_int8, many)
    refused("at most 1073741824", int8.dequantize_int8, int8.Int8Rows(torch.zeros(1, 1, dtype=torch.int8).expand(2 ** 31 + 5, 1), torch.ones(3)))


def test_a_weight_that_torch_changes_is_waited_for_again():
    w = int8.Int8Weight(ROWS.clone(), SCALES.clone())
    w.operands()
    w.stream = 7
    w.operands()
    assert w.stream == 7
    w.values.fill_(3)
    w.operands()
    assert w.stream is None
    w.stream = 7
    w.changed()
    assert w.stream is None
    with torch.inference_mode():
        w = int8.Int8Weight(ROWS.clone(), SCALES.clone())
    w.stream = 7
    w.operands()
    assert w.stream == 7


def test_norm():
    def norm(x=X, w=torch.ones(32), **kw):
        int8.rmsnorm_int8(x, w, 1e-6, **kw)
    refused("weight of 32 numbers", norm, w=torch.ones(31))
    refused("weight of 32 numbers", norm, w=torch.ones(32).half())
    refused("weight of 32 numbers", norm, w=torch.ones(64)[::2])
    refused("must share", norm, delta=X.bfloat16())
    refused("must share", norm, delta=X[:2])
    refused("cannot take a sum", norm, x=torch.zeros(1, 32).expand(3, 32), delta=X)
    both = torch.zeros(4, 32)
    refused("not overlap", norm, x=both[:3], delta=both[1:])
    refused("not on a CUDA device", norm, x=both[:2], delta=both[2:])
    refused("not on a CUDA device", norm, x=X, delta=X)


def test_gate():
    refused("33 numbers", int8.silu_mul_int8, torch.zeros(3, 33))
    refused("blocks of 5", int8.silu_mul_int8, X, block=5)
    refused("blocks of 0", int8.silu_mul_int8, X, block=0)
    refused("has no kernel", int8.silu_mul_int8, X, act="relu")


def test_weight_and_product():
    refused("a scale for each channel", int8.Int8Weight, ROWS, torch.ones(2))
    refused("a scale for each channel", int8.Int8Weight, ROWS.float(), SCALES)
    refused("exact in 32 bits", int8.Int8Weight, torch.zeros(1, int8.MAX_WIDTH + 1, dtype=torch.int8), torch.ones(1))
    refused("exact in 32 bits", int8.Int8Weight, ROWS[:, :0], SCALES)
    refused("float32 scales", int8.Int8Weight, ROWS, SCALES.bfloat16())
    w = int8.Int8Weight(torch.ones(5, 33, dtype=torch.int8), torch.ones(10)[::2])     # laid out in rows of 64
    assert w.values.stride() == (64, 1) and bool((w.values == 1).all()) and w.scales.is_contiguous()
    wide = int8.Int8Weight(torch.arange(4 * 80).view(4, 80).to(torch.int8), torch.ones(4))
    assert wide.values.stride() == (128, 1) and torch.equal(wide.values, torch.arange(4 * 80).view(4, 80).to(torch.int8))
    kept = int8.Int8Weight(ROWS, SCALES)
    assert kept.values.data_ptr() == ROWS.data_ptr()
    rows = int8.Int8Rows(ROWS, SCALES)
    refused("rows of 32 on cpu and a weight of 5 x 33", int8.linear_int8, rows, w)
    refused("3 float32 numbers of bias", int8.linear_int8, rows, kept, bias=torch.ones(3).bfloat16())
    refused("3 float32 numbers of bias", int8.linear_int8, rows, kept, bias=torch.ones(4))
    refused("float16 is not supported", int8.linear_int8, rows, kept, out_dtype=torch.float16)
    refused(r"results \[3, 3\]", int8.linear_int8, rows, kept, out=torch.empty(3, 4))
    refused("must not overlap", int8.linear_int8, rows, kept, out=torch.empty(3, 3).t())
    refused("must not overlap", int8.linear_int8, rows, kept, out=torch.empty(1, 3).expand(3, 3))
    refused("not on a CUDA device", int8.linear_int8, rows, kept)


@pytest.mark.parametrize("name,args", [
    ("oi_quantize_int8", (1, 32, 1, 1, 7, 32, 1, 32, 1)),                     # an unknown dtype
    ("oi_quantize_int8", (1, 32, 1, 1, 0, 32, -1, 32, 1)),
    ("oi_quantize_int8", (1, 32, 1, 1, 0, 32, 1, 0, 1)),
    ("oi_quantize_int8", (0, 32, 1, 1, 0, 32, 1, 32, 1)),
    ("oi_quantize_int8", (1, 16, 1, 1, 0, 32, 2, 32, 1)),                     # rows that overlap
    ("oi_quantize_int8", (1, 1 << 31, 1, 1, 0, 32, 1, (1 << 30) + 1, 1)),
    ("oi_dequantize_int8", (1, 0, 1 << 31, 1, 1 << 31, 1, 1, (1 << 30) + 1)),
    ("oi_linear_int8", (16, 1, 8, 16, 32, 16, 16, 32, 16, 0, (1 << 30) + 1, 8, 32)),
    ("oi_rmsnorm_int8", (1, 32, 1, 1, 16, 1, 32, 0, 1, 0, 2, 32, 1e-6, 0.0, 1)),
    ("oi_rmsnorm_int8", (1, 32, 1, 1, 32, 0, 0, 0, 1, 5, 2, 32, 1e-6, 0.0, 1)),
    ("oi_silu_mul_int8", (1, 32, 1, 1, 0, 64, 1, 32, 5, 1, 1)),
    ("oi_silu_mul_int8", (1, 32, 1, 1, 0, 64, 1, 32, 32, 9, 1)),
    ("oi_dequantize_int8", (1, 5, 32, 1, 32, 1, 1, 32)),
    ("oi_dequantize_int8", (1, 0, 16, 1, 32, 1, 2, 32)),
    ("oi_linear_int8", (16, 1, 8, 16, 32, 16, 16, 32, 16, 0, 4, 8, 131072)),   # a sum that 32 bits may not hold
    ("oi_linear_int8", (16, 1, 8, 8, 32, 16, 16, 32, 16, 0, 4, 8, 32)),        # off the 16-byte border
    ("oi_linear_int8", (16, 1, 8, 16, 33, 16, 16, 32, 16, 0, 4, 8, 32)),
    ("oi_linear_int8", (16, 1, 8, 16, 32, 16, 16, 16, 16, 0, 4, 8, 32)),
    ("oi_linear_int8", (16, 1, 4, 16, 32, 16, 16, 32, 16, 0, 4, 8, 32)),       # result rows that overlap
    ("oi_linear_int8", (16, 6, 8, 16, 32, 16, 16, 32, 16, 0, 4, 8, 32)),
])
def test_the_library_refuses_before_it_launches(name, args):
    L = klib.load(verbose=False)
    assert getattr(L, name)(*args, None) == 1
    assert name[3:].encode() in L.oi_last_error()


def test_a_weight_given_other_tensors_is_waited_for_again():
    w = int8.Int8Weight(ROWS.clone(), SCALES.clone())
    for name in ("values", "scales"):
        w.stream = 7
        setattr(w, name, getattr(w, name).clone())
        assert w.stream is None
    w.stream = 7
    w.operands()
    assert w.stream is None                          # the new values' place is seen
    w.stream = 7
    w.operands()
    assert w.stream == 7


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: the launches have to fail")
def test_the_kernel_behind_a_way_back_starts_when_that_has_finished():
    """What ``dequantize_int8`` writes may be a weight, which products fetch ahead: the next launch on its stream, and on no other, is in
    plain stream order."""
    L = klib.load(verbose=False)
    null, legacy, own = None, 1, 2                   # streams that are there without a device
    for stream, others in ((null, (legacy, own)), (own, (null, legacy))):
        L.oi_dequantize_int8(16, 1, 32, 16, 32, 16, 1, 32, stream)
        assert L.oi_stream_fence_pending(stream) == 1
        for other in others:
            L.oi_quantize_int8(16, 32, 16, 16, 0, 32, 1, 32, 1, other)
            assert L.oi_stream_fence_pending(other) == 0 and L.oi_stream_fence_pending(stream) == 1
        L.oi_quantize_int8(16, 32, 16, 16, 0, 32, 1, 32, 1, stream)
        assert L.oi_stream_fence_pending(stream) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: the launches have to fail")
@pytest.mark.parametrize("name,args", [
    ("oi_quantize_int8", (16, 32, 16, 16, 0, 32, 1, 32, 1)),
    ("oi_rmsnorm_int8", (16, 32, 16, 16, 32, 0, 0, 0, 16, 0, 1, 32, 1e-6, 0.0, 1)),
    ("oi_silu_mul_int8", (16, 32, 16, 16, 0, 64, 1, 32, 32, 1, 1)),
    ("oi_dequantize_int8", (16, 1, 32, 16, 32, 16, 1, 32)),
    ("oi_dequantize_int8", (16, 0, 32, 16, 32, 16, 1, 32)),
    ("oi_linear_int8", (16, 1, 8, 16, 32, 16, 16, 32, 16, 0, 1, 8, 32)),
])
def test_a_launch_that_fails_is_an_error_of_its_call(name, args):
    L = klib.load(verbose=False)
    assert getattr(L, name)(*args, None) > 1


def test_a_weight_given_tensors_of_another_kind():
    def product(w, x=ROWS, words="not on a CUDA device"):
        refused(words, int8.linear_int8, int8.Int8Rows(x, torch.ones(len(x))), w)

    b = torch.arange(1.0, 7.0)
    w = int8.Int8Weight(ROWS.clone(), b[:3])
    product(w)
    w.scales = b[::2]                                          # at the same address, every other one
    product(w, words="3 scales")
    w.scales = b[:3]
    w.scales.data = b[::2]                                     # the same without an assignment to the weight
    product(w, words="3 scales")
    w.scales = b[:3]
    w.values = w.values.view(torch.uint8)                      # the same bytes, other numbers
    product(w, words="int8 with float32 scales")
    w.values = ROWS.clone()
    w.values.data = w.values.view(torch.uint8)
    product(w, words="int8 with float32 scales")
    w.values, w.scales = torch.zeros(5, 64, dtype=torch.int8), torch.ones(5)
    assert (w.channels, w.width, w.device) == (5, 64, torch.device("cpu"))
    product(w, words="a weight of 5 x 64")
    product(w, x=torch.zeros(3, 64, dtype=torch.int8))


@pytest.mark.parametrize("first,second", [(False, True), (True, False)])
def test_a_weight_given_tensors_of_inference_mode_or_other_ones(first, second):
    """Changes of ordinary tensors are seen whatever the weight was made with; those of inference mode are told with ``changed``."""
    def made(inference):
        with torch.inference_mode(inference):
            return ROWS.clone()
    w = int8.Int8Weight(made(first), SCALES.clone())
    w.values = made(second)
    w.operands()
    w.stream = 7
    w.operands()
    assert w.stream == 7
    with torch.inference_mode(second):
        w.values.fill_(3)
    w.operands()
    assert w.stream == (7 if second else None)


def choice(dtype, on_borders, rows, channels, width):
    """(kernel, rows of x a tile, slices of the sum, tiles, stages, partial sums over the ring) of a product"""
    L, said = klib.load(verbose=False), (ctypes.c_int * 6)()
    assert L.oi_linear_int8_choice(int8._DT[dtype], on_borders, rows, channels, width, said) == 0
    return tuple(said)


def test_no_tile_of_a_product_lies_behind_the_last_row():
    """Tiles are a multiple of sixteen rows high: as many as were asked for of that height may be more than there are rows for."""
    for rows in [*range(1, 1200), *range(1200, 4097, 13)]:
        for channels, width in ((128, 16384), (4096, 4096), (1000, 7000), (300, 1000)):
            kernel, tile, slices, tiles, stages, over = choice(torch.bfloat16, True, rows, channels, width)
            along = tiles // -(-channels // (16, 128, 256)[kernel])
            assert (along - 1) * tile < rows <= along * tile and stages >= 1


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: the launches have to fail")
@pytest.mark.parametrize("rows,width", [(1, 1 << 30), (1, (1 << 28) + 5), (3, 1 << 30), (1 << 30, 1)])
def test_rows_of_every_length_that_are_made_are_brought_back(rows, width):
    """The launch is come to (and fails): no size that ``quantize_int8`` takes is refused."""
    L = klib.load(verbose=False)
    assert L.oi_quantize_int8(16, width, 16, 16, 1, width, rows, width, 1, None) > 1
    for code in (0, 1):
        assert L.oi_dequantize_int8(16, code, width, 16, width, 16, rows, width, None) > 1


def test_one_row_is_itself_whatever_its_stride():
    wide = torch.zeros(4, 64)
    x = wide[2:3, :32]
    same = x.as_strided((1, 32), (32, 1))
    for a, b in ((x, same), (same, x)):
        refused("not on a CUDA device", lambda: int8.rmsnorm_int8(a, torch.ones(32), 1e-6, delta=b))
    refused("not overlap", lambda: int8.rmsnorm_int8(x, torch.ones(32), 1e-6, delta=wide[2:3, 16:48]))
