"""8-bit rows and their products on the GPU against plain statements in 64 bits and in exact integers.

What is tested bit for bit: products (their sums are whole numbers, and float32(sum) * sx * sw + bias is three float32
operations in a stated order), the rows of ``quantize_int8`` and ``dequantize_int8`` (likewise). Norms and gates are held to
bounds that follow from their roundings.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24                  # half a step of float32, relative
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def int8():
    from openinfer_b200.kernels import int8, lib
    lib.load()
    yield int8
    assert int8.status() == 0          # no bounded wait has run out


def randn(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed + 1000 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def strided(t, pad, dtype=None):
    """The same numbers on the device in rows that lie further apart, the room between them filled with what must not be read."""
    t = t if dtype is None else t.to(dtype)
    wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan") if t.is_floating_point() else 99, dtype=t.dtype, device=DEV)
    wide[:, :t.shape[1]] = t.to(DEV)
    return wide[:, :t.shape[1]]


def held_exactly(y):
    """What the definition says of float32 rows, in float32 operations: q = round(y * (127 / m)), scale = m / 127."""
    m = y.abs().amax(dim=1)
    top = torch.full_like(m, 127)            # a tensor: torch takes 127 / m as 127 times a rounded reciprocal
    q = torch.round(y * torch.where(m > 0, top / m, torch.zeros(()))[:, None])
    return q.to(torch.int8), m / top


def check_held(rows, y, err):
    """``rows`` against numbers y in 64 bits, of which the kernel's differ by at most ``err`` (relative, per element): the scale is
    off by the largest number's error and one rounding; q lies within half of y / scale and what the errors of y and of the two
    float32 roundings of y * (127 / m) add."""
    q, s = rows.values.cpu().double(), rows.scales.cpu().double()
    m = y.abs().amax(dim=1)
    worst = (err * y.abs() / m[:, None]).amax(dim=1) + 2 * U       # of m, relative
    assert ((s - m / 127).abs() <= (worst + U) * m / 127).all()
    room = 0.5 + (y.abs() * 127 / m[:, None]) * (err + worst[:, None] + 3 * U)
    off = (q - y * (127 / m)[:, None]).abs()
    assert (off <= room).all(), (off - room).max()
    assert int(q.abs().max()) <= 127


# ------------------------------------------------------------------------------------------------------------ plain rows
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (5, 64), (2, 100), (7, 1000), (1, 4096), (130, 257), (3, 5001), (2, 12288), (1, 40000), (2, 70001)])
def test_rows(int8, dtype, rows, width):
    x = randn(rows, width, scale=3.0).to(dtype)
    q, s = held_exactly(x.float())
    for at in (x.to(DEV), strided(x, 3), strided(x, 8)):
        held = int8.quantize_int8(at)
        assert torch.equal(held.values.cpu(), q) and torch.equal(held.scales.cpu(), s)
        assert held.values.data_ptr() % 16 == 0 and (rows == 1 or held.values.stride(0) % 16 == 0)
    for to in DTYPES:
        assert torch.equal(int8.dequantize_int8(held, to).cpu(), (q.float() * s[:, None]).to(to))
    out = strided(torch.zeros(rows, width), 5)
    int8.dequantize_int8(held, out=out)
    assert torch.equal(out.cpu(), q.float() * s[:, None])
    if rows > 1:
        assert bool(torch.isnan(out.as_strided((rows - 1, 5), out.stride(), out.storage_offset() + width)).all())   # the room between rows


@pytest.mark.parametrize("width", [33, 64, 512, 4096, 40000])
def test_rows_of_extreme_numbers(int8, width):
    big, small, sub = 3.0e38, 2.0e-36, 1.0e-41
    x = randn(9, width)
    x[0] = 0.0
    x[1, -1] = float("inf")
    x[2, width // 2] = float("nan")
    x[3, 0], x[3, 1] = float("-inf"), float("nan")
    x[4] *= big / x[4].abs().max()
    x[5] *= small / x[5].abs().max()
    x[6] = 0.0
    x[6, 3] = -sub                       # below the normal numbers: 127 / m alone would be infinite
    x[7, 5] = -0.0
    held = int8.quantize_int8(x.to(DEV))
    q, s = held.values.cpu(), held.scales.cpu()
    assert not q[0].any() and s[0] == 0
    for r in (1, 2, 3):
        assert not q[r].any() and torch.isnan(s[r])
    ref_q, ref_s = held_exactly(x)
    for r in (4, 7, 8):                  # a row beside one that is not finite is what it is alone
        assert torch.equal(q[r], ref_q[r]) and torch.equal(s[r], ref_s[r])
    # row 5 is multiplied by a power of two first, which changes no rounding; its scale is normal
    assert torch.equal(q[5], held_exactly((x[5:6].double() * 2.0 ** 80).float())[0][0]) and abs(float(s[5]) * 127 / small - 1) < 4 * U
    # row 6: the integer is exact, the scale a subnormal number, off by half a step of those (2^-150) and the roundings
    assert q[6, 3] == -127 and int(q[6].abs().sum()) == 127
    assert abs(float(s[6]) - float(x[6, 3].abs()) / 127) <= 2.0 ** -149
    back = int8.dequantize_int8(held, torch.float32).cpu()
    assert torch.isnan(back[1:4]).all() and not torch.isnan(back[[0, 4, 5, 6, 7, 8]]).any()


# ------------------------------------------------------------------------------------------------------------ norms
def norm_error(width):
    """Relative error of a norm's output in float32: squares added by at least 32 threads in turn and then in a tree (at most
    width / 32 + 20 roundings, halved by the root), the root's 2 units, three products, an addition."""
    return ((width / 32 + 20) / 2 + 12) * U


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("w_dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (4, 24), (3, 100), (9, 512), (2, 1000), (1, 4096), (5, 4104), (130, 768), (3, 5001), (1, 16384), (2, 33000)])
def test_norm(int8, dtype, w_dtype, rows, width):
    x, d = (randn(rows, width, seed=s, scale=3.0).to(dtype) for s in (1, 2))
    w = (1 + 0.1 * randn(width, seed=3)).to(w_dtype)

    def ref(v, offset):
        v = v.double()
        return v / torch.sqrt(v.pow(2).mean(dim=1, keepdim=True) + 1e-5) * (offset + w.double())
    for pad in (0, 3, 8):
        at, dt = strided(x, pad), strided(d, pad)
        held = int8.rmsnorm_int8(at, w.to(DEV), 1e-5)
        check_held(held, ref(x, 0.0), norm_error(width))
        assert torch.equal(at.cpu(), x)
        held = int8.rmsnorm_int8(at, w.to(DEV), 1e-5, delta=dt, weight_offset=1.0)
        total = (x.float() + d.float()).to(dtype)
        assert torch.equal(at.cpu(), total) and torch.equal(dt.cpu(), d)           # the sum is stored, rounded once
        check_held(held, ref(total, 1.0), norm_error(width))
        if pad and rows > 1:                                                       # and nothing behind a row
            assert bool(torch.isnan(at.as_strided((rows, pad), at.stride(), at.storage_offset() + width)).all())


def test_norm_of_rows_that_are_zero_or_not_finite(int8):
    for width in (40, 4096, 40000):
        x = randn(4, width, dtype=torch.bfloat16)
        x[0] = 0
        x[1, 7] = float("inf")
        x[2, 0] = float("nan")
        held = int8.rmsnorm_int8(x.to(DEV), torch.ones(width, device=DEV), 1e-6)
        alone = int8.rmsnorm_int8(x[3:].to(DEV), torch.ones(width, device=DEV), 1e-6)
        s = held.scales.cpu()
        assert s[0] == 0 and torch.isnan(s[1:3]).all() and not held.values[:3].any()
        assert torch.equal(held.values[3:], alone.values) and torch.equal(held.scales[3:], alone.scales)


def test_norm_takes_itself_as_the_residual_and_one_row_for_all(int8):
    x, one, w = randn(6, 256).to(DEV), randn(1, 256, seed=4).to(DEV), torch.ones(256, device=DEV)
    a, b = x.clone(), x.clone()
    held = int8.rmsnorm_int8(a, w, 1e-6, delta=a)
    assert torch.equal(a, x + x)
    check_held(held, (a.cpu().double() / a.cpu().double().pow(2).mean(dim=1, keepdim=True).add(1e-6).sqrt()), norm_error(256))
    int8.rmsnorm_int8(b, w, 1e-6, delta=one.expand(6, 256))
    assert torch.equal(b, x + one)


@pytest.mark.parametrize("first", [0, 1])
def test_norm_of_rows_and_residuals_that_lie_in_turn(int8, first):
    """x and delta are the halves of one matrix's rows: they share a range of memory and no number."""
    both, w = randn(7, 512, dtype=torch.bfloat16).to(DEV), torch.ones(256, device=DEV)
    halves = both[:, :256], both[:, 256:]
    x, delta = halves[first], halves[1 - first]
    alone, d = x.clone(), delta.clone()
    want = int8.rmsnorm_int8(alone, w, 1e-6, delta=d)
    held = int8.rmsnorm_int8(x, w, 1e-6, delta=delta)
    assert torch.equal(x, alone) and torch.equal(delta, d)
    assert torch.equal(held.values, want.values) and torch.equal(held.scales, want.scales)
    with pytest.raises(int8.KernelError, match="not overlap"):
        int8.rmsnorm_int8(both[:, :256], w, 1e-6, delta=both[:, 128:384])


@pytest.mark.parametrize("width", [64, 256, 1024, 4096, 5001])
def test_a_row_does_not_depend_on_the_rows_around_it(int8, width):
    x = randn(3000, width, dtype=torch.bfloat16).to(DEV)
    w = (1 + 0.1 * randn(width, seed=5)).to(DEV)
    whole = int8.rmsnorm_int8(x, w, 1e-6)
    gates = int8.silu_mul_int8(x[:, :width // 2 * 2])
    for r in (0, 1777, 2999):
        one = int8.rmsnorm_int8(x[r:r + 1], w, 1e-6)
        assert torch.equal(one.values[0], whole.values[r]) and torch.equal(one.scales[0], whole.scales[r])
        one = int8.silu_mul_int8(x[r:r + 1, :width // 2 * 2])
        assert torch.equal(one.values[0], gates.values[r]) and torch.equal(one.scales[0], gates.scales[r])


@pytest.mark.parametrize("op,dtype,residual,rows,width,pad", [
    ("norm", torch.bfloat16, True, 600, 12288, 0), ("norm", torch.bfloat16, True, 450, 16384, 8), ("norm", torch.bfloat16, False, 450, 10248, 24),
    ("norm", torch.float32, True, 600, 8200, 4), ("norm", torch.float32, False, 450, 16376, 0), ("norm", torch.bfloat16, True, 4000, 8704, 0),
    ("rows", torch.bfloat16, False, 4097, 8200, 0), ("rows", torch.bfloat16, False, 2100, 16384, 8)])
def test_many_wide_rows(int8, op, dtype, residual, rows, width, pad):
    """Wide rows, many at a time and one at a time: the same bits; some are zero, tiny or not finite."""
    w = (1 + 0.1 * randn(width, seed=5)).to(DEV)
    x, d = (torch.randn(rows, width, generator=torch.Generator(device=DEV).manual_seed(s), device=DEV).to(dtype) for s in (1, 2))
    wide = torch.full((rows, width + pad), float("nan"), dtype=dtype, device=DEV)
    x[5], d[5], x[151, 8], x[300, width - 1] = 0, 0, float("inf"), float("nan")
    x[7] *= 1e-36
    d[7] = 0
    wide[:, :width] = x
    room = torch.full((rows + 1, width + 24 - width % 8 + 64), 99, dtype=torch.int8, device=DEV)
    room = room.as_strided((rows + 1, width), (room.shape[1] // 16 * 16, 1))
    scales = torch.full((rows + 1,), 7.0, device=DEV)
    out = int8.Int8Rows(room[:rows], scales[:rows])

    def call(at, delta, **kw):
        return int8.quantize_int8(at, **kw) if op == "rows" else int8.rmsnorm_int8(at, w, 1e-6, delta=delta, **kw)
    whole = call(wide[:, :width], d if residual else None, out=out)
    assert torch.equal(wide[:, :width].nan_to_num(), ((x.float() + d.float()).to(dtype) if residual else x).nan_to_num())
    assert bool((room[rows:] == 99).all()) and float(scales[rows]) == 7.0 and bool(torch.isnan(wide[:, width:]).all())
    for r in [0, 5, 7, 147, 148, 151, 295, 296, 300, 301, rows - 2, rows - 1]:
        one = call(x[r:r + 1].clone(), d[r:r + 1] if residual else None)
        assert torch.equal(one.values[0], whole.values[r]), r
        assert torch.equal(one.scales[0].nan_to_num(), whole.scales[r].nan_to_num()), r
    s = whole.scales
    assert float(s[5]) == 0 and bool(torch.isnan(s[[151, 300]]).all()) and not bool(whole.values[[5, 151, 300]].any())
    assert int(torch.isfinite(s).sum()) == rows - 2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(2559, 640), (2560, 640), (2560, 513), (2561, 767), (2048, 769), (4099, 1024)])
def test_many_rows_of_half_a_block(int8, dtype, rows, width):
    """Rows of 513 to 1,024 numbers, many at a time and one at a time: the same bits."""
    x = torch.randn(rows, 2 * width, generator=torch.Generator(device=DEV).manual_seed(width), device=DEV).to(dtype)
    held, gates = int8.quantize_int8(x[:, :width]), int8.silu_mul_int8(x)
    for r in (0, 7, 8, rows // 2, rows - 1):
        for many, one in ((held, int8.quantize_int8(x[r:r + 1, :width])), (gates, int8.silu_mul_int8(x[r:r + 1]))):
            assert torch.equal(one.values[0], many.values[r]) and torch.equal(one.scales[0], many.scales[r])


def test_many_wide_rows_take_themselves_as_the_residual_and_one_row_for_all(int8):
    x, w = torch.randn(500, 12288, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).bfloat16(), torch.ones(12288, device=DEV)
    a, b, one = x.clone(), x.clone(), x[3:4].clone()
    held = int8.rmsnorm_int8(a, w, 1e-6, delta=a)
    assert torch.equal(a, x + x)
    alone = int8.rmsnorm_int8((x + x)[499:].clone(), w, 1e-6)
    assert torch.equal(alone.values[0], held.values[499]) and torch.equal(alone.scales[0], held.scales[499])
    int8.rmsnorm_int8(b, w, 1e-6, delta=one.expand(500, 12288))
    assert torch.equal(b, (x.float() + one.float()).bfloat16())


# ------------------------------------------------------------------------------------------------------------ gates
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("rows,inter,block", [(1, 1, 1), (3, 5, 5), (4, 64, 64), (2, 96, 32), (5, 1000, 8), (3, 1000, 4), (1, 12288, 64), (130, 640, 640), (2, 12288, 12288),
                                              (1, 36000, 36000), (1, 36000, 16), (2, 5001, 5001)])
def test_gate(int8, dtype, act, rows, inter, block):
    gu = randn(rows, 2 * inter, scale=4.0).to(dtype)
    pairs = gu.double().view(rows, inter // block, 2, block)
    g, u = pairs[:, :, 0].reshape(rows, inter), pairs[:, :, 1].reshape(rows, inter)
    t = 2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3) if act == "gelu_tanh" else g
    y = g * torch.sigmoid(t) * u
    # t is off by at most 8 roundings; e^-t by that times |t|, and 2 units of its own; then a sum, a quotient, a product
    err = (8 * t.abs() + 8) * U
    for pad in (0, 3, 8):
        check_held(int8.silu_mul_int8(strided(gu, pad), block=block, act=act), y, err)


def test_gates_that_are_far_out_and_not_finite(int8):
    g = torch.tensor([[-200.0, 200.0, 0.0, -88.8, 89.0, 1.0, -1e30, 1.0], [float("inf"), 1, 1, 1, 1, 1, 1, 1], [1, 1, float("nan"), 1, 1, 1, 1, 1]])
    u = torch.ones(3, 8)
    u[0, 7] = -3.0
    held = int8.silu_mul_int8(torch.cat([g, u], dim=1).to(DEV))
    y = g[:1].double() * torch.sigmoid(g[:1].double()) * u[:1].double()
    check_held(int8.Int8Rows(held.values[:1], held.scales[:1]), y, (8 * g[:1].double().abs().clamp(max=200) + 8) * U)
    assert torch.isnan(held.scales[1:].cpu()).all() and not held.values[1:].any()


# ------------------------------------------------------------------------------------------------------------ products
def product_exactly(x, sx, w, sw, bias, dtype):
    total = (x.cuda().double() @ w.cuda().double().t()).cpu()          # whole numbers below 2^53: exact in any order
    y = total.to(torch.int64).float() * sx[:, None] * sw
    return (y if bias is None else y + bias).to(dtype)


def integers(rows, width, seed):
    g = torch.Generator().manual_seed(seed + rows + 7 * width)
    return torch.randint(-128, 128, (rows, width), generator=g, dtype=torch.int8), torch.rand(rows, generator=g) * 0.02 + 1e-4


def on_device(int8, x, sx):
    room = -(-x.shape[1] // 16) * 16
    wide = torch.full((x.shape[0], room), 77, dtype=torch.int8, device=DEV)      # what lies behind an odd width must not count
    held = int8.Int8Rows(wide[:, :x.shape[1]], torch.empty(x.shape[0], device=DEV))
    held.values.copy_(x)
    held.scales.copy_(sx)
    return held


# rows on both sides of every size at which another tile is taken; sums that fill a stage, miss it by one, and leave slices empty
SHAPES = [(1, 1, 1), (1, 128, 128), (1, 5, 16), (2, 33, 31), (3, 130, 129), (8, 256, 127), (15, 1000, 64), (16, 128, 4096), (17, 256, 500), (31, 300, 1024), (32, 1536, 4096),
          (33, 257, 2048), (48, 640, 1000), (64, 1024, 4096), (65, 384, 96), (100, 4096, 777), (127, 129, 8192), (128, 1024, 1024), (129, 999, 2048), (200, 128, 300),
          (256, 512, 512), (257, 2049, 333), (300, 6144, 256), (512, 513, 1025), (777, 1000, 2001), (1024, 2048, 640), (2050, 300, 4100), (5000, 130, 72), (1, 9000, 14000), (4, 64, 60000)]
# Every kernel, width of its tiles, number of slices, of warps that read results, and place of the partial sums; result rows on 16-byte
# borders, on four-byte borders, and on none; more tiles than pairs of CTAs.
# (By the rule that chose when they were drawn. By the rule as it is, sizes for all of this are in test_int8_tiles.py, which asks it.)
TILES = [(370, 2972, 7657), (574, 7354, 3863), (309, 8746, 3887), (629, 8798, 2673), (1532, 671, 7446), (1367, 3287, 3872), (442, 5427, 4611),
          (1789, 2761, 2951), (464, 4400, 7640), (1599, 1672, 2630), (1784, 3048, 757), (763, 4112, 1824), (2003, 5096, 186), (624, 5560, 2014),
          (1570, 9128, 55), (2496, 1736, 1546), (1845, 6736, 139), (616, 2552, 8097), (67, 10187, 33), (194, 9522, 546), (140, 15241, 130),
          (1, 32, 33), (34, 10895, 37), (276, 9555, 408), (137, 13516, 33), (197, 5048, 33), (427, 6948, 519), (262, 8322, 134), (83, 9769, 33),
          (18, 32, 33), (127, 9708, 32), (389, 33, 32), (108, 5112, 7677), (66, 4827, 4703), (1, 32, 692), (36, 4895, 2498), (3232, 178, 7209),
          (2455, 147, 3658), (1765, 513, 9245), (17, 34, 1061), (3053, 32, 3017), (105, 3407, 6918), (71, 2413, 5902), (129, 2256, 14702),
          (1, 32, 401), (33, 2092, 2422), (3112, 32, 5562), (2099, 32, 2845), (269, 1898, 7347), (21, 32, 786), (389, 36, 1449), (105, 1506, 10930),
          (65, 1113, 9920), (130, 1413, 14655), (1, 33, 917), (33, 830, 4806), (1164, 34, 14005), (812, 33, 5825), (22, 32, 977), (409, 36, 2770)]
# The same for the sums that are cut, with columns that leave some of the CTAs without a part
SLICES = [(1, 5145, 38), (73, 5536, 3470), (147, 6767, 4895), (142, 4907, 6373), (1, 4849, 390), (2332, 148, 2878), (2949, 287, 5675),
          (4067, 158, 5709), (668, 46, 1779), (120, 2166, 9557), (140, 3095, 6274), (1, 2626, 4885), (33, 2561, 3541), (3653, 33, 5702),
          (1370, 321, 6947), (123, 1374, 14983), (1, 32, 8836), (34, 814, 8161), (1454, 34, 12852), (1610, 72, 16138), (195, 9696, 1188),
          (139, 11726, 762), (140, 11008, 534), (155, 10696, 33), (4, 4786, 8161), (35, 4300, 2844), (1870, 517, 4856), (30, 3497, 2275),
          (1, 2441, 7291), (3695, 35, 9257), (2393, 142, 9751), (18, 34, 1533), (1, 32, 12445), (1369, 78, 13866), (18, 43, 1998)]
# Up to 16 rows: every length of the registers that hold x, one and two groups of eight rows, rows of w that the ring holds and that it does not
FEW = [(8, 32, 8836), (7, 126, 9360), (1, 32, 33), (5, 46, 32), (8, 34, 2234), (3, 39, 2064), (2, 33, 4292), (8, 47, 5408), (10, 42, 34), (13, 34, 32),
       (16, 37, 2310), (14, 32, 2736), (9, 38, 4452), (16, 32, 5328), (8, 3650, 9116), (2, 4034, 8944), (1, 14218, 1377), (5, 14860, 1312),
       (8, 7377, 2220), (1, 13154, 2544), (4, 3073, 6529), (8, 4796, 4720), (16, 8629, 2049), (12, 2369, 8192), (16, 2368, 4096), (6, 150, 12288)]


@pytest.mark.parametrize("rows,channels,width", SHAPES)
def test_product(int8, rows, channels, width):
    (x, sx), (w, sw) = integers(rows, width, 1), integers(channels, width, 2)
    bias = randn(channels, seed=3)
    held, weight = on_device(int8, x, sx), int8.Int8Weight(w.to(DEV), sw.to(DEV))
    for dtype in DTYPES:
        assert torch.equal(int8.linear_int8(held, weight, out_dtype=dtype).cpu(), product_exactly(x, sx, w, sw, None, dtype))
    want = product_exactly(x, sx, w, sw, bias, torch.bfloat16)
    assert torch.equal(int8.linear_int8(held, weight, bias=bias.to(DEV)).cpu(), want)
    for pad in (1, 8):                                    # result rows further apart, on and off 16-byte borders; nothing behind them
        for dtype in DTYPES:
            out = torch.full((rows, channels + pad), -7.0, dtype=dtype, device=DEV)
            int8.linear_int8(held, weight, bias=bias.to(DEV), out=out[:, :channels])
            assert torch.equal(out[:, :channels].cpu(), product_exactly(x, sx, w, sw, bias, dtype)) and bool((out[:, channels:] == -7.0).all())


@pytest.mark.parametrize("rows,channels,width", TILES + SLICES + FEW)
def test_product_by_every_kind_of_tile(int8, rows, channels, width):
    (x, sx), (w, sw) = integers(rows, width, 1), integers(channels, width, 2)
    bias = randn(channels, seed=3)
    held, weight = on_device(int8, x, sx), int8.Int8Weight(w.to(DEV), sw.to(DEV))
    assert torch.equal(int8.linear_int8(held, weight).cpu(), product_exactly(x, sx, w, sw, None, torch.bfloat16))
    out = torch.full((rows, channels + 1), -7.0, device=DEV)
    for dtype, room in ((torch.float32, out[:, :channels]), (torch.float32, None)):
        got = int8.linear_int8(held, weight, bias=bias.to(DEV), out_dtype=dtype, out=room)
        assert torch.equal(got.cpu(), product_exactly(x, sx, w, sw, bias, dtype))
    assert bool((out[:, channels:] == -7.0).all())


def test_the_longest_and_largest_sums(int8):
    """131071 products of -128 and -128: the largest sum there is, one step below 2^31."""
    width = int8.MAX_WIDTH
    for rows in (1, 40):
        x = torch.full((rows, width), -128, dtype=torch.int8)
        w = torch.full((3, width), -128, dtype=torch.int8)
        w[1] = 127
        held, weight = on_device(int8, x, torch.ones(rows)), int8.Int8Weight(w.to(DEV), torch.ones(3, device=DEV))
        got = int8.linear_int8(held, weight, out_dtype=torch.float32).cpu()
        want = torch.tensor([128 * 128 * width, -128 * 127 * width, 128 * 128 * width], dtype=torch.int64).float()
        assert torch.equal(got, want.expand(rows, 3))


@pytest.mark.parametrize("rows", [2, 40, 300])
def test_scales_that_are_zero_or_not_finite_stay_in_their_row_and_channel(int8, rows):
    (x, sx), (w, sw) = integers(rows, 256, 5), integers(200, 256, 6)
    sx[0], sx[1] = 0.0, float("nan")
    sw[3], sw[150] = float("inf"), 0.0
    got = int8.linear_int8(on_device(int8, x, sx), int8.Int8Weight(w.to(DEV), sw.to(DEV)), out_dtype=torch.float32).cpu()
    want = product_exactly(x, sx, w, sw, None, torch.float32)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got, nan=1.0), torch.nan_to_num(want, nan=1.0))


def test_no_rows_and_no_channels(int8):
    weight = int8.Int8Weight(torch.ones(5, 32, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV))
    none = int8.quantize_int8(torch.empty(0, 32, device=DEV))
    assert none.values.shape == (0, 32) and none.scales.shape == (0,)
    assert int8.linear_int8(none, weight).shape == (0, 5)
    assert int8.dequantize_int8(none).shape == (0, 32)
    assert int8.silu_mul_int8(torch.empty(0, 32, device=DEV)).values.shape == (0, 16)
    assert int8.rmsnorm_int8(torch.empty(0, 32, device=DEV), torch.ones(32, device=DEV), 1e-6).values.shape == (0, 32)
    empty = int8.Int8Weight(torch.ones(0, 32, dtype=torch.int8, device=DEV), torch.ones(0, device=DEV))
    assert int8.linear_int8(int8.quantize_int8(torch.ones(3, 32, device=DEV)), empty).shape == (3, 0)


@pytest.mark.parametrize("rows", [1, 20, 70, 700])
def test_one_tensor_as_rows_and_as_weight(int8, rows):
    """Rows that the kernel just ahead wrote may be a weight: the product waits for them."""
    x = randn(rows, 512, dtype=torch.bfloat16).to(DEV)
    for _ in range(20):
        held = int8.quantize_int8(x)
        got = int8.linear_int8(held, int8.Int8Weight(*held), out_dtype=torch.float32)
        q, s = held_exactly(x.float().cpu())
        assert torch.equal(got.cpu(), product_exactly(q, s, q, s, None, torch.float32))
        x = x.roll(1, dims=0) * 1.5 if rows > 1 else -x * 1.5


@pytest.mark.parametrize("rows", [1, 100])
def test_a_weight_that_is_written_again(int8, rows):
    """New values in a weight's own memory, by torch and through ``out``, between products that follow at once."""
    big = [randn(2048, 1024, seed=s).to(DEV) for s in range(3)]
    x = int8.quantize_int8(randn(rows, 1024).to(DEV))
    want = [int8.linear_int8(x, int8.Int8Weight.quantize(w)) for w in big]
    weight = int8.Int8Weight.quantize(big[0])
    held = int8.Int8Rows(weight.values, weight.scales)
    got = []
    for i in range(30):
        if i % 2:
            fresh = int8.quantize_int8(big[i % 3])
            weight.values.copy_(fresh.values)
            weight.scales.copy_(fresh.scales)
        else:
            int8.quantize_int8(big[i % 3], out=held)
        got.append(int8.linear_int8(x, weight))
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 3])


@pytest.mark.parametrize("write", ["quantize", "norm", "gate"])
def test_a_weight_written_through_out_is_not_fetched_ahead_on_its_stream(int8, write):
    """Another stream's launch comes between the write and the weight's next product on the writing stream."""
    ws = [randn(64, 256, seed=s).to(DEV) for s in range(2)]
    norm_w = torch.ones(128, device=DEV)
    make = {"quantize": lambda x, **kw: int8.quantize_int8(x, **kw), "gate": lambda x, **kw: int8.silu_mul_int8(x, **kw),
            "norm": lambda x, **kw: int8.rmsnorm_int8(x[:, :128], norm_w, 1e-6, **kw)}[write]
    width = 256 if write == "quantize" else 128
    x = int8.quantize_int8(randn(3, width).to(DEV))
    weight = int8.Int8Weight(*make(ws[0]))
    want = int8.linear_int8(x, int8.Int8Weight(*make(ws[1])))
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        int8.linear_int8(x, weight)
        weight.operands()
        assert weight.stream is not None
        make(ws[1], out=int8.Int8Rows(weight.values, weight.scales))
        with torch.cuda.stream(torch.cuda.Stream()):
            int8.quantize_int8(x.values.float())
        weight.operands()
        assert weight.stream is None                 # the next product starts behind what is ahead of it
        got = int8.linear_int8(x, weight)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_a_product_that_is_refused_leaves_the_weight_to_be_waited_for(int8, monkeypatch):
    x = int8.quantize_int8(randn(3, 64).to(DEV))
    weight = int8.Int8Weight.quantize(randn(8, 64).to(DEV))
    library = int8._lib.load()

    class Refusing:
        oi_launch_fence = staticmethod(library.oi_launch_fence)
        oi_linear_int8 = staticmethod(lambda *args: 1)

    with monkeypatch.context() as m:
        m.setattr(int8._lib, "load", lambda: Refusing)
        m.setattr(int8._lib, "check", lambda rc, what: (_ for _ in ()).throw(RuntimeError(what)))
        with pytest.raises(RuntimeError, match="linear_int8"):
            int8.linear_int8(x, weight)
    assert weight.stream is None
    int8.linear_int8(x, weight)
    assert weight.stream is not None


# ------------------------------------------------------------------------------------------------------------ together
def layer(int8, h, branch, norm_w, gate_up, down, block):
    """A feed-forward layer as a model runs it: norm of the sum, gate and up, activation, down."""
    rows = int8.rmsnorm_int8(h, norm_w, 1e-6, delta=branch)
    gu = int8.linear_int8(rows, gate_up)
    act = int8.silu_mul_int8(gu, block=block)
    return rows, gu, act, int8.linear_int8(act, down)


@pytest.mark.parametrize("tokens", [1, 7, 40, 150, 600])
def test_a_feed_forward_layer(int8, tokens):
    width, inter, block = 512, 1536, 64
    h, branch = (randn(tokens, width, seed=s, dtype=torch.bfloat16) for s in (1, 2))
    norm_w = (1 + 0.1 * randn(width, seed=3)).bfloat16()
    wgu, wd = randn(2 * inter, width, seed=4, scale=width ** -0.5), randn(width, inter, seed=5, scale=inter ** -0.5)
    gate_up, down = int8.Int8Weight.quantize(wgu.to(DEV)), int8.Int8Weight.quantize(wd.to(DEV))
    on = h.to(DEV)
    rows, gu, act, out = layer(int8, on, branch.to(DEV), norm_w.to(DEV), gate_up, down, block)
    # each link from what the one before it gave: products bit for bit, norm and gate within their bounds
    total = (h.float() + branch.float()).bfloat16()
    assert torch.equal(on.cpu(), total)
    v = total.double()
    y = v / torch.sqrt(v.pow(2).mean(dim=1, keepdim=True) + 1e-6) * norm_w.double()
    check_held(rows, y, norm_error(width))
    assert torch.equal(gu.cpu(), product_exactly(rows.values.cpu(), rows.scales.cpu(), *held_exactly(wgu), None, torch.bfloat16))
    pairs = gu.cpu().double().view(tokens, inter // block, 2, block)
    g, u = pairs[:, :, 0].reshape(tokens, inter), pairs[:, :, 1].reshape(tokens, inter)
    check_held(act, g * torch.sigmoid(g) * u, (8 * g.abs() + 8) * U)
    assert torch.equal(out.cpu(), product_exactly(act.values.cpu(), act.scales.cpu(), *held_exactly(wd), None, torch.bfloat16))
    # and the whole against the layer without 8-bit integers. Rounding to steps of m / 127 is noise of m / 127 / sqrt(12) in each
    # operand: 0.0023 m of a root mean square of m / 4 (normal numbers, widths near 500) or m / 8 (activations: products of two
    # such) is 0.9 % and 1.8 %; weights 0.9 %. First product sqrt(2) * 0.9 = 1.3 %; the activation passes on the gate's and the up's
    # share, about 1.3 * sqrt(2) = 1.8 %; with its own 1.8 % and the weights' 0.9 %: 2.7 %. Twice that is never reached.
    full = y @ wgu.double().t()
    pairs = full.view(tokens, inter // block, 2, block)
    g, u = pairs[:, :, 0].reshape(tokens, inter), pairs[:, :, 1].reshape(tokens, inter)
    full = (g * torch.sigmoid(g) * u) @ wd.double().t()
    assert float((out.cpu().double() - full).norm() / full.norm()) < 0.054


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_a_layer_in_a_recorded_graph_and_on_another_stream(int8, tokens):
    width, inter = 256, 768
    norm_w = torch.ones(width, device=DEV)
    gate_up = int8.Int8Weight.quantize(randn(2 * inter, width, seed=4).to(DEV))
    down = int8.Int8Weight.quantize(randn(width, inter, seed=5).to(DEV))
    h, branch = (torch.zeros(tokens, width, dtype=torch.bfloat16, device=DEV) for _ in range(2))

    def fill(seed):
        h.copy_(randn(tokens, width, seed=seed))
        branch.copy_(randn(tokens, width, seed=seed + 50))

    def eager(seed):
        fill(seed)
        return layer(int8, h, branch, norm_w, gate_up, down, 64)[3].clone(), h.clone()
    want = [eager(s) for s in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in range(4):
            got = eager(s)
            assert torch.equal(got[0], want[s][0]) and torch.equal(got[1], want[s][1])
    torch.cuda.current_stream().wait_stream(side)
    fill(0)
    graphs = []
    for _ in range(2):                          # two graphs of the same layer, replayed in turn, eager calls between them
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer(int8, h, branch, norm_w, gate_up, down, 64)[3]
        graphs.append((g, out))
    for s in (3, 1, 2, 0, 3):
        fill(s)
        graphs[s % 2][0].replay()
        assert torch.equal(graphs[s % 2][1], want[s][0]) and torch.equal(h, want[s][1])
        assert torch.equal(eager(s)[0], want[s][0])


def test_two_streams_at_once(int8):
    width = 1024
    weight = int8.Int8Weight.quantize(randn(2048, width, seed=1).to(DEV))
    xs = [randn(r, width, seed=r, dtype=torch.bfloat16).to(DEV) for r in (5, 90, 400)]
    want = [int8.linear_int8(int8.quantize_int8(x), weight) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]
    for _ in range(10):
        for i, (x, s) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(s):
                got[i].append(int8.linear_int8(int8.quantize_int8(x), weight))
    torch.cuda.synchronize()
    for w, several in zip(want, got):
        assert all(torch.equal(w, g) for g in several)


def test_tensors_on_another_device_than_the_current_one(int8, monkeypatch):
    """Each call is made under the tensors' own device, and only there."""
    current, entered = [5], []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)
            self.was, current[0] = current[0], self.device

        def __exit__(self, *exc):
            current[0] = self.was

    x, w = randn(6, 512).to(DEV), randn(40, 512, seed=1).to(DEV)
    weight = int8.Int8Weight.quantize(w)
    norm_w = torch.ones(512, device=DEV)
    calls = (lambda: int8.quantize_int8(x).values, lambda: int8.rmsnorm_int8(x, norm_w, 1e-6).values, lambda: int8.silu_mul_int8(x, block=8).values,
             lambda: int8.dequantize_int8(int8.Int8Rows(weight.values, weight.scales)), lambda: int8.linear_int8(held, weight))
    held = int8.quantize_int8(x)
    want = [c() for c in calls]
    monkeypatch.setattr(int8._lib, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    got = [c() for c in calls]
    assert entered == [0] * len(calls) and current == [5]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_results_that_lie_beyond_2_to_the_31(int8):
    """70,000 rows of 32,768 results: the last ones begin 2.3e9 numbers behind the first."""
    rows, channels = 70000, 32768
    (x, sx), (w, sw) = integers(rows, 32, 1), integers(channels, 32, 2)
    out = int8.linear_int8(on_device(int8, x, sx), int8.Int8Weight(w.to(DEV), sw.to(DEV)))
    for at in (0, 65535, 69990):
        assert torch.equal(out[at:at + 10].cpu(), product_exactly(x[at:at + 10], sx[at:at + 10], w, sw, None, torch.bfloat16))
    held = int8.quantize_int8(out)
    ref = held_exactly(out[-5:].float().cpu())
    assert torch.equal(held.values[-5:].cpu(), ref[0]) and torch.equal(held.scales[-5:].cpu(), ref[1])
    back = int8.dequantize_int8(held, out=out)
    assert torch.equal(back[-5:].cpu(), (ref[0].float() * ref[1][:, None]).bfloat16())


def test_refusals_on_the_device(int8):
    from openinfer_b200.kernels.lib import KernelError
    weight = int8.Int8Weight(torch.ones(5, 32, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV))
    held = int8.quantize_int8(torch.ones(3, 32, device=DEV))
    for bad in (lambda: int8.linear_int8(held, int8.Int8Weight(torch.ones(5, 32, dtype=torch.int8), torch.ones(5))),
                lambda: int8.linear_int8(held, weight, bias=torch.ones(5)),
                lambda: int8.linear_int8(held, weight, out=torch.empty(3, 5)),
                lambda: int8.linear_int8(int8.Int8Rows(held.values, held.scales.cpu()), weight),
                lambda: int8.rmsnorm_int8(torch.ones(3, 32, device=DEV), torch.ones(32), 1e-6),
                lambda: int8.rmsnorm_int8(torch.ones(3, 32, device=DEV), torch.ones(32, device=DEV), 1e-6, delta=torch.ones(3, 32)),
                lambda: int8.quantize_int8(torch.ones(3, 32, device=DEV), out=int8.empty_rows(3, 31, DEV)),
                lambda: int8.silu_mul_int8(torch.ones(3, 32, device=DEV), out=int8.empty_rows(3, 32, DEV))):
        with pytest.raises(KernelError):
            bad()


@pytest.mark.parametrize("rows", [1, 8, 32])
def test_a_weight_brought_back_is_not_fetched_ahead(int8, rows):
    """A bfloat16 weight is written by ``dequantize_int8`` and multiplied at once, behind a kernel that takes a while: in a recorded
    graph that is replayed with new values, and call by call with another stream's launch in between."""
    from openinfer_b200.kernels.linear import linear
    channels, width = 1024, 512
    x = randn(rows, width, seed=1, dtype=torch.bfloat16).to(DEV)
    held = [int8.quantize_int8(randn(channels, width, seed=s).to(DEV)) for s in range(4)]
    want = []
    for h in held:
        w = int8.dequantize_int8(h)
        torch.cuda.synchronize()
        want.append(linear(x, w))
    now, weight, busy = int8.empty_rows(channels, width, DEV), torch.zeros(channels, width, dtype=torch.bfloat16, device=DEV), randn(8192, 4096).to(DEV)

    def chain():
        for _ in range(4):
            int8.quantize_int8(busy)
        int8.dequantize_int8(now, out=weight)
        return linear(x, weight)

    def put(i):
        now.values.copy_(held[i].values)
        now.scales.copy_(held[i].scales)
    put(0)
    chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for i in (1, 2, 3, 0, 2, 1):
        put(i)
        graph.replay()
        assert torch.equal(got, want[i])
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in (1, 2, 3, 0, 2, 1):
        with torch.cuda.stream(side):
            put(i)
            int8.quantize_int8(busy)
            int8.dequantize_int8(now, out=weight)
        with torch.cuda.stream(other):
            int8.quantize_int8(x)
        with torch.cuda.stream(side):
            again = linear(x, weight)
        torch.cuda.synchronize()
        assert torch.equal(again, want[i])


@pytest.mark.parametrize("rows", [1, 16, 40])
def test_a_product_behind_kernels_that_take_longer_than_its_own_waits_may(int8, rows):
    """Its waits are bounded (two seconds) from when the kernels ahead have finished, not from when it has been started."""
    x = int8.quantize_int8(randn(rows, 4096, seed=1).to(DEV))
    weight = int8.Int8Weight.quantize(randn(24576, 4096, seed=2).to(DEV))
    want = int8.linear_int8(x, weight)
    width = 1 << 30                                    # one block's work for a second
    zeros, norm_w = (torch.zeros(*shape, width, dtype=torch.bfloat16, device=DEV) for shape in ((1,), ()))
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))

    def busy(times):
        start.record()
        for _ in range(times):
            int8.rmsnorm_int8(zeros, norm_w, 1e-6, delta=zeros)
    busy(1)
    end.record()
    torch.cuda.synchronize()
    times = int(3000 / start.elapsed_time(end)) + 1
    busy(times)
    got = int8.linear_int8(x, weight)
    end.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) > 2500
    assert torch.equal(got, want) and int8.status() == 0


@pytest.mark.parametrize("rows,channels,width,code,all_of_it", [
    (3, 24576, 4096, 21, False), (3, 500, 4096, 22, True), (16, 1000, 2048, 22, True),                                     # up to 16 rows
    (40, 130, 60000, 1, True), (40, 130, 8192, 2, True), (40, 130, 8192, 3, True), (70, 24576, 1000, 2, True), (70, 24576, 1000, 3, True),      # few
    (2050, 4999, 3000, 11, False), (2050, 4999, 3000, 12, True), (2050, 5000, 3000, 13, True), (2050, 5000, 3000, 14, False)])              # many
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_wait_that_runs_out_makes_results_that_are_no_numbers(int8, dtype, rows, channels, width, code, all_of_it):
    """The kernel behaves as if its wait ``code`` had lasted too long: what it did not come to is NaN, the status names the wait, and
    the next product is as ever."""
    (x, sx), (w, sw) = integers(rows, width, 1), integers(channels, width, 2)
    held, weight = on_device(int8, x, sx), int8.Int8Weight(w.to(DEV), sw.to(DEV))
    want = product_exactly(x, sx, w, sw, None, dtype)
    out = torch.full((rows, channels + 8), -7.0, dtype=dtype, device=DEV)
    L = int8._lib.load()
    torch.cuda.synchronize()
    try:
        L.oi_linear_int8_run_out(code)
        int8.linear_int8(held, weight, out=out[:, :channels])
    finally:
        L.oi_linear_int8_run_out(0)
    assert int8.status() == code and int8.status() == 0
    got = out[:, :channels].cpu()
    none = torch.isnan(got)
    assert bool(none.any()) and (not all_of_it or bool(none.all()))
    assert torch.equal(got[~none], want[~none]) and bool((out[:, channels:] == -7.0).all())
    assert torch.equal(int8.linear_int8(held, weight, out_dtype=dtype).cpu(), want) and int8.status() == 0


@pytest.mark.parametrize("rows,width,off", [(1, (1 << 28) + 21, 0), (1, (1 << 28) + 21, 1), (2, 3 << 27, 0)])
def test_rows_that_one_launch_does_not_bring_back(int8, rows, width, off):
    """More than 2^27 numbers a row, on 16-byte borders and off."""
    g = torch.Generator(device=DEV).manual_seed(3)
    held = int8.empty_rows(rows, width, DEV)
    held.values.copy_(torch.randint(-127, 128, (rows, width), generator=g, dtype=torch.int8, device=DEV))
    held.scales.copy_(torch.rand(rows, generator=g, device=DEV) + 0.1)
    room = torch.full((rows, width + 8), -7.0, dtype=torch.bfloat16, device=DEV)
    out = room[:, off:off + width]
    int8.dequantize_int8(held, out=out)
    assert bool((room[:, off + width:] == -7.0).all()) and bool((room[:, :off] == -7.0).all())
    for first in range(0, width, 1 << 26):
        part = slice(first, first + (1 << 26))
        assert torch.equal(out[:, part], (held.values[:, part].float() * held.scales[:, None]).bfloat16())
