"""Every kernel, tile and slice that the rule of the 8-bit products chooses: the rule is asked for its choice (without a GPU), and each
size is multiplied and compared bit for bit, all of it (on the GPU)."""
import ctypes

import pytest
import torch

from openinfer_b200.kernels import int8
from openinfer_b200.kernels import lib as klib

DEV = "cuda:0"
FEW_ROWS, ROWS, PAIRS = 0, 1, 2
DTYPES = [torch.bfloat16, torch.float32]

# Many rows. (rows of x a tile, float32 results, results on 16-byte borders): sizes with one tile, two, and three or more for a pair of
# CTAs; of the third on, tensor memory is filled again when it has been drained. Sums of two turns of the ring and more.
BY_PAIRS = {
    (32, 0, 0): [(64, 7811, 5310), (58, 16361, 17013), (59, 24415, 10751)],
    (32, 0, 1): [(61, 7880, 5540), (52, 16320, 25903), (63, 57248, 3312)],
    (32, 1, 0): [(59, 7985, 5635), (59, 16351, 17700), (60, 24271, 13610)],
    (32, 1, 1): [(61, 7872, 5526), (57, 16352, 22406), (64, 57144, 3269)],
    (64, 0, 0): [(4349, 33, 2198), (105, 18487, 4229), (76, 27991, 4594)],
    (64, 0, 1): [(4177, 32, 2299), (127, 18672, 2871), (99, 27824, 2188)],
    (64, 1, 0): [(4205, 33, 2192), (120, 18599, 3180), (95, 28211, 2700)],
    (64, 1, 1): [(4695, 32, 2178), (121, 18624, 3178), (100, 28072, 2194)],
    (96, 0, 0): [(4741, 33, 2193), (89, 26431, 3016), (265, 28465, 2971)],
    (96, 0, 1): [(4927, 32, 2296), (259, 11864, 2188), (96, 40288, 2334)],
    (96, 1, 0): [(5069, 33, 2183), (86, 20997, 4108), (257, 29675, 2208)],
    (96, 1, 1): [(5168, 32, 2217), (259, 11800, 2198), (94, 43208, 2258)],
    (128, 0, 0): [(7386, 33, 1957), (6224, 515, 1994), (594, 14683, 3685)],
    (128, 0, 1): [(7630, 32, 2067), (113, 23256, 1984), (104, 39056, 1929)],
    (128, 1, 0): [(7251, 33, 1977), (6211, 515, 1932), (225, 19093, 2474)],
    (128, 1, 1): [(7579, 32, 1987), (113, 23848, 2018), (98, 38304, 1932)],
    (160, 0, 0): [(4776, 275, 1667), (6517, 521, 1708), (259, 19201, 3285)],
    (160, 0, 1): [(4756, 272, 1704), (131, 18992, 1676), (91, 40040, 1797)],
    (160, 1, 0): [(5060, 267, 1693), (6346, 521, 1674), (279, 18979, 2268)],
    (160, 1, 1): [(4926, 264, 1761), (133, 19128, 1691), (95, 43928, 1672)],
    (192, 0, 0): [(6061, 259, 1674), (8067, 513, 1692), (6321, 1303, 1675)],
    (192, 0, 1): [(5960, 280, 1674), (163, 19000, 1698), (89, 45360, 1678)],
    (192, 1, 0): [(6040, 257, 1755), (7906, 521, 1794), (7481, 1029, 1667)],
    (192, 1, 1): [(6092, 264, 1712), (162, 19200, 1681), (85, 49144, 1690)],
    (224, 0, 0): [(7136, 265, 1674), (7113, 781, 1685), (8635, 1039, 1716)],
    (224, 0, 1): [(7131, 280, 1671), (108, 32576, 1686), (86, 49136, 1672)],
    (224, 1, 0): [(7157, 257, 1735), (222, 18967, 2193), (422, 19041, 1739)],
    (224, 1, 1): [(7210, 264, 1694), (101, 35760, 1696), (83, 54192, 1695)],
    (256, 0, 0): [(8534, 271, 1419), (8374, 795, 1419), (6963, 1567, 1455)],
    (256, 0, 1): [(8449, 264, 1443), (97, 35208, 1702), (82, 52720, 1689)],
    (256, 1, 0): [(8688, 263, 1434), (6549, 1027, 1430), (7046, 1549, 1413)],
    (256, 1, 1): [(8330, 264, 1437), (91, 34840, 2157), (81, 54056, 1922)],
}
# Few rows. (rows of x a tile, slices of the sum, partial sums over the ring, more stages than the ring holds): float32 results, on
# borders, size
BY_ROWS = {
    (16, 1, 0, 0): (0, 0, (17, 33, 34)), (16, 1, 0, 1): (1, 0, (29, 33, 1417)), (16, 2, 0, 0): (0, 0, (9, 4761, 2806)),
    (16, 2, 0, 1): (1, 0, (1, 4753, 7280)), (16, 4, 0, 0): (0, 1, (17, 32, 1416)), (16, 4, 0, 1): (1, 1, (17, 32, 6173)),
    (16, 8, 0, 0): (0, 0, (17, 33, 1801)), (16, 8, 0, 1): (1, 1, (1, 32, 12431)), (32, 1, 0, 0): (0, 0, (135, 33, 32)),
    (32, 1, 0, 1): (1, 0, (129, 33, 1285)), (32, 2, 0, 0): (0, 0, (33, 3397, 2190)), (32, 2, 0, 1): (1, 1, (17, 4224, 2457)),
    (32, 4, 0, 0): (0, 1, (131, 32, 1450)), (32, 4, 0, 1): (1, 0, (132, 33, 5158)), (32, 8, 0, 0): (0, 0, (129, 33, 1805)),
    (32, 8, 0, 1): (1, 0, (133, 35, 9230)), (32, 8, 1, 1): (0, 0, (18, 4155, 35444)), (48, 1, 0, 0): (1, 1, (401, 32, 33)),
    (48, 1, 0, 1): (0, 1, (402, 32, 1158)), (48, 2, 0, 1): (1, 0, (1044, 131, 2215)), (48, 2, 1, 1): (0, 0, (47, 18957, 27152)),
    (48, 4, 0, 0): (1, 0, (396, 33, 1685)), (48, 4, 0, 1): (0, 1, (389, 32, 4271)), (48, 8, 0, 0): (1, 1, (388, 32, 1890)),
    (48, 8, 0, 1): (0, 1, (387, 32, 8510)), (48, 8, 1, 1): (1, 1, (34, 4328, 37722)), (64, 1, 0, 0): (0, 0, (991, 33, 34)),
    (64, 1, 0, 1): (1, 1, (976, 32, 1079)), (64, 2, 0, 1): (0, 0, (2238, 33, 2226)), (64, 2, 1, 1): (1, 0, (49, 19121, 33496)),
    (64, 4, 0, 0): (0, 1, (964, 32, 1910)), (64, 4, 0, 1): (1, 0, (976, 33, 3587)), (64, 8, 0, 0): (0, 1, (591, 32, 2789)),
    (64, 8, 0, 1): (1, 1, (587, 32, 7480)), (64, 8, 1, 1): (0, 1, (50, 4128, 44668)), (80, 1, 0, 0): (1, 1, (65, 9856, 33)),
    (80, 1, 0, 1): (0, 0, (65, 8555, 913)), (80, 2, 0, 1): (1, 0, (2378, 131, 2540)), (80, 2, 1, 1): (0, 1, (65, 19024, 20234)),
    (80, 4, 0, 0): (1, 1, (2056, 32, 2214)), (80, 4, 0, 1): (0, 1, (2139, 32, 3092)), (80, 8, 0, 0): (1, 0, (770, 33, 5881)),
    (80, 8, 0, 1): (0, 1, (772, 32, 6470)), (80, 8, 1, 1): (1, 1, (67, 4216, 52696)), (96, 1, 0, 0): (0, 0, (82, 9981, 34)),
    (96, 1, 0, 1): (1, 0, (84, 20005, 387)), (96, 2, 0, 1): (0, 0, (3042, 129, 3060)), (96, 4, 0, 0): (1, 1, (2606, 32, 2977)),
    (96, 4, 0, 1): (0, 0, (2623, 33, 3127)), (96, 8, 0, 1): (1, 1, (980, 32, 6840)), (96, 8, 1, 1): (0, 0, (83, 4261, 55214)),
    (112, 1, 0, 0): (1, 1, (99, 9600, 32)), (112, 1, 0, 1): (0, 0, (97, 8995, 789)), (112, 2, 0, 1): (1, 0, (3614, 131, 3564)),
    (112, 2, 1, 1): (0, 1, (100, 18984, 17386)), (112, 4, 0, 1): (1, 1, (3159, 32, 4392)), (112, 4, 1, 1): (0, 1, (100, 9504, 55900)),
    (112, 8, 0, 1): (1, 1, (1159, 32, 10397)), (128, 1, 0, 0): (0, 0, (114, 9717, 33)), (128, 1, 0, 1): (1, 1, (116, 9816, 776)),
    (128, 2, 0, 1): (0, 0, (113, 4997, 5045)), (128, 2, 1, 1): (1, 0, (115, 18995, 24278)), (128, 4, 1, 1): (0, 0, (3596, 33, 5437)),
    (128, 8, 1, 1): (1, 0, (1346, 35, 13910)), (144, 1, 0, 0): (0, 0, (3805, 521, 393)), (144, 1, 0, 1): (1, 1, (130, 9776, 798)),
    (144, 2, 0, 1): (0, 0, (130, 4807, 5882)), (144, 4, 1, 1): (1, 0, (2088, 129, 7567)), (144, 8, 1, 1): (0, 1, (1631, 32, 20441)),
    (160, 1, 0, 0): (1, 1, (476, 4792, 513)), (160, 1, 0, 1): (0, 1, (148, 10056, 775)), (160, 2, 1, 1): (1, 1, (145, 4888, 6034)),
    (160, 4, 1, 1): (0, 0, (2315, 131, 8550)), (160, 8, 1, 1): (1, 0, (1740, 35, 20012)), (176, 1, 0, 0): (0, 0, (4064, 641, 530)),
    (176, 1, 0, 1): (1, 0, (165, 9533, 897)), (176, 2, 1, 1): (0, 1, (162, 4864, 6890)), (176, 4, 1, 1): (1, 0, (2571, 135, 9730)),
    (176, 8, 1, 1): (0, 1, (2024, 32, 25404)), (192, 1, 0, 1): (1, 1, (184, 9504, 1031)), (192, 2, 1, 1): (0, 1, (179, 4776, 7565)),
    (192, 4, 1, 1): (1, 0, (2851, 135, 11652)), (192, 8, 1, 1): (0, 0, (2122, 33, 26398)), (208, 1, 0, 1): (1, 1, (193, 9816, 1037)),
    (208, 2, 1, 1): (0, 1, (195, 4784, 8160)), (208, 4, 1, 1): (1, 0, (3096, 133, 11546)), (208, 8, 1, 1): (0, 0, (2350, 35, 29257)),
    (224, 1, 0, 1): (1, 1, (212, 11672, 1028)), (224, 2, 1, 1): (0, 0, (212, 4871, 8869)), (224, 4, 1, 1): (1, 0, (3384, 131, 13515)),
    (224, 8, 1, 1): (0, 0, (2511, 33, 31311)), (240, 1, 0, 1): (1, 1, (3591, 1056, 770)), (240, 2, 1, 1): (0, 1, (228, 5384, 8877)),
    (240, 4, 1, 1): (1, 0, (3628, 129, 15751)), (240, 8, 1, 1): (0, 0, (2703, 33, 36309)), (256, 1, 0, 1): (1, 1, (245, 11560, 1172)),
    (256, 2, 1, 1): (0, 0, (250, 5479, 9853)), (256, 4, 1, 1): (1, 0, (3904, 137, 16165)), (256, 8, 1, 1): (0, 0, (3011, 33, 40458)),
}
# Up to 16 rows. (groups of eight rows, stages of a row of w as registers of x are laid out, the ring holds all rows of a CTA): size
BY_FEW_ROWS = {
    (1, 1, 0): (1, 15948, 1157), (1, 1, 1): (1, 32, 32), (1, 2, 0): (1, 7201, 2051), (1, 2, 1): (1, 32, 2049), (1, 4, 0): (1, 2380, 6221),
    (1, 4, 1): (1, 32, 4140), (1, 6, 0): (1, 2709, 8214), (1, 6, 1): (1, 32, 8226), (2, 1, 1): (9, 32, 32), (2, 2, 1): (9, 32, 2062),
    (2, 4, 0): (9, 6366, 4152), (2, 4, 1): (9, 32, 4164),
}


def choice(f32, on_borders, size):
    """(kernel, rows of x a tile, slices of the sum, tiles, stages of the ring, partial sums over the ring) of a product"""
    said = (ctypes.c_int * 6)()
    assert klib.load(verbose=False).oi_linear_int8_choice(int8._DT[DTYPES[f32]], on_borders, *size, said) == 0
    return tuple(said)


def blocks(width):
    return -(-width // 128)


def test_the_rule_chooses_what_these_sizes_stand_for():
    for (tile, f32, on), sizes in BY_PAIRS.items():
        for turns, size in enumerate(sizes, 1):
            kernel, bn, _, tiles, stages, _ = choice(f32, on, size)
            assert (kernel, bn, min(3, -(-tiles // 74))) == (PAIRS, tile, turns) and blocks(size[2]) >= 2 * stages + 2, size
            assert on == (size[1] % 8 == 0)
    for (tile, slices, over, again), (f32, on, size) in BY_ROWS.items():
        kernel, bn, c, _, stages, at = choice(f32, on, size)
        assert (kernel, bn, c, at, -(-blocks(size[2]) // c) > stages) == (ROWS, tile, slices, over, bool(again)), size
        assert on == (size[1] % 8 == 0)
    for (groups, stages, at_once), size in BY_FEW_ROWS.items():
        for f32 in (0, 1):
            assert choice(f32, size[1] % 8 == 0, size)[0] == FEW_ROWS, size
        chunks, mine = -(-size[2] // 2048), -(-size[1] // 16)
        assert (-(-size[0] // 8), chunks if chunks <= 2 else 4 if chunks <= 4 else 6, -(-mine // min(mine, 148)) * chunks <= 6) == (groups, stages, bool(at_once))


def test_every_choice_is_among_these_sizes():
    """Tiles of 32 to 256 rows in pairs, each with both types, on and off borders, with one to three tiles a pair; of few rows every
    height of a tile and every number of slices; up to 16 rows both groups and every length of the registers."""
    assert set(BY_PAIRS) == {(bn, f32, on) for bn in range(32, 257, 32) for f32 in (0, 1) for on in (0, 1)}
    assert {(bn, c) for bn, c, _, _ in BY_ROWS} == {(bn, c) for bn in range(16, 257, 16) for c in (1, 2, 4, 8)}
    assert {(over, c) for _, c, over, _ in BY_ROWS} == {(0, c) for c in (1, 2, 4, 8)} | {(1, c) for c in (2, 4, 8)}
    assert {(groups, stages) for groups, stages, _ in BY_FEW_ROWS} == {(1, s) for s in (1, 2, 4, 6)} | {(2, s) for s in (1, 2, 4)}


def exactly(x, sx, w, sw, bias, dtype):
    total = x.double() @ w.double().t()                     # whole numbers below 2^53: exact in any order
    y = total.to(torch.int64).float() * sx[:, None] * sw
    return (y if bias is None else y + bias).to(dtype)


def product(f32, size, seed):
    rows, channels, width = size
    g = torch.Generator(device=DEV).manual_seed(seed)

    def integers(n):
        wide = torch.full((n, -(-width // 16) * 16), 77, dtype=torch.int8, device=DEV)     # what lies behind an odd width must not count
        wide[:, :width] = torch.randint(-128, 128, (n, width), generator=g, dtype=torch.int8, device=DEV)
        return int8.Int8Rows(wide[:, :width], torch.rand(n, generator=g, device=DEV) * 0.02 + 1e-4)
    x, w = integers(rows), integers(channels)
    bias = torch.randn(channels, generator=g, device=DEV) if seed % 2 else None
    room = torch.full((rows + 1, channels), -7.0, dtype=DTYPES[f32], device=DEV)             # nothing behind the last row
    got = int8.linear_int8(x, int8.Int8Weight(*w), bias=bias, out=room[:rows])
    assert torch.equal(got, exactly(*x, *w, bias, DTYPES[f32])) and bool((room[rows] == -7.0).all())


@pytest.fixture(scope="module")
def waits():
    klib.load()
    yield
    assert int8.status() == 0                               # no bounded wait has run out


@pytest.mark.gpu
@pytest.mark.parametrize("tile,f32,on,size", [(*k, size) for k, sizes in BY_PAIRS.items() for size in sizes])
def test_many_rows(waits, tile, f32, on, size):
    product(f32, size, sum(size))


@pytest.mark.gpu
@pytest.mark.parametrize("tile,slices,over,again,f32,size", [(*k, f32, size) for k, (f32, _, size) in BY_ROWS.items()])
def test_few_rows(waits, tile, slices, over, again, f32, size):
    product(f32, size, sum(size))


@pytest.mark.gpu
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("size", BY_FEW_ROWS.values())
def test_up_to_16_rows(waits, size, f32):
    product(f32, size, sum(size))
