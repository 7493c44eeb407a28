"""The lines between the experts' kernels (csrc/moe.hip) against both sides' times."""
import ctypes as C

import pytest

import edgexpu_amd as E

SORT = 5.0

# experts, pairs, elements of an expert's weights in the product, measured us of a workgroup a token and of tiles
# without their sort
MEASURED = [
    # gate and up of 14336 x 4096 (Q4_K, Q8_0, Q5_K), 8192 x 4096 (Q4_K, Q5_K, Q8_0), 4096 x 4096 (Q4_K, Q8_0)
    (8, 6, 2 * 14336 * 4096, 91.6, 90.1), (8, 8, 2 * 14336 * 4096, 118.8, 90.2), (8, 8, 2 * 14336 * 4096, 313.8, 251.2),
    (8, 8, 2 * 14336 * 4096, 160.9, 110.4), (4, 4, 2 * 14336 * 4096, 63.7, 57.8), (4, 6, 2 * 14336 * 4096, 87.9, 58.0),
    (2, 4, 2 * 14336 * 4096, 60.3, 40.8), (8, 6, 2 * 8192 * 4096, 53.4, 55.5), (8, 8, 2 * 8192 * 4096, 72.3, 60.1),
    (8, 8, 2 * 8192 * 4096, 95.4, 70.4), (8, 8, 2 * 8192 * 4096, 177.0, 176.3), (6, 6, 2 * 8192 * 4096, 54.8, 41.8),
    (8, 8, 2 * 4096 * 4096, 39.3, 38.9), (4, 6, 2 * 4096 * 4096, 28.2, 24.4), (4, 8, 2 * 4096 * 4096, 37.0, 25.6),
    (4, 8, 2 * 4096 * 4096, 88.8, 73.7), (2, 4, 2 * 4096 * 4096, 18.0, 22.1), (2, 8, 2 * 4096 * 4096, 33.1, 23.8),
    (4, 8, 2 * 4096 * 2048, 21.2, 17.1),
    # down of the same (Q4_K, Q6_K, Q8_0, ...)
    (8, 8, 14336 * 4096, 58.9, 65.3), (8, 8, 14336 * 4096, 124.7, 141.7), (4, 6, 14336 * 4096, 46.2, 46.0),
    (4, 8, 14336 * 4096, 59.7, 47.0), (4, 8, 14336 * 4096, 115.3, 91.9), (8, 8, 8192 * 4096, 74.9, 86.1),
    (4, 6, 8192 * 4096, 57.9, 58.7), (4, 8, 8192 * 4096, 72.7, 58.8), (4, 8, 4096 * 4096, 20.9, 21.8),
    # 128 experts of 768 x 2560: gate and up Q4_K, down Q6_K
    (128, 48, 2 * 768 * 2560, 25.3, 27.9), (128, 96, 2 * 768 * 2560, 45.0, 38.0), (128, 48, 768 * 2560, 28.6, 31.3),
    (128, 96, 768 * 2560, 53.0, 47.5),
]


def one(pairs, experts, weights, lds=304):
    f = E.hip().lib._ZN3exq13moe_takes_oneExixm
    f.restype, f.argtypes = C.c_bool, [C.c_longlong, C.c_int, C.c_longlong, C.c_size_t]
    return f(pairs, experts, weights, lds)


@pytest.mark.parametrize("experts,pairs,weights,alone,tiles", MEASURED)
def test_the_line_takes_the_faster(experts, pairs, weights, alone, tiles):
    """What it takes is within 10 % of the faster one."""
    tiles += SORT
    assert (alone if one(pairs, experts, weights) else tiles) <= 1.1 * min(alone, tiles)


def test_the_line_bounds():
    assert all(one(1, n, 1 << 40) for n in (1, 2, 512))
    assert one(256, 512, 1 << 30) and not one(257, 512, 1 << 10)
    assert one(8, 4, 1 << 20) and not one(9, 4, 1 << 20)
    assert one(1, 8, 1 << 20, 60 * 1024) and not one(1, 8, 1 << 20, 60 * 1024 + 1)


# type, experts, pairs, measured us of gate, up and down with tiles of 64 and of 128 pairs
TILES = [
    (14, 32, 1536, 141.8, 153.9), (14, 32, 2048, 151.4, 142.5), (14, 32, 4096, 226.9, 198.9), (14, 128, 6400, 393.7, 368.8),
    (14, 128, 8192, 443.2, 406.1), (14, 128, 32768, 1290.4, 1097.5), (14, 8, 1024, 377.7, 338.1),
    (8, 32, 2048, 207.8, 236.6), (8, 32, 4096, 281.4, 289.2), (8, 32, 6144, 345.6, 327.9), (8, 32, 16384, 762.4, 660.5),
    (8, 128, 6400, 499.4, 478.8), (8, 128, 12288, 734.0, 721.2), (8, 128, 16384, 886.3, 791.5), (8, 8, 768, 362.8, 459.4),
    (8, 8, 1024, 534.8, 480.8), (8, 8, 1536, 664.2, 519.8),
    (6, 32, 2048, 252.5, 296.4), (6, 32, 6144, 465.1, 436.7), (6, 128, 8192, 780.5, 772.1),
    (6, 128, 12288, 962.5, 882.0), (6, 128, 32768, 2057.9, 1725.6), (6, 8, 768, 644.9, 578.7),
    (2, 32, 4096, 273.8, 285.6), (2, 32, 16384, 692.8, 705.4), (2, 128, 8192, 512.1, 568.8), (2, 128, 16384, 820.3, 902.3),
    (12, 32, 4096, 133.3, 154.0), (12, 32, 16384, 368.4, 373.4), (13, 32, 4096, 146.6, 172.3), (13, 32, 16384, 422.6, 406.0),
]


def wide(qt, pairs, experts):
    f = E.hip().lib._ZN3exq14moe_takes_wideEixi
    f.restype, f.argtypes = C.c_bool, [C.c_int, C.c_longlong, C.c_int]
    return f(qt, pairs, experts)


@pytest.mark.parametrize("qt,experts,pairs,narrow,broad", TILES)
def test_the_tiles_are_the_faster_ones(qt, experts, pairs, narrow, broad):
    """The tile that a type and a number of pairs take is within 10 % of the faster one."""
    assert (broad if wide(qt, pairs, experts) else narrow) <= 1.1 * min(broad, narrow)
