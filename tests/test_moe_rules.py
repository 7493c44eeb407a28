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
