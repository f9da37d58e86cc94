"""8-bit products through every variant of their kernels: the columns and rows of a workgroup, rows by
DMA or through registers, one part of K or several, operands as they are or as padded copies, and as
many steps of K as the rings of LDS hold, fewer and more, K that ends inside a step or with it.
(tests/test_int8_plans.py asks the rule that picks a variant whether any is missing here.)
Tolerances as in tests/test_gpu_int8_linear.py."""

import pytest
import torch

import mrsa
from oracle import int8_oracle as O8
from test_gpu_int8_linear import DEV, U, _operands

pytestmark = pytest.mark.gpu

# rows, columns, length, whether both operands' rows are at multiples of 16 bytes
PRODUCTS = [
    # few cols 16 rows 16 dma 0
    (2, 40, 128, False), (2, 40, 16, False), (3, 40, 640, False), (2, 40, 514, False), (2, 40,
    1152, False), (2, 40, 1042, False), (2, 42, 1664, False), (2, 40, 1552, False), (2, 40,
    2304, False), (2, 40, 2064, False),
    # few cols 16 rows 16 dma 1
    (2, 40, 128, True), (2, 40, 144, True), (2, 41, 640, True), (2, 40, 528, True), (2, 41,
    1152, True), (2, 40, 1056, True), (3, 40, 1664, True), (2, 40, 1568, True), (2, 40, 2176,
    True), (2, 40, 2096, True),
    # few cols 16 rows 32 dma 0
    (18, 40, 128, False), (17, 40, 16, False), (19, 40, 640, False), (17, 41, 523, False), (19,
    40, 1152, False), (18, 40, 1040, False), (19, 42, 1792, False), (17, 41, 1567, False), (18,
    44, 2176, False), (17, 41, 2064, False),
    # few cols 16 rows 32 dma 1
    (17, 41, 128, True), (17, 40, 144, True), (18, 40, 640, True), (17, 41, 528, True), (20, 42,
    1152, True), (20, 40, 1056, True), (17, 41, 1664, True), (17, 40, 1600, True), (18, 44,
    2176, True), (17, 42, 2064, True),
    # few cols 16 rows 64 dma 0
    (66, 40, 128, False), (66, 40, 16, False), (66, 42, 640, False), (68, 40, 523, False), (66,
    40, 1152, False), (67, 41, 1065, False), (72, 42, 1664, False), (70, 41, 1550, False), (68,
    43, 2304, False), (67, 42, 2064, False),
    # few cols 16 rows 64 dma 1
    (69, 40, 128, True), (67, 40, 144, True), (66, 45, 640, True), (66, 40, 528, True), (66, 45,
    1152, True), (73, 41, 1056, True), (72, 42, 1792, True), (72, 40, 1552, True), (72, 44,
    2304, True), (67, 42, 2096, True),
    # few cols 32 rows 16 dma 0
    (2, 4110, 128, False), (2, 4097, 16, False), (2, 4114, 640, False), (5, 4127, 513, False),
    (5, 4121, 1152, False), (3, 4100, 1032, False), (2, 4108, 1664, False), (3, 4132, 1546,
    False), (13, 4127, 2176, False), (9, 4099, 2064, False),
    # few cols 32 rows 16 dma 1
    (2, 4101, 128, True), (3, 4104, 144, True), (7, 4106, 640, True), (4, 4107, 528, True), (3,
    4109, 1152, True), (2, 4185, 1040, True), (2, 4143, 1664, True), (2, 4124, 1552, True), (3,
    4366, 2176, True), (2, 4149, 2064, True),
    # few cols 32 rows 32 dma 0
    (20, 4136, 128, False), (17, 4105, 16, False), (27, 4341, 640, False), (24, 4153, 515,
    False), (18, 4221, 1152, False), (18, 4116, 1040, False), (19, 4207, 1664, False), (20,
    4151, 1537, False), (21, 4388, 2304, False), (20, 4155, 2052, False),
    # few cols 32 rows 32 dma 1
    (18, 4130, 128, True), (23, 4106, 144, True), (28, 4129, 640, True), (18, 4103, 528, True),
    (21, 4349, 1152, True), (20, 4142, 1040, True), (17, 4131, 1664, True), (20, 4107, 1552,
    True), (26, 4236, 2176, True), (25, 4142, 2064, True),
    # few cols 32 rows 64 dma 0
    (258, 825, 128, False), (66, 2057, 16, False), (477, 522, 640, False), (398, 585, 528,
    False), (513, 476, 1152, False), (449, 517, 1035, False), (452, 514, 1664, False), (451,
    523, 1540, False), (392, 597, 2176, False), (395, 588, 2080, False),
    # few cols 32 rows 64 dma 1
    (322, 677, 128, True), (392, 586, 144, True), (326, 692, 640, True), (471, 515, 528, True),
    (530, 488, 1152, True), (398, 582, 1040, True), (472, 531, 1664, True), (482, 519, 1552,
    True), (900, 175, 2304, True), (523, 449, 2112, True),
    # tile 128x128 256 dma 1 parts 0 copies 0
    (1301, 1539, 128, True), (1510, 1352, 256, True), (1028, 1932, 144, True), (1711, 1153, 384,
    True), (1671, 1188, 272, True), (1676, 1186, 512, True), (1154, 1707, 400, True), (1925,
    1050, 640, True), (1557, 1282, 528, True),
    # tile 128x128 256 dma 1 parts 0 copies 1
    (1614, 1237, 517, False),
    # tile 128x128 256 dma 1 parts 1 copies 0
    (722, 739, 6016, True), (596, 868, 6064, True),
    # tile 128x128 256 dma 1 parts 1 copies 1
    (577, 822, 5098, False),
    # tile 128x128 512 dma 0 parts 0 copies 0
    (1347, 1484, 128, False), (129, 10915, 16, False), (1175, 1667, 256, False), (1187, 1682,
    133, False), (1282, 1544, 384, False), (1231, 1628, 260, False), (1096, 1804, 512, False),
    (1258, 1607, 385, False), (1154, 1680, 640, False), (1155, 1669, 560, False),
    # tile 128x128 512 dma 0 parts 1 copies 0
    (474, 1352, 3840, False), (795, 834, 3872, False), (998, 692, 4096, False), (1118, 903,
    3040, False), (623, 869, 4352, False), (855, 616, 4336, False),
    # tile 128x128 512 dma 1 parts 0 copies 0
    (1665, 2346, 128, True), (2804, 1425, 256, True), (2706, 1414, 144, True), (2751, 1442, 384,
    True), (2695, 1432, 272, True), (2067, 1956, 512, True), (1565, 2567, 400, True), (2957,
    1282, 640, True), (1693, 2306, 528, True),
    # tile 128x128 512 dma 1 parts 0 copies 1
    (2836, 10828, 129, False), (5382, 2979, 264, False), (4873, 3241, 387, False), (2989, 2578,
    1037, False),
    # tile 128x128 512 dma 1 parts 1 copies 0
    (1175, 2140, 10624, True), (2196, 1068, 10144, True),
    # tile 128x128 512 dma 1 parts 1 copies 1
    (1290, 1851, 10312, False),
    # tile 128x256 256 dma 1 parts 0 copies 0
    (2518, 1550, 768, True), (2094, 1923, 656, True),
    # tile 128x256 256 dma 1 parts 0 copies 1
    (2728, 1429, 774, False),
    # tile 128x256 256 dma 1 parts 1 copies 0
    (1196, 1717, 7808, True), (1358, 1503, 7536, True),
    # tile 128x256 256 dma 1 parts 1 copies 1
    (1352, 906, 9533, False),
    # tile 256x256 256 dma 0 parts 0 copies 0
    (2334, 3344, 128, False), (259, 21822, 16, False), (2212, 3623, 256, False), (3586, 2185,
    136, False), (2331, 3364, 384, False), (3355, 2321, 270, False), (2215, 3635, 512, False),
    (2339, 3337, 386, False), (2697, 2956, 640, False), (3925, 2053, 519, False),
    # tile 256x256 256 dma 0 parts 1 copies 0
    (2421, 1668, 4096, False), (1584, 2451, 3744, False),
    # tile 256x256 256 dma 1 parts 0 copies 0
    (2453, 3203, 128, True), (2329, 3337, 256, True), (3222, 2446, 144, True), (3731, 2180, 384,
    True), (2455, 3236, 272, True), (3257, 2452, 512, True), (2314, 3329, 416, True), (3683,
    2221, 640, True), (3369, 2352, 528, True),
    # tile 256x256 256 dma 1 parts 0 copies 1
    (6676, 9538, 17, False), (10427, 3208, 133, False), (5545, 4399, 270, False), (3364, 7177,
    388, False), (3086, 2563, 518, False),
    # tile 256x256 256 dma 1 parts 1 copies 0
    (1659, 2476, 8448, True), (2504, 1562, 8400, True),
    # tile 256x256 256 dma 1 parts 1 copies 1
    (2544, 1561, 8358, False),
    # tile 64x128 512 dma 1 parts 0 copies 0
    (1236, 776, 128, True), (1244, 780, 256, True), (1160, 851, 144, True), (901, 1109, 384,
    True), (978, 1028, 272, True), (1102, 908, 512, True), (774, 1240, 400, True), (865, 1167,
    640, True), (979, 1026, 528, True),
    # tile 64x128 512 dma 1 parts 0 copies 1
    (965, 1030, 1038, False),
    # tile 64x128 512 dma 1 parts 1 copies 0
    (328, 332, 13568, True), (326, 329, 12944, True),
    # tile 64x128 512 dma 1 parts 1 copies 1
    (778, 626, 4927, False),
    # tile 64x64 512 dma 0 parts 0 copies 0
    (588, 899, 128, False), (65, 4504, 16, False), (656, 945, 256, False), (641, 933, 132,
    False), (968, 721, 384, False), (646, 1045, 259, False), (1139, 710, 512, False), (794, 994,
    388, False), (841, 659, 640, False), (715, 780, 541, False),
    # tile 64x64 512 dma 0 parts 1 copies 0
    (86, 68, 5760, False), (65, 67, 5749, False),
    # tile 64x64 512 dma 1 parts 0 copies 0
    (837, 818, 128, True), (707, 1029, 256, True), (642, 1129, 144, True), (964, 818, 384,
    True), (785, 1019, 272, True), (1032, 846, 512, True), (1039, 851, 400, True), (862, 816,
    640, True), (839, 837, 528, True),
    # tile 64x64 512 dma 1 parts 0 copies 1
    (837, 678, 1566, False),
    # tile 64x64 512 dma 1 parts 1 copies 0
    (77, 73, 9984, True), (67, 68, 9840, True),
    # tile 64x64 512 dma 1 parts 1 copies 1
    (69, 69, 11268, False),
    # sizes of the package's model, more rows of tiles than one band, rows of fewer than 16 values
    (2049, 4611, 144, True), (4097, 8195, 240, True), (8200, 8200, 128, True), (733, 6753,
    15184, True), (1047, 4117, 15347, False), (32, 4608, 1003, False), (17, 4097, 3584, True),
    (32, 4608, 3584, True), (1, 37888, 3584, True), (32, 37888, 3584, True), (1003, 3584, 18944,
    True), (1, 1, 15, False), (70, 90, 9, False),
]


def _check(out, exact, product):
    """The bound of check_linear, for a result that is known."""

    half = torch.finfo(out.dtype).eps / 2
    bound = (3 * U * product.abs() + U * exact.abs()) * 1.001
    bound = bound + half * (exact.abs() + bound) + 2.0 ** -25
    bad = (out.double() - exact).abs() > bound
    assert not bad.any(), (bad.nonzero()[:4].tolist(), int(bad.sum()))


def _placed(t, left, right):
    """t inside wider rows of other values."""

    big = torch.full((t.shape[0], t.shape[1] + left + right), 77, dtype=torch.int8, device=DEV)
    big[:, left:left + t.shape[1]] = t
    return big[:, left:left + t.shape[1]]


@pytest.mark.parametrize("M,N,K,aligned", PRODUCTS)
def test_products_through_every_variant(M, N, K, aligned):
    print(f"[gpu-case] int8_linear {M} {N} {K} {aligned}", flush=True)
    x, sx, w, sw, bias = _operands(M, N, K, M + N + K, full=True)
    odd = (_placed(x, 3, 2), w) if N % 2 else (x, _placed(w, 1, 0))
    if not aligned and K % 16 == 0 and K >= 128:
        xs, ws = odd
    else:
        xs, ws = x, w
    _, product = O8.linear(x, sx, w, sw)
    _check(mrsa.int8_linear(xs, sx, ws, sw, dtype=torch.bfloat16), product, product)
    for dtype in (torch.float16, torch.float32):
        b = bias.to(dtype)
        out = mrsa.int8_linear(xs, sx, ws, sw, b, dtype=dtype)
        _check(out, product + b.double(), product)
    if aligned:   # (the same bits however the operands lie; here through other variants)
        for xs, ws in (odd, (_placed(x, 16, 32), _placed(w, 32, 16))):
            assert torch.equal(mrsa.int8_linear(xs, sx, ws, sw, bias, dtype=torch.float32), out)


def test_weights_past_32_bits():
    """Offsets inside the weights past 2^32 bytes: few rows and tiles, by DMA and through registers."""

    K, N = 16384, (1 << 32) // 16384 + 40
    w = torch.zeros(N, K, dtype=torch.int8, device=DEV)
    w[-40:] = _operands(40, 1, K, 3)[0]
    sw = torch.full((N,), 1e-3, device=DEV)
    for rows in (8, 30, 70, 300):
        x, sx, _, _, _ = _operands(rows, 1, K, rows)
        out = mrsa.int8_linear(x, sx, w, sw)
        _, product = O8.linear(x, sx, w[-40:], sw[-40:])
        _check(out[:, -40:], product, product)
        assert not out[:, :-40].any()
        out = mrsa.int8_linear(x[:, 1:], sx, w[:, 1:], sw)
        _, product = O8.linear(x[:, 1:], sx, w[-40:, 1:], sw[-40:])
        _check(out[:, -40:], product, product)
        assert not out[:, :-40].any()
