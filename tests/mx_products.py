"""MX products whose float32 sums are exact in every order, for the tests of each kernel, and the sizes that reach it.

Codes are e2m1 values (multiples of 1/2 up to 6), scales two neighbouring powers of two: a product of two values is a
multiple of a quarter, at most 144, in units of the scales' powers. A sum of k of them is at most 576 k quarters, below 2^24
for k below 29127, so that float32 holds every partial sum and a result is right to the last bit or wrong."""

import numpy as np

from oracle import mx

# rows, columns, K, epilogue, kernel: whole and cut slabs, whole and ragged tiles, with and without an activation
PRODUCTS = [
    (1, 500, 5000, "none", "few_16x16"), (16, 4099, 1056, "bias_gelu", "few_16x16"),
    (1, 8192, 64, "none", "few_16x32"), (9, 8200, 1056, "bias", "few_16x32"), (16, 8229, 4096, "silu", "few_16x32"),
    (7, 14336, 4128, "relu", "few_16x32"),
    (16, 28672, 544, "none", "few_16x64"), (9, 28701, 100, "bias_relu", "few_16x64"), (13, 30000, 2560, "gelu", "few_16x64"),
    (17, 700, 4096, "none", "few_32x16"), (32, 4095, 1500, "bias", "few_32x16"),
    (32, 8192, 544, "none", "few_32x32"), (20, 8301, 4096, "silu", "few_32x32"), (31, 14336, 96, "bias", "few_32x32"),
    (65, 129, 513, "none", "tile_64x64_short"), (1000, 1001, 1056, "bias_gelu", "tile_64x64_short"),
    (6000, 300, 8192, "none", "tile_64x64"), (33, 6000, 4096, "silu", "tile_64x64"), (130, 3000, 5000, "bias_relu", "tile_64x64"),
    (200, 200, 5000, "none", "tile_64x64_deep"), (100, 5000, 8192, "gelu", "tile_64x64_deep"),
    (33, 40, 8192, "bias_gelu", "tile_64x64_deep in 8 parts"), (33, 43, 5000, "relu", "tile_64x64_deep in 5 parts"),
    (130, 6000, 40, "none", "tile_64x128"), (130, 6001, 1056, "gelu", "tile_64x128"), (512, 4096, 4096, "bias", "tile_64x128"),
    (33, 4100, 8192, "none", "tile_64x128 in 6 parts"), (33, 4101, 5000, "bias_relu", "tile_64x128 in 5 parts"),
    (400, 5000, 40, "none", "tile_128x128"), (1000, 3000, 1024, "bias", "tile_128x128"),
    (1000, 3001, 1056, "none", "tile_128x128"), (600, 5000, 512, "bias_gelu", "tile_128x128"),
    (100, 4100, 14336, "none", "tile_128x128 in 7 parts"), (130, 6000, 3000, "silu", "tile_128x128 in 2 parts"),
    # 256 x 256 tiles: the last tile's rows end 4 and 160 rows into it, in a wave's first rows and past a whole quarter
    (4100, 2176, 512, "none", "quad_256x256"), (4000, 2176, 544, "bias", "quad_256x256"),
    (4100, 2100, 1056, "none", "quad_256x256"), (2304, 4112, 1024, "bias", "quad_256x256"),
    (3000, 4100, 544, "silu", "quad_256x256"), (3000, 4224, 1536, "bias_relu", "quad_256x256"),
    (4100, 2176, 6400, "none", "quad_256x256"), (4100, 2176, 6624, "bias", "quad_256x256"),
]  # fmt: skip

# slices of the 256 x 256 loop, which takes twelve a turn (six slabs) and the rest in pairs: K of every remainder, whole and
# ending in a slab's first, second and last block
SLABS = [1, 2, 3, 4, 5, 6, 7, 8, 13]
TAILS = [(s, k) for s in SLABS for k in ([512 * s, 512 * s - 31] if s == 1 else [512 * s, 512 * s - 479, 512 * s - 480, 512 * s - 33])]


def matrix(rng, rows, k, power=127):
    """(codes, scales) of random codes at scales 2^(power - 127) and twice that."""
    blocks = -(-k // 32)
    codes = rng.integers(0, 256, (rows, 16 * blocks), np.uint8)
    codes[:, k // 2 + k % 2:] = 0  # past k
    if k % 2:
        codes[:, k // 2] &= 15
    return codes, rng.integers(power, power + 2, (rows, blocks), np.uint8)


def centred(k):
    """The power at which the second operand's scales bring a sum of k products to about 1: a code's mean square is 8.6, with
    either scale 21."""
    return 127 - round(np.log2(21.4 * np.sqrt(k)))


def values(a, k):
    """The float32 values, which hold it exactly."""
    return mx.decode(*a, k).astype(np.float32)
