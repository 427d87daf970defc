"""Which kernel an MX product runs, and how large its launch is: host arithmetic, no GPU."""

import numpy as np
import pytest

from krn_amd.runtime import library
from tests import mx_products
from tests.test_library import LIBRARY

pytestmark = pytest.mark.skipif(not LIBRARY.exists(), reason="libkrn_amd.so is not built")

# rows and columns of a workgroup (rows 0: all of them), its threads
KERNELS = {"few_16x16": (0, 16, 512), "few_16x32": (0, 32, 512), "few_16x64": (0, 64, 256), "few_32x16": (0, 16, 256),
           "few_32x32": (0, 32, 512), "tile_64x64_short": (64, 64, 256), "tile_64x64": (64, 64, 256),
           "tile_64x64_deep": (64, 64, 256), "tile_64x128": (64, 128, 256), "tile_128x128": (128, 128, 256),
           "quad_256x256": (256, 256, 256)}
LAST = (1 << 28) - 1


@pytest.mark.parametrize("activation", [False, True])
@pytest.mark.parametrize("k", [1, 32, 512, 8192])
@pytest.mark.parametrize("m,n", [(1, LAST), (16, LAST), (17, LAST), (32, LAST), (32, LAST - 30), (32, LAST - 31), (33, 1 << 27),
                                 (1 << 27, 33), (LAST, 1), (LAST, 32), (LAST, 64), (64 * 4095, 64 * 4095)])
def test_a_launch_holds_fewer_than_2_to_the_32_threads(m, n, k, activation):
    rows, cols, threads = KERNELS[library.mx_gemm_kernel(m, n, k, activation, 0)]
    assert (-(-m // rows) if rows else 1) * -(-n // cols) * threads < 1 << 32


def test_no_kernel_runs_for_sizes_that_are_refused_or_empty():
    for m, n, k in [(0, 5, 32), (5, 0, 32), (-1, 5, 32), (5, 5, 0), (5, 5, 1 << 23), (1 << 28, 5, 32), (5, 1 << 28, 32)]:
        assert library.mx_gemm_kernel(m, n, k) == ""


def test_the_columns_of_a_few_rows():
    """One row to eight: 32 columns from 8192 on. Nine to sixteen: 64 where a CU gets two or a multiple of three of them."""
    cols = {16: "few_16x16", 32: "few_16x32", 64: "few_16x64"}
    for n in (1, 4096, 8191, 8192, 11008, 14336, 16384, 28672, 32768, 65536):
        assert library.mx_gemm_kernel(1, n, 4096) == library.mx_gemm_kernel(8, n, 1000) == cols[16 if n < 8192 else 32]
    for n, want in [(4096, 16), (8192, 32), (14336, 32), (16385, 32), (24576, 32), (24577, 64), (28672, 64), (32768, 64), (32769, 32),
                    (40960, 32), (49152, 64), (65536, 32), (81920, 32), (98304, 64), (131072, 32)]:
        assert library.mx_gemm_kernel(9, n, 4096) == library.mx_gemm_kernel(16, n, 777) == cols[want]


def test_the_products_of_the_gpu_tests_reach_every_kernel():
    """Each case runs the kernel it names, and each kernel has a case; the 256 x 256 loop runs each of its remainders."""
    for m, n, k, epilogue, kernel in mx_products.PRODUCTS:
        assert library.mx_gemm_kernel(m, n, k, epilogue.removeprefix("bias_") in library.ACTIVATIONS) == kernel
    assert {kernel.split(" ")[0] for *_, kernel in mx_products.PRODUCTS} == set(KERNELS)
    for _, k in mx_products.TAILS:
        assert library.mx_gemm_kernel(1412, 3000, k) == library.mx_gemm_kernel(2100, 2944, k) == "quad_256x256"
    assert {-(-k // 512) % 6 for _, k in mx_products.TAILS} == set(range(6))


@pytest.mark.parametrize("m,n,k", [(3, 40, 512), (5, 33, 1056), (4, 31, 5000), (2, 20, 14336)])
def test_the_exact_products_show_a_lost_block(m, n, k):
    """The inputs of the GPU tests: their float32 sums are the float64 ones, and without any one block of 32 every row of
    the result differs."""
    rng = np.random.default_rng(k)
    a, b = mx_products.matrix(rng, m, k), mx_products.matrix(rng, n, k, mx_products.centred(k))
    x, y = mx_products.values(a, k), mx_products.values(b, k)
    want = x.astype(np.float64) @ y.astype(np.float64).T
    np.testing.assert_array_equal((x @ y.T).astype(np.float64), want)
    assert 0.3 < np.sqrt(np.mean(want**2)) < 3
    for block in range(-(-k // 32)):
        without = want - x[:, 32 * block: 32 * block + 32].astype(np.float64) @ y[:, 32 * block: 32 * block + 32].T
        assert (without != want).any(axis=1).all()
