"""Every kernel of the MX product on inputs whose sums are exact: each result is the float64 one rounded once, to the last bit
(with a GELU or SiLU, within the float32 roundings of its formula), and the memory around it stays."""

import numpy as np
import pytest

from krn_amd.lib import mx_matmul
from krn_amd.runtime import library
from krn_amd.runtime.hip import HIPTensor
from tests import mx_products
from tests.test_gpu_mx import ERF, HALF_STEP, TINY, TYPES, to_device, values, words

pytestmark = pytest.mark.gpu

GUARD = 64  # elements before the result; 512 rows behind it


def guarded(device, kind, m, n):
    """A result inside a larger buffer, and that buffer."""
    host = np.full(GUARD + m * n + 512 * n, 77, np.uint16 if kind == "bf16" else {"f32": np.float32, "f16": np.float16}[kind])
    held = device.to_device(host, TYPES[kind])
    return HIPTensor(device, held.pointer + GUARD * host.itemsize, TYPES[kind], (m, n), owner=held), held


def product(device, kind, m, n, k, epilogue, seed, broken=()):
    """(got, the exact sums with the bias): `broken` names (operand, row, block) of scales that are 255."""
    rng = np.random.default_rng(seed)
    a, b = mx_products.matrix(rng, m, k), mx_products.matrix(rng, n, k, mx_products.centred(k))
    x = mx_products.values(a, k) @ mx_products.values(b, k).T  # float32: exact in every order
    bias = rng.integers(-8, 9, n) / 4
    for operand, row, block in broken:
        (a, b)[operand][1][row, block] = 255
    vector = device.to_device(words(bias, kind)[0], TYPES[kind]) if "bias" in epilogue else None
    out, held = guarded(device, kind, m, n)
    mx_matmul(to_device(device, *a, k), to_device(device, *b, k), epilogue=epilogue, bias=vector, out=out)
    around = held.to_host()
    assert (around[:GUARD] == 77).all() and (around[GUARD + m * n:] == 77).all()
    return values(out), x + bias.astype(np.float32) if "bias" in epilogue else x


def check(got, x, epilogue, kind):
    """Without an activation, and with relu: the exact sum (and the exact float32 sum of it and the bias: multiples of a power
    of two that 24 bits hold) rounded to the type. Otherwise, in units of 2^-24: gelu 0.5 x (1 + erf(x / sqrt 2)) has
    |x| (two roundings of the argument, slope at most 0.49 an argument; four of erf, one of the sum) <= 3 |x| and 2 |f|
    of its products, silu 6 |f| (four of exp, one of the sum, one of the quotient); 8 (|x| + |f|) holds both."""
    activation = epilogue.removeprefix("bias_")
    if activation not in ("gelu", "silu"):
        want = np.maximum(x, np.float32(0)) if activation == "relu" else x
        np.testing.assert_array_equal(got, words(want, kind)[1])
        return
    wide = x.astype(np.float64)
    f = 0.5 * wide * (1 + ERF(wide / np.sqrt(2))) if activation == "gelu" else wide / (1 + np.exp(-wide))
    bound = 8 * 2.0**-24 * (np.abs(wide) + np.abs(f))
    bound += (np.abs(f) + bound) * HALF_STEP[kind] + TINY[kind]
    error = np.abs(got - f)
    worst = np.unravel_index(np.argmax(error - bound), error.shape)
    assert np.all(error <= bound), f"error {error[worst]} > {bound[worst]} at {worst}"


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("m,n,k,epilogue,kernel", mx_products.PRODUCTS)
def test_every_kernel_gives_the_exact_product(device, kind, m, n, k, epilogue, kernel):
    assert library.mx_gemm_kernel(m, n, k, epilogue.removeprefix("bias_") in library.ACTIVATIONS) == kernel
    check(*product(device, kind, m, n, k, epilogue, m + n + k), epilogue, kind)


@pytest.mark.parametrize("slabs,k", mx_products.TAILS)
def test_the_256_x_256_loop_at_every_remainder_of_its_slices(device, slabs, k):
    """Through the patches (1412 x 3000: the last tile has 132 rows and 184 columns) and the direct store (2100 x 2944: 52
    rows), which only 16-bit results take."""
    for kind, m, n in (("f32", 1412, 3000), ("bf16", 2100, 2944)):
        assert library.mx_gemm_kernel(m, n, k) == "quad_256x256"
        check(*product(device, kind, m, n, k, "bias", slabs), "bias", kind)


@pytest.mark.parametrize("m,n,k", [(9, 8200, 1056), (9, 28701, 100), (20, 8301, 1500), (33, 6000, 4096), (130, 6001, 1056),
                                   (1000, 3001, 1056), (33, 4101, 5000), (2100, 2944, 1056), (1412, 3000, 512), (1412, 3000, 3618)])
def test_a_broken_block_reaches_its_row_or_column_and_no_other(device, m, n, k):
    """Scale 255 in the first and the last block of rows of A, and in the middle of a row of B, the matrices' last rows among
    them: their results are NaN, all others exact."""
    last = -(-k // 32) - 1
    broken = [(0, 1, 0), (0, m - 1, last), (1, 5, last // 2), (1, n - 1, last)]
    got, x = product(device, "f32", m, n, k, "none", k, broken)
    x[[1, m - 1]], x[:, [5, n - 1]] = np.nan, np.nan
    np.testing.assert_array_equal(got, x)
