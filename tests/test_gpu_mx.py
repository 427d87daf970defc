"""Microscaled 4-bit matrices on the GPU against oracle/mx.py in float64: codes, scales and values bit for bit, products
within the float32 accumulation bound and one rounding."""

import math

import numpy as np
import pytest

from krn_amd import T
from krn_amd.dtypes import BF16, F16, F32, U8
from krn_amd.lib import MxMatrix, mx_dequantize, mx_matmul, mx_quantize
from krn_amd.runtime import library
from krn_amd.runtime.hip import HIPTensor
from oracle import mx
from oracle.numerics import bf16_values, bf16_words

pytestmark = pytest.mark.gpu

TYPES = {"f32": F32, "f16": F16, "bf16": BF16}
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
TINY = {"f32": 2.0**-149, "f16": 2.0**-25, "bf16": 2.0**-133}  # half a subnormal step and more
ERF = np.vectorize(math.erf, otypes=[np.float64])


def words(x, kind):
    """x rounded to the type, as krn stores it, and those values."""
    if kind == "bf16":
        w = bf16_words(x.astype(np.float32))
        return w, bf16_values(w).astype(np.float64)
    w = x.astype({"f32": np.float32, "f16": np.float16}[kind])
    return w, w.astype(np.float64)


def values(t):
    host = t.to_host()
    return (bf16_values(host) if t.dtype == BF16 else host).astype(np.float64)


def to_device(device, codes, scales, k):
    return MxMatrix(device.to_device(codes), device.to_device(scales), k)


def random_mx(rng, rows, k, spread=4):
    codes, scales = mx.encode(rng.standard_normal((rows, k)))
    return codes, (scales.astype(int) + rng.integers(-spread, spread + 1, scales.shape)).astype(np.uint8)


SHAPES = [(1, 1), (1, 32), (3, 31), (2, 33), (7, 777), (64, 64), (5, 8192), (1000, 301), (33, 4096), (4100, 512), (900, 3001)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,k", SHAPES)
def test_codes_scales_and_values_are_the_oracles(device, kind, rows, k):
    rng = np.random.default_rng(rows * 7919 + k)
    x, exact = words(rng.standard_normal((rows, k)) * np.exp(2 * rng.standard_normal((1, k))), kind)
    got = mx_quantize(device.to_device(x, TYPES[kind]))
    codes, scales = mx.encode(exact)
    np.testing.assert_array_equal(got.codes.to_host(), codes)
    np.testing.assert_array_equal(got.scales.to_host(), scales)
    back = mx.decode(codes, scales, k)
    for out in TYPES:
        np.testing.assert_array_equal(values(mx_dequantize(got, dtype=TYPES[out])), words(back, out)[1])


@pytest.mark.parametrize("kind", list(TYPES))
def test_halves_signs_extremes_and_broken_blocks(device, kind):
    x = np.zeros((14, 64))
    x[0, :12] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -0.0, -5]
    x[1, :3] = [7.5, -7.99, 6.01]  # beyond 6 at the same scale
    x[2, 5], x[3, 40], x[4, 0], x[5, 63] = np.nan, np.inf, -np.inf, np.nan
    x[2, 40], x[3, 2] = 3.0, 1.0  # the other block of those rows is whole
    x[6, :4] = [2.0**-149, 2.0**-130, -(2.0**-127), 0]
    x[7, :4] = [2.0**-126, 2.0**-127, 2.0**-128, 2.0**-129]
    x[8, :3] = [2.0**127 * 1.9, 2.0**126, -(2.0**125)]
    x[9, :3] = [65504, 6e-8, -1]
    x[10], x[11] = 1.0, -(2.0**-14)
    x[12] = np.linspace(-8, 8, 64)
    with np.errstate(over="ignore"):
        w, exact = words(x, kind)
    got = mx_quantize(device.to_device(w, TYPES[kind]))
    codes, scales = mx.encode(exact)
    np.testing.assert_array_equal(got.scales.to_host(), scales)
    np.testing.assert_array_equal(got.codes.to_host(), codes)
    np.testing.assert_array_equal(values(mx_dequantize(got, dtype=F32)), mx.decode(codes, scales, 64))


def test_every_code_at_every_scale_has_its_value(device):
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8), 16).reshape(256, 16)
    a = to_device(device, codes, scales, 512)
    with np.errstate(over="ignore"):
        for out in TYPES:
            np.testing.assert_array_equal(values(mx_dequantize(a, dtype=TYPES[out])), words(mx.decode(codes, scales, 512), out)[1])


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("k", [40, 64])
def test_any_alignment_of_values_and_scales_and_nothing_else_is_written(device, offset, k):
    """x, the scales and the values inside larger buffers, at odd places: the bytes around them stay."""
    rng = np.random.default_rng(offset)
    rows, blocks = 37, -(-k // 32)
    x = rng.standard_normal((rows, k)).astype(np.float16)
    held = device.to_device(np.concatenate([np.zeros(offset, np.float16), x.ravel()]))
    source = HIPTensor(device, held.pointer + 2 * offset, F16, (rows, k), owner=held)
    scale_bytes = device.to_device(np.full(rows * blocks + offset + 5, 99, np.uint8))
    code_bytes = device.to_device(np.full(rows * blocks * 16 + 16, 99, np.uint8))
    out = MxMatrix(HIPTensor(device, code_bytes.pointer, U8, (rows, 16 * blocks), owner=code_bytes),
                   HIPTensor(device, scale_bytes.pointer + offset, U8, (rows, blocks), owner=scale_bytes), k)
    mx_quantize(source, out=out)
    codes, scales = mx.encode(x.astype(np.float64))
    np.testing.assert_array_equal(code_bytes.to_host(), np.append(codes.ravel(), np.full(16, 99)))
    np.testing.assert_array_equal(scale_bytes.to_host(), np.r_[[99] * offset, scales.ravel(), [99] * 5])
    y = device.to_device(np.full(rows * k + offset + 3, 7, np.float16))
    mx_dequantize(out, out=HIPTensor(device, y.pointer + 2 * offset, F16, (rows, k), owner=y))
    want = mx.decode(codes, scales, k).astype(np.float16).ravel()
    np.testing.assert_array_equal(y.to_host(), np.r_[[7] * offset, want, [7] * 3])


def test_no_rows(device):
    a = mx_quantize(device.to_device(np.zeros((0, 40), np.float32)))
    assert a.shape == (0, 40) and mx_dequantize(a, dtype=F32).to_host().shape == (0, 40)
    b = mx_quantize(device.to_device(np.ones((5, 40), np.float32)))
    assert mx_matmul(a, b, dtype=F32).to_host().shape == (0, 5) and mx_matmul(b, a, dtype=F32).to_host().shape == (5, 0)


def check(got, a, b, kind, bias=None, activation=None):
    """Within the float32 accumulation bound of any order, carried through the epilogue (slopes of at most 1.13, eight
    float32 roundings), plus one rounding to the type. The accumulation bound holds where no partial sum overflows:
    partial sums stay below the sum of magnitudes, so it has to be below float32's 2^128. Past that the order of the
    terms decides whether a sum of both signs is finite; one that is beyond 2^128 by more than the bound is not."""
    k = a.shape[1]
    x = a @ b.T
    size = np.abs(a) @ np.abs(b).T
    bound = 8 * 2.0**-24 * (k + 8) * size
    if bias is not None:
        x = x + bias
        bound = bound + np.abs(x) * 2.0**-24
    if activation:
        x = {"relu": lambda v: np.maximum(v, 0), "gelu": lambda v: 0.5 * v * (1 + ERF(v / math.sqrt(2))),
             "silu": lambda v: v / (1 + np.exp(-v))}[activation](x)
        bound = bound * 1.13 + np.abs(x) * 8 * 2.0**-24
    bound = bound + (np.abs(x) + bound) * HALF_STEP[kind] + TINY[kind]
    assert not np.isfinite(got[np.abs(x) - bound > 2.0**128]).any()
    error = np.where(size > 2.0**127, 0.0, np.abs(got - x))
    worst = np.unravel_index(np.argmax(error - bound), error.shape)
    assert np.all(error <= bound), f"error {error[worst]} > {bound[worst]} at {worst}"


PRODUCTS = [(1, 1, 1), (1, 16, 32), (2, 17, 33), (1, 300, 8192), (16, 33, 100), (5, 64, 992), (17, 130, 512), (32, 48, 544),
            (33, 96, 1500), (64, 100, 1000), (65, 129, 513), (128, 128, 512), (130, 257, 2080), (300, 70, 777),
            (256, 384, 1024), (520, 530, 288)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_products(device, kind, m, n, k):
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    a, b = random_mx(rng, m, k), random_mx(rng, n, k)
    got = mx_matmul(to_device(device, *a, k), to_device(device, *b, k), dtype=TYPES[kind])
    assert got.dtype == TYPES[kind] and got.shape == (m, n)
    check(values(got), mx.decode(*a, k), mx.decode(*b, k), kind)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("m,n,k,epilogue", [(70, 100, 8192, "none"), (128, 133, 14336, "bias_gelu"), (40, 260, 5000, "bias")])
def test_products_whose_k_is_split(device, kind, m, n, k, epilogue):
    """Few tiles and a long K: parts of K in planes of the workspace, added with the epilogue by a second kernel. Without
    a workspace another kernel gives the product."""
    assert library.mx_gemm_workspace(m, n, k) > 0
    rng = np.random.default_rng(m)
    a, b = random_mx(rng, m, k, 1), random_mx(rng, n, k, 1)
    bias, exact = words(rng.uniform(-2, 2, n), kind)
    left, right, vector = to_device(device, *a, k), to_device(device, *b, k), device.to_device(bias, TYPES[kind])
    got = mx_matmul(left, right, epilogue=epilogue, dtype=TYPES[kind], bias=vector if "bias" in epilogue else None)
    wide, activation = (mx.decode(*a, k), mx.decode(*b, k)), "gelu" if "gelu" in epilogue else None
    check(values(got), *wide, kind, exact if "bias" in epilogue else None, activation)
    out = device.empty(TYPES[kind], m, n)
    library.mx_gemm_call(left.pointers, right.pointers, out.pointer, TYPES[kind], m, n, k, [], 0)(
        0, device.default_stream.handle)
    check(values(out), *wide, kind)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("epilogue", ["bias", "relu", "gelu", "silu", "bias_relu", "bias_gelu"])
@pytest.mark.parametrize("m,n,k", [(3, 45, 192), (40, 70, 70), (100, 130, 640)])
def test_epilogues(device, kind, epilogue, m, n, k):
    rng = np.random.default_rng(len(epilogue) + m)
    a, b = random_mx(rng, m, k, 0), random_mx(rng, n, k, 0)
    bias, exact = words(rng.uniform(-2, 2, n), kind)
    got = mx_matmul(to_device(device, *a, k), to_device(device, *b, k), epilogue=epilogue, dtype=TYPES[kind],
                    bias=device.to_device(bias, TYPES[kind]) if "bias" in epilogue else None)
    activation = epilogue.removeprefix("bias_")
    check(values(got), mx.decode(*a, k), mx.decode(*b, k), kind, exact if "bias" in epilogue else None,
          None if activation == "bias" else activation)


@pytest.mark.parametrize("m,n,k", [(3, 40, 544), (20, 40, 96), (64, 40, 3000), (150, 140, 544), (150, 140, 512)])
def test_a_broken_block_reaches_its_row_or_column_and_no_other(device, m, n, k):
    """Scale 255 in the first block of a row of A and of B, and in the last of another row of A. Rows that end inside a
    slab lie next to the broken ones, whose scales must not reach them."""
    rng = np.random.default_rng(m)
    (ac, a_s), (bc, bs) = random_mx(rng, m, k), random_mx(rng, n, k)
    a_s[1, 0], a_s[m - 1, -1], bs[5, 0] = 255, 255, 255
    got = values(mx_matmul(to_device(device, ac, a_s, k), to_device(device, bc, bs, k), dtype=F32))
    broken = np.zeros((m, n), bool)
    broken[1], broken[m - 1], broken[:, 5] = True, True, True
    np.testing.assert_array_equal(np.isnan(got), broken)
    a, b = mx.decode(ac, a_s, k), mx.decode(bc, bs, k)
    rows, cols = ~broken.all(axis=1), ~broken.all(axis=0)
    check(got[rows][:, cols], a[rows], b[cols], "f32")


@pytest.mark.parametrize("m,n", [(4, 20), (130, 40)])
def test_smallest_and_largest_scales(device, m, n):
    rng = np.random.default_rng(n)
    (ac, _), (bc, _) = random_mx(rng, m, 96), random_mx(rng, n, 96)
    a_s, bs = np.full((m, 3), 0, np.uint8), np.full((n, 3), 127 + 100, np.uint8)
    a_s[::2] = 127 + 60
    bs[::3] = 40
    got = mx_matmul(to_device(device, ac, a_s, 96), to_device(device, bc, bs, 96), dtype=F32)
    check(values(got), mx.decode(ac, a_s, 96), mx.decode(bc, bs, 96), "f32")


@pytest.mark.parametrize("m,n,k", [(2, 37, 100), (70, 131, 100), (130, 133, 1056)])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_results_and_scales_at_any_alignment_and_nothing_else_is_written(device, m, n, k, kind):
    rng = np.random.default_rng(k)
    a, b = random_mx(rng, m, k), random_mx(rng, n, k)
    scales = device.to_device(np.append(np.full(1, 255, np.uint8), a[1].ravel()))
    left = MxMatrix(device.to_device(a[0]), HIPTensor(device, scales.pointer + 1, U8, a[1].shape, owner=scales), k)
    size = 4 if kind == "f32" else 2
    host = np.full(m * n + 8, 77, np.float32 if kind == "f32" else np.uint16)
    held = device.to_device(host, TYPES[kind])
    out = HIPTensor(device, held.pointer + size, TYPES[kind], (m, n), owner=held)
    assert mx_matmul(left, to_device(device, *b, k), out=out) is out
    after = held.to_host()
    assert after[0] == 77 and (after[1 + m * n:] == 77).all()
    check(values(out), mx.decode(*a, k), mx.decode(*b, k), kind)


def test_a_linear_layer_bound_recorded_and_replayed(device):
    """Activations quantised, multiplied by a weight and the result quantised for the next product: bound calls give the
    direct calls' bits, on another stream and replayed from a graph with new contents."""
    rng = np.random.default_rng(8)
    m, n, k = 24, 160, 1000
    weight = to_device(device, *random_mx(rng, n, k), k)
    back = to_device(device, *random_mx(rng, k, n), n)
    x = device.to_device(rng.standard_normal((m, k)).astype(np.float16))
    xs, hidden, hs = MxMatrix.empty(device, m, k), device.empty(F16, m, n), MxMatrix.empty(device, m, n)
    y = device.empty(F16, m, k)
    steps = [mx_quantize.bind(x, out=xs), mx_matmul.bind(xs, weight, epilogue="silu", out=hidden),
             mx_quantize.bind(hidden, out=hs), mx_matmul.bind(hs, back, out=y)]

    def layer():
        for step in steps:
            step()

    def direct(host):
        h = mx_matmul(mx_quantize(device.to_device(host)), weight, epilogue="silu", dtype=F16)
        return mx_matmul(mx_quantize(h), back, dtype=F16).to_host()

    layer()
    np.testing.assert_array_equal(y.to_host(), direct(x.to_host()))
    graph = device.graph(layer)
    for seed in range(3):
        host = np.random.default_rng(seed).standard_normal((m, k)).astype(np.float16)
        x.copy_from(host)
        graph()
        np.testing.assert_array_equal(y.to_host(), direct(host))
        stream = device.stream()
        x.copy_from(-host)
        with stream:
            layer()
        stream.sync()
        np.testing.assert_array_equal(y.to_host(), direct(-host))


def test_submit_and_rebind(device):
    rng = np.random.default_rng(9)
    a, b = to_device(device, *random_mx(rng, 4, 64), 64), to_device(device, *random_mx(rng, 8, 64), 64)
    bound = mx_matmul.bind(a, b)
    bound.submit().wait()
    first = bound.result.to_host()
    bound.rebind(b, a)
    bound()
    np.testing.assert_array_equal(bound.result.to_host(), first.T)
    mx_matmul.submit(a, b, out=bound.result.device.empty(T.bf16, 4, 8)).wait()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("m,n,k,epilogue", [(4096, 2176, 512, "none"), (2176, 4224, 544, "bias"), (4100, 2100, 1056, "silu"),
                                            (2304, 4112, 1024, "bias_relu")])
def test_many_tiles_and_nothing_else_is_written(device, kind, m, n, k, epilogue):
    """Products of the 256 x 256 tiles, whole and ragged, rows that end inside a slab; sizes that leave a quarter of the
    last tiles past the end of the result. The memory behind the result stays."""
    rng = np.random.default_rng(m + n)
    a, b = random_mx(rng, m, k, 1), random_mx(rng, n, k, 1)
    bias, exact = words(rng.uniform(-2, 2, n), kind)
    host = np.full(m * n + 512 * n, 77, np.uint16 if kind == "bf16" else {"f32": np.float32, "f16": np.float16}[kind])
    held = device.to_device(host, TYPES[kind])
    out = HIPTensor(device, held.pointer, TYPES[kind], (m, n), owner=held)
    mx_matmul(to_device(device, *a, k), to_device(device, *b, k), epilogue=epilogue, out=out,
              bias=device.to_device(bias, TYPES[kind]) if "bias" in epilogue else None)
    assert (held.to_host()[m * n:] == 77).all()
    activation = epilogue.removeprefix("bias_")
    rows = np.r_[0:3, 127:130, 255:258, m - 130:m]  # the first rows of blocks, and the last tile's
    check(values(out)[rows], mx.decode(*a, k)[rows], mx.decode(*b, k), kind, exact if "bias" in epilogue else None,
          activation if activation in ("silu", "relu") else None)
