"""The microscaled 4-bit operations on the host (no GPU): the oracle's format against closed forms, and what the calls
refuse before anything reaches the device."""

import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

from krn_amd.dtypes import BF16, F16, F32, F64, I8, U8
from krn_amd.lib import MxMatrix, moe, mx_dequantize, mx_matmul, mx_quantize
from krn_amd.runtime.hip import HIPTensor
from oracle import mx
from tests.test_library import LIBRARY

DEVICE = SimpleNamespace(arch="gfx950")
needs_library = pytest.mark.skipif(not LIBRARY.exists(), reason="libkrn_amd.so is not built")


def stand_in(dtype, *shape):
    return HIPTensor(DEVICE, 1 << 20, dtype, shape, owner=DEVICE)


def mx_stand_in(rows, k):
    blocks = -(-k // 32)
    return MxMatrix(stand_in(U8, rows, 16 * blocks), stand_in(U8, rows, blocks), k)


def test_the_oracles_codes_are_the_nearest_values_with_halves_to_even():
    x = np.zeros((1, 32))
    x[0, :13] = [6, 0.25, 0.26, 0.74, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 5.01, -0.0, -0.25]  # the 6 fixes the scale at 1
    codes, scales = mx.encode(x)
    n = np.stack([codes[0] & 15, codes[0] >> 4], -1).reshape(-1)
    assert scales[0, 0] == 127
    assert n[:13].tolist() == [7, 0, 1, 1, 2, 2, 4, 4, 6, 6, 7, 8, 8] and not n[13:].any()


@pytest.mark.parametrize("top,scale", [(6.0, 127), (4.0, 127), (7.99, 127), (8.0, 128), (3.99, 126), (2.0**127, 252),
                                       (2.0**-125, 0), (2.0**-126, 0), (2.0**-149, 0), (0.0, 0), (np.inf, 255),
                                       (np.nan, 255)])
def test_the_oracles_scale_brings_the_largest_into_4_to_8(top, scale):
    x = np.zeros((1, 33))
    x[0, 32] = top  # the second block's
    codes, scales = mx.encode(x)
    assert scales[0, 1] == scale and codes.shape == (1, 32)
    if 0 < top <= 2.0**127 and scale > 0:
        back = mx.decode(codes, scales, 33)[0, 32]
        assert abs(back - top) <= 2 * 2.0 ** (scale - 127) and top / 2.0 ** (scale - 127) < 8


def test_decoded_values_encode_to_themselves():
    rng = np.random.default_rng(3)
    codes, scales = rng.integers(0, 256, (5, 64), np.uint8), rng.integers(1, 250, (5, 4), np.uint8)
    codes[:, ::16] = 7 | (codes[:, ::16] & 0xF0)  # a six in every block
    x = mx.decode(codes, scales, 128)
    again = mx.encode(x)
    np.testing.assert_array_equal(again[0], codes)
    np.testing.assert_array_equal(again[1], scales)


def test_a_matrix_needs_codes_and_scales_of_its_row_length():
    assert mx_stand_in(3, 33).shape == (3, 33)
    for codes, scales, k in [((3, 16), (3, 1), 33), ((3, 32), (3, 1), 33), ((3, 32), (2, 2), 33), ((3, 32), (3, 2), 32)]:
        with pytest.raises(ValueError, match="rows of"):
            MxMatrix(stand_in(U8, *codes), stand_in(U8, *scales), k)
    with pytest.raises(ValueError, match="one value or more"):
        MxMatrix(stand_in(U8, 3, 0), stand_in(U8, 3, 0), 0)
    with pytest.raises(ValueError, match="u8"):
        MxMatrix(stand_in(I8, 3, 16), stand_in(U8, 3, 1), 32)
    with pytest.raises(TypeError, match="device tensor"):
        MxMatrix(np.zeros((3, 16), np.uint8), stand_in(U8, 3, 1), 32)


def test_quantisation_refuses_other_types_and_shapes():
    with pytest.raises(TypeError, match="device tensor"):
        mx_quantize(np.zeros((2, 32), np.float32))
    for x in (stand_in(I8, 2, 32), stand_in(F64, 2, 32), stand_in(F32, 2, 32, 1)):
        with pytest.raises(ValueError, match="x has 2 axes"):
            mx_quantize(x)
    with pytest.raises(ValueError, match="one value or more"):
        mx_quantize(stand_in(F32, 2, 0))
    with pytest.raises(ValueError, match="out has shape"):
        mx_quantize(stand_in(F32, 2, 32), out=mx_stand_in(2, 33))
    with pytest.raises(TypeError, match="MxMatrix"):
        mx_quantize(stand_in(F32, 2, 32), out=stand_in(U8, 2, 16))
    with pytest.raises(TypeError, match="MxMatrix"):
        mx_dequantize(stand_in(U8, 2, 16))
    with pytest.raises(ValueError, match="f64"):
        mx_dequantize(mx_stand_in(2, 32), dtype=F64)
    with pytest.raises(ValueError, match="out has shape"):
        mx_dequantize(mx_stand_in(2, 32), out=stand_in(F32, 2, 33))


def test_the_product_refuses_what_does_not_match():
    a, b = mx_stand_in(4, 64), mx_stand_in(6, 64)
    with pytest.raises(TypeError, match="MxMatrix"):
        mx_matmul(stand_in(BF16, 4, 64), b)
    with pytest.raises(ValueError, match="transposed"):
        mx_matmul(a, mx_stand_in(6, 65))
    with pytest.raises(ValueError, match="i8"):
        mx_matmul(a, b, dtype=I8)
    with pytest.raises(ValueError, match="out has shape"):
        mx_matmul(a, b, out=stand_in(BF16, 6, 4))
    with pytest.raises(ValueError, match="i8"):
        mx_matmul(a, b, out=stand_in(I8, 4, 6))
    with pytest.raises(ValueError, match="bias"):
        mx_matmul(a, b, epilogue="bias")
    with pytest.raises(ValueError, match="bias"):
        mx_matmul(a, b, epilogue="bias", bias=stand_in(F32, 6))  # the result is bf16
    with pytest.raises(ValueError, match="bias"):
        mx_matmul(a, b, epilogue="bias_relu", bias=stand_in(BF16, 5))
    with pytest.raises(ValueError, match="tanh"):
        mx_matmul(a, b, epilogue="tanh")


def test_the_layer_refuses_what_does_not_match():
    x, router, gate_up, down = stand_in(BF16, 3, 64), stand_in(BF16, 4, 64), mx_stand_in(4 * 2 * 48, 64), mx_stand_in(256, 48)
    cases = [((stand_in(F32, 3, 64), router, gate_up, down), 2, "x has 2 axes"),
             ((x, stand_in(F16, 4, 64), gate_up, down), 2, "router has 2 axes"),
             ((x, stand_in(BF16, 4, 63), gate_up, down), 2, "router has shape"),
             ((x, router, mx_stand_in(4 * 48, 64), down), 2, "need gate_up"),
             ((x, router, gate_up, mx_stand_in(255, 48)), 2, "need gate_up"),
             ((x, router, gate_up, down), 0, "top_k"), ((x, router, gate_up, down), 5, "top_k")]
    for args, top_k, message in cases:
        with pytest.raises(ValueError, match=message):
            moe(*args, top_k=top_k)
    with pytest.raises(TypeError, match="MxMatrix"):
        moe(x, router, stand_in(U8, 384, 32), down, top_k=2)
    with pytest.raises(ValueError, match="out has shape"):
        moe(x, router, gate_up, down, top_k=2, out=stand_in(BF16, 4, 64))


@needs_library
def test_the_entry_points_refuse_before_any_device_call():
    library = ctypes.CDLL(str(LIBRARY))
    library.krn_amd_last_error.restype = ctypes.c_char_p
    p, far, i64 = ctypes.c_void_p, ctypes.c_void_p(1 << 40), ctypes.c_int64

    def refused(name, *args):
        assert getattr(library, name)(*args) == -1
        return library.krn_amd_last_error().decode()

    x, codes, scales = p(1 << 20), p(1 << 30), p(1 << 32)
    assert "element kind" in refused("krn_mx_quantize", 4, x, codes, scales, i64(2), i64(32), None)
    assert "aligned" in refused("krn_mx_quantize", 0, x, p((1 << 30) + 8), scales, i64(2), i64(32), None)
    assert "2^31 blocks" in refused("krn_mx_quantize", 0, x, codes, scales, i64(1 << 31), i64(33), None)
    assert "2^31 blocks" in refused("krn_mx_quantize", 0, x, codes, scales, i64(2), i64(0), None)
    assert "share memory" in refused("krn_mx_quantize", 0, codes, codes, scales, i64(2), i64(32), None)
    assert "share memory" in refused("krn_mx_dequantize", codes, p((1 << 30) + 31), 0, far, i64(2), i64(32), None)

    def product(*, a=codes, c=far, out=2, m=4, n=8, k=64, nops=0, ops=None):
        b, bs = p(1 << 33), p(1 << 34)
        return refused("krn_mx_gemm", a, scales, b, bs, c, out, i64(m), i64(n), i64(k), nops, ops, None, None, None, i64(0), None)

    assert "output kind" in product(out=5)
    assert "aligned" in product(a=p((1 << 30) + 4))
    assert "shares memory" in product(c=codes)
    assert "shares memory" in product(c=p((1 << 32) - 1))
    assert "2^23" in product(k=1 << 23) and "2^23" in product(k=0) and "2^23" in product(m=-1)
    assert "2^24 tiles" in product(m=(1 << 31) - 1, n=1 << 20)
    assert "at most 4" in product(nops=5)
    assert "unknown epilogue" in product(nops=1, ops=(ctypes.c_int * 1)(9))
    assert "needs a vector" in product(nops=1, ops=(ctypes.c_int * 1)(5))

    workspace = library.krn_moe_workspace
    workspace.restype, workspace.argtypes = i64, [ctypes.c_int] + [i64] * 5

    def layer(*, kind=2, y=far, t=3, h=64, i=48, experts=4, top_k=2, ws=p(1 << 41), nbytes=1 << 30, down=p(1 << 36)):
        return refused("krn_moe", kind, x, p(1 << 21), codes, scales, down, p(1 << 37), y, i64(t), i64(h), i64(i),
                       i64(experts), i64(top_k), ws, i64(nbytes), None)

    assert "element kind" in layer(kind=0)
    for sizes in ({"t": 65}, {"top_k": 17, "experts": 32}, {"experts": 1025}, {"top_k": 5}, {"i": 0}, {"h": 1 << 24}):
        assert "at most 64 tokens" in layer(**sizes)
    assert "aligned" in layer(down=p((1 << 36) + 2))
    assert "workspace" in layer(ws=None) and "workspace" in layer(nbytes=workspace(2, 3, 64, 48, 4, 2) - 1)
    assert "shares memory" in layer(y=x)
    assert workspace(2, 65, 64, 48, 4, 2) == 0 and workspace(2, 64, 64, 48, 4, 2) > 0


@needs_library
def test_the_product_refuses_launches_of_too_many_threads_and_a_workspace_at_odd_places():
    """A launch holds fewer than 2^32 threads: 512 for 32 columns of a few rows, 256 for a tile of 64 x 64."""
    library = ctypes.CDLL(str(LIBRARY))
    library.krn_amd_last_error.restype = ctypes.c_char_p
    p, i64 = ctypes.c_void_p, ctypes.c_int64

    def refused(m, n, workspace=None):
        assert library.krn_mx_gemm(p(1 << 30), p(1 << 32), p(1 << 40), p(1 << 45), p(1 << 46), 2, i64(m), i64(n), i64(32), 0, None,
                                   None, None, workspace, i64(0), None) == -1
        return library.krn_amd_last_error().decode()

    assert "below 2^28" in refused(32, 1 << 28) and "below 2^28" in refused(1 << 28, 8)
    assert "2^24 tiles" in refused(64 * 4096, 64 * 4096)
    assert "aligned" in refused(70, 100, p((1 << 41) + 8))
