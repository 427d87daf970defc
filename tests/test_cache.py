"""The paged cache on the host (no GPU): the oracle against closed forms and against mistakes that its tests must see, the
frequencies of rotary positions, and what the calls refuse before anything reaches the device."""

import ctypes
import math
from fractions import Fraction
from types import SimpleNamespace

import numpy as np
import pytest

from krn_amd.dtypes import BF16, F16, F32, I32, I64
from krn_amd.lib import KvCache, Rotary, Sequences, cache_attention, rotary_append
from krn_amd.runtime.hip import HIPTensor
from oracle import cache as oracle
from tests.paged import Paged
from tests.test_library import LIBRARY

needs_library = pytest.mark.skipif(not LIBRARY.exists(), reason="libkrn_amd.so is not built")
DEVICE = SimpleNamespace(arch="gfx950")


def stand_in(dtype, *shape):
    return HIPTensor(DEVICE, 1 << 20, dtype, shape, owner=DEVICE)


DEVICE.to_device = lambda array, dtype: stand_in(dtype, *array.shape)


def cache_of(dtype=BF16, pages=9, kv_heads=2, page=16, d=64):
    return KvCache(stand_in(dtype, pages, kv_heads, page, d), stand_in(dtype, pages, kv_heads, page, d))


def sequences_of(n=3, width=4, **kwargs):
    return Sequences(stand_in(I32, n), stand_in(I32, n, width), **kwargs)


def test_a_pair_turns_by_its_angle():
    x = np.zeros((3, 1, 8))
    x[:, 0, 0], x[:, 0, 3], x[:, 0, 7] = 1, 1, 5
    y, _ = oracle.rotate(x, np.array([0, 1, 2]), [math.pi / 2, math.pi / 4, 0], False, 2.0)
    np.testing.assert_allclose(y[0, 0], [2, 0, 0, 2, 0, 0, 0, 5], atol=1e-15)
    np.testing.assert_allclose(y[1, 0], [-2, 0, 0, 2, 0, 0, 0, 5], atol=1e-15)  # (1, 1) by a quarter turn, times 2
    y, _ = oracle.rotate(x, np.array([0, 1, 2]), [math.pi / 2, math.pi / 2], True)
    np.testing.assert_allclose(y[1, 0], [0, 1, -1, 0, 0, 0, 0, 5], atol=1e-15)


def test_the_oracles_attention_is_softmax_over_what_a_token_sees():
    paged = Paged(None, np.random.default_rng(0), "f16", [40, 3], kv_heads=2, d=64)
    q = np.random.default_rng(1).standard_normal((5, 4, 64))
    starts = [0, 3, 5]
    y, _ = oracle.attention(q, paged.keys, paged.values, starts, paged.lengths, paged.table, 0.1, 5)
    i, t, h = 0, 1, 3  # position 38: keys 34 to 38, of key head 1
    rows = [(paged.table[i, j // 16], 1, j % 16) for j in range(34, 39)]
    k, v = (np.array([data[r] for r in rows]) for data in (paged.keys, paged.values))
    p = np.exp(0.1 * k @ q[t, h])
    np.testing.assert_allclose(y[t, h], p @ v / p.sum(), rtol=1e-12)
    assert oracle.owners([0, 3, 5], [40, 3], 6)[0].tolist() == [0, 0, 0, 1, 1, -1]
    assert oracle.owners([0, 3, 5], [40, 3], 6)[1].tolist() == [37, 38, 39, 1, 2, 0]


@pytest.mark.parametrize("mistake", ["a lost key", "a key too many", "a lost page", "another head", "another page order"])
def test_equal_weights_show_mistakes(mistake):
    """What the GPU tests with queries of zeros accept is less than any of these changes."""
    rng = np.random.default_rng(3)
    n = 2000
    v = rng.integers(-9, 10, (n + 1, 2, 64)).astype(float)
    right = v[:n, 0].mean(0)
    wrong = {"a lost key": v[1:n, 0].mean(0), "a key too many": v[:, 0].mean(0), "a lost page": v[16:n, 0].mean(0),
             "another head": v[:n, 1].mean(0), "another page order": v[16:n + 1, 0].mean(0)}[mistake]
    assert (np.abs(wrong - right) > np.abs(right) * (2.0**-22 + 2.0**-8)).any()


def test_frequencies_are_fractions_of_a_turn():
    """The device's 64-bit fractions stand for frequency / 2 pi to a double's rounding, and wrap with the position."""
    kept = []
    device = SimpleNamespace(to_device=lambda array, dtype: kept.append(array) or stand_in(dtype, *array.shape))
    rotary = Rotary(device, [1.0, 0.0, 2 * math.pi, -0.5, 1e-4, 7.0])
    turns = [Fraction(int(t), 2**64) for t in kept[0]]
    for f, turn in zip(rotary.frequencies, turns):
        want = Fraction(f) / Fraction(6.283185307179586476925286766559).limit_denominator(10**30)
        off = (turn - want) % 1
        assert min(off, 1 - off) < Fraction(4, 2**53)
    assert turns[1] == turns[2] == 0


def test_scaled_frequencies():
    plain, linear = Rotary.of(DEVICE, 64), Rotary.of(DEVICE, 64, factor=4.0)
    parts = Rotary.of(DEVICE, 64, factor=8.0, original=4096)
    np.testing.assert_allclose(plain.frequencies, [10000.0 ** (-2 * j / 64) for j in range(32)])
    np.testing.assert_allclose(linear.frequencies, plain.frequencies / 4)
    rounds = 4096 * plain.frequencies / (2 * math.pi)
    assert (parts.frequencies[rounds > 32] == plain.frequencies[rounds > 32]).all() and (rounds > 32).any()
    np.testing.assert_allclose(parts.frequencies[rounds < 1], plain.frequencies[rounds < 1] / 8)
    assert (rounds < 1).any() and plain.magnitude == linear.magnitude == 1 and parts.magnitude == 0.1 * math.log(8) + 1
    assert Rotary.of(DEVICE, 0).dim == 0 and plain.dim == 64


def test_rotary_positions_refuse_what_is_not_one():
    for frequencies in ([1.0, np.nan], [np.inf], [[1.0]]):
        with pytest.raises(ValueError, match="frequencies"):
            Rotary(DEVICE, frequencies)
    with pytest.raises(ValueError, match="magnitude"):
        Rotary(DEVICE, [1.0], magnitude=math.inf)
    for dim in (63, -2, 64.0):
        with pytest.raises(ValueError, match="even number"):
            Rotary.of(DEVICE, dim)
    for kwargs in ({"base": 0.0}, {"base": math.nan}, {"factor": 0.5}, {"factor": math.inf}):
        with pytest.raises(ValueError, match="factor"):
            Rotary.of(DEVICE, 64, **kwargs)
    with pytest.raises(ValueError, match="original"):
        Rotary.of(DEVICE, 64, factor=2.0, original=0)


def test_a_cache_refuses_what_is_not_one():
    one = stand_in(BF16, 9, 2, 16, 64)
    with pytest.raises(TypeError, match="device tensor"):
        KvCache(np.zeros((9, 2, 16, 64), np.float16), one)
    for keys, vals, message in [(stand_in(F32, 9, 2, 16, 64), one, "keys has 4 axes"), (one, stand_in(F16, 9, 2, 16, 64), "values"),
                                (one, stand_in(BF16, 9, 2, 16), "values"), (one, stand_in(BF16, 8, 2, 16, 64), "keys have shape")]:
        with pytest.raises(ValueError, match=message):
            KvCache(keys, vals)
    for shape, message in [((9, 2, 16, 96), "64 or 128"), ((9, 0, 16, 64), "key head"), ((9, 2, 24, 64), "power of two"),
                           ((9, 2, 8, 64), "power of two"), ((9, 2, 0, 64), "power of two")]:
        with pytest.raises(ValueError, match=message):
            KvCache(stand_in(BF16, *shape), stand_in(BF16, *shape))


def test_sequences_refuse_what_is_not_one():
    lengths, pages = stand_in(I32, 3), stand_in(I32, 3, 4)
    for args, kwargs, message in [((stand_in(I64, 3), pages), {}, "lengths has 1 axes"), ((lengths, stand_in(I32, 3)), {}, "pages has 2"),
                                  ((stand_in(I32, 2), pages), {}, "as many lengths"), ((lengths, pages), {"new": 0}, "new"),
                                  ((lengths, pages), {"new": 1.0}, "new"), ((lengths, pages), {"starts": stand_in(I32, 3)}, "4 starts"),
                                  ((lengths, pages), {"starts": stand_in(I32, 4), "new": 2}, "without starts")]:  # fmt: skip
        with pytest.raises(ValueError, match=message):
            Sequences(*args, **kwargs)
    with pytest.raises(TypeError, match="device tensor"):
        Sequences(np.zeros(3, np.int32), pages)


def test_the_append_refuses_what_does_not_match():
    cache, sequences, qkv = cache_of(), sequences_of(), stand_in(BF16, 3, 8 * 64)
    with pytest.raises(TypeError, match="KvCache"):
        rotary_append(qkv, qkv, sequences)
    with pytest.raises(TypeError, match="Sequences"):
        rotary_append(qkv, cache, qkv)
    with pytest.raises(TypeError, match="Rotary"):
        rotary_append(qkv, cache, sequences, rotary=64)
    cases = [(stand_in(F16, 3, 512), {}, "qkv has 2 axes of bf16"), (stand_in(BF16, 3, 500), {}, "rows of qkv"),
             (stand_in(BF16, 3, 4 * 64), {}, "rows of qkv"), (stand_in(BF16, 3, 7 * 64), {}, "rows of qkv"),
             (stand_in(BF16, 4, 512), {}, "are 3 tokens"), (qkv, {"rotary": Rotary.of(DEVICE, 66)}, "cannot be rotated"),
             (qkv, {"out": stand_in(BF16, 3, 4, 63)}, "out has shape"), (qkv, {"out": stand_in(F16, 3, 4, 64)}, "out has 3 axes")]
    for x, kwargs, message in cases:
        with pytest.raises(ValueError, match=message):
            rotary_append(x, cache, sequences, **kwargs)


def test_the_attention_refuses_what_does_not_match():
    cache, sequences, q = cache_of(), sequences_of(new=2), stand_in(BF16, 6, 4, 64)
    with pytest.raises(TypeError, match="KvCache"):
        cache_attention(q, None, sequences)
    with pytest.raises(TypeError, match="Sequences"):
        cache_attention(q, cache, None)
    cases = [(stand_in(F16, 6, 4, 64), {}, "q has 3 axes"), (stand_in(BF16, 6, 4, 128), {}, "a multiple as many"),
             (stand_in(BF16, 6, 3, 64), {}, "a multiple as many"), (stand_in(BF16, 6, 0, 64), {}, "a multiple as many"),
             (stand_in(BF16, 5, 4, 64), {}, "are 6 tokens"), (q, {"scale": 0.0}, "positive finite"),
             (q, {"scale": -1.0}, "positive finite"), (q, {"scale": math.nan}, "positive finite"), (q, {"scale": math.inf}, "positive"),
             (q, {"window": 0}, "window"), (q, {"window": -1}, "window"), (q, {"window": 2.5}, "window"),
             (q, {"out": stand_in(BF16, 6, 4, 63)}, "out has shape"), (q, {"out": stand_in(F16, 6, 4, 64)}, "out has 3 axes")]
    for x, kwargs, message in cases:
        with pytest.raises(ValueError, match=message):
            cache_attention(x, cache, sequences, **kwargs)


@needs_library
def test_the_entry_points_refuse_before_any_device_call():
    library = ctypes.CDLL(str(LIBRARY))
    library.krn_amd_last_error.restype = ctypes.c_char_p
    p, i64, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float
    places = {"x": 1 << 40, "keys": 1 << 41, "values": 1 << 42, "out": 1 << 43, "starts": None, "lengths": 1 << 21, "table": 1 << 22,
              "turns": 1 << 23}

    def refused(name, *, kind=2, tokens=3, heads=4, kv_heads=2, d=64, pages=9, page=16, step=1, sequences=3, width=4, rotary=64,
                magnitude=1.0, scale=0.125, window=0, workspace=None, **where):
        at = {**places, **where}
        head = [kind, p(at["x"])]
        if name == "krn_rotary_append":
            head += [p(at["out"]), p(at["keys"]), p(at["values"])]
            tail = [p(at["turns"]), i64(rotary), 0, f32(magnitude), None]
        else:
            head += [p(at["keys"]), p(at["values"]), p(at["out"])]
            tail = [f32(scale), i64(window), p(workspace), i64(1 << 30 if workspace else 0), None]
        sizes = [i64(v) for v in (tokens, heads, kv_heads, d, pages, page)]
        assert getattr(library, name)(*head, *sizes, p(at["starts"]), i64(step), p(at["lengths"]), p(at["table"]), i64(sequences),
                                      i64(width), *tail) == -1
        return library.krn_amd_last_error().decode()

    for name in ("krn_rotary_append", "krn_cache_attention"):
        assert "element kind" in refused(name, kind=0) and "element kind" in refused(name, kind=3)
        assert "head dimension" in refused(name, d=96)
        assert "negative" in refused(name, tokens=-1) and "negative" in refused(name, width=-1)
        for sizes in ({"heads": 3}, {"heads": 0}, {"kv_heads": 0}, {"kv_heads": 8}):
            assert "evenly" in refused(name, **sizes)
        assert "4096" in refused(name, heads=8192)
        for page in (8, 24, 0, -16, 1 << 17):
            assert "power of two" in refused(name, page=page)
        for sizes in ({"pages": 1 << 31}, {"pages": 1 << 30, "page": 2048}, {"width": 1 << 31}, {"sequences": 1 << 23, "tokens": 1 << 23},
                      {"tokens": 1 << 23, "starts": 1 << 24}):
            assert "at most" in refused(name, **sizes)
        assert "a sequence" in refused(name, width=(1 << 27) - 15) and "a sequence" in refused(name, width=1 << 15, page=1 << 16, pages=1)
        assert "are not" in refused(name, tokens=4) and "are not" in refused(name, step=0) and "are not" in refused(name, step=-1)
        assert "cache must be" in refused(name, keys=(1 << 41) + 8) and "cache must be" in refused(name, values=(1 << 42) + 2)
        for what in ("lengths", "table"):
            assert "4-byte" in refused(name, **{what: places[what] + 2})
        assert "4-byte" in refused(name, starts=(1 << 24) + 1)
        assert "16-byte" in refused(name, x=(1 << 40) + 8) and "16-byte" in refused(name, out=(1 << 43) + 8)
        row = 4 * 64 * 2
        for over in ("keys", "values", "lengths", "table"):
            assert "shares memory" in refused(name, out=places[over] // 16 * 16)
            assert "shares memory" in refused(name, out=places[over] - 3 * row + 16)
    assert "shares memory" in refused("krn_rotary_append", out=places["x"])
    assert "shares memory" in refused("krn_rotary_append", out=places["turns"])
    assert "shares memory" in refused("krn_rotary_append", values=places["keys"])
    assert "shares memory" in refused("krn_rotary_append", x=places["values"] + 9 * 2 * 16 * 64 * 2 - 16)
    assert "shares memory" in refused("krn_cache_attention", out=places["x"] + 16)
    for rotary in (-2, 66, 3):
        assert "rotated columns" in refused("krn_rotary_append", rotary=rotary)
    assert "magnitude" in refused("krn_rotary_append", magnitude=math.nan) and "magnitude" in refused("krn_rotary_append", magnitude=math.inf)
    for scale in (0.0, -1.0, math.nan, math.inf):
        assert "scale" in refused("krn_cache_attention", scale=scale)
    assert "window" in refused("krn_cache_attention", window=-1)
