"""Rotary positions and the append to a paged cache on the GPU, against oracle/cache.py in float64 within the bound derived there
and one rounding."""

import numpy as np
import pytest

from krn_amd.dtypes import BF16, F16
from krn_amd.lib import KvCache, Rotary, Sequences, rotary_append
from krn_amd.runtime.hip import HIPTensor
from oracle import cache as oracle
from tests.paged import HALF_STEP, TINY, TYPES, Paged, assert_within, values, words

pytestmark = pytest.mark.gpu


def check(paged, rotary, qkv, exact, starts, got, heads, lengths=None, new=0):
    """The queries, the rows that were stored, and that no other row of the cache changed."""
    lengths = paged.lengths if lengths is None else lengths
    kv = paged.cache.kv_heads
    tokens, d = qkv.shape[0], paged.cache.d
    starts = [i * new for i in range(len(lengths) + 1)] if new else starts
    seq, position = oracle.owners(starts, lengths, tokens)
    f = rotary.frequencies if rotary is not None else []
    interleaved, magnitude = (rotary.interleaved, rotary.magnitude) if rotary is not None else (False, 1.0)
    x = exact.reshape(tokens, heads + 2 * kv, d)
    y, bound = oracle.rotate(x[:, : heads + kv], position, f, interleaved, magnitude)
    bound = bound + (np.abs(y) + bound) * HALF_STEP[paged.kind] + TINY[paged.kind]
    owned = seq >= 0
    q = values(got)
    assert_within(q[owned], y[owned, :heads], bound[owned, :heads], "q")
    keys, vals = paged.cache.keys.to_host(), paged.cache.values.to_host()
    wide = values(paged.cache.keys)
    want_keys, want_values = paged.key_words.copy(), paged.value_words.copy()
    for t in range(tokens):
        at = oracle.place(paged.table, paged.page, seq[t], position[t], len(keys)) if owned[t] else None
        if at is None:
            continue
        number, row = at
        assert_within(wide[number, :, row], y[t, heads:], bound[t, heads:], f"key of token {t}")
        want_keys[number, :, row] = keys[number, :, row]
        want_values[number, :, row] = qkv.reshape(tokens, -1, d)[t, heads + kv:]
    np.testing.assert_array_equal(keys.view(np.uint16), want_keys.view(np.uint16))
    np.testing.assert_array_equal(vals.view(np.uint16), want_values.view(np.uint16))


CASES = [  # counts, before, heads, kv_heads, d, page, rotary, interleaved
    ([1], [0], 1, 1, 64, 16, 64, False),
    ([1], [999], 32, 8, 128, 16, 128, False),
    ([3, 1, 0, 7], [5, 0, 9, 40], 6, 2, 64, 16, 64, True),
    ([17, 33], [15, 64], 7, 1, 128, 32, 128, True),
    ([5, 2], [100, 31], 4, 4, 64, 64, 36, True),
    ([5, 2], [100, 31], 4, 4, 64, 64, 38, False),
    ([9], [3], 3, 3, 128, 128, 48, False),
    ([9], [3], 3, 3, 128, 16, 2, False),
    ([4, 6], [0, 2], 8, 2, 128, 16, 32, True),
    ([1] * 300, [7] * 300, 2, 1, 64, 16, 64, False),
    ([257, 1, 300], [0, 500, 13], 5, 5, 64, 256, 64, False),
    ([0, 0, 11, 0], [3, 0, 0, 0], 2, 2, 64, 16, 62, False),
    ([6], [2], 4, 2, 64, 16, 0, False),
]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("counts,before,heads,kv_heads,d,page,rotary,interleaved", CASES)
def test_queries_keys_and_values(device, kind, counts, before, heads, kv_heads, d, page, rotary, interleaved):
    rng = np.random.default_rng(sum(counts) * 31 + rotary)
    lengths = [c + b for c, b in zip(counts, before)]
    paged = Paged(device, rng, kind, lengths, kv_heads=kv_heads, d=d, page=page)
    tokens = sum(counts)
    qkv, exact = words(rng.standard_normal((tokens, (heads + 2 * kv_heads) * d)), kind)
    turn = Rotary.of(device, rotary, interleaved=interleaved) if rotary else None
    starts = [0, *np.cumsum(counts).tolist()]
    got = rotary_append(paged.tensor(qkv), paged.cache, paged.sequences(starts=starts), rotary=turn)
    assert got.shape == (tokens, heads, d) and got.dtype == TYPES[kind]
    check(paged, turn, qkv, exact, starts, got, heads)


@pytest.mark.parametrize("new", [1, 3, 4, 5])
def test_new_tokens_of_every_sequence(device, new):
    rng = np.random.default_rng(new)
    paged = Paged(device, rng, "bf16", [new, 20, 77, 16, 1000, 33, 48], kv_heads=2, d=128)
    qkv, exact = words(rng.standard_normal((7 * new, 8 * 128)), "bf16")
    turn = Rotary.of(device, 128)
    got = rotary_append(paged.tensor(qkv), paged.cache, paged.sequences(new=new), rotary=turn)
    check(paged, turn, qkv, exact, None, got, 4, new=new)


@pytest.mark.parametrize("position", [0, 1, 65535, 10**6, 2**24 + 1, 2**30 + 7])
@pytest.mark.parametrize("scaled", [{}, {"factor": 4.0}, {"factor": 8.0, "original": 4096}, {"base": 5e5}])
def test_far_positions_and_scaled_frequencies(device, position, scaled):
    """Angles of any size: one page stands at the end of a table whose other entries are not pages."""
    rng = np.random.default_rng(position % 97)
    page = 65536 if position > 2**20 else 16
    paged = Paged(device, rng, "f16", [1], kv_heads=1, d=64, page=page, width=position // page + 1, spare=0)
    paged.lengths, paged.table[0, 0], paged.table[0, -1] = [position + 1], -1, 0
    paged.on_table = device.to_device(paged.table)
    qkv, exact = words(rng.standard_normal((1, 4 * 64)), "f16")
    turn = Rotary.of(device, 64, **scaled)
    got = rotary_append(paged.tensor(qkv), paged.cache, paged.sequences(), rotary=turn)
    check(paged, turn, qkv, exact, None, got, 2, new=1)


def test_tokens_of_no_sequence_and_pages_that_are_not_there(device):
    """Rows before the first start and behind the last one stay as they were; a token of a negative position, beyond its table or
    on a page outside of the cache gets its query and is not stored."""
    rng = np.random.default_rng(8)
    paged = Paged(device, rng, "bf16", [40, 64, 20, 30], kv_heads=2, d=64)
    paged.table[0, 2] = 10**6  # keys 32 to 39 of sequence 0
    paged.table[2, 1] = -5     # keys 16 to 19 of sequence 2
    paged.on_table = device.to_device(paged.table)
    lengths = [40, 66, 20, 2]  # sequence 1 has four pages, sequence 3 fewer keys than tokens
    starts = [3, 13, 19, 25, 30]
    qkv, exact = words(rng.standard_normal((37, 8 * 64)), "bf16")
    out = paged.tensor(np.full((37, 4, 64), 0x4040, np.uint16))
    turn = Rotary.of(device, 64)
    got = rotary_append(paged.tensor(qkv), paged.cache, paged.sequences(starts=starts, lengths=lengths), rotary=turn, out=out)
    check(paged, turn, qkv, exact, starts, got, 4, lengths=lengths)
    host = out.to_host()
    assert (host[:3] == 0x4040).all() and (host[30:] == 0x4040).all() and not (host[3:30] == 0x4040).all(axis=(1, 2)).any()


def test_starts_that_make_no_sense_stay_in_bounds(device):
    """Starts that decrease, or lie outside of the tokens, give some tokens no sequence, and nothing else is written."""
    rng = np.random.default_rng(9)
    paged = Paged(device, rng, "f16", [20, 20, 20], kv_heads=1, d=64)
    qkv, _ = words(rng.standard_normal((12, 3 * 64)), "f16")
    held = device.to_device(np.full(14 * 64, 7, np.float16))
    out = HIPTensor(device, held.pointer + 128, F16, (12, 1, 64), owner=held)
    for starts in ([-4, 5, 2, 100], [50, 60, 70, 80], [-9, -8, -7, -6], [8, 4, 2, 0], [2**31 - 1, -(2**31), 3, 12]):
        rotary_append(paged.tensor(qkv), paged.cache, paged.sequences(starts=starts, lengths=[-3, 2**31 - 1, 20]), out=out)
    host = held.to_host()
    assert (host[:64] == 7).all() and (host[-64:] == 7).all()


def test_infinities_and_nan_stay_in_their_pairs(device):
    rng = np.random.default_rng(10)
    paged = Paged(device, rng, "bf16", [8], kv_heads=1, d=64)
    x = rng.standard_normal((8, 3 * 64))
    x[2, 5], x[3, 64 + 40], x[4, 130] = np.nan, np.inf, np.nan
    with np.errstate(invalid="ignore"):
        qkv, _ = words(x, "bf16")
    turn = Rotary.of(device, 64)
    got = rotary_append(paged.tensor(qkv), paged.cache, paged.sequences(new=8), rotary=turn)
    bad = ~np.isfinite(values(got))
    assert np.argwhere(bad).tolist() == [[2, 0, 5], [2, 0, 37]]
    keys, vals = values(paged.cache.keys), values(paged.cache.values)
    number = paged.table[0, 0]
    assert np.argwhere(~np.isfinite(keys[number, 0, :8])).tolist() == [[3, 8], [3, 40]]
    assert np.argwhere(~np.isfinite(vals[number, 0, :8])).tolist() == [[4, 2]]


def test_nothing_to_append(device):
    paged = Paged(device, np.random.default_rng(1), "bf16", [], kv_heads=1, d=64)
    empty = device.empty(BF16, 0, 192)
    assert rotary_append(empty, paged.cache, paged.sequences()).shape == (0, 1, 64)
    paged = Paged(device, np.random.default_rng(1), "bf16", [5], kv_heads=1, d=64)
    assert rotary_append(empty, paged.cache, paged.sequences(starts=[0, 0])).to_host().shape == (0, 1, 64)


def test_a_cache_beyond_32_bits(device):
    """Rows of a cache of more than 2^31 elements: the last page and the first one."""
    pages, page = 2**31 // (256 * 128) + 2, 256
    cache = KvCache.empty(device, pages, 1, page, 128)
    from krn_amd.dtypes import I32

    table = device.to_device(np.array([[pages - 1], [0]], np.int32))
    rng = np.random.default_rng(3)
    qkv, exact = words(rng.standard_normal((2, 3 * 128)), "bf16")
    got = rotary_append(device.to_device(qkv, BF16), cache, Sequences(device.to_device(np.array([256, 1], np.int32)), table))
    np.testing.assert_array_equal(values(got)[:, 0], exact[:, :128])
    size = 128 * 2
    for number, row, t in ((pages - 1, 255, 0), (0, 0, 1)):
        for data, at in ((cache.keys, 128), (cache.values, 256)):
            one = HIPTensor(device, data.pointer + (number * page + row) * size, BF16, (128,), owner=data)
            np.testing.assert_array_equal(one.to_host(), qkv[t, at:at + 128])
    assert table.dtype == I32
