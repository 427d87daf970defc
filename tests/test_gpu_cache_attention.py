"""Attention over a paged cache on the GPU, packed prompts and new tokens, against oracle/cache.py in float64 within the bound
derived there, and on inputs whose weights are exact: equal ones, which show every key that is lost or seen too much, and single
ones, which show a key in a wrong place."""

import numpy as np
import pytest

from krn_amd.dtypes import BF16
from krn_amd.lib import KvCache, Sequences, cache_attention
from krn_amd.runtime.hip import HIPTensor
from tests.paged import HALF_STEP, TINY, TYPES, Paged, assert_within, values, words

pytestmark = pytest.mark.gpu

# counts of new tokens, keys before them, heads, kv_heads, d, page, window
PACKED = [
    ([1], [0], 1, 1, 64, 16, 0), ([2], [0], 2, 1, 128, 16, 0), ([33], [0], 4, 4, 64, 16, 0), ([100], [0], 8, 2, 128, 16, 0),
    ([64, 64], [0, 0], 4, 1, 128, 64, 0), ([5, 0, 130, 1], [0, 7, 3, 200], 6, 2, 64, 16, 0), ([300], [211], 7, 1, 128, 32, 0),
    ([17] * 9, list(range(9)), 3, 3, 128, 16, 0), ([70, 9], [500, 1000], 5, 1, 64, 128, 0), ([257], [0], 2, 2, 128, 256, 0),
    ([90], [40], 4, 2, 128, 16, 1), ([90], [40], 4, 2, 64, 16, 33), ([200, 31], [400, 0], 8, 2, 128, 32, 100),
    ([1] * 70, [11] * 70, 16, 1, 64, 16, 0), ([40], [0], 48, 1, 64, 16, 0), ([513], [70], 1, 1, 64, 16, 64),
    # few rows, many keys: the keys of a tile of rows in several parts
    ([40], [3000], 4, 1, 128, 16, 0), ([150, 5], [2500, 4000], 8, 2, 64, 32, 0), ([60, 0, 90], [5000, 9, 1], 4, 2, 128, 64, 3000),
    ([3, 200], [7000, 1500], 3, 3, 64, 128, 0), ([1] * 5, [2000, 1, 1500, 40, 3000], 8, 1, 128, 16, 0),
]  # fmt: skip
# lengths, new tokens each, heads, kv_heads, d, page, window
TOKENS = [
    ([1], 1, 1, 1, 64, 16, 0), ([2, 1], 1, 2, 2, 128, 16, 0), ([16, 17, 15], 1, 4, 1, 128, 16, 0), ([1000], 1, 8, 2, 128, 16, 0),
    ([33, 1, 700, 64, 65], 1, 7, 1, 64, 32, 0), ([4000, 1, 2], 1, 4, 4, 64, 16, 0), ([129, 2000], 1, 32, 2, 128, 128, 0),
    ([5000], 1, 16, 1, 128, 64, 0), ([300, 40], 1, 17, 1, 64, 16, 0), ([200, 3], 1, 40, 1, 128, 16, 0),
    ([700, 9, 31], 3, 4, 2, 128, 16, 0), ([64, 2000], 4, 16, 2, 64, 32, 0), ([1500, 40], 1, 4, 2, 128, 16, 100),
    ([1500, 40, 3], 3, 9, 9, 64, 32, 500), ([900], 2, 6, 3, 128, 256, 1), ([31] * 40, 1, 4, 2, 64, 16, 0),
    ([50, 2, 1], 8, 8, 1, 128, 16, 0), ([4000, 200], 20, 8, 1, 128, 16, 0), ([3000], 100, 2, 2, 64, 16, 1000), ([2100], 1, 2, 2, 64, 1024, 0),
]  # fmt: skip


def small(rng, shape):
    return rng.integers(-9, 10, shape)


def signs(rng, shape):
    return rng.choice([-1.0, 1.0], shape)


def case_of(device, rng, kind, sizes, packed, fill=None):
    if packed:
        counts, before, heads, kv_heads, d, page, window = sizes
        lengths, new = [c + b for c, b in zip(counts, before)], 0
        starts = [0, *np.cumsum(counts).tolist()]
    else:
        lengths, new, heads, kv_heads, d, page, window = sizes
        starts = [i * new for i in range(len(lengths) + 1)]
    paged = Paged(device, rng, kind, lengths, kv_heads=kv_heads, d=d, page=page, fill=fill)
    return paged, paged.sequences(starts=starts) if packed else paged.sequences(new=new), starts, heads, window


FORMS = [(sizes, True) for sizes in PACKED] + [(sizes, False) for sizes in TOKENS]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,packed", FORMS)
def test_attention_is_the_oracles(device, kind, sizes, packed):
    rng = np.random.default_rng(len(sizes[0]) * 7 + sizes[4])
    paged, sequences, starts, heads, window = case_of(device, rng, kind, sizes, packed)
    q, exact = words(2 * rng.standard_normal((starts[-1], heads, paged.cache.d)), kind)
    got = cache_attention(paged.tensor(q), paged.cache, sequences, window=window or None)
    assert got.shape == q.shape and got.dtype == TYPES[kind]
    assert_within(values(got), *paged.attention(exact, starts, window=window))
    np.testing.assert_array_equal(cache_attention(paged.tensor(q), paged.cache, sequences, window=window or None).to_host(),
                                  got.to_host())  # the same bits again


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,packed", FORMS)
def test_equal_weights_count_every_key_once(device, kind, sizes, packed):
    """Queries of zeros: every weight is 1, the sums of small whole values are exact, and the mean is off by the reciprocal of the
    count, a product and the result's rounding. The oracle's own float64 sum of n weights 1 / n times at most 9 is off by at most
    9 (n + 3) 2^-52 < 1e-10, also where the exact mean is zero."""
    rng = np.random.default_rng(len(sizes[0]) * 11 + sizes[3])
    paged, sequences, starts, heads, window = case_of(device, rng, kind, sizes, packed, fill=(signs, small))
    q = np.zeros((starts[-1], heads, paged.cache.d), np.uint16 if kind == "bf16" else np.float16)
    got = values(cache_attention(paged.tensor(q), paged.cache, sequences, window=window or None))
    y, _ = paged.attention(q.astype(np.float64), starts, window=window)
    assert_within(got, y, np.abs(y) * (2.0**-22 + HALF_STEP[kind]) + 1e-10 + TINY[kind])


@pytest.mark.parametrize("sizes,packed", FORMS)
def test_a_single_weight_finds_its_key(device, sizes, packed):
    """Keys of random signs and a query of eight times one of those it sees: the others' weights are below 2^-100 of its own (at
    scale 1, scores of 8 d against 8 (d - 2 m), m the columns that differ), and the result is its value."""
    rng = np.random.default_rng(len(sizes[0]) * 13 + sizes[3])
    paged, sequences, starts, heads, window = case_of(device, rng, "f16", sizes, packed, fill=(signs, _normal))
    group, d = heads // paged.cache.kv_heads, paged.cache.d
    q, want = np.zeros((starts[-1], heads, d)), np.zeros((starts[-1], heads, d))
    for i, length in enumerate(paged.lengths):
        for t in range(starts[i], starts[i + 1]):
            position = length - (starts[i + 1] - t)
            if position < 0:
                continue
            low = max(0, position + 1 - window) if window else 0
            for h in range(heads):
                j = position if h == 0 else low if h == heads - 1 else int(rng.integers(low, position + 1))
                number, row = paged.table[i, j // paged.page], j % paged.page
                q[t, h], want[t, h] = 8 * paged.keys[number, h // group, row], paged.values[number, h // group, row]
    got = values(cache_attention(paged.tensor(words(q, "f16")[0]), paged.cache, sequences, scale=1.0, window=window or None))
    assert_within(got, want, np.abs(want) * (2 * HALF_STEP["f16"] + 2.0**-20) + TINY["f16"])


def _normal(rng, shape):
    return rng.standard_normal(shape)


@pytest.mark.parametrize("packed", [True, False])
def test_tokens_of_no_sequence_keep_their_rows_and_tokens_of_no_keys_get_zeros(device, packed):
    rng = np.random.default_rng(2)
    paged = Paged(device, rng, "bf16", [40, 64, 0, 20], kv_heads=2, d=64)
    lengths = [40, 66, 0, -7]  # sequence 1 has four pages of 16; the last two have no keys
    starts = [3, 13, 80, 82, 85] if packed else [0, 1, 2, 3, 4]
    tokens = 91 if packed else 4
    q, exact = words(rng.standard_normal((tokens, 4, 64)), "bf16")
    out = paged.tensor(np.full((tokens, 4, 64), 0x4040, np.uint16))
    sequences = paged.sequences(starts=starts, lengths=lengths) if packed else paged.sequences(lengths=lengths)
    got = values(cache_attention(paged.tensor(q), paged.cache, sequences, out=out))
    y, bound = paged.attention(exact, starts, lengths=lengths)
    owned = ~np.isnan(y).any(axis=(1, 2))
    assert_within(got[owned], y[owned], bound[owned])
    assert (out.to_host()[~owned] == 0x4040).all() and owned.sum() == starts[-1] - starts[0]
    assert (got[starts[2]:starts[4]] == 0).all()


@pytest.mark.parametrize("packed", [True, False])
def test_pages_that_are_not_there_read_as_zeros(device, packed):
    rng = np.random.default_rng(3)
    paged = Paged(device, rng, "f16", [100, 500], kv_heads=1, d=128, page=32)
    paged.table[0, 1], paged.table[1, 3], paged.table[1, 15] = -1, 2**31 - 1, -(2**31)
    paged.on_table = device.to_device(paged.table)
    starts = [0, 2, 4]
    q, exact = words(rng.standard_normal((4, 4, 128)), "f16")
    sequences = paged.sequences(starts=starts) if packed else paged.sequences(new=2)
    assert_within(values(cache_attention(paged.tensor(q), paged.cache, sequences)), *paged.attention(exact, starts))


@pytest.mark.parametrize("packed", [True, False])
def test_starts_and_lengths_that_make_no_sense_stay_in_bounds(device, packed):
    rng = np.random.default_rng(4)
    paged = Paged(device, rng, "f16", [20, 20, 20], kv_heads=1, d=64)
    q = paged.tensor(words(rng.standard_normal((12, 2, 64)), "f16")[0])
    held = device.to_device(np.full(14 * 128, 7, np.float16))
    out = HIPTensor(device, held.pointer + 256, TYPES["f16"], (12, 2, 64), owner=held)
    for lengths in ([-3, 2**31 - 1, 20], [-(2**31), 2, 33]):
        for starts in ([-4, 5, 2, 100], [50, 60, 70, 80], [-9, -8, -7, -6], [8, 4, 2, 0], [2**31 - 1, -(2**31), 3, 12]):
            sequences = paged.sequences(starts=starts, lengths=lengths) if packed else paged.sequences(lengths=lengths, new=4)
            cache_attention(q, paged.cache, sequences, out=out)
    host = held.to_host()
    assert (host[:128] == 7).all() and (host[-128:] == 7).all()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("packed", [True, False])
def test_large_scores_and_infinite_ones(device, kind, packed):
    """Scores in the thousands, growing and falling along the keys, and keys of minus infinity, which have no weight."""
    rng = np.random.default_rng(5)
    paged = Paged(device, rng, kind, [333, 150], kv_heads=1, d=64, fill=(_normal, _normal))
    for i, length in enumerate(paged.lengths):
        for j in range(length):
            paged.keys[paged.table[i, j // 16], 0, j % 16] = (j % 100 if i else length - j) / 4
    paged.keys[paged.table[0, 3], 0, 5, 7] = -np.inf
    paged.key_words, paged.keys = words(paged.keys, kind)
    paged.cache = KvCache(paged.tensor(paged.key_words), paged.cache.values)
    q, exact = words(rng.integers(1, 5, (6, 2, 64)), kind)
    starts = [0, 3, 6]
    sequences = paged.sequences(starts=starts) if packed else paged.sequences(new=3)
    got = values(cache_attention(paged.tensor(q), paged.cache, sequences))
    where = (paged.table[0, 3], 0, 5)
    paged.keys[where] = 0
    paged.keys[where][7] = -60000  # as good as minus infinity, and the oracle's arithmetic stays finite
    y, bound = paged.attention(exact, starts)
    assert_within(got, y, bound)


@pytest.mark.parametrize("packed,counts", [(True, [3]), (True, [200]), (False, [4]), (False, [100])])
def test_scores_far_below_zero(device, packed, counts):
    """Equal scores of -7200: the weights are equal, in every part that the keys are shared out to, but for roundings of exponents
    of that size: 7200 * 2^-24 of a weight, in the maximum that it is taken from too, and for both once more where parts are
    joined; values are at most 9."""
    rng = np.random.default_rng(11)
    paged = Paged(device, rng, "f16", [5000], kv_heads=1, d=64, fill=(lambda rng, shape: np.full(shape, -30.0), small))
    starts = [0, *np.cumsum(counts).tolist()]
    q = np.full((starts[-1], 2, 64), 30, np.float16)
    sequences = paged.sequences(starts=starts) if packed else paged.sequences(new=counts[0])
    got = values(cache_attention(paged.tensor(q), paged.cache, sequences))
    y, _ = paged.attention(q.astype(np.float64), starts)
    assert_within(got, y, 4 * 7200 * 2.0**-24 * 9 + np.abs(y) * 2 * HALF_STEP["f16"])


@pytest.mark.parametrize("packed", [True, False])
def test_nan_reaches_its_own_head_and_sequence_only(device, packed):
    rng = np.random.default_rng(6)
    paged = Paged(device, rng, "bf16", [90, 80], kv_heads=2, d=64)
    paged.keys[paged.table[0, 2], 1, 3, 9] = np.nan  # key 35
    paged.values[paged.table[1, 4], 0, 1, 63] = np.nan  # value 65
    with np.errstate(invalid="ignore"):
        cache = KvCache(paged.tensor(words(paged.keys, "bf16")[0]), paged.tensor(words(paged.values, "bf16")[0]))
    q, exact = words(rng.standard_normal((8, 4, 64)), "bf16")
    starts = [0, 4, 8]
    sequences = paged.sequences(starts=starts) if packed else paged.sequences(new=4)
    got = values(cache_attention(paged.tensor(q), cache, sequences))
    bad = np.zeros((8, 4, 64), bool)
    bad[:4, 2:], bad[4:, :2, 63] = True, True
    np.testing.assert_array_equal(np.isnan(got), bad)
    y, bound = paged.attention(exact, starts)
    assert np.all(np.abs(got - y)[~bad] <= bound[~bad])


# packed or new tokens each, lengths, counts of new tokens, heads, kv_heads, d, page, window
UNSEEN = [
    (True, [100], [90], 4, 2, 128, 16, 0), (True, [500, 31], [300, 31], 8, 2, 64, 32, 0), (True, [3040], [40], 4, 1, 128, 16, 0),
    (True, [600, 40], [200, 31], 8, 2, 128, 32, 100), (True, [513], [313], 1, 1, 64, 16, 33), (True, [2000], [60], 6, 2, 64, 64, 900),
    (False, [70, 300], [4, 4], 4, 2, 128, 16, 0), (False, [3000], [8], 8, 1, 64, 32, 0), (False, [1500, 90], [1, 1], 4, 2, 128, 16, 100),
    (False, [1500], [20], 9, 3, 64, 16, 37), (False, [400], [100], 4, 4, 64, 32, 70),
]  # fmt: skip


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("packed,lengths,counts,heads,kv_heads,d,page,window", UNSEEN)
def test_what_a_token_does_not_see_does_not_reach_it(device, kind, packed, lengths, counts, heads, kv_heads, d, page, window):
    """NaN and infinities in some of the new keys and values, in a column of theirs or a head, and in all that lies before the
    first window, whose pages may be another sequence's by then. A token that sees none of them gets what it gets without."""
    rng = np.random.default_rng(12)
    paged = Paged(device, rng, kind, lengths, kv_heads=kv_heads, d=d, page=page)
    starts, group = [0, *np.cumsum(counts).tolist()], heads // kv_heads
    bad = np.zeros((starts[-1], heads, d), bool)
    put = []
    for i, (length, count) in enumerate(zip(lengths, counts)):
        positions = np.arange(length - count, length)
        lows = np.maximum(0, positions + 1 - window) if window else 0 * positions
        at = lambda k: (paged.table[i, k // page], slice(None), k % page)  # noqa: B023, E731
        for k in range(lows[0]):
            put += [(paged.keys, at(k), np.nan), (paged.values, at(k), rng.choice([np.nan, np.inf, -np.inf]))]
        some = np.arange(1 + (lows if window else positions)[0], length)  # not all tokens see these
        for n, k in enumerate(sorted(rng.choice(some, min(5, len(some)), replace=False))):
            page_, _, row = at(k)
            head, col = rng.integers(kv_heads), rng.integers(d)
            sees = (starts[i] + np.flatnonzero((positions >= k) & (lows <= k)))[:, None]
            of_head = np.arange(head * group, (head + 1) * group)
            if n == 3:
                put.append((paged.keys, (page_, head, row), np.nan))
                bad[sees, of_head] = True
            else:
                put.append((paged.values, (page_, head, row, col), [np.nan, np.inf, -np.inf][n % 3]))
                bad[sees, of_head, col] = True
    assert 0 < bad.sum() < bad.size
    for data, where, value in put:
        data[where] = value
    with np.errstate(invalid="ignore"):
        cache = KvCache(paged.tensor(words(paged.keys, kind)[0]), paged.tensor(words(paged.values, kind)[0]))
    for data, where, _ in put:
        data[where] = 0
    q, exact = words(rng.standard_normal((starts[-1], heads, d)), kind)
    sequences = paged.sequences(starts=starts) if packed else paged.sequences(new=counts[0])
    got = values(cache_attention(paged.tensor(q), cache, sequences, window=window or None))
    y, bound = paged.attention(exact, starts, window=window)
    np.testing.assert_array_equal(~np.isfinite(got), bad)
    assert np.all(np.abs(got - y)[~bad] <= bound[~bad])


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("scale", [1e-30, 0.01, 3.0])
def test_scales(device, packed, scale):
    rng = np.random.default_rng(7)
    paged = Paged(device, rng, "f16", [70, 200], kv_heads=2, d=64)
    q, exact = words(rng.standard_normal((4, 6, 64)), "f16")
    sequences = paged.sequences(starts=[0, 2, 4]) if packed else paged.sequences(new=2)
    got = cache_attention(paged.tensor(q), paged.cache, sequences, scale=scale)
    assert_within(values(got), *paged.attention(exact, [0, 2, 4], scale=scale))


@pytest.mark.parametrize("packed", [True, False])
def test_a_result_over_its_queries(device, packed):
    rng = np.random.default_rng(8)
    paged = Paged(device, rng, "bf16", [700, 30, 1000], kv_heads=2, d=128)
    starts = [0, 4, 8, 12]
    sequences = paged.sequences(starts=starts) if packed else paged.sequences(new=4)
    q, exact = words(rng.standard_normal((12, 4, 128)), "bf16")
    held = paged.tensor(q)
    got = cache_attention(held, paged.cache, sequences, out=held)
    assert got is held
    assert_within(values(held), *paged.attention(exact, starts))


@pytest.mark.parametrize("packed,n", [(True, 2), (True, 20), (True, 64), (True, 65), (False, 20), (False, 64)])
def test_more_rows_than_run_at_once_are_those_of_each_sequence_alone(device, packed, n):
    """Workgroups may take rows in any order: every row is the same to the last bit, and the others stay as they were."""
    rng = np.random.default_rng(n)
    counts = np.array([4000, 2500]) if n == 2 else rng.integers(0, 12000 // n, n) if packed else np.full(n, 100)
    if packed and n > 2:
        counts[3], counts[n - 1] = 0, 1
    lengths = [int(c + b) for c, b in zip(counts, rng.integers(0, 400, n))]
    if not packed:
        lengths[2], lengths[5] = 30, 0  # fewer keys than new tokens
    paged = Paged(device, rng, "bf16", lengths, kv_heads=16, d=64)
    starts = [2, *(2 + np.cumsum(counts)).tolist()] if packed else [0, *np.cumsum(counts).tolist()]
    tokens = starts[-1] + (3 if packed else 0)
    q, _ = words(rng.standard_normal((tokens, 32, 64)), "bf16")
    out = paged.tensor(np.full((tokens, 32, 64), 0x4040, np.uint16))
    cache_attention(paged.tensor(q), paged.cache, paged.sequences(starts=starts) if packed else paged.sequences(new=100), out=out)
    got = out.to_host()
    assert (got[: starts[0]] == 0x4040).all() and (got[starts[-1] :] == 0x4040).all()
    for i in range(n):
        rows = slice(starts[i], starts[i + 1])
        if counts[i] == 0:
            continue
        one = Sequences(device.to_device(np.array(lengths[i : i + 1], np.int32)), device.to_device(paged.table[i : i + 1].copy()),
                        starts=device.to_device(np.array([0, counts[i]], np.int32)))
        np.testing.assert_array_equal(got[rows], cache_attention(paged.tensor(q[rows].copy()), paged.cache, one).to_host())


@pytest.mark.parametrize("prompt", [2000, 1300, 100])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_few_tokens_before_many_keys_beside_a_prompt(device, kind, prompt):
    """The keys of some rows in parts, and rows that see fewer key tiles than their sequence has parts, beside whole ones."""
    rng = np.random.default_rng(prompt)
    counts, before = [1, prompt, 40, 0, 3, 30], [9000, 0, 8500, 7, 12000, 0]
    lengths = [c + b for c, b in zip(counts, before)]
    paged = Paged(device, rng, kind, lengths, kv_heads=8, d=64, page=32)
    starts = [0, *np.cumsum(counts).tolist()]
    q, exact = words(rng.standard_normal((starts[-1], 32, 64)), kind)
    got = values(cache_attention(paged.tensor(q), paged.cache, paged.sequences(starts=starts)))
    for i in (0, 2, 4, 5):
        rows = slice(starts[i], starts[i + 1])
        part = exact[rows]
        one = Paged.__new__(Paged)
        one.__dict__ = {**paged.__dict__, "table": paged.table[i : i + 1], "lengths": lengths[i : i + 1]}
        assert_within(got[rows], *one.attention(part, [0, counts[i]]))
    own = Sequences(device.to_device(np.array([prompt], np.int32)), device.to_device(paged.table[1:2, : -(-prompt // 32)].copy()),
                    starts=device.to_device(np.array([0, prompt], np.int32)))
    alone = values(cache_attention(paged.tensor(q[starts[1] : starts[2]].copy()), paged.cache, own))
    np.testing.assert_array_equal(got[starts[1] : starts[2]], alone)


def test_nothing_to_attend(device):
    paged = Paged(device, np.random.default_rng(1), "bf16", [], kv_heads=1, d=64)
    empty = device.empty(BF16, 0, 3, 64)
    assert cache_attention(empty, paged.cache, paged.sequences()).shape == (0, 3, 64)
    paged = Paged(device, np.random.default_rng(1), "bf16", [5], kv_heads=1, d=64)
    assert cache_attention(empty, paged.cache, paged.sequences(starts=[0, 0])).to_host().shape == (0, 3, 64)


@pytest.mark.parametrize("packed", [True, False])
def test_a_cache_beyond_32_bits(device, packed):
    """Pages whose rows start beyond 2^31 elements."""
    pages, page = 2**31 // (256 * 128) + 3, 256
    cache = KvCache.empty(device, pages, 1, page, 128)
    rng = np.random.default_rng(3)
    kk, vv = (words(rng.standard_normal((2, page, 128)), "bf16") for _ in range(2))
    for data, (host, _) in ((cache.keys, kk), (cache.values, vv)):
        HIPTensor(device, data.pointer + (pages - 2) * page * 256, BF16, (2, page, 128), owner=data).copy_from(host)
    table = np.array([[pages - 1, pages - 2]], np.int32)
    q, exact = words(rng.standard_normal((1, 2, 128)), "bf16")
    lengths = device.to_device(np.array([500], np.int32))
    if packed:
        sequences = Sequences(lengths, device.to_device(table), starts=device.to_device(np.array([0, 1], np.int32)))
    else:
        sequences = Sequences(lengths, device.to_device(table))
    got = values(cache_attention(device.to_device(q, BF16), cache, sequences))
    from oracle import cache as oracle

    y, bound = oracle.attention(exact, kk[1][:, None], vv[1][:, None], [0, 1], [500], np.array([[1, 0]]), 128**-0.5, 0, 2.0**-8)
    assert_within(got, y, bound + (np.abs(y) + bound) * 2.0**-8)
