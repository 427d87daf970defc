"""The softmax weights of attention over a paged cache where their 16-bit forms could lose them: many small ones beside a
large one, and sums that nearly cancel, which show whether a weight has one 16-bit part or two. Keys and values repeat every
sixteen keys, so wherever the keys are shared out, each share has the large weights too."""

import math

import numpy as np
import pytest

from krn_amd.lib import cache_attention
from oracle import cache as oracle
from tests.paged import HALF_STEP, TINY, Paged, assert_within, values, words

# packed, lengths, counts of new tokens, heads, kv_heads, d
FORMS = [
    (True, [16], [1], 1, 1, 64), (True, [3040], [40], 4, 2, 128), (True, [600, 39], [200, 31], 8, 2, 64), (True, [1000], [1000], 2, 1, 128),
    (False, [16], [1], 1, 1, 64), (False, [1000], [1], 8, 2, 128), (False, [500, 33, 2], [3, 3, 3], 4, 4, 64),
    (False, [1000, 64], [4, 4], 8, 1, 64), (False, [320] * 5, [1] * 5, 17, 1, 128),
]  # fmt: skip
# What a weight may be off by, relative, and near zero in units of the largest: one 16-bit part or two, f16 ones multiplied by
# 2^7, so that half of their last step, 2^-25, is 2^-32 of the largest.
ONE_PART = HALF_STEP
TWO_PARTS = {"bf16": 2.0**-17, "f16": 2.0**-23}
NEAR_ZERO = {"bf16": 2.0**-133, "f16": 2.0**-32}


def repeated(device, kind, lengths, kv_heads, d, keys, vals):
    """A cache whose sequences have the rows `keys`, of the first columns, and one of `vals` in every column, again and again."""
    def fill_keys(rng, shape):
        k = np.zeros(shape)
        k[:, :, : keys.shape[1]] = keys[: shape[1]]
        return k

    def fill_values(rng, shape):
        return np.broadcast_to(vals[: shape[1], None], shape)

    return Paged(device, np.random.default_rng(1), kind, lengths, kv_heads=kv_heads, d=d, fill=(fill_keys, fill_values))


def sinks(device, kind, lengths, kv_heads, d):
    """One key in sixteen has the weight 1 and the value 0, the others the weight e^-17.625, below 2^-25, and the value 1000."""
    keys = np.zeros((16, 1))
    keys[0] = 17.625
    return repeated(device, kind, lengths, kv_heads, d, keys, np.where(np.arange(16) == 0, 0.0, 1000.0))


def halves(kind):
    """A weight just below the middle between one half and the type's next value, and the logarithm as a sum of its values."""
    weight, parts = 0.5 * (1 + 0.98 * HALF_STEP[kind]), []
    left = math.log(weight)
    for _ in range(4):
        parts.append(float(words(np.array([left]), kind)[1][0]))
        left -= parts[-1]
    return weight, parts


def cancelling(device, kind, lengths, kv_heads, d):
    """Keys in turns of the weight 1 and the value 1, and of a weight that one part rounds to 1/2 and the value -2."""
    keys = np.zeros((16, 4))
    keys[1::2] = halves(kind)[1]
    return repeated(device, kind, lengths, kv_heads, d, keys, np.where(np.arange(16) % 2 == 0, 1.0, -2.0))


def queries(kind, tokens, heads, d, columns):
    q = np.zeros((tokens, heads, d))
    q[:, :, :columns] = 1
    return words(q, kind)


def starts_of(counts):
    return [0, *np.cumsum(counts).tolist()]


def rounded(y, bound, kind):
    return y, bound + (np.abs(y) + bound) * HALF_STEP[kind] + TINY[kind]


def call(paged, packed, counts, q, **kwargs):
    sequences = paged.sequences(starts=starts_of(counts)) if packed else paged.sequences(new=counts[0])
    return values(cache_attention(paged.tensor(q), paged.cache, sequences, **kwargs))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("packed,lengths,counts,heads,kv_heads,d", FORMS)
def test_many_small_weights_count_beside_a_large_one(device, kind, packed, lengths, counts, heads, kv_heads, d):
    """A token sees at most fifteen small weights for each large one: what they lose near zero is 15 * 1000 of it."""
    paged = sinks(device, kind, lengths, kv_heads, d)
    q, exact = queries(kind, sum(counts), heads, d, 1)
    got = call(paged, packed, counts, q, scale=1.0)
    y, bound = oracle.attention(exact, np.nan_to_num(paged.keys), np.nan_to_num(paged.values), starts_of(counts), lengths,
                                paged.table, 1.0, weight=ONE_PART[kind])
    assert_within(got, *rounded(y, bound + 15 * 1000 * NEAR_ZERO[kind], kind))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("packed,lengths,counts,heads,kv_heads,d", [form for form in FORMS if not form[0]])
def test_weights_of_new_tokens_have_two_parts(device, kind, packed, lengths, counts, heads, kv_heads, d):
    paged = cancelling(device, kind, lengths, kv_heads, d)
    q, exact = queries(kind, sum(counts), heads, d, 4)
    assert_within(call(paged, packed, counts, q, scale=1.0), *rounded(*oracle.attention(
        exact, np.nan_to_num(paged.keys), np.nan_to_num(paged.values), starts_of(counts), lengths, paged.table, 1.0,
        weight=TWO_PARTS[kind], tiny=NEAR_ZERO[kind]), kind))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("n", [16, 320, 1000])
def test_one_part_is_more_than_two_parts_may_be_off(kind, n):
    """On the host: weights of one part give zero where the test above accepts no such thing. (The logarithm's last part is off
    by half of f16's last step, 2^-25.)"""
    paged = cancelling(None, kind, [n], 1, 64)
    _, exact = queries(kind, 1, 1, 64, 4)
    y, bound = rounded(*oracle.attention(exact, paged.keys, paged.values, [0, 1], [n], paged.table, 1.0, weight=TWO_PARTS[kind],
                                         tiny=NEAR_ZERO[kind]), kind)
    weight = halves(kind)[0]
    np.testing.assert_allclose(y, (1 - 2 * weight) / (1 + weight), rtol=0, atol=2.0**-25)
    one = words(np.array([weight]), kind)[1][0]
    assert one == 0.5 and (np.abs((1 - 2 * one) / (1 + weight) - y) > bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("packed,lengths,counts,heads,kv_heads,d", FORMS)
def test_scores_of_minus_infinity_alone_give_zeros(device, kind, packed, lengths, counts, heads, kv_heads, d):
    paged = repeated(device, kind, lengths, kv_heads, d, np.full((16, 1), -np.inf), np.ones(16))
    got = call(paged, packed, counts, queries(kind, sum(counts), heads, d, 1)[0])
    np.testing.assert_array_equal(got, np.zeros(got.shape))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("size", [1e5, 3e7, 7e7, 1e8, 2e8])
@pytest.mark.parametrize("packed,lengths,counts,heads,kv_heads,d", FORMS)
def test_scores_whose_steps_are_large_give_a_mean(device, kind, size, packed, lengths, counts, heads, kv_heads, d):
    """Scores of up to 10^8 differ by float32's steps, 8 and 16 there: the weights are what they come to, but a mean of equal
    values is that value, off by a weight's rounding, of n sums' 2^-23 (n + 64), and the result's."""
    rng = np.random.default_rng(int(size) % 1009)
    vals = rng.integers(1, 9, d).astype(float)

    def fill_keys(rng, shape):
        k = np.zeros(shape)
        k[:, :, 0], k[:, :, 1] = size / 30000, rng.integers(0, 60, shape[:2])
        return k

    paged = Paged(device, rng, kind, lengths, kv_heads=kv_heads, d=d, fill=(fill_keys, lambda rng, shape: np.broadcast_to(vals, shape)))
    q = np.zeros((sum(counts), heads, d))
    q[:, :, 0], q[:, :, 1] = rng.integers(25000, 32000, q.shape[:2]), rng.integers(-1, 2, q.shape[:2])
    got = call(paged, packed, counts, words(q, kind)[0], scale=1.0)
    n = max(lengths)
    _, position = oracle.owners(starts_of(counts), lengths, sum(counts))
    want = np.broadcast_to(vals, got.shape) * (position >= 0)[:, None, None]  # a token before all keys has none
    assert_within(got, *rounded(want, want * (ONE_PART[kind] + n * NEAR_ZERO[kind] + (n + 64) * 2.0**-23), kind))
