"""Sizes at which the paged cache's calls take other paths: projections of 128 MiB and more, against the same tokens in smaller
calls, and more sequences than are shared out or found in two looks."""

import numpy as np
import pytest

from krn_amd.lib import KvCache, Rotary, Sequences, cache_attention, rotary_append
from oracle import cache as oracle
from tests.paged import HALF_STEP, TINY, TYPES, Paged, assert_within, values, words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("d,interleaved", [(128, False), (128, True), (64, False), (64, True)])
def test_a_large_projection_is_its_parts(device, kind, d, interleaved):
    """Both kernels do the same arithmetic: the same bits in queries, keys, values and what lies between them."""
    rng = np.random.default_rng(d + interleaved)
    heads, kv_heads, page, counts = 12, 4, 64, [c * 128 // d for c in (9001, 0, 13000, 5000, 7013)]
    tokens, n, row = sum(counts), len(counts), (heads + 2 * kv_heads) * d
    assert tokens * row * 2 >= 1 << 27 and 2 * max(sum(counts[:3]), sum(counts[3:])) * row < 1 << 27
    lengths = [c + b for c, b in zip(counts, (0, 5, 100, 63, 1000))]
    width = -(-max(lengths) // page)
    owned = [-(-length // page) for length in lengths]
    table = np.full((n, width), -1, np.int32)
    order = rng.permutation(sum(owned)).astype(np.int32)
    for i, count in enumerate(owned):
        table[i, :count] = order[sum(owned[:i]) : sum(owned[:i]) + count]
    # any values below 2: the highest bit of the exponent is clear
    qkv = rng.integers(0, 1 << 16, (tokens, row), np.uint16) & np.uint16(0xBFFF)
    host = qkv if kind == "bf16" else qkv.view(np.float16)
    turn = Rotary.of(device, d, interleaved=interleaved, factor=2.0, original=4096)

    def appended(groups):
        cache = KvCache(*(device.to_device(np.zeros((sum(owned), kv_heads, page, d), host.dtype), TYPES[kind]) for _ in range(2)))
        q = []
        for first, last in groups:
            starts = np.concatenate([[0], np.cumsum(counts[first:last])]).astype(np.int32)
            at = sum(counts[:first])
            sequences = Sequences(device.to_device(np.array(lengths[first:last], np.int32)),
                                  device.to_device(table[first:last].copy()), starts=device.to_device(starts))
            part = device.to_device(np.ascontiguousarray(host[at : at + starts[-1]]), TYPES[kind])
            q.append(rotary_append(part, cache, sequences, rotary=turn).to_host())
        return [np.concatenate(q).view(np.uint16), cache.keys.to_host().view(np.uint16), cache.values.to_host().view(np.uint16)]

    for got, want in zip(appended([(0, n)]), appended([(0, 3), (3, n)])):
        np.testing.assert_array_equal(got, want)
        assert got.any()


@pytest.mark.parametrize("packed", [True, False])
def test_more_sequences_than_are_shared_out(device, packed):
    """8300 sequences, two of them long: each stays in one workgroup."""
    rng = np.random.default_rng(8300)
    n, long = 8300, {4097: 2000, 8299: 900}
    lengths = rng.integers(0, 30, n)
    counts = rng.integers(0, 3, n) if packed else np.ones(n, int)
    for i, length in long.items():
        lengths[i], counts[i] = length, 1
    paged = Paged(device, rng, "bf16", lengths.tolist(), kv_heads=1, d=64)
    starts = [0, *np.cumsum(counts).tolist()]
    sequences = paged.sequences(starts=starts) if packed else paged.sequences()
    q, exact = words(rng.standard_normal((starts[-1], 2, 64)), "bf16")
    got = values(cache_attention(paged.tensor(q), paged.cache, sequences))
    assert_within(got, *paged.attention(exact, starts))
    qkv, exact = words(rng.standard_normal((starts[-1], 4 * 64)), "bf16")
    turn = Rotary.of(device, 64)
    got = values(rotary_append(paged.tensor(qkv), paged.cache, sequences, rotary=turn))
    y, bound = oracle.rotate(exact.reshape(-1, 4, 64)[:, :2], oracle.owners(starts, paged.lengths, starts[-1])[1], turn.frequencies)
    assert_within(got, y, bound + (np.abs(y) + bound) * HALF_STEP["bf16"] + TINY["bf16"])


def test_keys_stay_in_one_workgroup_of_many_packed_sequences(device):
    """300 sequences of a wide table whose rows fill the chip, one of them long, beside a prompt."""
    rng = np.random.default_rng(300)
    counts, before = np.ones(300, int), rng.integers(0, 50, 300)
    counts[7], before[200] = 500, 9000
    lengths = (counts + before).tolist()
    paged = Paged(device, rng, "f16", lengths, kv_heads=8, d=64, page=32)
    starts = [0, *np.cumsum(counts).tolist()]
    q, exact = words(rng.standard_normal((starts[-1], 16, 64)), "f16")
    got = values(cache_attention(paged.tensor(q), paged.cache, paged.sequences(starts=starts)))
    for i in (0, 6, 8, 199, 200, 201, 299):
        one = Paged.__new__(Paged)
        one.__dict__ = {**paged.__dict__, "table": paged.table[i : i + 1], "lengths": lengths[i : i + 1]}
        assert_within(got[starts[i] : starts[i + 1]], *one.attention(exact[starts[i] : starts[i + 1]], [0, counts[i]]))
