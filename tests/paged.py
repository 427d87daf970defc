"""Paged caches for the tests: sequences of given lengths on pages in random order, on the host and on the device."""

import numpy as np

from krn_amd.dtypes import BF16, F16, I32
from krn_amd.lib import KvCache, Sequences
from oracle import cache as oracle
from oracle.numerics import bf16_values, bf16_words

TYPES = {"bf16": BF16, "f16": F16}
HALF_STEP = {"bf16": 2.0**-8, "f16": 2.0**-11}
TINY = {"bf16": 2.0**-133, "f16": 2.0**-25}


def words(x, kind):
    """x rounded to the type, as it is stored, and those values."""
    if kind == "bf16":
        w = bf16_words(np.asarray(x, np.float32))
        return w, bf16_values(w).astype(np.float64)
    w = np.asarray(x, np.float16)
    return w, w.astype(np.float64)


def values(t):
    host = t.to_host()
    return (bf16_values(host) if t.dtype == BF16 else host).astype(np.float64)


class Paged:
    """A cache with room for `lengths`, its spare pages and the rows behind every sequence NaN."""

    def __init__(self, device, rng, kind, lengths, *, kv_heads=2, d=64, page=16, spare=3, fill=None, width=0):
        self.device, self.kind, self.lengths, self.page = device, kind, list(lengths), page
        counts = [-(-max(n, 0) // page) for n in lengths]
        total = sum(counts) + spare
        order = rng.permutation(total)
        self.table = np.full((len(lengths), max([*counts, width, 1])), -1, np.int32)
        shape = (total, kv_heads, page, d)
        keys, vals = np.full(shape, np.nan), np.full(shape, np.nan)
        at = 0
        for i, count in enumerate(counts):
            self.table[i, :count] = order[at:at + count]
            at += count
            for j in range(count):
                rows = min(page, lengths[i] - j * page)
                for data, which in ((keys, 0), (vals, 1)):
                    some = rng.standard_normal((kv_heads, rows, d)) if fill is None else fill[which](rng, (kv_heads, rows, d))
                    data[self.table[i, j], :, :rows] = some
        with np.errstate(invalid="ignore"):
            (self.key_words, self.keys), (self.value_words, self.values) = words(keys, kind), words(vals, kind)
        if device is not None:
            self.cache = KvCache(device.to_device(self.key_words, TYPES[kind]), device.to_device(self.value_words, TYPES[kind]))
            self.on_table = device.to_device(self.table)

    def sequences(self, *, starts=None, new=1, lengths=None):
        on = self.device.to_device(np.array(self.lengths if lengths is None else lengths, np.int32))
        if starts is None:
            return Sequences(on, self.on_table, new=new)
        return Sequences(on, self.on_table, starts=self.device.to_device(np.array(starts, np.int32)))

    def tensor(self, host):
        return self.device.to_device(host, TYPES[self.kind])

    def attention(self, q, starts, *, scale=None, window=0, lengths=None, weight=None):
        """The oracle's (y, bound) with the result's rounding in it."""
        half = HALF_STEP[self.kind]
        d = q.shape[2]
        y, bound = oracle.attention(q, np.nan_to_num(self.keys), np.nan_to_num(self.values), starts,
                                    self.lengths if lengths is None else lengths, self.table, scale or d**-0.5, window,
                                    half if weight is None else weight, TINY[self.kind])
        return y, bound + (np.abs(y) + bound) * half + TINY[self.kind]


def assert_within(got, y, bound, what=""):
    error = np.abs(got - y)
    assert not np.isnan(got).any(), f"{what}: NaN at {np.argwhere(np.isnan(got))[0]}"
    worst = np.unravel_index(np.argmax(error - bound), error.shape)
    assert np.all(error <= bound), f"{what}: error {error[worst]} > {bound[worst]} at {worst}"
