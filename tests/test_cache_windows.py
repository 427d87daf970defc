"""Windows of any number of keys, as the library's call passes them to the C entry, which has 64 bits for them."""

from types import SimpleNamespace

import pytest

from krn_amd.dtypes import BF16, I32
from krn_amd.lib import KvCache, Sequences, cache_attention
from krn_amd.runtime import library
from krn_amd.runtime.hip import HIPTensor


@pytest.mark.parametrize("window", [1, 100, 2**31 - 1, 2**31, 2**63 - 1, 2**63, 2**64, 2**64 + 5, 3 * 2**64 + 2**31, 10**30])
def test_a_window_is_never_a_smaller_one(monkeypatch, window):
    device = SimpleNamespace(arch="gfx950")

    def stand_in(dtype, *shape):
        return HIPTensor(device, 1 << 20, dtype, shape, owner=device)

    passed = []

    class Entry:
        def krn_cache_attention(self, *arguments):
            passed.extend(arguments)
            return 0

    monkeypatch.setattr(library, "lib", Entry)
    monkeypatch.setattr(library, "cache_attention_workspace", lambda *sizes: 0)
    cache = KvCache(stand_in(BF16, 9, 2, 16, 64), stand_in(BF16, 9, 2, 16, 64))
    q = stand_in(BF16, 3, 4, 64)
    work = cache_attention.check(q, cache, Sequences(stand_in(I32, 3), stand_in(I32, 3, 4)), window=window, out=stand_in(BF16, 3, 4, 64))
    work.run(SimpleNamespace(handle=0))
    got = passed[18].value  # after the scale
    assert passed[17].value == 0.125 and (got == window if window < 2**31 else got >= 2**31)
