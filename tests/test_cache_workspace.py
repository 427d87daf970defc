"""The scratch of attention over a paged cache: how much a call asks for, and that it keeps to it."""

import ctypes

import numpy as np
import pytest

from krn_amd.dtypes import BF16, I32
from tests.paged import TYPES, Paged, assert_within, values, words
from tests.test_library import LIBRARY

needs_library = pytest.mark.skipif(not LIBRARY.exists(), reason="libkrn_amd.so is not built")


@needs_library
@pytest.mark.parametrize("sequences", [1, 128, 129, 2048, 8192, 8193])
@pytest.mark.parametrize("step,heads,kv_heads,d", [(1, 32, 8, 128), (4, 64, 8, 128), (4, 128, 16, 128), (32, 1, 1, 64), (1, 512, 16, 64)])
def test_scratch_of_new_tokens_does_not_grow_with_their_number(sequences, step, heads, kv_heads, d):
    """At most 1024 parts beyond the first of each sequence, and as many first ones of the sequences that have several: planes of
    rows * (d + 4) floats. Besides them 16 bytes for each of those sequences and of the workgroups of a key head."""
    workspace = ctypes.CDLL(str(LIBRARY)).krn_cache_attention_workspace
    workspace.restype = ctypes.c_int64
    for width in (1, 100, 1 << 20):
        sizes = [ctypes.c_int64(v) for v in (sequences * step, heads, kv_heads, d, 16)]
        need = workspace(*sizes, 0, ctypes.c_int64(sequences), ctypes.c_int64(width))
        rows = step * heads // kv_heads
        assert 0 <= need <= 2 * 1024 * rows * (d + 4) * 4 + 16 * (1025 + sequences + 1024)
        assert need > 0 or sequences > 8192 or width * 16 <= 1024


# lengths, new tokens each, heads, kv_heads, d: all sequences in several parts, some, one, none, and more than a wave counts
SPLIT = [
    ([1000] * 3, 1, 4, 1, 64), ([5000, 3, 900, 20], 2, 8, 2, 128), ([40] * 100 + [8000] + [0] * 27, 1, 4, 4, 64), ([30] * 50, 4, 8, 1, 64),
    ([20] * 200 + [3000, 2500] + [50] * 98, 1, 2, 2, 64), ([900] * 300, 1, 1, 1, 64), ([2000] * 130, 1, 16, 8, 64),
]  # fmt: skip


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,new,heads,kv_heads,d", SPLIT)
def test_a_call_keeps_to_its_scratch(device, lengths, new, heads, kv_heads, d):
    """The C entry with exactly what it asks for, and the memory behind it unchanged."""
    from ctypes import c_float, c_int, c_int64, c_void_p

    from krn_amd.runtime import library

    rng = np.random.default_rng(len(lengths))
    n = len(lengths)
    paged = Paged(device, rng, "bf16", lengths, kv_heads=kv_heads, d=d, width=70)
    q, exact = words(rng.standard_normal((n * new, heads, d)), "bf16")
    on, o = paged.tensor(q), device.empty(TYPES["bf16"], n * new, heads, d)
    at = device.to_device(np.array(lengths, np.int32))
    width = paged.table.shape[1]
    need = library.lib().krn_cache_attention_workspace(n * new, heads, kv_heads, d, 16, 0, n, width)
    assert need > 0 and need % 4 == 0
    held = device.empty(I32, need // 4 + 4096)
    held.copy_from(np.full(held.shape, 77, np.int32))
    library.check(library.lib().krn_cache_attention(
        c_int(library.kind(BF16)), c_void_p(on.pointer), *map(c_void_p, paged.cache.pointers), c_void_p(o.pointer),
        *map(c_int64, (n * new, heads, kv_heads, d, len(paged.keys), 16)), c_void_p(0), c_int64(new), c_void_p(at.pointer),
        c_void_p(paged.on_table.pointer), c_int64(n), c_int64(width), c_float(d**-0.5), c_int64(0), c_void_p(held.pointer),
        c_int64(need), c_void_p(device.default_stream.handle)), "krn_cache_attention")
    assert_within(values(o), *paged.attention(exact, list(range(0, n * new + 1, new))))
    assert (held.to_host()[need // 4:] == 77).all()
