"""A paged key-value cache: the rotated queries, keys and values of a step's tokens, and causal attention over the cache. No
counterpart in the reference, whose attention is a tile program on dense tensors (examples/04_libraries/08_flash_attention.py)."""

import math
from collections.abc import Sequence

import numpy as np

from krn_amd.dtypes import BF16, F16, I32, U64
from krn_amd.lib.calls import LibraryCall, Work, tensor
from krn_amd.runtime import library
from krn_amd.runtime.hip import HIPDevice, HIPTensor

HEADS = (64, 128)  # head dimensions
ALL_KEYS = 2**31  # a window that holds any sequence


class KvCache:
    """`keys` and `values`, each (pages, kv_heads, page, d) of f16 or bf16: pages of `page` keys (a power of two, 16 or more)
    that sequences own, d 64 or 128. Which page holds what is up to the program (`Sequences`)."""

    def __init__(self, keys: HIPTensor, values: HIPTensor) -> None:
        tensor(keys, "keys", 4, (F16, BF16))
        tensor(values, "values", 4, (keys.dtype,))
        if keys.shape != values.shape:
            raise ValueError(f"keys have shape {keys.shape}, values {values.shape}")
        self.pages, self.kv_heads, self.page, self.d = keys.shape
        if self.d not in HEADS:
            raise ValueError(f"heads of a cache have 64 or 128 columns, not {self.d}")
        if self.kv_heads < 1:
            raise ValueError("a cache has one key head or more")
        if self.page < 16 or self.page & (self.page - 1):
            raise ValueError(f"a page holds a power of two of keys, 16 or more, not {self.page}")
        self.keys, self.values, self.dtype, self.device = keys, values, keys.dtype, keys.device

    @classmethod
    def empty(cls, device: HIPDevice, pages: int, kv_heads: int, page: int, d: int, dtype=BF16) -> "KvCache":
        """Uninitialized: what is not written yet is not read."""
        return cls(device.empty(dtype, pages, kv_heads, page, d), device.empty(dtype, pages, kv_heads, page, d))

    @property
    def pointers(self) -> tuple[int, int]:
        return self.keys.pointer, self.values.pointer

    @property
    def sizes(self) -> tuple[int, int, int, int]:
        return self.kv_heads, self.d, self.pages, self.page

    def __repr__(self) -> str:
        return f"KvCache({self.pages} pages of {self.page} keys, {self.kv_heads} heads of {self.d} {self.dtype})"


class Sequences:
    """The sequences of a step, on the device, all i32: `lengths` (n), the keys of each, those of its newest tokens included;
    `pages` (n, width), the pages that it owns: key j lies in row j % page of page pages[i, j // page]. The step's tokens are
    packed: with `starts` (n + 1) those of sequence i are starts[i] to starts[i + 1] - 1, without it every sequence has `new`.
    The last token of sequence i has position lengths[i] - 1.

    The kernels read these at every call or replay, so a program changes their contents between them as it likes. Tokens
    before starts[0] or from starts[n] on belong to no sequence, and what a call would write for them is left as it was.
    starts do not decrease. Keys beyond width pages are not there, a page number outside of the cache reads as zeros and
    is not written."""

    def __init__(self, lengths: HIPTensor, pages: HIPTensor, *, starts: HIPTensor | None = None, new: int = 1) -> None:
        tensor(lengths, "lengths", 1, (I32,))
        tensor(pages, "pages", 2, (I32,))
        self.count, self.width = pages.shape
        if lengths.shape != (self.count,):
            raise ValueError(f"{self.count} rows of pages need as many lengths, got {lengths.shape}")
        if starts is not None and tensor(starts, "starts", 1, (I32,)).shape != (self.count + 1,):
            raise ValueError(f"{self.count} sequences need {self.count + 1} starts, got {starts.shape}")
        if not isinstance(new, int) or new < 1 or (starts is not None and new != 1):
            raise ValueError(f"sequences without starts have one new token or more each, got new = {new!r}")
        self.lengths, self.pages, self.starts, self.new = lengths, pages, starts, new

    @property
    def arguments(self) -> tuple[int, int, int, int, int, int]:
        starts = self.starts.pointer if self.starts is not None else 0
        return starts, self.new, self.lengths.pointer, self.pages.pointer, self.count, self.width

    def check(self, tokens: int) -> None:
        if self.starts is None and tokens != self.new * self.count:
            raise ValueError(f"{self.count} sequences of {self.new} new tokens are {self.new * self.count} tokens, not {tokens}")

    def __repr__(self) -> str:
        return f"Sequences({self.count}, {'packed' if self.starts is not None else f'{self.new} new tokens each'})"


class Rotary:
    """Rotary positions: pair j of a head turns by position * frequencies[j] radians and is multiplied by `magnitude`. Pairs
    are columns (j, j + dim / 2) or, `interleaved`, (2j, 2j + 1) of the head's first dim = 2 len(frequencies); the other
    columns stay as they are. On the device a frequency is a 64-bit fraction of a turn, so angles are exact at any position."""

    def __init__(self, device: HIPDevice, frequencies: Sequence[float], *, interleaved: bool = False,
                 magnitude: float = 1.0) -> None:
        self.frequencies = np.array(frequencies, dtype=np.float64)
        if self.frequencies.ndim != 1 or not np.isfinite(self.frequencies).all():
            raise ValueError("frequencies are finite numbers, one for each pair")
        if not math.isfinite(magnitude):
            raise ValueError(f"the magnitude is a finite number, not {magnitude}")
        turns = [round(math.fmod(f / (2 * math.pi), 1.0) * 2**64) % 2**64 for f in self.frequencies.tolist()]
        self.turns = device.to_device(np.array(turns, dtype=np.uint64), U64)
        self.dim, self.interleaved, self.magnitude = 2 * len(turns), bool(interleaved), float(magnitude)

    @classmethod
    def of(cls, device: HIPDevice, dim: int, *, base: float = 10000.0, factor: float = 1.0, original: int | None = None,
           interleaved: bool = False) -> "Rotary":
        """frequencies[j] = base^(-2j / dim), for contexts `factor` times as long as those of training: all of them divided
        by `factor` or, with the `original` context length, only those of pairs that turn less than once in it, those beyond
        32 turns as they are and between these a mix linear in the turns, with the magnitude 0.1 ln factor + 1. Models whose
        mix is linear in the pair's index, or that have other limits or magnitudes, pass theirs to `Rotary` itself."""
        if not isinstance(dim, int) or dim < 0 or dim % 2:
            raise ValueError(f"an even number of columns is rotated, not {dim!r}")
        if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor >= 1):
            raise ValueError(f"the base is positive and the factor 1 or more, got {base} and {factor}")
        f = base ** (-np.arange(dim // 2, dtype=np.float64) / max(dim // 2, 1))
        if original is None:
            return cls(device, f / factor, interleaved=interleaved)
        if original < 1:
            raise ValueError(f"the original context has one position or more, not {original}")
        kept = np.clip((original * f / (2 * np.pi) - 1) / 31, 0, 1)
        return cls(device, f * kept + f / factor * (1 - kept), interleaved=interleaved, magnitude=0.1 * math.log(factor) + 1)

    def __repr__(self) -> str:
        return f"Rotary({self.dim}{', interleaved' if self.interleaved else ''})"


def _checked(cache: object, sequences: object) -> None:
    if not isinstance(cache, KvCache):
        raise TypeError(f"cache is a KvCache, not {type(cache).__name__}")
    if not isinstance(sequences, Sequences):
        raise TypeError(f"sequences are Sequences, not {type(sequences).__name__}")


@LibraryCall
def rotary_append(qkv, cache: KvCache, sequences: Sequences, *, rotary: Rotary | None = None, out=None) -> Work:
    """The queries (tokens, heads, d) of a step from its fused projection `qkv`, (tokens, (heads + 2 kv_heads) d) of the cache's
    type: heads query heads, then the cache's key heads, then its value heads. Queries and keys are rotated by their tokens'
    positions (not at all without `rotary`), float32 arithmetic and one rounding; keys and values go to their places in the
    cache, which no two tokens share. A token whose position is negative or beyond its sequence's pages is not stored. `out`
    shares no memory with `qkv`."""
    _checked(cache, sequences)
    tensor(qkv, "qkv", 2, (cache.dtype,))
    tokens, width = qkv.shape
    heads = width // cache.d - 2 * cache.kv_heads
    if width % cache.d or heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"rows of qkv hold heads * {cache.d} queries, heads a multiple of {cache.kv_heads}, and "
                         f"{2 * cache.kv_heads * cache.d} keys and values, got {width}")
    sequences.check(tokens)
    if rotary is not None and not isinstance(rotary, Rotary):
        raise TypeError(f"rotary is a Rotary, not {type(rotary).__name__}")
    dim = rotary.dim if rotary is not None else 0
    if dim > cache.d:
        raise ValueError(f"{dim} columns of heads of {cache.d} cannot be rotated")
    if out is not None and tensor(out, "out", 3, (cache.dtype,)).shape != (tokens, heads, cache.d):
        raise ValueError(f"out has shape {out.shape}, the queries {(tokens, heads, cache.d)}")
    result = out if out is not None else qkv.device.empty(cache.dtype, tokens, heads, cache.d)
    turns = (rotary.turns.pointer, dim, rotary.interleaved, rotary.magnitude) if rotary is not None else (0, 0, False, 1.0)
    call = library.rotary_append_call(cache.dtype, qkv.pointer, result.pointer, *cache.pointers, tokens, heads, *cache.sizes,
                                      *sequences.arguments, *turns)
    return Work("rotary_append", qkv.device, result, (qkv, cache, sequences, rotary, result),
                lambda stream: call(stream.handle))


@LibraryCall
def cache_attention(q, cache: KvCache, sequences: Sequences, *, scale: float | None = None, window: int | None = None,
                    out=None) -> Work:
    """softmax(scale q K^T) V of a step's tokens over their sequences' keys, causal: a token at position p attends to keys up
    to p, to the last `window` of them if that is given. q is (tokens, heads, d) of the cache's type; heads / kv_heads query
    heads share a key head; scale is 1 / sqrt(d) unless given. A token without keys gets zeros. Keys and values that a token
    does not see have no part in its result, NaN and infinities included; pages wholly before the windows of all new tokens
    may be another sequence's. Scores, maxima and sums are float32; softmax weights are rounded to 16 bits before they multiply
    values, to two 16-bit parts where sequences have up to 32 rows, new tokens times query heads of a key head; in f16, weights
    below 2^-32 of a token's largest are lost. A token whose scores are all minus infinity gets zeros too. `out` may be q itself and
    shares no other memory. Sequences of as many new tokens each, a few, are faster without `starts`, and new tokens with a long
    past are faster in a call of their own than packed beside prompts."""
    _checked(cache, sequences)
    tensor(q, "q", 3, (cache.dtype,))
    tokens, heads, d = q.shape
    if d != cache.d or heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"q has {heads} heads of {d}, the cache {cache.kv_heads} of {cache.d}: a multiple as many, of one size")
    sequences.check(tokens)
    if scale is not None and not (math.isfinite(scale) and scale > 0):
        raise ValueError(f"the scale is a positive finite number, not {scale}")
    if window is not None and (not isinstance(window, int) or window < 1):
        raise ValueError(f"a window holds one key or more, not {window!r}")
    if out is not None and tensor(out, "out", 3, (cache.dtype,)).shape != q.shape:
        raise ValueError(f"out has shape {out.shape}, q {q.shape}")
    result = out if out is not None else q.device.empty(cache.dtype, *q.shape)
    sizes = (tokens, heads, *cache.sizes)
    need = library.cache_attention_workspace(*sizes, *sequences.arguments)
    call = library.cache_attention_call(cache.dtype, q.pointer, *cache.pointers, result.pointer, *sizes, *sequences.arguments,
                                        scale if scale is not None else d**-0.5, min(window or 0, ALL_KEYS), need)

    def run(stream) -> None:
        if need:
            stream.with_workspace("cache_attention", need, call)
        else:
            call(0, stream.handle)

    return Work("cache_attention", q.device, result, (q, cache, sequences, result), run)
