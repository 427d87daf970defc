"""A paged cache as a server uses it: steps of prompts and new tokens one after the other against attention over everything so
far, calls recorded and replayed with other lengths, on several streams and by several threads at once."""

import threading

import numpy as np
import pytest

from krn_amd.dtypes import BF16, I32
from krn_amd.lib import KvCache, Rotary, Sequences, cache_attention, rotary_append
from oracle import cache as oracle
from tests.paged import HALF_STEP, TINY, TYPES, Paged, assert_within, values, words

pytestmark = pytest.mark.gpu


class Server:
    """Sequences that grow, on pages handed out as they need them; the host keeps what was projected."""

    def __init__(self, device, rng, kind, n, *, heads=4, kv_heads=2, d=64, page=16, width=40, **rotary):
        self.device, self.rng, self.kind, self.n, self.heads = device, rng, kind, n, heads
        self.cache = KvCache.empty(device, n * width, kv_heads, page, d, TYPES[kind])
        self.turn = Rotary.of(device, d, **rotary)
        self.table = rng.permutation(n * width).reshape(n, width).astype(np.int32)
        self.pages = device.to_device(self.table)
        self.lengths = [0] * n
        self.seen = [np.zeros((0, heads + 2 * kv_heads, d)) for _ in range(n)]

    def step(self, counts):
        """One step of so many new tokens a sequence: (result, its oracle's value and bound)."""
        d, kv = self.cache.d, self.cache.kv_heads
        qkv, exact = words(self.rng.standard_normal((sum(counts), (self.heads + 2 * kv) * d)), self.kind)
        starts = [0, *np.cumsum(counts).tolist()]
        for i, count in enumerate(counts):
            self.lengths[i] += count
            self.seen[i] = np.concatenate([self.seen[i], exact[starts[i]:starts[i + 1]].reshape(count, self.heads + 2 * kv, d)])
        lengths = self.device.to_device(np.array(self.lengths, np.int32))
        if len(set(counts)) == 1:
            sequences = Sequences(lengths, self.pages, new=counts[0])
        else:
            sequences = Sequences(lengths, self.pages, starts=self.device.to_device(np.array(starts, np.int32)))
        q = rotary_append(self.device.to_device(qkv, TYPES[self.kind]), self.cache, sequences, rotary=self.turn)
        got = values(cache_attention(q, self.cache, sequences))
        want = [self.attend(i, count) for i, count in enumerate(counts) if count]
        return got, np.concatenate([w[0] for w in want]), np.concatenate([w[1] for w in want])

    def attend(self, i, count):
        """Attention of the last `count` tokens over all, from the projections. Queries and keys are rounded once: a score is off
        by half a step of both, a weight by twice that, besides what the oracle allows."""
        half, d = HALF_STEP[self.kind], self.cache.d
        x, position = self.seen[i], np.arange(len(self.seen[i]))
        turned, _ = oracle.rotate(x[:, : -self.cache.kv_heads], position, self.turn.frequencies, self.turn.interleaved,
                                  self.turn.magnitude)
        q, k, v = turned[len(x) - count:, : self.heads], turned[:, self.heads:], x[:, -self.cache.kv_heads:]
        y, bound = oracle.attention(q, k[None].transpose(0, 2, 1, 3), v[None].transpose(0, 2, 1, 3), [0, count], [len(x)],
                                    np.zeros((1, 1), int), d**-0.5, 0, half, TINY[self.kind])
        group = self.heads // self.cache.kv_heads
        for t in range(count):
            for h in range(self.heads):
                kk, vv = k[: len(x) - count + t + 1, h // group], v[: len(x) - count + t + 1, h // group]
                s = d**-0.5 * kk @ q[t, h]
                w = np.exp(s - s.max())
                w /= w.sum()
                off = d**-0.5 * (np.abs(kk) @ np.abs(q[t, h])) * 2.1 * half
                bound[t, h] += (w * (np.exp(off + off.max()) - 1)) @ np.abs(vv)
        return y, bound + (np.abs(y) + bound) * half + TINY[self.kind]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("sizes", [{}, {"heads": 6, "kv_heads": 1, "d": 128, "page": 32, "interleaved": True},
                                   {"heads": 3, "kv_heads": 3, "factor": 4.0, "original": 64}])
def test_steps_of_a_server(device, kind, sizes):
    server = Server(device, np.random.default_rng(len(sizes)), kind, 4, **sizes)
    for counts in ([33, 1, 0, 70], [1, 1, 1, 1], [2, 2, 2, 2], [0, 130, 5, 1], [1, 1, 1, 1], [1, 1, 1, 1], [100, 100, 100, 100]):
        assert_within(*server.step(counts), str(counts))


def step_of(device, rng, lengths, new=1, heads=8, kv_heads=2, d=128, width=0):
    """Bound calls of one step and the tensors that a program changes between them."""
    paged = Paged(device, rng, "bf16", lengths, kv_heads=kv_heads, d=d, page=16, width=width)
    sequences = paged.sequences(new=new)
    tokens = new * len(lengths)
    qkv = device.empty(BF16, tokens, (heads + 2 * kv_heads) * d)
    q, o = device.empty(BF16, tokens, heads, d), device.empty(BF16, tokens, heads, d)
    append = rotary_append.bind(qkv, paged.cache, sequences, rotary=Rotary.of(device, d), out=q)
    attend = cache_attention.bind(q, paged.cache, sequences, out=o)

    def both():
        append()
        attend()

    return paged, sequences, qkv, o, both


def test_recorded_steps_with_other_lengths_between_eager_calls(device):
    """Two graphs and eager calls share a stream; lengths and projections change between the replays of the same graph."""
    rng = np.random.default_rng(5)
    lengths = [[900, 40, 17, 3], [901, 600, 1, 33], [5, 6, 7, 2000], [1, 1, 1, 1], [2001, 2002, 2003, 16]]
    paged, sequences, qkv, o, both = step_of(device, rng, [2003] * 4)
    other, other_sequences, other_qkv, other_o, others = step_of(device, rng, [500, 1500], new=3, heads=6)
    graphs = [device.graph(both), device.graph(others)]
    tokens = words(rng.standard_normal((6, 10 * 128)), "bf16")[0]
    for round, now in enumerate(lengths):
        sequences.lengths.copy_from(np.array(now, np.int32))
        qkv.copy_from(words(np.random.default_rng(round).standard_normal((4, 12 * 128)), "bf16")[0])
        other_qkv.copy_from(tokens)
        both()
        want = o.to_host()
        others()
        other_want = other_o.to_host()
        for _ in range(2):
            for out in (o, other_o):
                out.copy_from(np.zeros(out.shape, np.uint16))
            graphs[0]()
            graphs[1]()
            np.testing.assert_array_equal(o.to_host(), want)
            np.testing.assert_array_equal(other_o.to_host(), other_want)
        stream = device.stream()
        o.copy_from(np.zeros(o.shape, np.uint16))
        with stream:
            both()
        stream.sync()
        np.testing.assert_array_equal(o.to_host(), want)


def test_a_recorded_prompt_whose_keys_are_shared_out(device):
    rng = np.random.default_rng(6)
    paged = Paged(device, rng, "f16", [3000, 2100], kv_heads=1, d=64)
    lengths, starts = device.to_device(np.array([3000, 2100], np.int32)), device.to_device(np.array([0, 40, 100], np.int32))
    q, o = paged.tensor(words(rng.standard_normal((110, 4, 64)), "f16")[0]), device.empty(TYPES["f16"], 110, 4, 64)
    attend = cache_attention.bind(q, paged.cache, Sequences(lengths, paged.on_table, starts=starts), out=o)
    graph = device.graph(attend)
    for now, at in (([3000, 2100], [0, 40, 100]), ([2999, 64], [10, 10, 11]), ([50, 2100], [0, 50, 50]), ([3000, 2000], [0, 1, 110])):
        lengths.copy_from(np.array(now, np.int32))
        starts.copy_from(np.array(at, np.int32))
        o.copy_from(np.zeros(o.shape, np.float16))
        attend()
        want = o.to_host()
        y, bound = paged.attention(values(q), at, lengths=now)
        owned = ~np.isnan(y).any(axis=(1, 2))
        assert_within(want.astype(np.float64)[owned], y[owned], bound[owned])
        for _ in range(2):
            o.copy_from(np.zeros(o.shape, np.float16))
            graph()
            np.testing.assert_array_equal(o.to_host(), want)


@pytest.mark.parametrize("streams", [1, 3])
def test_threads_that_call_at_once(device, streams):
    """Six threads, eight calls each of split attentions, on one stream's workspace or on three: the result of a call alone."""
    rng = np.random.default_rng(7)
    paged = Paged(device, rng, "bf16", [1500, 30, 700], kv_heads=2, d=64)
    tokens = [paged.tensor(words(rng.standard_normal((3, 4, 64)), "bf16")[0]) for _ in range(6)]
    prompts = [paged.tensor(words(rng.standard_normal((60, 4, 64)), "bf16")[0]) for _ in range(6)]
    one, packed = paged.sequences(), paged.sequences(starts=[0, 40, 41, 60])
    alone = [(cache_attention(t, paged.cache, one).to_host(), cache_attention(p, paged.cache, packed).to_host())
             for t, p in zip(tokens, prompts)]
    outs = [[(device.empty(BF16, 3, 4, 64), device.empty(BF16, 60, 4, 64)) for _ in range(8)] for _ in range(6)]
    on = [device.stream() for _ in range(streams)]
    device.sync()
    failed = []

    def work(t):
        try:
            with on[t % streams]:
                for a, b in outs[t]:
                    cache_attention(tokens[t], paged.cache, one, out=a)
                    cache_attention(prompts[t], paged.cache, packed, out=b)
        except BaseException as error:
            failed.append(error)

    threads = [threading.Thread(target=work, args=(t,)) for t in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for stream in on:
        stream.sync()
    for t in range(6):
        for a, b in outs[t]:
            np.testing.assert_array_equal(a.to_host(), alone[t][0])
            np.testing.assert_array_equal(b.to_host(), alone[t][1])


def test_without_a_workspace_the_keys_stay_in_one_workgroup(device):
    """The C entry with no workspace, or with too little, gives the same rows but for the order of sums."""
    from ctypes import c_float, c_int, c_int64, c_void_p

    from krn_amd.runtime import library

    rng = np.random.default_rng(8)
    paged = Paged(device, rng, "f16", [3000, 70], kv_heads=2, d=64)
    for starts in (None, [0, 40, 41]):
        tokens = 41 if starts else 2
        q, exact = words(rng.standard_normal((tokens, 4, 64)), "f16")
        on, o = paged.tensor(q), device.empty(TYPES["f16"], tokens, 4, 64)
        lengths, at = device.to_device(np.array([3000, 70], np.int32)), device.to_device(np.array(starts or [0], np.int32))
        sizes = [c_int64(v) for v in (tokens, 4, 2, 64, len(paged.keys), 16)]
        need = library.lib().krn_cache_attention_workspace(tokens, 4, 2, 64, 16, int(starts is not None), 2, paged.table.shape[1])
        assert need > 0
        held = device.empty(I32, need // 4 + 4)
        for pointer, nbytes in ((0, 0), (held.pointer, need - 1), (held.pointer, need)):
            o.copy_from(np.zeros(o.shape, np.float16))
            library.check(library.lib().krn_cache_attention(
                c_int(1), c_void_p(on.pointer), c_void_p(paged.cache.keys.pointer), c_void_p(paged.cache.values.pointer),
                c_void_p(o.pointer), *sizes, c_void_p(at.pointer if starts else 0), c_int64(1), c_void_p(lengths.pointer),
                c_void_p(paged.on_table.pointer), c_int64(2), c_int64(paged.table.shape[1]), c_float(0.125), c_int64(0),
                c_void_p(pointer), c_int64(nbytes), c_void_p(device.default_stream.handle)), "krn_cache_attention")
            assert_within(values(o), *paged.attention(exact, starts or [0, 1, 2]))


@pytest.mark.parametrize("n", [63, 65, 127, 128, 129, 256, 1030])
@pytest.mark.parametrize("new", [1, 2])
def test_many_sequences_some_of_them_long(device, n, new):
    rng = np.random.default_rng(n)
    lengths = rng.integers(0, 60, n).tolist()
    lengths[0], lengths[n // 2], lengths[n - 1] = 3000, 1000, 5000
    paged = Paged(device, rng, "bf16", lengths, kv_heads=2, d=64)
    q, exact = words(rng.standard_normal((n * new, 4, 64)), "bf16")
    got = values(cache_attention(paged.tensor(q), paged.cache, paged.sequences(new=new)))
    assert_within(got, *paged.attention(exact, list(range(0, n * new + 1, new))))


def test_many_sequences(device):
    """More sequences than are shared out or searched in one look, of one token and of a few."""
    rng = np.random.default_rng(9)
    n = 2500
    lengths = rng.integers(0, 40, n).tolist()
    lengths[17], lengths[2400] = 700, 900
    paged = Paged(device, rng, "f16", lengths, kv_heads=1, d=64)
    q, exact = words(rng.standard_normal((n, 2, 64)), "f16")
    got = values(cache_attention(paged.tensor(q), paged.cache, paged.sequences()))
    assert_within(got, *paged.attention(exact, list(range(n + 1))))
    counts = rng.integers(0, 3, n)
    counts[5] = 300
    starts = [0, *np.cumsum(counts).tolist()]
    q, exact = words(rng.standard_normal((starts[-1], 2, 64)), "f16")
    got = values(cache_attention(paged.tensor(q), paged.cache, paged.sequences(starts=starts, lengths=paged.lengths)))
    assert_within(got, *paged.attention(exact, starts))
    turn = Rotary.of(device, 64)
    qkv, exact = words(rng.standard_normal((starts[-1], 4 * 64)), "f16")
    q = values(rotary_append(paged.tensor(qkv), paged.cache, paged.sequences(starts=starts, lengths=paged.lengths), rotary=turn))
    _, position = oracle.owners(starts, paged.lengths, starts[-1])
    y, bound = oracle.rotate(exact.reshape(-1, 4, 64)[:, :2], position, turn.frequencies)
    assert_within(q, y, bound + (np.abs(y) + bound) * HALF_STEP["f16"] + TINY["f16"])
