"""The expert layer on the GPU against oracle/mx.py in float64, within the bound derived there: float32 sums, one rounding
of the inner values to two bf16 parts (2^-8 of at most 2^-8 of a value is left) and one of the result."""

import numpy as np
import pytest

from krn_amd.dtypes import BF16, F16, U8
from krn_amd.lib import MxMatrix, moe
from krn_amd.runtime.hip import HIPTensor
from oracle import mx
from tests.test_gpu_mx import HALF_STEP, TINY, TYPES, to_device, values, words

pytestmark = pytest.mark.gpu

INNER = 2.0**-16


class Layer:
    """Random weights, on the host and on the device."""

    def __init__(self, device, rng, kind, hidden, inner, experts):
        self.device, self.kind, self.sizes = device, kind, (hidden, inner, experts)
        self.router, self.router_values = words(rng.standard_normal((experts, hidden)) / np.sqrt(hidden), kind)
        gate_up = mx.encode(rng.standard_normal((experts * 2 * inner, hidden)) / np.sqrt(hidden))
        down = mx.encode(rng.standard_normal((experts * hidden, inner)) / np.sqrt(inner))
        self.codes = gate_up, down
        self.gate_up, self.down = to_device(device, *gate_up, hidden), to_device(device, *down, inner)
        self.wide = (mx.decode(*gate_up, hidden).reshape(experts, 2 * inner, hidden),
                     mx.decode(*down, inner).reshape(experts, hidden, inner))
        self.router_on = device.to_device(self.router, TYPES[kind])

    def tensor(self, host):
        return self.device.to_device(host, TYPES[self.kind])

    def __call__(self, x, top_k, **kwargs):
        return moe(self.tensor(x), self.router_on, self.gate_up, self.down, top_k=top_k, **kwargs)

    def check(self, got, exact, top_k):
        y, bound = mx.moe(exact, self.router_values, *self.wide, top_k, INNER)
        bound = bound + (np.abs(y) + bound) * HALF_STEP[self.kind] + TINY[self.kind]
        error = np.abs(got - y)
        worst = np.unravel_index(np.argmax(error - bound), error.shape)
        assert np.all(error <= bound), f"error {error[worst]} > {bound[worst]} at {worst}"


CASES = [(1, 32, 32, 1, 1), (1, 64, 48, 4, 2), (3, 31, 17, 5, 3), (2, 1000, 777, 6, 2), (7, 520, 100, 12, 3),
         (16, 256, 544, 8, 4), (17, 100, 64, 3, 3), (33, 96, 130, 70, 5), (64, 160, 96, 130, 16), (64, 64, 33, 2, 1),
         (5, 2100, 1056, 4, 2), (1, 4096, 96, 64, 4)]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", CASES)
def test_the_layer_is_the_oracles(device, kind, tokens, hidden, inner, experts, top_k):
    rng = np.random.default_rng(tokens * 101 + hidden)
    layer = Layer(device, rng, kind, hidden, inner, experts)
    x, exact = words(rng.standard_normal((tokens, hidden)), kind)
    got = layer(x, top_k)
    assert got.shape == (tokens, hidden) and got.dtype == TYPES[kind]
    layer.check(values(got), exact, top_k)
    np.testing.assert_array_equal(layer(x, top_k).to_host(), got.to_host())  # the same bits again


@pytest.mark.parametrize("tokens", [16, 40, 64])
def test_all_tokens_on_the_same_experts(device, tokens):
    """Many tokens an expert, in several runs of sixteen; the other experts have none."""
    rng = np.random.default_rng(tokens)
    layer = Layer(device, rng, "bf16", 128, 80, 9)
    x, exact = words(np.abs(rng.standard_normal((tokens, 128))), "bf16")
    router = np.full((9, 128), -1.0) / 16
    router[6], router[2] = 1 / 8, 1 / 16
    layer.router, layer.router_values = words(router, "bf16")
    layer.router_on = layer.tensor(layer.router)
    layer.check(values(layer(x, 2)), exact, 2)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_ties_go_to_the_lower_expert(device, kind):
    rng = np.random.default_rng(4)
    layer = Layer(device, rng, kind, 64, 32, 70)
    layer.router, layer.router_values = words(np.repeat(rng.integers(-2, 3, (10, 64)) / 8, 7, axis=0), kind)
    layer.router_on = layer.tensor(layer.router)
    x, exact = words(rng.integers(-3, 4, (20, 64)) / 2, kind)  # logits are exact: ties are ties
    layer.check(values(layer(x, 5)), exact, 5)
    layer.router, layer.router_values = words(np.zeros((70, 64)), kind)
    layer.router_on = layer.tensor(layer.router)
    assert mx.choose(exact, layer.router_values, 5)[0].tolist() == [[0, 1, 2, 3, 4]] * 20
    layer.check(values(layer(x, 5)), exact, 5)


def test_a_nan_or_infinite_token_breaks_its_own_row_only(device):
    rng = np.random.default_rng(5)
    layer = Layer(device, rng, "bf16", 96, 64, 6)
    x, exact = words(rng.standard_normal((18, 96)), "bf16")
    exact[4, 3], exact[17, 95] = np.nan, np.inf
    with np.errstate(invalid="ignore"):
        x, _ = words(exact, "bf16")
    got = values(layer(x, 2))
    assert np.isnan(got[4]).all() and not np.isfinite(got[17]).any()
    rows = [t for t in range(18) if t not in (4, 17)]
    layer.check(got[rows], exact[rows], 2)


def test_a_broken_weight_block_reaches_the_tokens_of_its_expert_only(device):
    rng = np.random.default_rng(6)
    hidden, inner, experts = 64, 40, 5
    layer = Layer(device, rng, "bf16", hidden, inner, experts)
    (gc, gs), (dc, ds) = layer.codes
    ds = ds.copy()
    ds[3 * hidden + 7, 1] = 255  # expert 3's output 7; its neighbours' rows end inside a slab
    layer.down = to_device(device, dc, ds, inner)
    x, exact = words(rng.standard_normal((12, hidden)), "bf16")
    got = values(layer(x, 2))
    chosen = mx.choose(exact, layer.router_values, 2)[0]
    broken = np.zeros((12, hidden), bool)
    broken[(chosen == 3).any(axis=1), 7] = True
    assert broken.any()
    np.testing.assert_array_equal(np.isnan(got), broken)
    whole = ~broken.any(axis=1)
    layer.check(got[whole], exact[whole], 2)


def test_nothing_but_the_result_is_written_at_any_alignment(device):
    rng = np.random.default_rng(7)
    layer = Layer(device, rng, "f16", 75, 40, 4)
    x, exact = words(rng.standard_normal((9, 75)), "f16")
    held_x, held_y = layer.tensor(np.append(np.float16(3), x.ravel())), layer.tensor(np.full(9 * 75 + 6, 5, np.float16))
    router = layer.tensor(np.append(np.float16(3), layer.router.ravel()))
    scales = device.to_device(np.append(np.full(3, 255, np.uint8), layer.codes[1][1].ravel()))
    down = MxMatrix(layer.down.codes, HIPTensor(device, scales.pointer + 3, U8, layer.down.scales.shape, owner=scales), 40)
    out = HIPTensor(device, held_y.pointer + 2, F16, (9, 75), owner=held_y)
    got = moe(HIPTensor(device, held_x.pointer + 2, F16, (9, 75), owner=held_x),
              HIPTensor(device, router.pointer + 2, F16, (4, 75), owner=router), layer.gate_up, down, top_k=3, out=out)
    assert got is out
    after = held_y.to_host()
    assert after[0] == 5 and (after[1 + 9 * 75:] == 5).all()
    layer.check(values(out), exact, 3)


def test_no_tokens(device):
    layer = Layer(device, np.random.default_rng(1), "bf16", 64, 32, 4)
    assert layer(np.zeros((0, 64), np.uint16), 2).to_host().shape == (0, 64)


def test_bound_recorded_and_replayed_on_several_streams(device):
    """Two layers share a stream's workspace; graphs hold their own, and replay between eager calls."""
    rng = np.random.default_rng(11)
    first, second = Layer(device, rng, "bf16", 256, 96, 8), Layer(device, rng, "bf16", 256, 640, 16)
    x = device.empty(BF16, 6, 256)
    middle, y = device.empty(BF16, 6, 256), device.empty(BF16, 6, 256)
    one = moe.bind(x, first.router_on, first.gate_up, first.down, top_k=2, out=middle)
    two = moe.bind(middle, second.router_on, second.gate_up, second.down, top_k=3, out=y)

    def both():
        one()
        two()

    graphs = [device.graph(both), device.graph(both)]
    for seed in range(4):
        host = words(np.random.default_rng(seed).standard_normal((6, 256)), "bf16")[0]
        want = second(first(host, 2).to_host(), 3).to_host()
        x.copy_from(host)
        both()
        np.testing.assert_array_equal(y.to_host(), want)
        y.copy_from(np.zeros((6, 256), np.uint16))
        graphs[seed % 2]()
        np.testing.assert_array_equal(y.to_host(), want)
        stream = device.stream()
        y.copy_from(np.zeros((6, 256), np.uint16))
        with stream:
            both()
        stream.sync()
        np.testing.assert_array_equal(y.to_host(), want)
