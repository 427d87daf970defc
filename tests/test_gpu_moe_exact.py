"""The expert layer on weights and tokens whose logits, gate and up values are exact in float32 (tests/moe_layers.py), within a
bound that accepts no lost block, weight or expert (tests/test_moe_layers.py); every form of its routing."""

import numpy as np
import pytest

from krn_amd.lib import moe
from krn_amd.runtime.hip import HIPTensor
from oracle import mx
from tests import moe_layers
from tests.test_gpu_mx import HALF_STEP, TINY, TYPES, to_device, values, words

pytestmark = pytest.mark.gpu


class OnDevice:
    def __init__(self, device, layer):
        hidden, inner, _ = layer.sizes
        self.device, self.layer, self.kind = device, layer, layer.kind
        self.gate_up, self.down = to_device(device, *layer.gate_up, hidden), to_device(device, *layer.down, inner)

    def __call__(self, x, top_k):
        """The result for the tokens x, inside a larger buffer whose other bytes stay."""
        held_words, exact = words(x, self.kind)
        np.testing.assert_array_equal(exact, x)  # NaN among them
        host = np.full(x.size + 128, 77, held_words.dtype)
        held = self.device.to_device(host, TYPES[self.kind])
        out = HIPTensor(self.device, held.pointer + 128, TYPES[self.kind], x.shape, owner=held)
        router = self.device.to_device(words(self.layer.router, self.kind)[0], TYPES[self.kind])
        moe(self.device.to_device(held_words, TYPES[self.kind]), router, self.gate_up, self.down, top_k=top_k, out=out)
        after = held.to_host()
        assert (after[:64] == 77).all() and (after[64 + x.size:] == 77).all()
        return values(out)

    def check(self, got, x, top_k):
        y, bound = self.layer(x, top_k)
        bound = bound + (np.abs(y) + bound) * HALF_STEP[self.kind] + TINY[self.kind]
        error = np.abs(got - y)
        worst = np.unravel_index(np.argmax(error - bound), error.shape)
        assert np.all(error <= bound), f"error {error[worst]} > {bound[worst]} at {worst}"


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", moe_layers.CASES)
def test_the_layer_within_a_bound_that_accepts_no_mistake(device, kind, tokens, hidden, inner, experts, top_k):
    rng = np.random.default_rng(tokens + hidden)
    layer = OnDevice(device, moe_layers.Layer(rng, kind, hidden, inner, experts))
    x = layer.layer.tokens(rng, tokens)
    layer.check(layer(x, top_k), x, top_k)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("experts,top_k", [(70, 5), (300, 16), (9, 9)])
@pytest.mark.parametrize("tokens", [1, 2, 3, 20])
def test_ties_go_to_the_lower_expert(device, kind, tokens, experts, top_k):
    """Seven experts of one logit after the other, then all experts of one."""
    rng = np.random.default_rng(tokens + experts)
    layer = OnDevice(device, moe_layers.Layer(rng, kind, 64, 48, experts))
    x = layer.layer.tokens(rng, tokens)
    layer.layer.router = layer.layer.router[np.arange(experts) // 7]
    layer.check(layer(x, top_k), x, top_k)
    layer.layer.router = np.zeros((experts, 64))
    layer.check(layer(x, top_k), x, top_k)


@pytest.mark.parametrize("tokens", [1, 2, 16, 17, 64])
@pytest.mark.parametrize("experts", [9, 100, 400])
def test_all_tokens_on_the_same_experts(device, tokens, experts):
    rng = np.random.default_rng(tokens)
    layer = OnDevice(device, moe_layers.Layer(rng, "bf16", 128, 80, experts))
    x = np.abs(layer.layer.tokens(rng, tokens))
    layer.layer.router = np.full((experts, 128), -1 / 16)
    layer.layer.router[6], layer.layer.router[2] = 1 / 64, 1 / 128
    layer.check(layer(x, 2), x, 2)


@pytest.mark.parametrize("broken", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,experts", [(1, 6), (2, 6), (2, 100), (2, 400), (18, 6), (18, 400)])
def test_a_broken_token_breaks_its_own_row_only(device, kind, tokens, experts, broken):
    """Every expert has the last token's infinity or NaN in some of its inner values, and the row no finite result."""
    rng = np.random.default_rng(5)
    layer = OnDevice(device, moe_layers.Layer(rng, kind, 96, 64, experts))
    x = layer.layer.tokens(rng, tokens)
    x[-1, 95] = broken
    got = layer(x, 2)
    assert not np.isfinite(got[-1]).any()
    if tokens > 1:
        layer.check(got[:-1], x[:-1], 2)


@pytest.mark.parametrize("tokens,experts", [(1, 5), (2, 5), (2, 100), (12, 5), (12, 400)])
def test_a_broken_weight_block_reaches_the_tokens_of_its_expert_only(device, tokens, experts):
    rng = np.random.default_rng(6)
    hidden, inner = 64, 40
    layer = OnDevice(device, moe_layers.Layer(rng, "bf16", hidden, inner, experts))
    x = layer.layer.tokens(rng, tokens)
    chosen = mx.choose(x, layer.layer.router, 2)[0]
    expert = int(chosen[0, 1])
    codes, scales = layer.layer.down
    scales = scales.copy()
    scales[expert * hidden + 7, 1] = 255  # that expert's output 7; its neighbours' rows end inside a slab
    layer.down = to_device(device, codes, scales, inner)
    got = layer(x, 2)
    nan = np.zeros((tokens, hidden), bool)
    nan[(chosen == expert).any(axis=1), 7] = True
    np.testing.assert_array_equal(np.isnan(got), nan)
    y = layer.layer(x, 2)[0]
    layer.check(np.where(nan, y, got), x, 2)
