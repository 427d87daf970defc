"""The expert layers of the GPU tests on the host: their sums are exact, and their bound accepts no mistake."""

import numpy as np
import pytest

from tests import moe_layers

HALF_STEP = {"bf16": 2.0**-8, "f16": 2.0**-11}


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("case", moe_layers.CASES, ids=lambda c: "x".join(map(str, c)))
def test_the_bound_accepts_no_mistake(case, kind):
    tokens, hidden, inner, experts, top_k = case
    rng = np.random.default_rng(tokens + hidden)
    layer = moe_layers.Layer(rng, kind, hidden, inner, experts)
    x = layer.tokens(rng, tokens)
    layer.assert_exact(x)
    y, bound = layer(x, top_k)
    bound = bound + (np.abs(y) + bound) * HALF_STEP[kind]
    assert np.median(bound) < 0.05 * np.sqrt(np.mean(y**2))
    for mistake in moe_layers.MISTAKES:
        if moe_layers.seen(case, mistake):
            wrong = np.abs(layer(x, top_k, mistake)[0] - y)
            seen = (wrong > 2 * bound).any(axis=1)  # in a token's row, with the bound on either side
            assert seen.mean() > 0.9, mistake  # one choice may weigh next to nothing in a token


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("case", [(1, 64, 48, 4, 2), (3, 31, 17, 5, 3), (7, 520, 100, 12, 3), (17, 100, 64, 3, 3), (1, 4096, 96, 64, 4),
                                  (1, 64, 32, 100, 8), (1, 8224, 64, 3, 2)], ids=lambda c: "x".join(map(str, c)))  # fmt: skip
def test_the_bound_of_few_terms_accepts_no_inner_values_in_one_bf16(case, kind):
    tokens, hidden, inner, experts, top_k = case
    assert case in moe_layers.CASES
    rng = np.random.default_rng(tokens + hidden)
    layer = moe_layers.Layer(rng, kind, hidden, inner, experts)
    x = layer.tokens(rng, tokens)
    y, bound = layer(x, top_k)
    bound = bound + (np.abs(y) + bound) * HALF_STEP[kind]
    wrong = np.abs(layer(x, top_k, "inner values in one bf16")[0] - y)
    assert (wrong > 2 * bound).any(axis=1).all()
