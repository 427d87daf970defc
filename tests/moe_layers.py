"""Expert layers whose logits, gate and up values are exact in float32 in every order, for tests of `lib.moe` with a bound that
leaves no room for a lost block: tokens and router rows are small integers times a power of two, weights e2m1 codes at two
neighbouring scales."""

import numpy as np

from oracle import mx
from oracle.numerics import bf16_values, bf16_words
from tests import mx_products

# tokens, hidden, inner, experts, top_k: rows of one to sixteen slabs, tokens of one run and of several, every form of the routing
# (one or two tokens and more; up to 64, 256 and 1024 experts)
CASES = [(1, 32, 32, 1, 1), (1, 64, 48, 4, 2), (3, 31, 17, 5, 3), (2, 1000, 777, 6, 2), (7, 520, 100, 12, 3), (16, 256, 544, 8, 4),
         (17, 100, 64, 3, 3), (33, 96, 130, 70, 5), (64, 160, 96, 130, 16), (64, 64, 33, 2, 1), (5, 2100, 1056, 4, 2),
         (1, 4096, 96, 64, 4), (1, 64, 32, 100, 8), (2, 520, 100, 128, 8), (2, 64, 32, 300, 16), (2, 32, 32, 1024, 16),
         (20, 32, 32, 1000, 16), (40, 1056, 1600, 6, 3), (64, 2100, 544, 4, 2), (3, 4128, 2080, 5, 2), (1, 8224, 64, 3, 2)]  # fmt: skip

LARGEST = {"bf16": 127, "f16": 300}  # a token's integers: 8 bits in bf16; 9 in f16, which takes two bf16 parts


class Layer:
    """Weights and the values they stand for, float64."""

    def __init__(self, rng, kind, hidden, inner, experts):
        self.kind, self.sizes = kind, (hidden, inner, experts)
        self.unit = 2.0 ** -round(np.log2(LARGEST[kind] / np.sqrt(3)))  # tokens of about 1
        self.router = rng.integers(-15, 16, (experts, hidden)) * 2.0 ** -round(np.log2(9 * np.sqrt(hidden)))
        self.gate_up = mx_products.matrix(rng, experts * 2 * inner, hidden, self.power(hidden))
        self.down = mx_products.matrix(rng, experts * hidden, inner, self.power(inner))
        self.wide_up = mx.decode(*self.gate_up, hidden).reshape(experts, 2 * inner, hidden)
        self.wide_down = mx.decode(*self.down, inner).reshape(experts, hidden, inner)

    @staticmethod
    def power(k):
        """The scales at which a sum of k weights times values of about 1 is about 1: with either scale a code's root mean
        square is 4.6."""
        return 127 - round(np.log2(4.6 * np.sqrt(k)))

    def tokens(self, rng, count):
        largest = LARGEST[self.kind]
        return rng.integers(-largest, largest + 1, (count, self.sizes[0])) * self.unit

    def assert_exact(self, x):
        """Sums of magnitudes below 2^24 units, so that float32 holds every partial sum."""
        hidden = self.sizes[0]
        x, unit = np.abs(x) / self.unit, 2.0 ** (self.power(hidden) - 128)  # half a code at the lower scale
        assert (x @ np.abs(self.wide_up / unit).sum(axis=(0, 1)) / self.wide_up.shape[1] / self.wide_up.shape[0]).max() < 2**23
        assert max((np.abs(e / unit) @ x.T).max() for e in self.wide_up) < 2**24
        assert (np.abs(self.router) / np.abs(self.router)[self.router != 0].min() @ x.T).max() < 2**24

    def __call__(self, x, top_k, mistake=None):
        """(y, bound). In units of 2^-24, of a rounding to float32: the weights' softmax has 4 of exp, 8 of its sum and 1 of
        the quotient, silu(gate) up w 4 of exp and 4 more operations: at most 24. The inner values are rounded to two bf16 parts,
        2^-8 of at most 2^-8 of a value. Then any order of additions of at most 2 top_k inner terms, in up to 256 parts, each off
        by at most 2^-23 of the sum of magnitudes (matrix cores may cut where they do not round). `mistake`: a wrong layer."""
        hidden, inner, experts = self.sizes
        chosen, weights = mx.choose(x, self.router, top_k)
        y, bound = np.zeros((2, x.shape[0], hidden))
        if mistake == "equal weights":
            weights = np.full_like(weights, 1 / top_k)
        if mistake == "the next expert":
            chosen = (chosen + 1) % experts
        if mistake == "a lost choice":
            weights = weights * (np.arange(top_k) < top_k - 1)
        x = x.copy()
        if mistake == "a lost hidden block":
            x[:, (hidden - 1) // 32 * 32:] = 0
        if mistake == "a lost first hidden block":
            x[:, :32] = 0
        for t in range(x.shape[0]):
            for e, w in zip(chosen[t], weights[t]):
                both = self.wide_up[e] @ x[t]
                gate, up = (both[inner:], both[:inner]) if mistake == "gate and up swapped" else (both[:inner], both[inner:])
                h = w * up * gate / (1 + np.exp(-gate))
                if mistake == "a lost inner block":
                    h[(inner - 1) // 32 * 32:] = 0
                if mistake == "a lost first inner block":
                    h[:32] = 0
                if mistake == "inner values in one bf16":
                    h = bf16_values(bf16_words(h.astype(np.float32))).astype(np.float64)
                size = np.abs(self.wide_down[e]) @ np.abs(h)
                y[t] += self.wide_down[e] @ h
                bound[t] += size * (24 * 2.0**-24 + 2.0**-16 + (2 * top_k * inner + 256) * 2.0**-23)
        return (y * 0 if mistake == "zero" else y), bound


MISTAKES = ["zero", "equal weights", "the next expert", "a lost choice", "a lost hidden block", "a lost first hidden block",
            "a lost inner block", "a lost first inner block", "gate and up swapped"]  # fmt: skip


def seen(case, mistake):
    """Whether the mistake changes the layer."""
    _, _, _, experts, top_k = case
    return {"equal weights": top_k > 1, "the next expert": experts > top_k}.get(mistake, True)
