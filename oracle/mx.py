"""Microscaled 4-bit matrices and the layer built on them, restated in numpy and float64."""

import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def encode(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes, scales) of the values x (rows, k), exact in float64: each element's nearest e2m1 value is looked up among
    all eight, an exact half going to the even code."""
    rows, k = x.shape
    v = np.zeros((rows, -(-k // BLOCK) * BLOCK))
    v[:, :k] = x
    v = v.reshape(rows, -1, BLOCK)
    top = np.abs(v).max(axis=2)
    broken = ~np.isfinite(top)
    with np.errstate(invalid="ignore"):
        exponent = np.frexp(np.where(broken, 0.0, top))[1] - 1 + 127  # floor(log2) with float32's bias
    scales = np.where(top < 2.0**-126, 0, np.maximum(exponent - 2, 0))
    magnitude = np.abs(np.where(broken[..., None], 0.0, v)) * 2.0 ** (127.0 - scales)[..., None]
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])  # even codes first: argmin takes the first of two equal distances
    codes = order[np.abs(np.minimum(magnitude, 6.0)[..., None] - MAGNITUDES[order]).argmin(axis=-1)]
    codes = np.where(broken[..., None], 0, codes | np.where(np.signbit(v), 8, 0)).astype(np.uint8).reshape(rows, -1)
    return codes[:, 0::2] | codes[:, 1::2] << 4, np.where(broken, 255, scales).astype(np.uint8)


def decode(codes: np.ndarray, scales: np.ndarray, k: int) -> np.ndarray:
    """The float64 values of an MX matrix."""
    n = np.stack([codes & 15, codes >> 4], axis=-1).reshape(*scales.shape, BLOCK)
    power = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (np.where(n & 8, -1.0, 1.0) * MAGNITUDES[n & 7] * power[..., None]).reshape(scales.shape[0], -1)[:, :k]


def choose(x: np.ndarray, router: np.ndarray, top_k: int) -> tuple[np.ndarray, np.ndarray]:
    """The experts of each token, largest logit first and ties to the lower index, and their softmax weights."""
    logits = x @ router.T
    experts = np.argsort(-logits, axis=1, kind="stable")[:, :top_k]
    best = np.take_along_axis(logits, experts, axis=1)
    weights = np.exp(best - best[:, :1])
    return experts, weights / weights.sum(axis=1, keepdims=True)


def moe(x: np.ndarray, router: np.ndarray, gate_up: np.ndarray, down: np.ndarray, top_k: int, rounding: float):
    """(y, bound) of the layer on float64 values: gate_up (experts, 2 inner, hidden), down (experts, hidden, inner). The
    bound follows the float32 sums (any order: 8 * 2^-24 * (terms + 8) times the sum of magnitudes), silu's slope of at
    most 1.1 and 16 float32 roundings in it, and the inner values' one rounding of at most `rounding` relative."""
    step = 8 * 2.0**-24
    inner, hidden = down.shape[2], x.shape[1]
    experts, weights = choose(x, router, top_k)
    y, bound = np.zeros((x.shape[0], down.shape[1])), np.zeros((x.shape[0], down.shape[1]))
    for t in range(x.shape[0]):
        off = step * (hidden + 8) * (np.abs(router[experts[t]]) @ np.abs(x[t])).max()  # of a logit
        for e, w in zip(experts[t], weights[t]):
            both, error = gate_up[e] @ x[t], step * (hidden + 8) * (np.abs(gate_up[e]) @ np.abs(x[t]))
            gate, up = both[:inner], both[inner:]
            act = gate / (1 + np.exp(-gate))
            h = w * act * up
            e_h = w * (1.1 * error[:inner] * (np.abs(up) + error[inner:]) + np.abs(act) * error[inner:])
            e_h += np.abs(h) * (16 * 2.0**-24 + 4 * off + rounding)
            y[t] += down[e] @ h
            bound[t] += np.abs(down[e]) @ (e_h + step * (top_k * inner + 8) * np.abs(h))
    return y, bound
