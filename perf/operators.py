"""The microscaled 4-bit operators, as a user's program calls them, and their plain forms.

An MX matrix holds rows of K values in blocks of 32: `codes` (rows, 16 blocks), two e2m1 codes a byte with the first in the
low nibble, and `scales` (rows, blocks), the exponent byte of the power of two that each block is scaled by. Both are
row-major uint8; what a last block has past K is zero.

Operators (`"op"`):
  quantize  values to MX (`lib.mx_quantize`) and back (`lib.mx_dequantize`), since what is held in 4 bits is returned as the
            values it stands for: bfloat16 for 16-bit inputs, float32 for float32 ones (both hold them exactly)
  product   C = f(A @ B^T) of two MX matrices (`lib.mx_matmul`), f being the epilogue
  moe       a mixture-of-experts layer with MX experts (`lib.moe`): y = sum_j w_j down_e(silu(gate_e x) * up_e x) over the
            top_k experts e of a token, w the softmax of their router logits

A program that serves keeps its weights, its output and the bound call, so `prepare` makes those, and `run` is one replay.
"""

import math
import os

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
BLOCK = 32
ELEMENTS = 4096 * 14336  # of the largest quantisation
FLOPS = 2.0 * 8192**3  # of the largest product
EXPERT_VALUES = 64 * 3 * 2048 * 4096  # of the largest layer's weights
CHOSEN_VALUES = 256 * 3 * 1024 * 4096  # of its tokens' experts, counted once for each token


def listed():
    return [
        # one token's activations before a layer: a launch and little else
        {"name": "quantize_token", "op": "quantize", "dtype": "bf16", "rows": 1, "k": 8192},
        # a float32 weight of sizes that fill no block, at its conversion
        {"name": "quantize_odd", "op": "quantize", "dtype": "f32", "rows": 1000, "k": 3001},
        # the activations of a prefill before a down-projection
        {"name": "quantize_prefill", "op": "quantize", "dtype": "bf16", "rows": 4096, "k": 14336},
        # one token through a square layer: the weight is read once, nothing else matters
        {"name": "product_token", "op": "product", "dtype": "bf16", "m": 1, "n": 8192, "k": 8192, "epilogue": "none"},
        # a decoding batch through an up-projection
        {"name": "product_batch", "op": "product", "dtype": "bf16", "m": 16, "n": 14336, "k": 4096, "epilogue": "none"},
        # a larger batch through a down-projection: few output tiles, a long K
        {"name": "product_long_k", "op": "product", "dtype": "bf16", "m": 256, "n": 4096, "k": 14336, "epilogue": "none"},
        # a feed-forward layer of sizes that fit no tile and no block, with its bias and activation
        {"name": "product_odd", "op": "product", "dtype": "f16", "m": 1000, "n": 3001, "k": 777, "epilogue": "bias_gelu"},
        # a large prefill: the matrix cores' rate
        {"name": "product_8192", "op": "product", "dtype": "bf16", "m": 8192, "n": 8192, "k": 8192, "epilogue": "none"},
        # the next token of one sequence: four experts of 64 are read
        {"name": "moe_token", "op": "moe", "dtype": "bf16", "tokens": 1, "hidden": 4096, "inner": 2048, "experts": 64,
         "top_k": 4},
        # the next tokens of sixteen sequences: two thirds of the experts are read
        {"name": "moe_batch", "op": "moe", "dtype": "bf16", "tokens": 16, "hidden": 4096, "inner": 2048, "experts": 64,
         "top_k": 4},
        # a small layer of sizes that fill no block, in float16
        {"name": "moe_odd", "op": "moe", "dtype": "f16", "tokens": 7, "hidden": 1000, "inner": 777, "experts": 12,
         "top_k": 3},
        # a full decoding batch: every expert is read, each by several tokens
        {"name": "moe_full", "op": "moe", "dtype": "bf16", "tokens": 64, "hidden": 4096, "inner": 1024, "experts": 32,
         "top_k": 4},
    ]


def _size(rng, low, high):
    """A size between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _inner(rng, low, high):
    """A size as layers have them: mostly a multiple of 128, sometimes of 32, sometimes anything."""
    step = rng.choice([128, 128, 128, 32, 1])
    return max(step, _size(rng, low, high) // step * step)


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "moe", "moe"])
    if op == "quantize":
        k = _inner(rng, 32, 16384)
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "rows": _size(rng, 1, ELEMENTS // k), "k": k}
    if op == "product":
        n, k = _inner(rng, 256, 16384), _inner(rng, 256, 16384)
        m = max(1, min(_size(rng, 1, 8192), int(FLOPS / (2 * n * k))))
        return {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "m": m, "n": n, "k": k,
                "epilogue": rng.choice(["none", "none", "bias", "relu", "bias_gelu", "silu"])}
    hidden, inner = _inner(rng, 256, 4096), _inner(rng, 128, 2048)
    experts = _size(rng, 4, max(4, min(128, EXPERT_VALUES // (3 * hidden * inner))))
    top_k = rng.randint(1, min(8, experts))
    tokens = _size(rng, 1, max(1, min(64, CHOSEN_VALUES // (3 * hidden * inner * top_k))))
    return {"op": op, "dtype": rng.choice(["bf16", "f16"]), "tokens": tokens, "hidden": hidden, "inner": inner,
            "experts": experts, "top_k": top_k}


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale


def _encode(x):
    """(codes, scales) of the MX matrix of float32 values."""
    rows, k = x.shape
    v = torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(rows, -1, BLOCK)
    a = v.abs()
    exponent = a.amax(2).view(torch.int32) >> 23  # a finite magnitude's biased exponent: floor(log2) + 127
    scale = torch.where(exponent == 255, 255, (exponent - 2).clamp(min=0))
    a = torch.ldexp(a, 127 - scale.unsqueeze(2))
    code = (a > 0.25).to(torch.uint8)  # ties go to the even code
    code += a >= 0.75
    code += a > 1.25
    code += a >= 1.75
    code += a > 2.5
    code += a >= 3.5
    code += a > 5
    code += torch.signbit(v).to(torch.uint8) * 8
    code = torch.where(scale.unsqueeze(2) == 255, 0, code).to(torch.uint8).reshape(rows, -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), scale.to(torch.uint8)


def _decode(codes, scales, k):
    """The float32 values of an MX matrix (a scale of 255 is NaN)."""
    magnitudes = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    table = torch.tensor(magnitudes + [-m for m in magnitudes], device=codes.device)
    pairs = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1)
    power = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    power = torch.where(scales == 255, math.nan, power)
    values = pairs.reshape(*scales.shape, BLOCK) * power.unsqueeze(-1)
    return values.reshape(*scales.shape[:-1], -1)[..., :k]


def _inputs(case, seed):
    """The tensors of a case, from its seed alone."""
    g, op, dtype = torch.Generator(device="cuda").manual_seed(seed), case["op"], TORCH[case["dtype"]]
    if op == "quantize":  # activations whose channels differ in size, as a layer's do
        k = case["k"]
        return {"x": (_normal(g, case["rows"], k) * torch.exp(_normal(g, 1, k))).to(dtype)}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a, b = _encode(_normal(g, m, k)), _encode(_normal(g, n, k, scale=k**-0.5))
        return {"a": a[0], "a_scales": a[1], "b": b[0], "b_scales": b[1], "bias": _normal(g, n).to(dtype)}
    t, h, i, e = case["tokens"], case["hidden"], case["inner"], case["experts"]
    gate_up, down = _encode(_normal(g, e * 2 * i, h, scale=h**-0.5)), _encode(_normal(g, e * h, i, scale=i**-0.5))
    return {"x": _normal(g, t, h).to(dtype), "router": _normal(g, e, h, scale=h**-0.5).to(dtype), "gate_up": gate_up[0],
            "gate_up_scales": gate_up[1], "down": down[0], "down_scales": down[1]}


def _bind(case, x, out):
    """The framework's call on these tensors: torch memory as its tensors, without a copy."""
    os.environ["ROCM_PATH"] = os.path.dirname(torch.__file__)  # one HIP runtime in a process: torch's own
    from krn_amd.dtypes import BF16, F16, F32, U8
    from krn_amd.lib import MxMatrix, moe, mx_dequantize, mx_matmul, mx_quantize
    from krn_amd.runtime.api import device_of
    from krn_amd.runtime.hip import HIPTensor

    device = device_of("gfx950")
    kinds = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32, torch.uint8: U8}

    def tensor(t):
        return HIPTensor(device, t.data_ptr(), kinds[t.dtype], tuple(t.shape), owner=t)

    def matrix(name, k):
        return MxMatrix(tensor(x[name]), tensor(x[name + "_scales"]), k)

    if case["op"] == "quantize":
        held = MxMatrix.empty(device, case["rows"], case["k"])
        forth, back = mx_quantize.bind(tensor(x["x"]), out=held), mx_dequantize.bind(held, out=tensor(out))

        def both():
            forth()
            back()

        return both
    if case["op"] == "product":
        bias = tensor(x["bias"]) if "bias" in case["epilogue"] else None
        return mx_matmul.bind(matrix("a", case["k"]), matrix("b", case["k"]), epilogue=case["epilogue"], bias=bias,
                              out=tensor(out))
    return moe.bind(tensor(x["x"]), tensor(x["router"]), matrix("gate_up", case["hidden"]),
                    matrix("down", case["inner"]), top_k=case["top_k"], out=tensor(out))


def prepare(case, seed):
    x, dtype = _inputs(case, seed), TORCH[case["dtype"]]
    if case["op"] == "quantize":
        shape, dtype = (case["rows"], case["k"]), torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    else:
        shape = (case["m"], case["n"]) if case["op"] == "product" else (case["tokens"], case["hidden"])
    out = torch.empty(shape, device="cuda", dtype=dtype)
    state = {"case": case, "inputs": x, "out": out}
    if own:
        state["call"] = _bind(case, x, out)
        torch.cuda.synchronize()  # the framework has streams of its own
    return state


def run(state):
    if own:
        state["call"]()
        return state["out"]
    case, x, out = state["case"], state["inputs"], state["out"]
    if case["op"] == "quantize":
        return _decode(*_encode(x["x"].float()), case["k"]).to(out.dtype)
    if case["op"] == "product":
        c = _decode(x["a"], x["a_scales"], case["k"]) @ _decode(x["b"], x["b_scales"], case["k"]).T
        if "bias" in case["epilogue"]:
            c = c + x["bias"].float()
        if "relu" in case["epilogue"]:
            c = torch.where(c < 0, 0.0, c)
        if "gelu" in case["epilogue"]:
            c = 0.5 * c * (1 + torch.erf(c * 0.7071067811865476))
        if "silu" in case["epilogue"]:
            c = c / (1 + torch.exp(-c))
        return c.to(out.dtype)
    t, h, i, e, top_k = (case[n] for n in ("tokens", "hidden", "inner", "experts", "top_k"))
    # 64 bits for the logits: which experts are chosen goes by them
    logits, chosen = torch.sort(x["router"].double() @ x["x"].double().T, dim=0, descending=True, stable=True)
    logits, chosen = logits[:top_k].T, chosen[:top_k].T.reshape(-1)  # of each token's experts
    weights = torch.exp(logits - logits[:, :1])
    weights = (weights / weights.sum(1, keepdim=True)).float()
    gate_up = _decode(x["gate_up"].reshape(e, 2 * i, -1)[chosen], x["gate_up_scales"].reshape(e, 2 * i, -1)[chosen], h)
    tokens = x["x"].float().repeat_interleave(top_k, 0)
    both = torch.bmm(gate_up, tokens.unsqueeze(2)).squeeze(2)
    gate, up = both[:, :i], both[:, i:]
    inner = gate / (1 + torch.exp(-gate)) * up
    down = _decode(x["down"].reshape(e, h, -1)[chosen], x["down_scales"].reshape(e, h, -1)[chosen], i)
    y = torch.bmm(down, inner.unsqueeze(2)).reshape(t, top_k, h)
    return (weights.unsqueeze(2) * y).sum(1).to(out.dtype)


def _mx_bytes(rows, k):
    return rows * -(-k // BLOCK) * 17


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "quantize":  # values in, codes and scales out and in again, values out
        values = case["rows"] * case["k"]
        return {"bytes": 2 * _mx_bytes(case["rows"], case["k"]) + values * (8 if size == 4 else 4), "flops": 0}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        bias = size * n if "bias" in case["epilogue"] else 0
        return {"bytes": _mx_bytes(m + n, k) + size * m * n + bias, "flops": 2 * m * n * k}
    t, h, i, e, top_k = (case[n] for n in ("tokens", "hidden", "inner", "experts", "top_k"))
    read = e * (1 - (1 - top_k / e) ** t)  # experts that t tokens choose, on average
    weights = read * (_mx_bytes(2 * i, h) + _mx_bytes(h, i))
    return {"bytes": weights + size * (e * h + 2 * t * h), "flops": 2 * t * (e * h + top_k * 3 * h * i)}


def _wide(codes, scales, k):
    """The float64 values of an MX matrix, from the fields of its codes."""
    c = torch.empty(codes.shape[0], 2 * codes.shape[1], device=codes.device, dtype=torch.float64)
    for half in (0, 1):
        n = (codes >> (4 * half)) & 15
        exponent, mantissa = ((n >> 1) & 3).double(), (n & 1).double()
        magnitude = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * 2 ** (exponent - 1))
        c[:, half::2] = torch.where(n > 7, -magnitude, magnitude)
    return (c * (2.0 ** (scales.double() - 127)).repeat_interleave(BLOCK, 1))[:, :k]


def exact(case, seed):
    x, op = _inputs(case, seed), case["op"]
    if op == "quantize":
        v = x["x"].double()
        rows, k = v.shape
        blocks = torch.nn.functional.pad(v, (0, -k % BLOCK)).unflatten(1, (-1, BLOCK))
        top = torch.frexp(blocks.abs().amax(2, keepdim=True)).exponent - 1  # floor(log2), of a block that is not all zero
        power = 2.0 ** (top - 2).clamp(min=-127).double()
        scaled = (blocks / power).abs()
        step = torch.where(scaled < 2, 0.5, torch.where(scaled < 4, 1.0, 2.0)).double()  # between neighbours there
        near = (torch.round(scaled / step) * step).clamp(max=6)  # halves to even
        return (torch.sign(blocks) * near * power).flatten(1)[:, :k]
    if op == "product":
        c = _wide(x["a"], x["a_scales"], case["k"]) @ _wide(x["b"], x["b_scales"], case["k"]).T
        if "bias" in case["epilogue"]:
            c += x["bias"]
        if "relu" in case["epilogue"]:
            c = c.clamp(min=0)
        if "gelu" in case["epilogue"]:
            c = c * 0.5 * torch.erfc(-c / math.sqrt(2))
        if "silu" in case["epilogue"]:
            c = c * torch.sigmoid(c)
        return c
    t, h, i, top_k = (case[n] for n in ("tokens", "hidden", "inner", "top_k"))
    y = torch.zeros(t, h, device="cuda", dtype=torch.float64)
    for token in range(t):
        v = x["x"][token].double()
        logits = x["router"].double() @ v
        best = torch.topk(logits, top_k)
        for expert, weight in zip(best.indices.tolist(), torch.softmax(best.values, 0)):
            rows = slice(expert * 2 * i, (expert + 1) * 2 * i)
            gate, up = (_wide(x["gate_up"][rows], x["gate_up_scales"][rows], h) @ v).split(i)
            rows = slice(expert * h, (expert + 1) * h)
            y[token] += weight * (_wide(x["down"][rows], x["down_scales"][rows], i) @ (gate * torch.sigmoid(gate) * up))
    return y
