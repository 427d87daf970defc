"""The operators of a paged key-value cache, as a user's program calls them, and their plain forms.

A cache holds `keys` and `values`, each (pages, kv_heads, page, d). Sequence i owns the pages that its row of `pages`
(sequences, width) numbers: key j lies in row j % page of page pages[i, j // page]. `lengths` (sequences) counts a sequence's
keys, those of its newest tokens included. The tokens of a step are packed: those of sequence i are starts[i] to
starts[i + 1] - 1, or, without `starts`, `new` for every sequence. The last token of a sequence has position
lengths[i] - 1.

Operators (`"op"`):
  append    the fused projection qkv (tokens, (heads + 2 kv_heads) d) of a step: queries and keys rotated by their positions,
            keys and values written into the cache, queries returned (`lib.rotary_append`). Pair j of a head turns by
            position * frequency[j]; pairs are (j, j + rotary / 2) or, interleaved, (2j, 2j + 1); columns from `rotary` on
            stay as they are
  prompt    causal attention of packed prompts over the cache (`lib.cache_attention`, sequences with `starts`): a token at
            position p attends to the keys up to p, to the last `window` of them if that is not 0; heads / kv_heads query
            heads share a key head
  token     the same for the `new` newest tokens of every sequence (`lib.cache_attention`, sequences without `starts`)

A program that serves keeps its cache, its tables, its output and the bound call, so `prepare` makes those, and `run` is one
replay. Lengths follow from a case alone, values from the seed.
"""

import math
import os
import random
from itertools import accumulate

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}
VALUES = 16384 * 48 * 128  # of the largest append's projection
FLOPS = 4.0 * 128 * 32 * 16384 * 16384 / 2  # of the longest prompt
KEY_VALUES = 64 * 4096 * 8 * 128  # keys of the largest batch of new tokens


def listed():
    common = {"dtype": "bf16", "heads": 32, "kv_heads": 8, "d": 128, "page": 16, "window": 0, "rotary": 128,
              "interleaved": False, "scaling": "none", "new": 0, "mix": 0}
    return [
        # the next token of one sequence: a launch and little else
        {**common, "name": "append_token", "op": "append", "sequences": 1, "tokens": 1, "context": 1000, "new": 1},
        # the next token of each of many sequences, at far positions of an extended context
        {**common, "name": "append_batch", "op": "append", "sequences": 128, "tokens": 128, "context": 128 * 20000, "new": 1,
         "scaling": "parts", "mix": 1},
        # ragged prompts, interleaved pairs in part of the head, float16
        {**common, "name": "append_odd", "op": "append", "dtype": "f16", "heads": 12, "kv_heads": 4, "d": 64, "page": 32,
         "sequences": 5, "tokens": 777, "context": 1001, "rotary": 36, "interleaved": True, "scaling": "linear", "mix": 2},
        # a large prefill: memory's rate
        {**common, "name": "append_prompt", "op": "append", "sequences": 4, "tokens": 16384, "context": 0, "mix": 3},
        # short prompts together: most tiles are partly filled
        {**common, "name": "prompt_short", "op": "prompt", "sequences": 16, "tokens": 500, "context": 0, "mix": 4},
        # the next part of one long prompt, seven query heads to a key head, float16
        {**common, "name": "prompt_part", "op": "prompt", "dtype": "f16", "heads": 28, "kv_heads": 4, "page": 64, "sequences": 1,
         "tokens": 512, "context": 15900},
        # packed prompts of different lengths, some of them with a prefix in the cache
        {**common, "name": "prompt_packed", "op": "prompt", "sequences": 12, "tokens": 8192, "context": 5000, "mix": 5},
        # one long prompt: the matrix cores' rate
        {**common, "name": "prompt_long", "op": "prompt", "sequences": 1, "tokens": 16384, "context": 0},
        # the next token of one sequence: latency
        {**common, "name": "token_one", "op": "token", "sequences": 1, "tokens": 1, "context": 4095, "new": 1},
        # a decoding batch of different lengths: memory's rate
        {**common, "name": "token_batch", "op": "token", "sequences": 64, "tokens": 64, "context": 64 * 4095, "new": 1, "mix": 6},
        # two very long sequences: one has to be shared by the whole chip
        {**common, "name": "token_long", "op": "token", "heads": 32, "kv_heads": 4, "page": 64, "sequences": 2, "tokens": 2,
         "context": 2 * 131000, "new": 1, "mix": 7},
        # three drafted tokens a sequence, no shared heads, a window, float16, sizes that fill nothing
        {**common, "name": "token_odd", "op": "token", "dtype": "f16", "heads": 9, "kv_heads": 9, "d": 64, "page": 32,
         "sequences": 7, "tokens": 21, "context": 20011, "new": 3, "window": 1500, "mix": 8},
    ]


def _size(rng, low, high):
    """A size between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["append", "prompt", "prompt", "token", "token"])
    d, kv_heads = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 8, _size(rng, 1, 16)])
    group = rng.choice([1, 2, 4, 4, 7, 8, rng.randint(1, 16)])
    group = max(1, min(group, 64 // kv_heads))
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16"]), "heads": kv_heads * group, "kv_heads": kv_heads, "d": d,
            "page": rng.choice([16, 16, 32, 64, 128, 256]), "mix": rng.randint(0, 1000), "new": 0,
            "window": rng.choice([0, 0, 0, _size(rng, 16, 4096)]), "rotary": d, "interleaved": rng.random() < 0.3,
            "scaling": rng.choice(["none", "none", "linear", "parts"])}
    if op == "append":
        if rng.random() < 0.3:
            case["rotary"] = 2 * rng.randint(1, d // 2)
        largest = min(16384, VALUES // ((kv_heads * (group + 2)) * d))
        case["tokens"] = _size(rng, 1, largest)
        case["sequences"] = _size(rng, 1, min(256, case["tokens"]))
        case["context"] = case["sequences"] * _size(rng, 1, 100000)
        if rng.random() < 0.5:
            case["new"] = rng.randint(1, 4)
            case["tokens"] = case["new"] * case["sequences"]
        return case
    if op == "prompt":
        case["tokens"] = _size(rng, 16, 16384)
        case["sequences"] = _size(rng, 1, min(64, case["tokens"]))
        case["context"] = rng.choice([0, 0, _size(rng, 1, 20000)])
        while work(case)["flops"] > FLOPS:
            case["tokens"], case["context"] = max(case["sequences"], case["tokens"] // 2), case["context"] // 2
        return case
    case["sequences"] = _size(rng, 1, 256)
    case["new"] = rng.choice([1, 1, 1, rng.randint(2, 4)])
    case["tokens"] = case["new"] * case["sequences"]
    case["context"] = _size(rng, case["sequences"], max(case["sequences"], min(500000, KEY_VALUES // (kv_heads * d) - 2000)))
    return case


def _split(total, parts, mix, least):
    """`total` in `parts` of different sizes (of one for mix = 0), each of `least` or more."""
    rng = random.Random(mix)
    weights = [math.exp(rng.gauss(0, 0.7)) if mix else 1.0 for _ in range(parts)]
    free = total - least * parts
    sizes = [least + int(free * w / sum(weights)) for w in weights]
    sizes[0] += total - sum(sizes)
    return sizes


def _tokens(case):
    """(first, count, before) of every sequence: its tokens in the step, and the keys that it had before them."""
    n = case["sequences"]
    counts = [case["new"]] * n if case["new"] else _split(case["tokens"], n, case["mix"], 1)
    before = _split(case["context"], n, case["mix"] + 1 if case["mix"] else 0, 0)
    return list(zip(accumulate(counts, initial=0), counts, before))


def _frequencies(case):
    """Radians a position of every pair, float64."""
    half = case["rotary"] // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    if case["scaling"] == "linear":
        f = f / 4
    if case["scaling"] == "parts":  # pairs that turn less than once in 8192 positions are slowed by 8, beyond 32 turns by nothing
        kept = ((8192 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * kept + f / 8 * (1 - kept)
    return f


def _magnitude(case):
    return 0.1 * math.log(8) + 1 if case["scaling"] == "parts" else 1.0


def _inputs(case, seed):
    """The tensors of a case: sizes from the case, values from the seed alone."""
    g, dtype, d, page = torch.Generator(device="cuda").manual_seed(seed), TORCH[case["dtype"]], case["d"], case["page"]
    heads, kv_heads, n, t = case["heads"], case["kv_heads"], case["sequences"], case["tokens"]
    plan = _tokens(case)
    lengths = [count + before for _, count, before in plan]
    width = max(-(-length // page) for length in lengths)
    # pages in the order in which a server handed them out; an append needs only those that its tokens reach
    needed = [(i, p) for i, (_, count, before) in enumerate(plan)
              for p in range(before // page if case["op"] == "append" else 0, -(-lengths[i] // page))]
    order = torch.randperm(len(needed), generator=torch.Generator().manual_seed(seed))
    table = torch.zeros(n, width, dtype=torch.int32)
    where = torch.tensor(needed)
    table[where[:, 0], where[:, 1]] = order.to(torch.int32)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    x = {"lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "pages": table.cuda()}
    if not case["new"]:
        x["starts"] = torch.tensor([first for first, _, _ in plan] + [t], dtype=torch.int32, device="cuda")
    if case["op"] == "append":
        x["qkv"] = normal(t, (heads + 2 * kv_heads) * d)
        x["keys"] = torch.zeros(len(needed), kv_heads, page, d, device="cuda", dtype=dtype)
        x["values"] = torch.zeros_like(x["keys"])
    else:
        x["q"] = normal(t, heads, d, scale=2.0)  # scores of a standard deviation of 2: a few keys in a hundred matter
        x["keys"], x["values"] = normal(len(needed), kv_heads, page, d), normal(len(needed), kv_heads, page, d)
    return x


def _bind(case, x, out):
    """The framework's call on these tensors: torch memory as its tensors, without a copy."""
    os.environ["ROCM_PATH"] = os.path.dirname(torch.__file__)  # one HIP runtime in a process: torch's own
    from krn_amd.dtypes import BF16, F16, I32
    from krn_amd.lib import KvCache, Rotary, Sequences, cache_attention, rotary_append
    from krn_amd.runtime.api import device_of
    from krn_amd.runtime.hip import HIPTensor

    device = device_of("gfx950")
    kinds = {torch.bfloat16: BF16, torch.float16: F16, torch.int32: I32}

    def tensor(t):
        return HIPTensor(device, t.data_ptr(), kinds[t.dtype], tuple(t.shape), owner=t)

    cache = KvCache(tensor(x["keys"]), tensor(x["values"]))
    if case["new"]:
        sequences = Sequences(tensor(x["lengths"]), tensor(x["pages"]), new=case["new"])
    else:
        sequences = Sequences(tensor(x["lengths"]), tensor(x["pages"]), starts=tensor(x["starts"]))
    if case["op"] == "append":
        scaled = {"none": {}, "linear": {"factor": 4.0}, "parts": {"factor": 8.0, "original": 8192}}[case["scaling"]]
        rotary = Rotary.of(device, case["rotary"], interleaved=case["interleaved"], **scaled)
        return rotary_append.bind(tensor(x["qkv"]), cache, sequences, rotary=rotary, out=tensor(out))
    return cache_attention.bind(tensor(x["q"]), cache, sequences, window=case["window"] or None, out=tensor(out))


def prepare(case, seed):
    x = _inputs(case, seed)
    out = torch.empty(case["tokens"], case["heads"], case["d"], device="cuda", dtype=TORCH[case["dtype"]])
    state = {"case": case, "inputs": x, "out": out, "tokens": _tokens(case)}
    if own:
        state["call"] = _bind(case, x, out)
        torch.cuda.synchronize()  # the framework has streams of its own
    return state


def _rotated(x, angles, case):
    """Heads (tokens, heads, d) in 32 bits, turned by angles (tokens, rotary / 2) in 64."""
    r, half, m = case["rotary"], case["rotary"] // 2, _magnitude(case)
    cos, sin = (torch.cos(angles) * m).float().unsqueeze(1), (torch.sin(angles) * m).float().unsqueeze(1)
    y = x.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, half), slice(half, r))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    return y


def _append(state):
    case, x, out = state["case"], state["inputs"], state["out"]
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["d"], case["page"]
    counts = torch.tensor([count for _, count, _ in state["tokens"]], device="cuda")
    owner = torch.repeat_interleave(torch.arange(case["sequences"], device="cuda"), counts, output_size=case["tokens"])
    ends = torch.cumsum(counts, 0)
    position = x["lengths"].long()[owner] - ends[owner] + torch.arange(case["tokens"], device="cuda")
    angles = position.double().unsqueeze(1) * _frequencies(case).cuda()
    qkv = x["qkv"].reshape(case["tokens"], heads + 2 * kv_heads, d)
    out.copy_(_rotated(qkv[:, :heads].float(), angles, case))
    numbers, rows = x["pages"][owner, position // page].long(), position % page
    x["keys"][numbers, :, rows] = _rotated(qkv[:, heads : heads + kv_heads].float(), angles, case).to(out.dtype)
    x["values"][numbers, :, rows] = qkv[:, heads + kv_heads :]
    return {"q": out, "keys": x["keys"], "values": x["values"]}


def _attention(state):
    case, x, out = state["case"], state["inputs"], state["out"]
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["d"]
    group = heads // kv_heads
    for i, (first, count, before) in enumerate(state["tokens"]):
        numbers = x["pages"][i, : -(-(before + count) // case["page"])].long()
        keys, values = (x[name][numbers].transpose(0, 1).reshape(kv_heads, -1, d).float() for name in ("keys", "values"))
        for at in range(0, count, 1024):  # so many queries at a time
            rows = min(1024, count - at)
            low, high = 0, before + at + rows
            if case["window"]:
                low = max(0, before + at + 1 - case["window"])
            q = x["q"][first + at : first + at + rows].float().reshape(rows, kv_heads, group, d)
            q = q.permute(1, 2, 0, 3).reshape(kv_heads, group * rows, d)
            s = torch.bmm(q, keys[:, low:high].transpose(1, 2).contiguous()) * d**-0.5
            s = s.view(kv_heads, group, rows, high - low)
            position = torch.arange(before + at, high, device="cuda").unsqueeze(1)
            key = torch.arange(low, high, device="cuda")
            hidden = key > position
            if case["window"]:
                hidden |= key <= position - case["window"]
            s.masked_fill_(hidden, -math.inf)
            p = torch.exp(s - s.amax(3, keepdim=True))
            p /= p.sum(3, keepdim=True)
            o = torch.bmm(p.view(kv_heads, group * rows, -1), values[:, low:high]).view(kv_heads, group, rows, d)
            out[first + at : first + at + rows] = o.permute(2, 0, 1, 3).reshape(rows, heads, d).to(out.dtype)
    return out


def run(state):
    x = state["inputs"]
    if own:
        state["call"]()
        if state["case"]["op"] == "append":
            return {"q": state["out"], "keys": x["keys"], "values": x["values"]}
        return state["out"]
    return _append(state) if state["case"]["op"] == "append" else _attention(state)


def work(case):
    heads, kv_heads, d, t, window = (case[name] for name in ("heads", "kv_heads", "d", "tokens", "window"))
    plan = _tokens(case)
    if case["op"] == "append":  # the projection in, queries, keys and values out
        return {"bytes": 4 * t * (heads + 2 * kv_heads) * d + 8 * case["sequences"],
                "flops": 3 * t * (heads + kv_heads) * case["rotary"]}
    pairs = read = 0
    for _, count, before in plan:
        if window:
            full = max(0, min(count, before + count - window))  # queries that see a whole window
            short = count - full
            pairs += full * window + short * before + short * (short + 1) // 2
            read += min(before + count, window + count - 1)
        else:
            pairs += count * before + count * (count + 1) // 2
            read += before + count
    return {"bytes": 4 * (t * heads + read * kv_heads) * d, "flops": 4 * d * heads * pairs}


def exact(case, seed):
    x, d, page, group = _inputs(case, seed), case["d"], case["page"], case["heads"] // case["kv_heads"]
    if case["op"] == "append":
        heads, kv_heads, r = case["heads"], case["kv_heads"], case["rotary"]
        f = _frequencies(case).cuda()
        q = torch.empty(case["tokens"], heads, d, device="cuda", dtype=torch.float64)
        keys, values = x["keys"].double(), x["values"].double()
        for i, (first, count, before) in enumerate(_tokens(case)):
            position = torch.arange(before, before + count, device="cuda")
            turn = torch.polar(torch.full((), _magnitude(case), device="cuda", dtype=torch.float64), position.double()[:, None] * f)
            z = x["qkv"][first : first + count].double().unflatten(1, (-1, d))
            if case["interleaved"]:
                c = torch.complex(z[:, : heads + kv_heads, 0:r:2], z[:, : heads + kv_heads, 1:r:2]) * turn[:, None]
                z[:, : heads + kv_heads, :r] = torch.view_as_real(c).flatten(2)
            else:
                c = torch.complex(z[:, : heads + kv_heads, : r // 2], z[:, : heads + kv_heads, r // 2 : r]) * turn[:, None]
                z[:, : heads + kv_heads, :r] = torch.cat([c.real, c.imag], 2)
            q[first : first + count] = z[:, :heads]
            at = x["pages"][i].long()[torch.div(position, page, rounding_mode="floor")]
            for h in range(kv_heads):
                keys[at, h, position % page], values[at, h, position % page] = z[:, heads + h], z[:, heads + kv_heads + h]
        return {"q": q, "keys": keys, "values": values}
    y = torch.empty(case["tokens"], case["heads"], d, device="cuda", dtype=torch.float64)
    for i, (first, count, before) in enumerate(_tokens(case)):
        j = torch.arange(before + count, device="cuda")
        at = x["pages"][i].long()[torch.div(j, page, rounding_mode="floor")]
        for h in range(case["kv_heads"]):
            k, v = x["keys"][at, h, j % page].double(), x["values"][at, h, j % page].double()
            for a in range(0, count, 2048):
                b = min(count, a + 2048)
                end, begin = before + b, max(0, before + a + 1 - case["window"]) if case["window"] else 0
                distance = torch.arange(before + a, before + b, device="cuda")[:, None] - j[begin:end]
                seen = (distance >= 0) & (distance < (case["window"] or distance.numel() + before + b))
                for e in range(h * group, (h + 1) * group):
                    s = (x["q"][first + a : first + b, e].double() / math.sqrt(d)) @ k[begin:end].T
                    y[first + a : first + b, e] = torch.softmax(torch.where(seen, s, -math.inf), 1) @ v[begin:end]
    return y
