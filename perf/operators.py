"""The operators for long contexts over a key / value cache, as cases with their inputs, one pass each in elementary
operations and through the framework's direct operators, the bytes and operations a pass cannot do without, and what the
definition gives in 64 bits.

Kinds of work
  rope        norms of queries and keys for each head and their rotation, in one pass
  window      attention with a sliding window and a few first tokens that stay visible
  prefix      attention of sequences that share a long prefix
  accumulate  attention that also adds up how much weight every cached token received
  evict       a cache cut to its first, its latest and its heaviest tokens

A batch's caches are [sequences, capacity, kv_heads, 128]; row r of a sequence of length n with R rows stands at position
n - R + r, so its own key and value are in the cache. Head layouts are those of this repository's benchmark
configurations (16 / 8, 32 / 8, 28 / 4 heads of 128). Lengths follow from the case alone, all values from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

WIDTH = 128          # of a head in all attention operators
POSITIONS = 40960    # rows of the rotation table


# ---- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # One decode step of 64 conversations at unequal positions: latency.
        {"name": "rope_step_64", "kind": "rope", "rows": 64, "heads": 32, "kv_heads": 8, "width": 128, "rotary": 128,
         "norm": True, "interleaved": False},
        # A prompt segment of 2048 rows with far positions, neighbouring pairs over half of the head.
        {"name": "rope_prompt_2048", "kind": "rope", "rows": 2048, "heads": 32, "kv_heads": 8, "width": 128, "rotary": 64,
         "norm": True, "interleaved": True},
        # One token of a small model deep in one conversation: latency again.
        {"name": "window_decode_1", "kind": "window", "sequences": 1, "rows": 1, "heads": 16, "kv_heads": 8,
         "shortest": 1501, "longest": 1501, "window": 1024, "sinks": 4},
        # A server's step: 64 conversations of unequal lengths.
        {"name": "window_decode_64", "kind": "window", "sequences": 64, "rows": 1, "heads": 32, "kv_heads": 8,
         "shortest": 256, "longest": 8192, "window": 4096, "sinks": 4},
        # A document's last segment behind what came before it.
        {"name": "window_prompt_2048", "kind": "window", "sequences": 1, "rows": 2048, "heads": 32, "kv_heads": 8,
         "shortest": 8192, "longest": 8192, "window": 2048, "sinks": 4},
        # Three conversations with one system prompt, four drafts each, seven query heads a key head.
        {"name": "prefix_verify_3x5", "kind": "prefix", "sequences": 3, "rows": 5, "heads": 28, "kv_heads": 4,
         "prefix": 2500, "shortest": 100, "longest": 407},
        # Many short answers about one document.
        {"name": "prefix_decode_64", "kind": "prefix", "sequences": 64, "rows": 1, "heads": 32, "kv_heads": 8,
         "prefix": 8192, "shortest": 17, "longest": 1024},
        # Verify steps about a long one: products of matrices.
        {"name": "prefix_verify_16x9", "kind": "prefix", "sequences": 16, "rows": 9, "heads": 32, "kv_heads": 8,
         "prefix": 30011, "shortest": 17, "longest": 512},
        # A token's weights over one long history.
        {"name": "accumulate_decode_1", "kind": "accumulate", "sequences": 1, "rows": 1, "heads": 32, "kv_heads": 8,
         "shortest": 30011, "longest": 30011},
        # A server's step over caches that are kept near their budget.
        {"name": "accumulate_decode_64", "kind": "accumulate", "sequences": 64, "rows": 1, "heads": 32, "kv_heads": 8,
         "shortest": 1900, "longest": 2304},
        # A prompt cut down after it was read.
        {"name": "evict_1", "kind": "evict", "sequences": 1, "kv_heads": 8, "shortest": 8191, "longest": 8191,
         "budget": 1024, "sinks": 4, "recent": 256},
        # 64 caches brought back to their budget.
        {"name": "evict_64", "kind": "evict", "sequences": 64, "kv_heads": 8, "shortest": 1900, "longest": 2304,
         "budget": 2048, "sinks": 4, "recent": 512},
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(["rope", "window", "window", "prefix", "accumulate", "evict"])
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (28, 4)])
    if kind == "rope":
        width = rng.choice([64, 128, 128, 256])
        return {"kind": kind, "rows": spread(1, 8192 * 16 // heads * 64 // width), "heads": heads, "kv_heads": kv_heads,
                "width": width, "rotary": rng.choice([width, width, width // 2]), "norm": rng.random() < 0.7,
                "interleaved": rng.random() < 0.5}
    if kind == "window" and rng.random() < 0.4:
        rows = spread(33, 2048)
        longest = rng.randint(rows, 8192)
        return {"kind": kind, "sequences": 1, "rows": rows, "heads": heads, "kv_heads": kv_heads, "shortest": longest,
                "longest": longest, "window": spread(64, 2048), "sinks": rng.choice([0, 1, 4, 64])}
    sequences = spread(1, 64)
    if kind == "window":
        longest = spread(64, 8192)
        return {"kind": kind, "sequences": sequences, "rows": rng.choice([1, 1, 1, 2, 5, 9, 16]), "heads": heads,
                "kv_heads": kv_heads, "shortest": rng.randint(16, longest), "longest": longest,
                "window": spread(32, 4096), "sinks": rng.choice([0, 1, 4, 64])}
    if kind == "prefix":
        sequences = max(2, sequences)
        longest = spread(32, 1024)
        return {"kind": kind, "sequences": sequences, "rows": rng.choice([1, 1, 2, 5, 9]) if sequences <= 16 else 1,
                "heads": heads, "kv_heads": kv_heads, "prefix": spread(100, 30000), "shortest": rng.randint(9, longest),
                "longest": longest}
    if kind == "accumulate":
        longest = spread(64, 65536 // sequences)
        return {"kind": kind, "sequences": sequences, "rows": rng.choice([1, 1, 2, 9, 16]), "heads": heads,
                "kv_heads": kv_heads, "shortest": rng.randint(16, longest), "longest": longest}
    longest = spread(64, 131072 // sequences)
    budget = rng.randint(32, longest)
    return {"kind": kind, "sequences": sequences, "kv_heads": kv_heads, "shortest": rng.randint(16, longest),
            "longest": longest, "budget": budget, "sinks": rng.choice([0, 4, 16]), "recent": rng.randint(0, budget - 16)}


def lengths_of(case):
    """Evenly spread between the shortest and the longest, in no order."""
    count = case["sequences"]
    step = next(s for s in (37, 41, 43) if math.gcd(s, count) == 1)
    span = case["longest"] - case["shortest"]
    return [case["longest"] - span * ((i * step) % count) // max(1, count - 1) for i in range(count)]


def seen(case, position):
    """Tokens that a row at `position` sees in a window case."""
    low = max(0, position - case["window"] + 1)
    return position + 1 - low + min(case["sinks"], low)


def work(case):
    kind = case["kind"]
    if kind == "rope":
        values = case["rows"] * (case["heads"] + case["kv_heads"]) * case["width"]
        table = case["rows"] * case["rotary"] * 4
        return {"bytes": 4 * values + table + 4 * case["rows"], "flops": values * (7 if case["norm"] else 3)}
    lengths = lengths_of(case)
    if kind == "evict":
        kept = sum(min(n, case["budget"]) for n in lengths) * case["kv_heads"]
        return {"bytes": sum(lengths) * case["kv_heads"] * 4 + kept * (4 * WIDTH * 2 + 8), "flops": sum(lengths) * case["kv_heads"]}
    rows, heads, kv_heads = case["rows"], case["heads"], case["kv_heads"]
    stacked = case["sequences"] * rows * heads
    bytes_ = stacked * WIDTH * 4 + 4 * len(lengths)
    token = kv_heads * WIDTH * 4
    if kind == "window":
        pairs = tokens = 0
        for n in lengths:
            pairs += sum(seen(case, p) for p in range(n - rows, n))
            low = max(0, n - rows - case["window"] + 1)
            tokens += n - low + min(case["sinks"], low)
    elif kind == "prefix":
        pairs = sum(p + 1 + case["prefix"] for n in lengths for p in range(n - rows, n))
        tokens = case["prefix"] + sum(lengths)
    else:
        pairs = sum(p + 1 for n in lengths for p in range(n - rows, n))
        tokens = sum(lengths)
        bytes_ += tokens * kv_heads * 8
    return {"bytes": bytes_ + tokens * token, "flops": pairs * heads * 4 * WIDTH}


# ---- what a program has in hand -----------------------------------------------------------------------------------------

def rotation_table(rotary):
    """[positions, rotary] FP32, sine and cosine of a pair side by side, from angles in 64 bits."""
    frequency = 1e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * frequency
    return torch.stack((angle.sin(), angle.cos()), -1).reshape(POSITIONS, rotary).float()


def prepare(case, seed):
    generator = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=generator, device="cuda", dtype=torch.bfloat16).mul_(scale)

    kind = case["kind"]
    state = {"case": case, "contexts": {}}
    if kind == "rope":
        rows, width = case["rows"], case["width"]
        # The queries and keys are slices of the fused projection's output [rows, (heads + 2 kv_heads) * width].
        fused = normal(rows, (case["heads"] + 2 * case["kv_heads"]), width)
        state["q"], state["k"] = fused[:, :case["heads"]], fused[:, case["heads"]:case["heads"] + case["kv_heads"]]
        state["positions"] = torch.randint(0, POSITIONS, (rows,), generator=generator, device="cuda", dtype=torch.int32)
        state["table"] = rotation_table(case["rotary"])
        if case["norm"]:
            state["q_weight"], state["k_weight"] = 1.0 + normal(width, scale=0.2), 1.0 + normal(width, scale=0.2)
        state["q_out"] = torch.empty((rows, case["heads"], width), dtype=torch.bfloat16, device="cuda")
        state["k_out"] = torch.empty((rows, case["kv_heads"], width), dtype=torch.bfloat16, device="cuda")
        return state
    sequences, kv_heads, capacity = case["sequences"], case["kv_heads"], case["longest"]
    state["lengths"] = torch.tensor(lengths_of(case), dtype=torch.int32, device="cuda")
    # Keys of unit size, values of the size the projections give.
    state["k"] = normal(sequences, capacity, kv_heads, WIDTH)
    state["v"] = normal(sequences, capacity, kv_heads, WIDTH, scale=0.5)
    if kind in ("accumulate", "evict"):
        # What earlier tokens left: few heavy tokens, many light ones.
        state["scores"] = torch.rand((sequences, kv_heads, capacity), generator=generator, device="cuda").pow_(8).mul_(4.0)
    if kind == "evict":
        budget = case["budget"]
        state["k_out"] = torch.zeros((sequences, budget, kv_heads, WIDTH), dtype=torch.bfloat16, device="cuda")
        state["v_out"] = torch.zeros_like(state["k_out"])
        state["scores_out"] = torch.zeros((sequences, kv_heads, budget), device="cuda")
        state["kept"] = torch.zeros((sequences, kv_heads, budget), dtype=torch.int32, device="cuda")
        state["lengths_out"] = torch.zeros_like(state["lengths"])
        return state
    # Scores spread as those of trained heads: a few tokens take most of the weight.
    state["q"] = normal(sequences * case["rows"], case["heads"], WIDTH, scale=2.0)
    state["output"] = torch.empty_like(state["q"])
    if kind == "prefix":
        state["prefix_k"] = normal(case["prefix"], kv_heads, WIDTH)
        state["prefix_v"] = normal(case["prefix"], kv_heads, WIDTH, scale=0.5)
    if kind == "accumulate":
        state["scores_out"] = torch.zeros_like(state["scores"])
    if own and kind in ("prefix", "accumulate"):
        operators = _operators()
        size = (operators.attention_shared_prefix_scratch_bytes(sequences * case["rows"], case["heads"], kv_heads, case["prefix"])
                if kind == "prefix" else
                operators.attention_accumulate_scratch_bytes(sequences, case["rows"], case["heads"], kv_heads, capacity))
        state["scratch"] = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _operators():
    import __graft_entry__ as entry
    return entry.load_package().operators


def _run_own(state):
    operators = _operators()
    stream = torch.cuda.current_stream().cuda_stream
    context = state["contexts"].get(stream)
    if context is None:
        context = state["contexts"][stream] = operators.prepare_execution_context(stream)
    case = state["case"]
    kind = case["kind"]
    if kind == "rope":
        operators.qk_norm_rope(context, state["q"], state["k"], state["table"], state["q_out"], state["k_out"],
                               positions=state["positions"], q_weight=state.get("q_weight"), k_weight=state.get("k_weight"),
                               epsilon=1e-6, interleaved=case["interleaved"])
        return state["q_out"], state["k_out"]
    if kind == "window":
        operators.attention_window(context, state["q"], state["k"], state["v"], state["output"], case["window"],
                                   case["sinks"], lengths=state["lengths"])
        return state["output"]
    if kind == "prefix":
        operators.attention_shared_prefix(context, state["q"], state["prefix_k"], state["prefix_v"], state["k"], state["v"],
                                          state["output"], state["scratch"], lengths=state["lengths"])
        return state["output"]
    if kind == "accumulate":
        operators.attention_accumulate(context, state["q"], state["k"], state["v"], state["output"], state["scores"],
                                       state["scores_out"], state["scratch"], lengths=state["lengths"])
        return state["output"], state["scores_out"]
    operators.evict_kv(context, state["k"], state["v"], state["scores"], state["k_out"], state["v_out"], state["scores_out"],
                       state["kept"], state["lengths_out"], case["sinks"], case["recent"], lengths=state["lengths"])
    return state["k_out"], state["v_out"], state["scores_out"], state["kept"], state["lengths_out"]


def _rotate_plain(x, weight, state):
    case = state["case"]
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    rotary = case["rotary"]
    turns = state["table"][state["positions"].long()].view(-1, 1, rotary // 2, 2)
    sine, cosine = turns[..., 0], turns[..., 1]
    turned, rest = x[..., :rotary], x[..., rotary:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cosine - b * sine, a * sine + b * cosine), -1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat((a * cosine - b * sine, a * sine + b * cosine), -1)
    return torch.cat((turned, rest), -1).bfloat16()


def _run_plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "rope":
        return (_rotate_plain(state["q"], state.get("q_weight"), state), _rotate_plain(state["k"], state.get("k_weight"), state))
    k, v, lengths = state["k"], state["v"], state["lengths"]
    sequences, capacity, kv_heads = k.shape[:3]
    tokens = torch.arange(capacity, device="cuda")
    if kind == "evict":
        budget, length = case["budget"], lengths.view(-1, 1, 1)
        scores = state["scores"]
        # First and latest tokens go before all others, what does not exist behind them; ties to the lowest index.
        rank = torch.where((tokens < case["sinks"]) | (tokens >= length - case["recent"]), math.inf, scores)
        rank = torch.where(tokens < length, rank, -math.inf)
        order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
        new = torch.minimum(lengths, torch.full_like(lengths, budget))
        alive = torch.arange(order.shape[-1], device="cuda") < new.view(-1, 1, 1)
        order = torch.where(alive, order, capacity).sort(dim=-1).values
        index = torch.where(alive, order, 0)
        scores_out = torch.where(alive, scores.gather(-1, index), 0.0)
        rows = index.transpose(1, 2).unsqueeze(-1).expand(-1, -1, -1, WIDTH)
        keep = alive.transpose(1, 2).unsqueeze(-1)
        return (torch.where(keep, k.gather(1, rows), 0), torch.where(keep, v.gather(1, rows), 0), scores_out,
                torch.where(alive, order, -1).int(), new)
    rows, heads = case["rows"], case["heads"]
    group = heads // kv_heads
    q = state["q"].float().view(sequences, rows, kv_heads, group, WIDTH)
    position = (lengths.view(-1, 1) - rows + torch.arange(rows, device="cuda")).view(-1, 1, rows, 1)
    visible = tokens <= position
    if kind == "window":
        visible = visible & ((tokens > position - case["window"]) | (tokens < case["sinks"]))
    output = torch.empty_like(state["q"])
    scores_out = torch.zeros_like(state["scores"]) if kind == "accumulate" else None
    for head in range(kv_heads):
        queries, keys, values = q[:, :, head].transpose(1, 2), k[:, :, head].float().unsqueeze(1), v[:, :, head].float().unsqueeze(1)
        scores = (queries @ keys.transpose(-1, -2)) / math.sqrt(WIDTH)
        scores = torch.where(visible, scores, -math.inf)
        if kind == "prefix":
            first = (queries @ state["prefix_k"][:, head].float().T) / math.sqrt(WIDTH)
            scores = torch.cat((first, scores), -1)
        weights = torch.exp(scores - scores.amax(-1, keepdim=True))
        weights = weights / weights.sum(-1, keepdim=True)
        if kind == "prefix":
            result = weights[..., :case["prefix"]] @ state["prefix_v"][:, head].float() + weights[..., case["prefix"]:] @ values
        else:
            result = weights @ values
        output.view(sequences, rows, kv_heads, group, WIDTH)[:, :, head] = result.transpose(1, 2).bfloat16()
        if kind == "accumulate":
            added = state["scores"][:, head] + weights.sum((1, 2))
            scores_out[:, head] = torch.where(tokens < lengths.view(-1, 1), added, 0.0)
    return (output, scores_out) if kind == "accumulate" else output


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        return _exact_rotation(state)
    if kind == "evict":
        return _exact_eviction(state)
    lengths, rows, heads, kv_heads = lengths_of(case), case["rows"], case["heads"], case["kv_heads"]
    output = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    scores = torch.zeros(state["scores"].shape, dtype=torch.float64, device="cuda") if kind == "accumulate" else None
    for s, n in enumerate(lengths):
        keys, values = state["k"][s, :n].double(), state["v"][s, :n].double()
        shift = 0
        if kind == "prefix":
            shift = case["prefix"]
            keys, values = torch.cat((state["prefix_k"].double(), keys)), torch.cat((state["prefix_v"].double(), values))
        if scores is not None:
            scores[s, :, :n] = state["scores"][s, :, :n].double()
        # Rows in blocks, over the tokens that one of a block's rows may see.
        for first in range(0, rows, 256):
            last = min(rows, first + 256)
            places = torch.arange(n - rows + first, n - rows + last, device="cuda") + shift
            token = torch.arange(n + shift, device="cuda")
            if kind == "window":
                low = max(0, n - rows + first - case["window"] + 1)
                token = token[(token < case["sinks"]) | (token >= low)]
            token = token[token <= int(n - rows + last - 1 + shift)]
            hidden = token[None] > places[:, None]
            if kind == "window":
                hidden |= (token[None] <= places[:, None] - case["window"]) & (token[None] >= case["sinks"])
            block = state["q"][s * rows + first:s * rows + last].double()
            for h in range(heads):
                j = h * kv_heads // heads
                logits = (block[:, h] @ keys[token, j].T * WIDTH ** -0.5).masked_fill(hidden, -math.inf)
                weights = torch.softmax(logits, -1)
                output[s * rows + first:s * rows + last, h] = weights @ values[token, j]
                if scores is not None:
                    scores[s, j, token] += weights.sum(0)
    return output if scores is None else (output, scores)


def _exact_rotation(state):
    case = state["case"]
    turns = state["table"].double()[state["positions"].long()]
    results = []
    for x, weight in ((state["q"], state.get("q_weight")), (state["k"], state.get("k_weight"))):
        y = x.double().clone()
        if weight is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / case["width"] + 1e-6).sqrt() * weight.double()
        z = y.clone()
        half = case["rotary"] // 2
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
            sine, cosine = turns[:, 2 * i, None], turns[:, 2 * i + 1, None]
            z[..., a] = y[..., a] * cosine - y[..., b] * sine
            z[..., b] = y[..., a] * sine + y[..., b] * cosine
        results.append(z)
    return tuple(results)


def _exact_eviction(state):
    case = state["case"]
    budget, lengths = case["budget"], lengths_of(case)
    scores = state["scores"].cpu().numpy()
    kept = np.full((case["sequences"], case["kv_heads"], budget), -1, dtype=np.int32)
    for s, n in enumerate(lengths):
        for h in range(case["kv_heads"]):
            if n <= budget:
                kept[s, h, :n] = np.arange(n)
                continue
            middle = np.arange(case["sinks"], n - case["recent"])
            heaviest = middle[np.lexsort((middle, -scores[s, h, middle].astype(np.float64)))][:budget - case["sinks"] - case["recent"]]
            kept[s, h] = np.concatenate((np.arange(case["sinks"]), np.sort(heaviest), np.arange(n - case["recent"], n)))
    index = torch.from_numpy(kept).cuda()
    moved = []
    for source in (state["k"], state["v"]):
        out = torch.zeros(state["k_out"].shape, dtype=torch.float64, device="cuda")
        for s, n in enumerate(lengths):
            for h in range(case["kv_heads"]):
                out[s, :min(n, budget), h] = source[s, index[s, h, :min(n, budget)].long(), h].double()
        moved.append(out)
    held = torch.where(index >= 0, state["scores"].double().gather(-1, index.clamp(min=0).long()), 0.0)
    return moved[0], moved[1], held, index, torch.tensor([min(n, budget) for n in lengths], dtype=torch.int32, device="cuda")
