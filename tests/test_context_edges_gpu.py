"""GPU checks of the operators for long contexts at the edges of what their documentation allows. Tolerances are those of
test_context_gpu.py."""
import math

import pytest

import context_cases
from test_context_gpu import attention_reference, ctx, evict_reference, expect_attention, normal, window_visible  # noqa: F401

pytestmark = pytest.mark.gpu


# rows, heads, kv_heads: one stacked row group of the few-row kernel; 36 and 1200 stacked rows; 300 rows that fill tensor-core tiles
@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 8, 2), (9, 8, 2), (300, 32, 8)])
def test_no_tokens_at_all(cuda, package, ctx, rows, heads, kv_heads):
    """No lengths and a length of 0, the default of both: every output row is zeros, accumulated weights stay as they were."""
    torch, ops = cuda, package.operators
    sequences, capacity = 4, 130
    q = normal(torch, 1, sequences * rows, heads, 128)
    k, v = (torch.full((sequences, capacity, kv_heads, 128), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    out = torch.full_like(q, 7.0)
    ops.attention_window(ctx, q, k, v, out, 100, 4)
    assert (out == 0).all()
    for prefix in (0, 70):
        pk, pv = normal(torch, 2, prefix, kv_heads, 128), normal(torch, 3, prefix, kv_heads, 128)
        size = ops.attention_shared_prefix_scratch_bytes(sequences * rows, heads, kv_heads, prefix)
        scratch = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
        out.fill_(7.0)
        ops.attention_shared_prefix(ctx, q, pk, pv, k, v, out, scratch)
        assert (out == 0).all()
    size = ops.attention_accumulate_scratch_bytes(sequences, rows, heads, kv_heads, capacity)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    for old in (None, torch.ones((sequences, kv_heads, capacity), device="cuda")):
        out.fill_(7.0)
        scores = torch.full((sequences, kv_heads, capacity), 9.0, device="cuda")
        ops.attention_accumulate(ctx, q, k, v, out, old, scores, scratch)
        torch.cuda.synchronize()
        assert (out == 0).all() and (scores == 9).all()


# Waits that run out. The first copy of every unit of the first sequence is told to expect 16 bytes more than it brings, with
# a short limit: nothing faults or hangs, the unit's blocks give up and leave.

@pytest.mark.parametrize("name", context_cases.GIVE_UP)
def test_window_waits_that_run_out(cuda, package, ctx, name):
    torch, ops, c = cuda, package.operators, context_cases.GIVE_UP[name]
    q = normal(torch, 1, c.sequences * c.rows, c.heads, 128)
    k, v = (normal(torch, seed, c.sequences, c.tokens, c.kv_heads, 128) for seed in (2, 3))
    want, out = torch.empty_like(q), torch.empty_like(q)
    ops.attention_window(ctx, q, k, v, want, c.window, c.sinks, length=c.tokens)
    for _ in range(2):
        ops.inject_wait_timeout(2000)
        ops.attention_window(ctx, q, k, v, out, c.window, c.sinks, length=c.tokens)
        torch.cuda.synchronize()
        assert out[:c.rows].isnan().all() and torch.equal(out[c.rows:], want[c.rows:])
        ops.attention_window(ctx, q, k, v, out, c.window, c.sinks, length=c.tokens)
        assert torch.equal(out, want)


@pytest.mark.parametrize("name", context_cases.PREFIX_GIVE_UP)
def test_prefix_waits_that_run_out(cuda, package, ctx, name):
    torch, ops, c = cuda, package.operators, context_cases.PREFIX_GIVE_UP[name]
    q = normal(torch, 1, c.sequences * c.rows, c.heads, 128)
    pk, pv = normal(torch, 2, c.prefix, c.kv_heads, 128), normal(torch, 3, c.prefix, c.kv_heads, 128)
    k, v = normal(torch, 4, c.sequences, 50, c.kv_heads, 128), normal(torch, 5, c.sequences, 50, c.kv_heads, 128)
    size = ops.attention_shared_prefix_scratch_bytes(c.sequences * c.rows, c.heads, c.kv_heads, c.prefix)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    want, out = torch.empty_like(q), torch.empty_like(q)
    ops.attention_shared_prefix(ctx, q, pk, pv, k, v, want, scratch, length=50)
    ops.inject_wait_timeout(2000)
    ops.attention_shared_prefix(ctx, q, pk, pv, k, v, out, scratch, length=50)
    torch.cuda.synchronize()
    assert out.isnan().all()
    ops.attention_shared_prefix(ctx, q, pk, pv, k, v, out, scratch, length=50)
    assert torch.equal(out, want) and torch.isfinite(want).all()


@pytest.mark.parametrize("rows,tokens,heads,kv_heads", [(1, 5000, 8, 8), (9, 300, 4, 4), (16, 700, 16, 4), (130, 500, 12, 4)])
def test_accumulated_weights_survive_waits_that_run_out(cuda, package, ctx, rows, tokens, heads, kv_heads):
    """What the first sequence has accumulated stays, in place and apart; the others' is added to as ever. With 390 stacked rows
    the second pass, which is not told to fail, adds what is its own."""
    torch, ops = cuda, package.operators
    q = normal(torch, 1, 2 * rows, heads, 128)
    k, v = normal(torch, 2, 2, tokens, kv_heads, 128), normal(torch, 3, 2, tokens, kv_heads, 128)
    old = torch.rand((2, kv_heads, tokens), generator=torch.Generator("cuda").manual_seed(4), device="cuda")
    scratch = torch.empty(ops.attention_accumulate_scratch_bytes(2, rows, heads, kv_heads, tokens), dtype=torch.uint8, device="cuda")
    want, new = torch.empty_like(q), torch.empty_like(old)
    ops.attention_accumulate(ctx, q, k, v, want, old, new, scratch, length=tokens)
    passes = -(-rows * (heads // kv_heads) // 256)
    for apart in (True, False):
        held, out = old.clone(), torch.empty_like(q)
        scores = torch.empty_like(old) if apart else held
        ops.inject_wait_timeout(2000)
        ops.attention_accumulate(ctx, q, k, v, out, held, scores, scratch, length=tokens)
        torch.cuda.synchronize()
        assert torch.equal(scores[1], new[1]) and torch.equal(out[rows:], want[rows:])
        assert torch.isfinite(scores).all()
        if passes == 1:
            assert torch.equal(scores[0], old[0]) and out[:rows].isnan().all()
        else:
            # Stacked rows of a KV head are row * group + head of the group: those from 256 on are as ever.
            failed = (torch.arange(rows * (heads // kv_heads), device="cuda") < 256).view(rows, 1, -1).expand(-1, kv_heads, -1).flatten(1)
            assert out[:rows][failed].isnan().all() and torch.equal(out[:rows][~failed], want[:rows][~failed])
            total = (scores[0] - old[0]).double().sum(-1)
            # As many rows' weights, which add up to one each: a weight's exponential and the one in the row's sum have arguments
            # up to 16 with three roundings of 2^-24 apart, below 2^-17; and per place some roundings of a value up to the total.
            left = (~failed).view(rows, kv_heads, -1).sum((0, 2))
            assert ((total - left).abs() <= left * 2.0 ** -17 + tokens * 2.0 ** -22 * float(scores.max())).all()
    ops.attention_accumulate(ctx, q, k, v, out, old, scores, scratch, length=tokens)
    assert torch.equal(scores, new) and torch.equal(out, want)


def test_the_host_learns_of_waits_that_ran_out(cuda, package):
    """By a count that grows with them and with nothing else, of both kernels, also from another thread and context."""
    import threading
    torch, ops = cuda, package.operators
    stream = torch.cuda.Stream()
    context, plain = ops.prepare_execution_context(stream.cuda_stream), ops.prepare_execution_context(0)
    k, v = normal(torch, 2, 1, 6000, 4, 128), normal(torch, 3, 1, 6000, 4, 128)
    before = ops.expired_waits(plain)
    for rows in (1, 300):
        q = normal(torch, 1, rows, 8, 128)
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        ops.attention_window(context, q, k, v, out, 1 << 20, 0, length=6000)
        assert ops.expired_waits(context) == before
        ops.inject_wait_timeout(2000)
        ops.attention_window(context, q, k, v, out, 1 << 20, 0, length=6000)
        after = ops.expired_waits(context)
        assert after > before and out.isnan().all()
        seen = []
        other = threading.Thread(target=lambda: seen.append(ops.expired_waits(plain)))
        other.start()
        other.join()
        assert seen == [after]
        before = after


# What is hard, on both kernels.

HARD = pytest.mark.parametrize("name", context_cases.HARD)


def window_call(torch, ops, context, c, q, k, v, out=None, **given):
    out = torch.empty_like(q) if out is None else out
    ops.attention_window(context, q, k, v, out, c.window, c.sinks, **(given or dict(length=c.tokens)))
    return out


def inputs_of(torch, c, scale=1.0):
    return (normal(torch, 1, c.sequences * c.rows, c.heads, 128, scale=scale),
            normal(torch, 2, c.sequences, c.tokens, c.kv_heads, 128, scale=scale), normal(torch, 3, c.sequences, c.tokens, c.kv_heads, 128))


def visible_of(torch, c, n=None):
    return window_visible(torch, c.tokens if n is None else n, c.rows, c.window, c.sinks, c.tokens)


@HARD
def test_random_scores_near_and_far_apart(cuda, package, ctx, name):
    torch, ops, c = cuda, package.operators, context_cases.HARD[name]
    for scale in (1.0, 1.5, 6.0, 40.0):
        q, k, v = inputs_of(torch, c, scale)
        out = window_call(torch, ops, ctx, c, q, k, v)
        for s in {0, c.sequences - 1}:
            mine = slice(s * c.rows, (s + 1) * c.rows)
            want, size, _, _ = attention_reference(torch, q[mine], k[s], v[s], visible_of(torch, c))
            expect_attention(torch, out[mine], want, size)


PATTERNS = ["ascending", "descending", "zigzag", "steps", "equal", "last", "lowest", "1e6", "1e12", "1e30", "1e36"]


def patterned_keys(torch, pattern, tokens):
    """First values of the keys; all others meet zeros of the queries, so that a score is one product, exact in FP32."""
    t = torch.arange(tokens, device="cuda", dtype=torch.float64)
    if pattern[0] == "1":  # two equal ones far above the others
        return torch.where(t % (tokens - 4) == 3, float(pattern), -float(pattern)).bfloat16()
    return {"ascending": t / 2, "descending": -t / 2, "zigzag": (t % 2 * 2 - 1) * 60, "steps": (t // 77) * 20, "equal": torch.full_like(t, 3.0),
            "lowest": torch.full_like(t, torch.finfo(torch.bfloat16).min), "last": torch.where(t == tokens - 1, 300.0, -300.0)}[pattern].bfloat16()


def exact_weights(torch, q, keys, visible):
    """Scores and weights in 64 bits of a head's queries."""
    s = (q.double() @ keys.double().T / math.sqrt(128)).masked_fill(~visible, -math.inf)
    return s, torch.softmax(s, -1)


def expect_exact_scores(torch, out, q, k, v, visible):
    """The reference's tolerance, but for scores that are exact: left are the exponential's argument, whose two roundings are of
    2^-24 of the score and of its distance from the maximum, and the joining of parts, two roundings of the maxima. A score
    beyond 16384 is at least 64 from any other (keys have eight bits) or equal to it, which no rounding takes apart."""
    n, heads = q.shape[:2]
    group = heads // k.shape[1]
    for h in range(heads):
        s, w = exact_weights(torch, q[:, h], k[:, h // group], visible)
        top = s.amax(-1, keepdim=True)
        error = 2.0 ** -21 + 2.0 ** -22 * (top.abs().clamp(max=16384.0) + torch.where(w > 2.0 ** -60, (s - top).abs(), 0.0))
        values = v[:, h // group].double()
        expect_attention(torch, out[:, h], w @ values, (w * (1 + error * 2.0 ** 8)) @ values.abs())


@HARD
@pytest.mark.parametrize("pattern", PATTERNS)
def test_scores_in_patterns(cuda, package, ctx, name, pattern):
    """Maxima that move every tile, never, or with the last token; equal scores; the lowest finite keys; scores as large
    as FP32 holds, whose products with the scale are rounded by more than weights' exponents reach."""
    torch, ops, c = cuda, package.operators, context_cases.HARD[name]
    _, k, v = inputs_of(torch, c)
    q = torch.zeros(c.sequences * c.rows, c.heads, 128, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0 if pattern in ("lowest", "1e36") else 8.0
    if pattern[0] == "1":
        q[..., 0] *= 1 + normal(torch, 8, *q.shape[:2]).abs() / 8
    k[..., 0] = patterned_keys(torch, pattern, c.tokens)[None, :, None]
    out = window_call(torch, ops, ctx, c, q, k, v)
    for s in {0, c.sequences - 1}:
        mine = slice(s * c.rows, (s + 1) * c.rows)
        expect_exact_scores(torch, out[mine], q[mine], k[s], v[s], visible_of(torch, c))


def clean(torch, got, want, size, wrong):
    """Rows and heads outside `wrong` are as ever."""
    got, want, size = got[~wrong], want[~wrong], size[~wrong]
    expect_attention(torch, got, want, size)


@HARD
def test_nan_keys_in_sight_stay_in_their_rows(cuda, package, ctx, name):
    """A key that is no number makes the rows that see it NaN, and no other: not the rows before it, those whose window has left it
    behind, other heads' or sequences'."""
    torch, ops, c = cuda, package.operators, context_cases.HARD[name]
    q, k, v = inputs_of(torch, c)
    base, visible = window_call(torch, ops, ctx, c, q, k, v), visible_of(torch, c)
    group, s, head = c.heads // c.kv_heads, c.sequences - 1, c.kv_heads - 1
    for token in (c.tokens - 1, c.tokens - 1 - c.rows // 2, max(c.sinks, c.tokens - c.window)):
        bad = k.clone()
        bad[s, token, head, 5] = math.nan
        out = window_call(torch, ops, ctx, c, q, bad, v)
        wrong = torch.zeros(out.shape[:2], dtype=torch.bool, device="cuda")
        wrong[s * c.rows:, head * group:] = visible[:, token, None]
        assert wrong.any()
        assert out[wrong].isnan().all() and torch.equal(out[~wrong], base[~wrong])


@HARD
def test_infinite_keys_in_sight(cuda, package, ctx, name):
    """A score of -inf is a weight of zero, one of +inf leaves nothing that is a number, as in the formula."""
    torch, ops, c = cuda, package.operators, context_cases.HARD[name]
    q, k, v = inputs_of(torch, c)
    q[..., 9] = torch.where(q[..., 9] == 0, 1.0, q[..., 9])
    visible = visible_of(torch, c)
    group, token = c.heads // c.kv_heads, c.tokens - 1 - c.rows // 3
    k[0, token, 0, 9] = math.inf
    out = window_call(torch, ops, ctx, c, q, k, v)[:c.rows]
    mine = q[:c.rows]
    infinite = visible[:, token, None] & (mine[..., 9] > 0)
    infinite[:, group:] = False
    assert infinite.any() and out[infinite].isnan().all()
    rest = visible.clone()
    rest[:, token] = False
    finite = k[0].clone()
    finite[token, 0, 9] = 0.0
    some, _, _, _ = attention_reference(torch, mine, finite, v[0], visible)
    without, size, _, _ = attention_reference(torch, mine, finite, v[0], rest)
    minus = visible[:, token, None] & (mine[..., 9] < 0)
    minus[:, group:] = False
    assert minus.any()
    want, wide, _, _ = attention_reference(torch, mine, finite, v[0], visible)
    want, wide = torch.where(minus[..., None], without, want), torch.where(minus[..., None], size, wide)
    clean(torch, out, want, wide, infinite)


@HARD
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_values_that_are_no_numbers_stay_in_their_column(cuda, package, ctx, name, value):
    """Rows that see the token lose that one column; of rows of the same call that do not see it, no other column, head or
    sequence is touched."""
    torch, ops, c = cuda, package.operators, context_cases.HARD[name]
    q, k, v = inputs_of(torch, c)
    base, visible = window_call(torch, ops, ctx, c, q, k, v), visible_of(torch, c)
    group, token = c.heads // c.kv_heads, c.tokens - 1 - c.rows // 2
    v[0, token, 0, 33] = value
    out = window_call(torch, ops, ctx, c, q, k, v)
    assert not torch.isfinite(out[:c.rows, :group, 33][visible[:, token]]).any()
    out[:c.rows, :group, 33] = base[:c.rows, :group, 33]
    assert torch.equal(out, base)


@HARD
def test_outputs_in_the_queries_place_and_wide_rows(cuda, package, ctx, name):
    """In place, as slices of wider rows, and over caches in another order: the same bits."""
    torch, ops, c = cuda, package.operators, context_cases.HARD[name]
    q, k, v = inputs_of(torch, c)
    base = window_call(torch, ops, ctx, c, q, k, v)
    mine = q.clone()
    assert torch.equal(window_call(torch, ops, ctx, c, mine, k, v, mine), base)
    wide = torch.full((q.shape[0], c.heads * 128 + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    rows = wide[:, 16:-8].unflatten(-1, (c.heads, 128))
    rows.copy_(q)
    turned = k.transpose(1, 2).contiguous().transpose(1, 2), torch.stack((v, v), 2)[:, :, 1]
    assert torch.equal(window_call(torch, ops, ctx, c, rows, *turned, rows), base)
    assert (wide[:, :16] == 7).all() and (wide[:, -8:] == 7).all()


@pytest.mark.parametrize("name", context_cases.GRAPH)
def test_graphs_follow_lengths(cuda, package, name):
    """Captured in a thread that has never called, replayed for other lengths (none, one, one below the rows, all) and queries."""
    import threading
    torch, ops, c = cuda, package.operators, context_cases.GRAPH[name]
    q, k, v = inputs_of(torch, c)
    lengths = torch.full((c.sequences,), c.tokens, dtype=torch.int32, device="cuda")
    out, stream, graph, errors = torch.empty_like(q), torch.cuda.Stream(), torch.cuda.CUDAGraph(), []
    context = ops.prepare_execution_context(stream.cuda_stream)
    with torch.cuda.stream(stream):
        window_call(torch, ops, context, c, q, k, v, out, lengths=lengths)
    torch.cuda.synchronize()

    def capture():
        try:
            with torch.cuda.graph(graph, stream=stream):
                window_call(torch, ops, context, c, q, k, v, out, lengths=lengths)
        except BaseException as error:  # noqa: BLE001
            errors.append(error)

    thread = threading.Thread(target=capture)
    thread.start()
    thread.join()
    assert not errors
    for n in ([c.tokens, c.tokens // 2], [0, c.tokens - 1], [1, c.rows - 1], [c.rows, c.tokens + 1], [c.rows + 1, -1]):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        q.copy_(normal(torch, sum(n), *q.shape))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for s, held in enumerate(n):
            mine = slice(s * c.rows, (s + 1) * c.rows)
            held = held if 0 <= held <= c.tokens else 0
            want, size, _, _ = attention_reference(torch, q[mine], k[s], v[s], visible_of(torch, c, held))
            expect_attention(torch, out[mine], want, size)
            assert (out[mine][:max(0, c.rows - held)] == 0).all()


@pytest.mark.parametrize("name", context_cases.PREFIX_HARD)
def test_shared_prefix_over_strided_caches(cuda, package, ctx, name):
    """Own tokens in another order and with gaps, outputs as slices of wider rows, two streams and threads at once with scratch of
    their own, in place: the same bits, and right."""
    import threading
    torch, ops, c = cuda, package.operators, context_cases.PREFIX_HARD[name]
    own = 61
    q = normal(torch, 1, c.sequences * c.rows, c.heads, 128, scale=1.5)
    pk, pv = normal(torch, 2, c.prefix, c.kv_heads, 128, scale=1.5), normal(torch, 3, c.prefix, c.kv_heads, 128)
    k, v = normal(torch, 4, c.sequences, own, c.kv_heads, 128, scale=1.5), normal(torch, 5, c.sequences, own, c.kv_heads, 128)
    lengths = torch.tensor([own - s % 7 for s in range(c.sequences)], dtype=torch.int32, device="cuda")
    size = ops.attention_shared_prefix_scratch_bytes(c.sequences * c.rows, c.heads, c.kv_heads, c.prefix)
    results = []

    def go(context, queries, keys, values, out):
        scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
        ops.attention_shared_prefix(context, queries, pk, pv, keys, values, out, scratch, lengths=lengths)
        results.append((out, scratch))

    go(ctx, q, k, v, torch.empty_like(q))
    wide = torch.full((q.shape[0] + 1, c.heads * 128 + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    rows = wide[:-1, 8:].unflatten(-1, (c.heads, 128))
    both = torch.full((c.sequences, own + 3, c.kv_heads, 2, 128), math.nan, dtype=torch.bfloat16, device="cuda")
    both[:, :own, :, 0], both[:, :own, :, 1] = k, v
    go(ctx, q, both[:, :own, :, 0], both[:, :own, :, 1], rows)
    mine = q.clone()
    go(ctx, mine, k.transpose(1, 2).contiguous().transpose(1, 2), v, mine)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(q) for _ in streams]
    torch.cuda.synchronize()
    threads = [threading.Thread(target=lambda s=s, o=o: [go(ops.prepare_execution_context(s.cuda_stream), q, k, v, o) for _ in range(20)])
               for s, o in zip(streams, outs)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert len(results) == 43
    for out, _ in results:
        assert torch.equal(out, results[0][0])
    assert (wide[-1] == 7).all() and (wide[:, :8] == 7).all()
    for s in {0, c.sequences - 1}:
        mine, n = slice(s * c.rows, (s + 1) * c.rows), int(lengths[s])
        place = torch.arange(n - c.rows, n, device="cuda")[:, None]
        visible = torch.cat(((place >= 0).expand(-1, c.prefix), torch.arange(own, device="cuda")[None] <= place), 1)
        want, allowance, _, _ = attention_reference(torch, q[mine], torch.cat((pk, k[s])), torch.cat((pv, v[s])), visible)
        expect_attention(torch, results[0][0][mine], want, allowance)


@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("name", context_cases.PREFIX_HARD)
def test_scores_in_patterns_behind_a_prefix(cuda, package, ctx, name, pattern):
    """The patterns over prefix and own tokens, the largest scores on both sides of the border."""
    torch, ops, c = cuda, package.operators, context_cases.PREFIX_HARD[name]
    own = 310
    q = torch.zeros(c.sequences * c.rows, c.heads, 128, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0 if pattern in ("lowest", "1e36") else 8.0
    pk, pv = normal(torch, 2, c.prefix, c.kv_heads, 128), normal(torch, 3, c.prefix, c.kv_heads, 128)
    k, v = normal(torch, 4, c.sequences, own, c.kv_heads, 128), normal(torch, 5, c.sequences, own, c.kv_heads, 128)
    keys = patterned_keys(torch, pattern, c.prefix + own - 4)
    if pattern[0] == "1":
        keys[3], keys[c.prefix - 1], keys[c.prefix] = float(pattern), float(pattern), float(pattern)
    keys = torch.cat((keys, keys[-4:]))
    pk[..., 0], k[..., 0] = keys[:c.prefix, None], keys[c.prefix:][None, :, None]
    size = ops.attention_shared_prefix_scratch_bytes(c.sequences * c.rows, c.heads, c.kv_heads, c.prefix)
    out = torch.empty_like(q)
    ops.attention_shared_prefix(ctx, q, pk, pv, k, v, out, torch.empty(size, dtype=torch.uint8, device="cuda"), length=own)
    place = torch.arange(own - c.rows, own, device="cuda")[:, None]
    visible = torch.cat(((place >= 0).expand(-1, c.prefix), torch.arange(own, device="cuda")[None] <= place), 1)
    for s in {0, c.sequences - 1}:
        mine = slice(s * c.rows, (s + 1) * c.rows)
        expect_exact_scores(torch, out[mine], q[mine], torch.cat((pk, k[s])), torch.cat((pv, v[s])), visible)


@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 16, 2), (9, 12, 4)])
def test_accumulated_weights_over_strided_caches_and_far_scores(cuda, package, ctx, rows, heads, kv_heads):
    """Caches in other orders and with gaps give the same bits; scores far apart give weights of one and zero."""
    torch, ops = cuda, package.operators
    sequences, tokens = 2, 700
    size = ops.attention_accumulate_scratch_bytes(sequences, rows, heads, kv_heads, tokens)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    old = torch.rand((sequences, kv_heads, tokens), generator=torch.Generator("cuda").manual_seed(9), device="cuda")

    def go(q, k, v, scores):
        out, new = torch.empty_like(q), torch.empty_like(old)
        ops.attention_accumulate(ctx, q, k, v, out, scores, new, scratch, length=tokens)
        return out, new

    for scale in (1.0, 40.0):
        q = normal(torch, 1, sequences * rows, heads, 128, scale=scale)
        k, v = normal(torch, 2, sequences, tokens, kv_heads, 128, scale=scale), normal(torch, 3, sequences, tokens, kv_heads, 128)
        out, new = go(q, k, v, old)
        both = torch.full((sequences, tokens + 5, 2, kv_heads, 128), math.nan, dtype=torch.bfloat16, device="cuda")
        both[:, :tokens, 0], both[:, :tokens, 1] = k, v
        turned = torch.rand((kv_heads, sequences, tokens + 1), device="cuda")[..., :tokens].transpose(0, 1)
        turned.copy_(old)
        for got in (go(q, both[:, :tokens, 0], both[:, :tokens, 1], turned), go(q, k.transpose(1, 2).contiguous().transpose(1, 2), v, old)):
            assert torch.equal(got[0], out) and torch.equal(got[1], new)
        for s in range(sequences):
            mine = slice(s * rows, (s + 1) * rows)
            want, allowance, weights, slack = attention_reference(torch, q[mine], k[s], v[s], window_visible(torch, tokens, rows, 1 << 30, 0, tokens))
            expect_attention(torch, out[mine], want, allowance)
            total = weights + old[s].double()
            assert ((new[s].double() - total).abs() <= slack + 2.0 ** -22 * total).all()


@pytest.mark.parametrize("pattern", ["lowest", "1e6", "1e12", "1e30", "1e36"])
@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 16, 2), (9, 12, 4)])
def test_accumulated_weights_of_far_scores(cuda, package, ctx, rows, heads, kv_heads, pattern):
    """Two equal scores above all others, or all of them equal: a half each, or one part each."""
    torch, ops = cuda, package.operators
    tokens = 700
    q = torch.zeros(rows, heads, 128, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1 + normal(torch, 8, rows, heads).abs() / 8
    if pattern == "lowest":
        q[..., 0] = 1.0
    k, v = normal(torch, 2, 1, tokens, kv_heads, 128), normal(torch, 3, 1, tokens, kv_heads, 128)
    k[..., 0] = patterned_keys(torch, pattern, tokens)[None, :, None]
    scratch = torch.empty(ops.attention_accumulate_scratch_bytes(1, rows, heads, kv_heads, tokens), dtype=torch.uint8, device="cuda")
    out, new = torch.empty_like(q), torch.empty((1, kv_heads, tokens), device="cuda")
    ops.attention_accumulate(ctx, q, k, v, out, None, new, scratch, length=tokens)
    visible = window_visible(torch, tokens, rows, 1 << 30, 0, tokens)
    expect_exact_scores(torch, out, q, k[0], v[0], visible)
    group = heads // kv_heads
    for j in range(kv_heads):
        want = sum(exact_weights(torch, q[:, h], k[0, :, j], visible)[1].sum(0) for h in range(j * group, (j + 1) * group))
        # A weight's exponential, its share and the additions: some roundings of 2^-24 and the exponential's 2^-22.
        assert ((new[0, j].double() - want).abs() <= 2.0 ** -20 * want + 1e-30).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_rotation_of_what_is_no_number(cuda, package, ctx, interleaved, norm):
    """NaN and infinities stay in their head; without a norm, in their pair."""
    torch, ops = cuda, package.operators
    q, k = normal(torch, 1, 6, 4, 128), normal(torch, 2, 6, 2, 128)
    weight = 1 + normal(torch, 3, 128, scale=0.1) if norm else None
    table = torch.from_numpy(ops.build_rope_table_scaled(100, 64, 1e4)).cuda()

    def go(x):
        out = torch.empty_like(x), torch.empty_like(k)
        ops.qk_norm_rope(ctx, x, k, table, *out, offset=3, q_weight=weight, k_weight=weight, interleaved=interleaved)
        return out

    base, keys = go(q)
    assert torch.isfinite(base).all()
    for at, value in ((10, math.nan), (100, math.inf), (63, -math.inf)):
        x = q.clone()
        x[2, 1, at] = value
        out, same = go(x)
        touched = torch.zeros(128, dtype=torch.bool)
        touched[at] = True
        if at < 64:
            touched[at ^ 1 if interleaved else at ^ 32] = True
        if norm and math.isnan(value):
            touched[:] = True
        assert torch.equal(same, keys)
        if norm and not math.isnan(value):  # divided by an infinite length: zeros beside it, which the rotation leaves zeros
            assert (out[2, 1, ~touched] == 0).all() and not torch.isfinite(out[2, 1, at])
        else:
            assert not torch.isfinite(out[2, 1, touched]).any()
            assert torch.equal(out[2, 1, ~touched], base[2, 1, ~touched])
        out[2, 1] = base[2, 1]
        assert torch.equal(out, base)


@pytest.mark.parametrize("name", ["window", "window of many rows", "prefix", "accumulate"])
def test_the_first_call_of_a_thread(cuda, package, ctx, name):
    """The driver's calls need the device's context, which a thread has from its first call of the runtime on."""
    import threading
    torch, ops = cuda, package.operators
    rows = 300 if "many" in name else 2
    q = normal(torch, 1, 2 * rows, 8, 128)
    k, v = normal(torch, 2, 2, 3000, 4, 128), normal(torch, 3, 2, 3000, 4, 128)
    scratch = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    scores = torch.zeros((2, 4, 3000), device="cuda")
    calls = {"prefix": lambda out: ops.attention_shared_prefix(ctx, q, k[0, :70], v[0, :70], k, v, out, scratch, length=3000),
             "accumulate": lambda out: ops.attention_accumulate(ctx, q, k, v, out, None, scores, scratch, length=3000)}
    call = calls.get(name, lambda out: ops.attention_window(ctx, q, k, v, out, 1 << 20, length=3000))
    want, out, errors = torch.empty_like(q), torch.zeros_like(q), []
    call(want)

    def first():
        try:
            call(out)
        except BaseException as error:  # noqa: BLE001
            errors.append(error)

    thread = threading.Thread(target=first)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert not errors and torch.equal(out, want)


def test_weights_eviction_and_rotation_in_a_graph(cuda, package):
    """One graph of a server's step behind an observation window: rotation into the cache, accumulated weights in one and in two
    passes, eviction; replayed for other lengths, positions, queries and scores, each time as the calls one by one."""
    torch, ops = cuda, package.operators
    sequences, rows, heads, kv_heads, capacity, budget = 3, 70, 16, 4, 500, 128  # 280 stacked rows
    q = normal(torch, 1, sequences * rows, heads, 128)
    k, v = normal(torch, 3, sequences, capacity, kv_heads, 128), normal(torch, 4, sequences, capacity, kv_heads, 128)
    table = torch.from_numpy(ops.build_rope_table_scaled(1000, 128, 1e4)).cuda()
    positions = torch.zeros(sequences * rows, dtype=torch.int32, device="cuda")
    lengths = torch.full((sequences,), capacity, dtype=torch.int32, device="cuda")
    scratch = torch.empty(ops.attention_accumulate_scratch_bytes(sequences, rows, heads, kv_heads, capacity), dtype=torch.uint8, device="cuda")
    keys = normal(torch, 5, sequences * rows, kv_heads, 128)

    def buffers():
        return dict(q=torch.zeros_like(q), k=torch.zeros_like(keys), out=torch.zeros_like(q),
                    scores=torch.zeros((sequences, kv_heads, capacity), device="cuda"),
                    k2=torch.zeros((sequences, budget, kv_heads, 128), dtype=torch.bfloat16, device="cuda"),
                    v2=torch.zeros((sequences, budget, kv_heads, 128), dtype=torch.bfloat16, device="cuda"),
                    scores2=torch.zeros((sequences, kv_heads, budget), device="cuda"),
                    kept=torch.zeros((sequences, kv_heads, budget), dtype=torch.int32, device="cuda"),
                    new=torch.zeros(sequences, dtype=torch.int32, device="cuda"))

    def step(context, b):
        ops.qk_norm_rope(context, q, keys, table, b["q"], b["k"], positions=positions)
        ops.attention_accumulate(context, b["q"], k, v, b["out"], b["scores"], b["scores"], scratch, lengths=lengths)
        ops.evict_kv(context, k, v, b["scores"], b["k2"], b["v2"], b["scores2"], b["kept"], b["new"], 4, 20, lengths=lengths)

    stream, held = torch.cuda.Stream(), buffers()
    context = ops.prepare_execution_context(stream.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step(context, held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(context, held)
    for turn, n in enumerate(([500, 300, 129], [128, 0, 60], [1, 501, -7], [333, 334, 500])):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        positions.copy_(torch.randint(-2, 1002, positions.shape, generator=torch.Generator("cuda").manual_seed(turn), device="cuda", dtype=torch.int32))
        q.copy_(normal(torch, 50 + turn, *q.shape))
        want = buffers()
        old = torch.rand(want["scores"].shape, generator=torch.Generator("cuda").manual_seed(90 + turn), device="cuda")
        want["scores"].copy_(old)
        for name in held:
            held[name].copy_(want[name])
        torch.cuda.synchronize()
        step(context, want)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in held:
            assert torch.equal(held[name], want[name]), name
        for s, tokens in enumerate(n):
            tokens = tokens if 0 <= tokens <= capacity else 0
            assert int(held["new"][s]) == min(tokens, budget)
            mine = slice(s * rows, (s + 1) * rows)
            visible = window_visible(torch, tokens, rows, 1 << 30, 0, capacity)
            exact, allowance, weights, slack = attention_reference(torch, held["q"][mine], k[s], v[s], visible)
            expect_attention(torch, held["out"][mine], exact, allowance)
            total = old[s].double() + weights
            assert ((held["scores"][s].double() - total).abs() <= slack + 2.0 ** -22 * total).all()


@pytest.mark.parametrize("lengths,capacity,budget,sinks,recent", [
    ([70, 3, 0], 70, 100, 40, 60),                # a budget beyond the capacity, first and latest beyond it too
    ([900, 64, 65], 150000, 64, 4, 60),           # caches far larger than what they hold; no place for any other
    ([2000, 1999], 100000, 700, 0, 1),
    ([41000, 100], 41000, 40, 0, 0),              # a little more than a block keeps, hardly any stay
    ([100], 100, 1, 1, 0), ([100], 100, 1, 0, 1), ([2], 2, 1, 0, 0),
])
def test_eviction_at_its_edges(cuda, package, ctx, lengths, capacity, budget, sinks, recent):
    torch, ops = cuda, package.operators
    sequences, kv_heads = len(lengths), 2
    generator = torch.Generator("cuda").manual_seed(5)
    k, v = (torch.full((sequences, capacity, kv_heads, 128), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    scores = torch.full((sequences, kv_heads, capacity), math.inf, device="cuda")  # of tokens that are not there
    for s, n in enumerate(lengths):
        k[s, :n], v[s, :n] = normal(torch, s, n, kv_heads, 128), normal(torch, 70 + s, n, kv_heads, 128)
        scores[s, :, :n] = torch.randint(0, 9, (kv_heads, n), generator=generator, device="cuda") * 2.0 ** -149  # the smallest numbers
    k_out, v_out = (torch.full((sequences, budget, kv_heads, 128), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    scores_out = torch.full((sequences, kv_heads, budget), 9.0, device="cuda")
    kept, new = torch.zeros((sequences, kv_heads, budget), dtype=torch.int32, device="cuda"), torch.zeros(sequences, dtype=torch.int32, device="cuda")
    ops.evict_kv(ctx, k, v, scores, k_out, v_out, scores_out, kept, new, sinks, recent, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    assert new.tolist() == [min(n, budget) for n in lengths]
    for s, n in enumerate(lengths):
        host = scores[s].cpu().tolist()
        for h in range(kv_heads):
            want = evict_reference(torch, host[h], n, budget, sinks, recent)
            assert kept[s, h].tolist() == want + [-1] * (budget - len(want))
            index = torch.tensor(want, dtype=torch.long, device="cuda")
            assert torch.equal(k_out[s, :len(want), h], k[s, index, h]) and torch.equal(v_out[s, :len(want), h], v[s, index, h])
            assert torch.equal(scores_out[s, h, :len(want)], scores[s, h, index])
        assert (k_out[s, len(want):] == 7).all() and (scores_out[s, :, len(want):] == 9).all()


def test_offsets_beyond_32_bits(cuda, package, ctx):
    """The last of five sequences starts beyond 2^32 elements: many rows, accumulated weights, eviction."""
    torch, ops = cuda, package.operators
    sequences, capacity, kv_heads, heads, n = 5, 65536 * 2, 8, 16, 3000
    k = torch.zeros((sequences * 8, capacity, kv_heads, 128), dtype=torch.bfloat16, device="cuda")[::8]
    assert k.stride(0) * 4 + 128 > 2 ** 32
    v = k.clone()
    k[-1, :n], v[-1, :n] = normal(torch, 1, n, kv_heads, 128), normal(torch, 2, n, kv_heads, 128)
    lengths = torch.tensor([0] * 4 + [n], dtype=torch.int32, device="cuda")
    q = normal(torch, 3, sequences * 300, heads, 128)
    out = torch.empty_like(q)
    ops.attention_window(ctx, q, k, v, out, 2500, 4, lengths=lengths)
    want, size, _, _ = attention_reference(torch, q[-300:], k[-1, :n], v[-1, :n], window_visible(torch, n, 300, 2500, 4, n))
    expect_attention(torch, out[-300:], want, size)
    assert (out[:-300] == 0).all()
    q, wide = q[:sequences * 2], torch.zeros((sequences * 1024, kv_heads, capacity), device="cuda")[::1024]
    assert wide.stride(0) * 4 >= 2 ** 32
    scratch = torch.empty(ops.attention_accumulate_scratch_bytes(sequences, 2, heads, kv_heads, capacity), dtype=torch.uint8, device="cuda")
    ops.attention_accumulate(ctx, q, k, v, torch.empty_like(q), wide, wide, scratch, lengths=lengths)
    _, _, weights, slack = attention_reference(torch, q[-2:], k[-1, :n], v[-1, :n], window_visible(torch, n, 2, 1 << 30, 0, n))
    assert ((wide[-1, :, :n].double() - weights).abs() <= slack + 2.0 ** -22 * weights).all()
    assert not wide[:4].any() and not wide[-1, :, n:].any()
    k_out, v_out = (torch.zeros((sequences, 64, kv_heads, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    scores_out, kept = torch.zeros((sequences, kv_heads, 64), device="cuda"), torch.zeros((sequences, kv_heads, 64), dtype=torch.int32, device="cuda")
    new = torch.zeros(sequences, dtype=torch.int32, device="cuda")
    ops.evict_kv(ctx, k, v, wide, k_out, v_out, scores_out, kept, new, 4, 8, lengths=lengths)
    assert new.tolist() == [0] * 4 + [64]
    host = wide[-1, :, :n].cpu().tolist()
    for h in range(kv_heads):
        want = evict_reference(torch, host[h], n, 64, 4, 8)
        assert kept[-1, h].tolist() == want
        index = torch.tensor(want, device="cuda")
        assert torch.equal(k_out[-1, :, h], k[-1, index, h]) and torch.equal(v_out[-1, :, h], v[-1, index, h])


def test_counting_expired_waits_leaves_a_capture_alone(cuda, package):
    """Refused while the stream is captured, and the capture goes on."""
    torch, ops, c = cuda, package.operators, context_cases.FEW
    q, k, v = inputs_of(torch, c)
    out, want, stream, graph = torch.zeros_like(q), torch.empty_like(q), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    context = ops.prepare_execution_context(stream.cuda_stream)
    with torch.cuda.stream(stream):
        window_call(torch, ops, context, c, q, k, v, want)
    torch.cuda.synchronize()
    before = ops.expired_waits(context)
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(ValueError, match="captured"):
            ops.expired_waits(context)
        window_call(torch, ops, context, c, q, k, v, out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and ops.expired_waits(context) == before
