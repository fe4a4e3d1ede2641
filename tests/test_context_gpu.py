"""GPU checks of the operators for long contexts against plain arithmetic in 64 bits on the same inputs.

Tolerances, per output, from the roundings there are:
  attention   weights are rounded to BF16 (a relative 2^-8 each, in the numerator and, as their sum, in the denominator) and the
              output once more: |a - e| <= 2^-8 |e| + 2.1 * 2^-8 * sum_t w_t |v_t|. FP32 scores add what `score_error` gives,
              relative to sum_t w_t |v_t| as well.
  weights     FP32 scores and sums: `score_error` twice (its own score and the row's sum) per row that adds to the place, and
              2^-22 of the place's total for the additions.
  rotation    FP32 throughout, one rounding: 2^-8 |e| + 2^-20 of the head's largest normalised value.
  eviction    exact.
`score_error`: a score is a sum of 128 products in FP32 in any order, 129 roundings of at most 2^-23 (the tensor core may cut off
instead of rounding) of the sum of the products' magnitudes; the exponential and its argument add 2^-21 and a relative 2^-23 of the
argument."""
import math

import pytest

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8


@pytest.fixture(scope="module")
def ctx(cuda, package):
    return package.operators.prepare_execution_context(0)


def normal(torch, seed, *shape, scale=1.0):
    generator = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=generator, device="cuda") * scale).bfloat16()


def attention_reference(torch, q, k, v, visible):
    """Rows q [n, heads, 128] over tokens k, v [t, kv_heads, 128]; visible [n, t]. Outputs, sum of w |v|, weights
    [kv_heads, t] and the allowance for them, in 64 bits."""
    n, heads = q.shape[:2]
    kv_heads = k.shape[1]
    group = heads // kv_heads
    out = torch.zeros(n, heads, 128, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    weights = torch.zeros(kv_heads, k.shape[0], dtype=torch.float64, device="cuda")
    slack = torch.zeros_like(weights)
    some = visible.any(0)
    kd = torch.where(some[:, None, None], k.double(), 0.0)
    vd = torch.where(some[:, None, None], v.double(), 0.0)
    for h in range(heads):
        j = h // group
        s = q[:, h].double() @ kd[:, j].T / math.sqrt(128)
        magnitude = (q[:, h].double().abs() @ kd[:, j].abs().T / math.sqrt(128))
        s = s.masked_fill(~visible, -math.inf)
        top = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
        error = 129 * 2.0 ** -23 * torch.where(visible, magnitude, 0.0).amax(-1, keepdim=True) + 2.0 ** -21
        error = error + 2.0 ** -22 * torch.where(visible, s - torch.where(top == -math.inf, 0.0, top), 0.0).abs()
        out[:, h] = w @ vd[:, j]
        size[:, h] = (w * (1 + error / HALF)) @ vd[:, j].abs()
        weights[j] += w.sum(0)
        slack[j] += (w * 2 * error.amax(-1, keepdim=True)).sum(0)
    return out, size, weights, slack


def expect_attention(torch, got, want, size):
    got = got.double()
    assert torch.isfinite(got).all()
    bad = (got - want).abs() > HALF * want.abs() + 2.1 * HALF * size + 1e-30
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}: {float((got - want).abs().max())}"


def window_visible(torch, n, rows, window, sinks, capacity):
    place = torch.arange(n - rows, n, device="cuda")[:, None]
    token = torch.arange(capacity, device="cuda")[None]
    return (token <= place) & ((token > place - window) | (token < sinks))


def cache_like(torch, layout, sequences, capacity, kv_heads, fill):
    """[sequences, capacity, kv_heads, 128] in one of several memory orders."""
    if layout == "tokens":
        base = torch.full((sequences, capacity, kv_heads, 128), fill, dtype=torch.bfloat16, device="cuda")
        return base
    if layout == "heads":
        return torch.full((sequences, kv_heads, capacity, 128), fill, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    wide = torch.full((capacity, sequences, 2 * kv_heads * 128 + 8), fill, dtype=torch.bfloat16, device="cuda")
    return wide[..., :kv_heads * 128].unflatten(-1, (kv_heads, 128)).transpose(0, 1)


WINDOW_CASES = [
    # lengths, capacity, rows, heads, kv_heads, window, sinks, layout
    ([1], 1, 1, 4, 4, 1, 0, "tokens"),                       # one token
    ([7], 40, 1, 8, 2, 3, 0, "tokens"),
    ([33, 64, 1, 0, 31], 64, 1, 8, 2, 16, 4, "tokens"),      # an empty sequence among others
    ([100, 3, 2], 128, 5, 28, 4, 10, 2, "heads"),            # sequences shorter than their rows
    ([257, 511], 600, 9, 32, 8, 100, 64, "wide"),
    ([1500], 1504, 1, 16, 8, 1024, 4, "tokens"),
    ([1500], 1500, 16, 32, 8, 4096, 0, "heads"),             # a window that reaches everything
    ([900, 901, 63], 901, 2, 32, 1, 128, 128, "tokens"),     # 32 query heads over one
    ([300], 300, 3, 5, 5, 1, 1, "tokens"),                   # a window of the own token and one sink
    ([300, 200], 320, 40, 12, 4, 33, 5, "wide"),             # many rows
    ([1000], 1000, 1000, 6, 3, 130, 3, "tokens"),            # a prompt
    ([2000], 2000, 333, 28, 4, 640, 70, "heads"),
    ([700, 90], 700, 300, 8, 8, 257, 0, "tokens"),           # prompts, one of them padded on the left
    ([8200], 8200, 1, 8, 8, 8000, 4, "tokens"),
    ([513], 513, 513, 4, 2, 1 << 40, 0, "tokens"),           # plain causal attention
    # Many-row kernel: clusters of eight, four, two blocks; odd last query tiles; queries that no box copies (groups of 7, 3)
    ([4100], 4100, 16, 32, 8, 4000, 4, "tokens"),
    ([4096], 4100, 64, 32, 8, 4096, 0, "heads"),
    ([2000, 1999], 2000, 100, 28, 4, 1900, 33, "tokens"),
    ([4000], 4001, 260, 12, 4, 3900, 64, "wide"),
    ([1300, 60, 0], 1300, 700, 16, 8, 1000, 5, "tokens"),
    ([3000], 3000, 129, 8, 8, 2900, 100, "tokens"),
    ([2000, 1500, 900, 20], 2000, 32, 32, 8, 2000, 0, "tokens"),
    ([2048 - 40 * i for i in range(24)], 2048, 32, 32, 8, 2048, 0, "tokens"),  # no cluster, both halves at one query tile
    ([500, 33], 500, 16, 64, 1, 300, 4, "tokens"),           # 64, 128 and 256 query heads over one
    ([2500], 2500, 7, 128, 1, 2400, 4, "heads"),
    ([700], 700, 5, 256, 1, 600, 1, "tokens"),
    ([40] * 300, 64, 1, 8, 2, 30, 2, "tokens"),              # many sequences
]


def window_inputs(torch, case, seed=1):
    lengths, capacity, rows, heads, kv_heads, window, sinks, layout = case
    sequences = len(lengths)
    q = normal(torch, seed, sequences * rows, heads, 128, scale=2.0)
    k, v = (cache_like(torch, layout, sequences, capacity, kv_heads, math.nan) for _ in range(2))
    visible = []
    for s, n in enumerate(lengths):
        see = window_visible(torch, n, rows, min(window, 1 << 30), sinks, capacity)
        visible.append(see)
        some = see.any(0)  # everything else stays NaN
        k[s, some] = normal(torch, seed + 10 + s, int(some.sum()), kv_heads, 128)
        v[s, some] = normal(torch, seed + 500 + s, int(some.sum()), kv_heads, 128)
    return q, k, v, visible


@pytest.mark.parametrize("case", WINDOW_CASES, ids=[str(i) for i in range(len(WINDOW_CASES))])
def test_attention_window(cuda, package, ctx, case):
    torch, ops = cuda, package.operators
    lengths, capacity, rows, heads, kv_heads, window, sinks, layout = case
    q, k, v, visible = window_inputs(torch, case)
    device_lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    wide = torch.full((q.shape[0] + 2, heads * 128 + 8), 7.0, dtype=torch.bfloat16, device="cuda")  # rows around stay
    out = wide[1:-1, :heads * 128].unflatten(-1, (heads, 128))
    ops.attention_window(ctx, q, k, v, out, window, sinks, lengths=device_lengths)
    again = torch.empty_like(q)
    ops.attention_window(ctx, q, k, v, again, window, sinks, lengths=device_lengths)
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    assert (wide[0] == 7).all() and (wide[-1] == 7).all() and (wide[:, heads * 128:] == 7).all()
    for s, n in enumerate(lengths):
        mine = slice(s * rows, (s + 1) * rows)
        want, size, _, _ = attention_reference(torch, q[mine], k[s], v[s], visible[s])
        expect_attention(torch, out[mine], want, size)
        if n < rows:
            assert (out[s * rows:s * rows + rows - n] == 0).all()
    if len(set(lengths)) == 1:
        same = torch.empty_like(q)
        ops.attention_window(ctx, q, k, v, same, window, sinks, length=lengths[0])
        assert torch.equal(same, out)


def test_attention_window_takes_lengths_outside_the_cache_as_empty(cuda, package, ctx):
    torch, ops = cuda, package.operators
    case = ([50, 50, 50], 50, 2, 8, 2, 20, 1, "tokens")
    q, k, v, _ = window_inputs(torch, case)
    out = torch.full_like(q, 7.0)
    ops.attention_window(ctx, q, k, v, out, 20, 1, lengths=torch.tensor([51, 50, -3], dtype=torch.int32, device="cuda"))
    assert (out[:2] == 0).all() and (out[4:] == 0).all() and (out[2:4] != 0).any()


def test_attention_window_extreme_scores(cuda, package, ctx):
    """Scores far apart, equal ones, and the lowest finite keys: the largest takes everything, without overflow."""
    torch, ops = cuda, package.operators
    for rows, n in ((1, 200), (150, 200)):
        q = normal(torch, 3, rows, 4, 128, scale=40.0)
        k, v = normal(torch, 4, 1, n, 2, 128, scale=40.0), normal(torch, 5, 1, n, 2, 128)
        k[0, 5] = torch.finfo(torch.bfloat16).min / 2 ** 20
        out = torch.empty_like(q)
        ops.attention_window(ctx, q, k, v, out, 150, 3, length=n)
        want, size, _, _ = attention_reference(torch, q, k[0], v[0], window_visible(torch, n, rows, 150, 3, n))
        expect_attention(torch, out, want, size)
        ops.attention_window(ctx, torch.zeros_like(q), k[:, :5], v[:, :5], out, 150, 3, length=5)
        assert (out[-1].double() - v[0, :5].double().mean(0).repeat_interleave(2, 0)).abs().max() <= 3 * HALF * v.abs().max()


def test_attention_window_nan_in_sight_stays_in_its_rows(cuda, package, ctx):
    torch, ops = cuda, package.operators
    q, k, v = normal(torch, 1, 3, 4, 128), normal(torch, 2, 3, 90, 4, 128), normal(torch, 3, 3, 90, 4, 128)
    k[1, 80, 2, 7] = math.nan
    out = torch.empty_like(q)
    ops.attention_window(ctx, q, k, v, out, 64, 0, length=90)
    wrong = out.isnan().all(-1)
    assert wrong[1, 2] and int(wrong.sum()) == 1 and int(out.isnan().sum()) == 128


@pytest.mark.parametrize("rows,n", [(3, 700), (300, 700)])
def test_attention_replaces_its_queries(cuda, package, ctx, rows, n):
    """The outputs may take the queries' place."""
    torch, ops = cuda, package.operators
    q, k, v = normal(torch, 1, 2 * rows, 12, 128), normal(torch, 2, 2, n, 4, 128), normal(torch, 3, 2, n, 4, 128)
    pk, pv = normal(torch, 4, 900, 4, 128), normal(torch, 5, 900, 4, 128)
    out = torch.empty_like(q)
    ops.attention_window(ctx, q, k, v, out, 200, 3, length=n)
    mine = q.clone()
    ops.attention_window(ctx, mine, k, v, mine, 200, 3, length=n)
    assert torch.equal(mine, out)
    scratch = torch.empty(ops.attention_shared_prefix_scratch_bytes(2 * rows, 12, 4, 900), dtype=torch.uint8, device="cuda")
    ops.attention_shared_prefix(ctx, q, pk, pv, k, v, out, scratch, length=n)
    mine = q.clone()
    ops.attention_shared_prefix(ctx, mine, pk, pv, k, v, mine, scratch, length=n)
    assert torch.equal(mine, out)


def test_attention_window_in_a_graph_follows_the_lengths(cuda, package):
    """Captured on a stream of its own, replayed for other lengths and queries, two graphs in turn."""
    torch, ops = cuda, package.operators
    case = ([200, 130], 300, 3, 16, 4, 90, 4, "tokens")
    lengths = torch.tensor([200, 130], dtype=torch.int32, device="cuda")
    q = normal(torch, 1, 6, 16, 128)
    k, v = normal(torch, 2, 2, 300, 4, 128), normal(torch, 3, 2, 300, 4, 128)
    out, prompt = torch.empty_like(q), normal(torch, 4, 2 * 260, 16, 128)
    prompt_out = torch.empty_like(prompt)
    stream = torch.cuda.Stream()
    context = ops.prepare_execution_context(stream.cuda_stream)
    with torch.cuda.stream(stream):
        ops.attention_window(context, q, k, v, out, 90, 4, lengths=lengths)
        ops.attention_window(context, prompt, k, v, prompt_out, 90, 4, lengths=lengths)
    stream.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0], stream=stream):
        ops.attention_window(context, q, k, v, out, 90, 4, lengths=lengths)
    with torch.cuda.graph(graphs[1], stream=stream):
        ops.attention_window(context, prompt, k, v, prompt_out, 90, 4, lengths=lengths)
    for n in ([200, 130], [7, 300], [0, 299]):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        q.copy_(normal(torch, sum(n), 6, 16, 128))
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for rows, result, queries in ((3, out, q), (260, prompt_out, prompt)):
            for s in range(2):
                mine = slice(s * rows, (s + 1) * rows)
                want, size, _, _ = attention_reference(torch, queries[mine], k[s], v[s], window_visible(torch, n[s], rows, 90, 4, 300))
                expect_attention(torch, result[mine], want, size)


def test_attention_window_beyond_32_bit_offsets(cuda, package, ctx):
    """The last sequence of a batch starts beyond 2^32 elements of the cache."""
    torch, ops = cuda, package.operators
    sequences, capacity, kv_heads = 5, 65536 * 2, 8
    k = torch.zeros((sequences * 8, capacity, kv_heads, 128), dtype=torch.bfloat16, device="cuda")[::8]
    assert k.stride(0) * 4 + 128 > 2 ** 32
    v = k.clone()
    for cache, seed in ((k, 1), (v, 2)):
        cache[-1, -300:] = normal(torch, seed, 300, kv_heads, 128)
        cache[-1, :4] = normal(torch, seed + 10, 4, kv_heads, 128)
    q = normal(torch, 3, sequences, 16, 128, scale=2.0)
    out = torch.empty_like(q)
    ops.attention_window(ctx, q, k, v, out, 290, 4, length=capacity)
    tokens = torch.cat((torch.arange(4), torch.arange(capacity - 290, capacity))).cuda()
    want, size, _, _ = attention_reference(torch, q[-1:], k[-1, tokens], v[-1, tokens], torch.ones(1, 294, dtype=torch.bool, device="cuda"))
    expect_attention(torch, out[-1:], want, size)


PREFIX_CASES = [
    # prefix, own lengths, capacity, rows, heads, kv_heads
    (1, [1], 1, 1, 2, 1),
    (63, [5, 9], 16, 1, 8, 2),
    (64, [1, 2, 3, 40, 0], 64, 1, 32, 8),                    # an empty one
    (65, [300, 30, 2], 300, 5, 28, 4),                       # one shorter than its rows
    (1000, [17], 20, 9, 32, 8),
    (2500, [100, 407, 222], 407, 5, 28, 4),
    (333, [20] * 24, 32, 1, 32, 8),                          # 96 stacked rows
    (4096, list(range(1, 65)), 64, 1, 32, 8),                # 256 stacked rows
    (700, [33, 50, 64], 64, 33, 12, 4),                      # 297 stacked rows, none a multiple of anything
    (5000, [70] * 7, 70, 16, 16, 8),
    (130, [256] * 3, 256, 250, 4, 4),                        # prompts behind a prefix
    (0, [40, 41], 41, 2, 8, 2),                              # no prefix
    (30011, [50] * 8, 64, 9, 16, 8),                         # 144 stacked rows: a pair of query tiles
    (9001, [33, 9, 2], 33, 40, 28, 4),                       # 840: three pairs and an odd tile
    (8192, [12] * 16, 16, 1, 32, 8),                         # 64
]


@pytest.mark.parametrize("case", PREFIX_CASES, ids=[str(i) for i in range(len(PREFIX_CASES))])
def test_attention_shared_prefix(cuda, package, ctx, case):
    torch, ops = cuda, package.operators
    prefix, lengths, capacity, rows, heads, kv_heads = case
    sequences = len(lengths)
    q = normal(torch, 1, sequences * rows, heads, 128, scale=2.0)
    pk = normal(torch, 2, prefix, kv_heads, 2, 128)[..., 0, :] if prefix % 2 else normal(torch, 2, kv_heads, prefix, 128).transpose(0, 1)
    pv = normal(torch, 3, prefix, kv_heads, 128)
    k = torch.full((sequences, capacity, kv_heads, 128), math.nan, dtype=torch.bfloat16, device="cuda")
    v = torch.full_like(k, math.inf)
    for s, n in enumerate(lengths):
        k[s, :n], v[s, :n] = normal(torch, 10 + s, n, kv_heads, 128), normal(torch, 300 + s, n, kv_heads, 128)
    device_lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    size = ops.attention_shared_prefix_scratch_bytes(sequences * rows, heads, kv_heads, prefix)
    results = []
    for fill in (0xff, 0x7f):  # whatever the scratch holds, all of it or none behind it
        scratch = torch.full((size + 64,), fill, dtype=torch.uint8, device="cuda")
        out = torch.full_like(q, 7.0)
        ops.attention_shared_prefix(ctx, q, pk, pv, k, v, out, scratch[:size] if size else None, lengths=device_lengths)
        torch.cuda.synchronize()
        assert (scratch[size:] == fill).all()
        results.append(out)
    assert torch.equal(*results)
    for s, n in enumerate(lengths):
        mine = slice(s * rows, (s + 1) * rows)
        place = torch.arange(n - rows, n, device="cuda")[:, None]
        own = torch.arange(capacity, device="cuda")[None] <= place
        visible = torch.cat(((place >= 0).expand(-1, prefix), own), 1)
        want, allowance, _, _ = attention_reference(torch, q[mine], torch.cat((pk, k[s])), torch.cat((pv, v[s])), visible)
        expect_attention(torch, results[0][mine], want, allowance)
        if n < rows:
            assert (results[0][s * rows:s * rows + rows - n] == 0).all()


def test_attention_shared_prefix_two_graphs_on_two_streams(cuda, package):
    """Graphs of their own scratch replay side by side."""
    torch, ops = cuda, package.operators
    q = normal(torch, 1, 20, 32, 128, scale=2.0)
    pk, pv = normal(torch, 2, 3000, 8, 128), normal(torch, 3, 3000, 8, 128)
    k, v = normal(torch, 4, 20, 64, 8, 128), normal(torch, 5, 20, 64, 8, 128)
    size = ops.attention_shared_prefix_scratch_bytes(20, 32, 8, 3000)
    sides = []
    for _ in range(2):
        stream = torch.cuda.Stream()
        context = ops.prepare_execution_context(stream.cuda_stream)
        scratch, out = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty_like(q)
        torch.cuda.synchronize()
        ops.attention_shared_prefix(context, q, pk, pv, k, v, out, scratch, length=50)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.attention_shared_prefix(context, q, pk, pv, k, v, out, scratch, length=50)
        sides.append((stream, graph, out, out.clone(), scratch))
    for _ in range(5):
        for stream, graph, out, _, _ in sides:
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, first, _ in sides:
        assert torch.equal(out, first)
    assert torch.equal(sides[0][2], sides[1][2])


ACCUMULATE_CASES = [
    # lengths, capacity, rows, heads, kv_heads, old scores
    ([1], 1, 1, 2, 1, True),
    ([64, 65, 0, 3], 70, 1, 32, 8, True),
    ([300, 2, 129], 300, 5, 28, 4, True),            # 35 stacked rows; one sequence shorter than its rows
    ([2000], 2001, 1, 16, 8, False),
    ([900, 45], 901, 32, 16, 4, True),               # an observation window of 128 stacked rows
    ([6000], 6000, 2, 32, 8, False),
    ([700, 129, 100], 701, 130, 12, 4, True),        # 390 stacked rows: two passes; padded on the left
    ([300], 300, 100, 16, 4, False),                 # 400 without old scores
    ([128, 0], 128, 16, 28, 4, True),                # 112
]


@pytest.mark.parametrize("case", ACCUMULATE_CASES, ids=[str(i) for i in range(len(ACCUMULATE_CASES))])
def test_attention_accumulate(cuda, package, ctx, case):
    torch, ops = cuda, package.operators
    lengths, capacity, rows, heads, kv_heads, old = case
    sequences = len(lengths)
    q = normal(torch, 1, sequences * rows, heads, 128, scale=2.0)
    k = torch.full((sequences, capacity, kv_heads, 128), math.nan, dtype=torch.bfloat16, device="cuda")
    v = torch.full_like(k, math.inf)
    for s, n in enumerate(lengths):
        k[s, :n], v[s, :n] = normal(torch, 10 + s, n, kv_heads, 128), normal(torch, 300 + s, n, kv_heads, 128)
    device_lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    before = torch.rand((sequences, kv_heads, capacity + 3), device="cuda")[..., :capacity] if old else None
    size = ops.attention_accumulate_scratch_bytes(sequences, rows, heads, kv_heads, capacity)
    scratch = torch.full((size + 64,), 0xff, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 7.0)
    after = torch.full((sequences, kv_heads, capacity), 9.0, device="cuda")
    ops.attention_accumulate(ctx, q, k, v, out, before, after, scratch[:size], lengths=device_lengths)
    torch.cuda.synchronize()
    assert (scratch[size:] == 0xff).all()
    # The same in place gives the same bits.
    held = before.clone() if old else torch.zeros_like(after)
    ops.attention_accumulate(ctx, q, k, v, torch.empty_like(out), held, held, scratch[:size], lengths=device_lengths)
    for s, n in enumerate(lengths):
        mine = slice(s * rows, (s + 1) * rows)
        visible = window_visible(torch, n, rows, 1 << 30, 0, capacity)
        want, allowance, weights, slack = attention_reference(torch, q[mine], k[s], v[s], visible)
        expect_attention(torch, out[mine], want, allowance)
        total = weights + (before[s].double() if old else 0.0)
        assert ((after[s, :, :n].double() - total[:, :n]).abs() <= slack[:, :n] + 2.0 ** -22 * total[:, :n] + 1e-30).all()
        assert (after[s, :, n:] == 9).all()
        assert torch.equal(held[s, :, :n], after[s, :, :n])


def evict_reference(torch, scores, n, budget, sinks, recent):
    if n <= budget:
        return list(range(n))
    middle = sorted(range(sinks, n - recent), key=lambda t: (-(scores[t] if scores[t] == scores[t] else -math.inf), scores[t] != scores[t], t))
    return list(range(sinks)) + sorted(middle[:budget - sinks - recent]) + list(range(n - recent, n))


EVICT_CASES = [
    # lengths, capacity, kv_heads, budget, sinks, recent, kind of scores
    ([1], 1, 1, 1, 0, 0, "random"),
    ([40, 33, 0, 32, 31], 40, 2, 32, 4, 8, "random"),
    ([500], 500, 8, 100, 4, 96, "random"),                   # no place for any other
    ([500, 499], 512, 3, 100, 0, 100, "ties"),
    ([1000, 700], 1000, 2, 333, 5, 17, "ties"),
    ([1000, 999], 1000, 2, 64, 0, 0, "equal"),
    ([777], 800, 4, 50, 1, 2, "odd"),                        # infinities, NaN, zeros of both signs, negatives
    ([8191], 8191, 8, 1024, 4, 256, "random"),
    ([50000], 50001, 2, 20000, 4, 100, "random"),            # more keys than a block keeps, more rows than a part holds
    ([2300, 2048, 1900], 2304, 8, 2048, 4, 512, "random"),
]


@pytest.mark.parametrize("case", EVICT_CASES, ids=[str(i) for i in range(len(EVICT_CASES))])
def test_evict_kv(cuda, package, ctx, case):
    torch, ops = cuda, package.operators
    lengths, capacity, kv_heads, budget, sinks, recent, kind = case
    sequences = len(lengths)
    k = normal(torch, 1, sequences, capacity, kv_heads, 128)
    v = normal(torch, 2, sequences, kv_heads, capacity, 128).transpose(1, 2)
    scores = torch.rand((sequences, kv_heads, capacity), generator=torch.Generator("cuda").manual_seed(3), device="cuda") ** 8
    if kind == "ties":
        scores = (scores * 4).floor()
    if kind == "equal":
        scores.fill_(0.25)
    if kind == "odd":
        choice = torch.randint(0, 8, scores.shape, generator=torch.Generator("cuda").manual_seed(4), device="cuda")
        for i, value in enumerate((0.0, -0.0, -1.0, math.inf, -math.inf, math.nan)):
            scores[choice == i] = value
    k_out = torch.full((sequences, budget + 2, kv_heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    v_out = torch.full((sequences, kv_heads, budget, 128), 7.0, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    scores_out = torch.full((sequences, kv_heads, budget), 9.0, device="cuda")
    kept = torch.full((sequences, kv_heads, budget), 99, dtype=torch.int32, device="cuda")
    new = torch.full((sequences,), 99, dtype=torch.int32, device="cuda")
    ops.evict_kv(ctx, k, v, scores, k_out[:, :budget], v_out, scores_out, kept, new, sinks, recent,
                 lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert new.tolist() == [min(n, budget) for n in lengths]
    assert (k_out[:, budget:] == 7).all()
    host = scores.cpu().tolist()
    for s, n in enumerate(lengths):
        for h in range(kv_heads):
            want = evict_reference(torch, host[s][h], n, budget, sinks, recent)
            assert kept[s, h].tolist() == want + [-1] * (budget - len(want))
            index = torch.tensor(want, dtype=torch.long, device="cuda")
            assert torch.equal(k_out[s, :len(want), h], k[s, index, h]) and torch.equal(v_out[s, :len(want), h], v[s, index, h])
            assert torch.equal(scores_out[s, h, :len(want)].view(torch.int32), scores[s, h, index].view(torch.int32))
        assert (k_out[s, min(n, budget):] == 7).all() and (v_out[s, min(n, budget):] == 7).all()
        assert (scores_out[s, :, min(n, budget):] == 9).all()


ROPE_CASES = [
    # rows, heads, kv_heads, width, rotary, norm, interleaved
    (1, 1, 1, 16, 16, True, False),
    (3, 2, 1, 48, 32, True, True),
    (5, 28, 4, 128, 128, True, False),
    (64, 32, 8, 128, 64, False, True),
    (7, 16, 8, 80, 80, True, False),
    (700, 8, 2, 256, 128, True, True),
    (601, 6, 3, 64, 64, False, False),
    (2, 3, 5, 512, 496, True, False),
]


@pytest.mark.parametrize("case", ROPE_CASES, ids=[str(i) for i in range(len(ROPE_CASES))])
def test_qk_norm_rope(cuda, package, ctx, case):
    torch, ops = cuda, package.operators
    rows, heads, kv_heads, width, rotary, norm, interleaved = case
    fused = normal(torch, 1, rows, heads + 2 * kv_heads, width, scale=3.0)
    q, k = fused[:, :heads], fused[:, heads:heads + kv_heads]
    q[0, 0] = 0.0  # a head of zeros stays one
    table = torch.from_numpy(ops.build_rope_table_scaled(40000, rotary, 1e6, "yarn", 4.0, 8192.0)).cuda()
    positions = torch.randint(0, 40000, (rows,), generator=torch.Generator("cuda").manual_seed(2), device="cuda", dtype=torch.int32)
    if rows > 4:
        positions[1], positions[2], positions[3] = 39999, 40000, -1  # the last row of the table, and two that it lacks
    weights = [normal(torch, 5 + i, width) if norm else None for i in range(2)]
    q_out = torch.full((rows, heads * width + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    k_out = torch.empty((rows, kv_heads, width), dtype=torch.bfloat16, device="cuda")
    out = q_out[:, :heads * width].unflatten(-1, (heads, width))
    go = dict(q_weight=weights[0], k_weight=weights[1], epsilon=1e-5, interleaved=interleaved)
    ops.qk_norm_rope(ctx, q, k, table, out, k_out, positions=positions, **go)
    torch.cuda.synchronize()
    assert (q_out[:, heads * width:] == 7).all()
    known = (positions >= 0) & (positions < 40000)
    turn = table.double()[positions.long().clamp(0, 39999)]
    for x, weight, got in ((q, weights[0], out), (k, weights[1], k_out)):
        y = x.double()
        if weight is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-5) * weight.double()
        want = y.clone()
        for i in range(rotary // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
            sine, cosine = turn[:, None, 2 * i], turn[:, None, 2 * i + 1]
            want[..., a] = y[..., a] * cosine - y[..., b] * sine
            want[..., b] = y[..., a] * sine + y[..., b] * cosine
        want[~known] = 0.0
        # The table's vectors are up to 1.14 long.
        assert ((got.double() - want).abs() <= HALF * want.abs() + 2.0 ** -20 * 1.5 * y.abs().amax(-1, keepdim=True)).all()
    # Consecutive positions behind an offset, and in place: the same bits.
    mine = torch.arange(100, 100 + rows, dtype=torch.int32, device="cuda")
    ops.qk_norm_rope(ctx, q, k, table, out, k_out, positions=mine, **go)
    v_before = fused[:, heads + kv_heads:].clone()
    ops.qk_norm_rope(ctx, q, k, table, q, k, offset=100, **go)
    assert torch.equal(q, out) and torch.equal(k, k_out) and torch.equal(fused[:, heads + kv_heads:], v_before)


def test_the_operators_together(cuda, package, ctx):
    """A prompt and steps as a server runs them: rotation into the cache, attention with accumulated weights, eviction, and
    windowed and shared-prefix attention over what stayed."""
    torch, ops = cuda, package.operators
    heads, kv_heads, capacity, budget, prompt = 16, 4, 400, 128, 300
    table = torch.from_numpy(ops.build_rope_table_scaled(1000, 128, 1e4, "linear", 2.0)).cuda()
    k, v = (torch.full((1, capacity, kv_heads, 128), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    scores = torch.zeros((1, kv_heads, capacity), device="cuda")
    weight = 1 + normal(torch, 9, 128, scale=0.1)
    scratch = torch.empty(ops.attention_accumulate_scratch_bytes(1, 16, heads, kv_heads, capacity), dtype=torch.uint8, device="cuda")

    def step(seed, first, rows):
        fused = normal(torch, seed, rows, heads + 2 * kv_heads, 128)
        q, new_k, new_v = fused.split((heads, kv_heads, kv_heads), 1)
        ops.qk_norm_rope(ctx, q, new_k, table, q, k[0, first:first + rows], offset=first, q_weight=weight, k_weight=weight)
        v[0, first:first + rows] = new_v
        return q

    q = step(1, 0, prompt)
    out = torch.empty_like(q)
    ops.attention_window(ctx, q, k, v, out, 1 << 20, length=prompt)
    want, size, _, _ = attention_reference(torch, q, k[0], v[0], window_visible(torch, prompt, prompt, 1 << 20, 0, capacity))
    expect_attention(torch, out, want, size)
    last = q[-16:].contiguous()
    ops.attention_accumulate(ctx, last, k, v, torch.empty_like(last), scores, scores, scratch, length=prompt)
    assert abs(float(scores.sum()) - 16 * heads) < 1e-3
    k2, v2 = (torch.full((1, budget, kv_heads, 128), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kept = torch.empty((1, kv_heads, budget), dtype=torch.int32, device="cuda")
    scores2, new = torch.empty((1, kv_heads, budget), device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    ops.evict_kv(ctx, k, v, scores, k2, v2, scores2, kept, new, 4, 32, length=prompt)
    host = scores.cpu().tolist()
    for h in range(kv_heads):
        assert kept[0, h].tolist() == evict_reference(torch, host[0][h], prompt, budget, 4, 32)
    one = normal(torch, 7, 1, heads, 128)
    got = torch.empty_like(one)
    ops.attention_window(ctx, one, k2, v2, got, 64, 4, lengths=new)
    want, size, _, _ = attention_reference(torch, one, k2[0], v2[0], window_visible(torch, budget, 1, 64, 4, budget))
    expect_attention(torch, got, want, size)
    shared = torch.empty(ops.attention_shared_prefix_scratch_bytes(2, heads, kv_heads, budget), dtype=torch.uint8, device="cuda")
    two, own = normal(torch, 8, 2, heads, 128), k[0, :40].unflatten(0, (2, 20))
    own_v, got = v[0, :40].unflatten(0, (2, 20)), torch.empty_like(two)
    ops.attention_shared_prefix(ctx, two, k2[0], v2[0], own, own_v, got, shared, length=20)
    for s in range(2):
        want, size, _, _ = attention_reference(torch, two[s:s + 1], torch.cat((k2[0], own[s])), torch.cat((v2[0], own_v[s])),
                                               torch.ones(1, budget + 20, dtype=torch.bool, device="cuda"))
        expect_attention(torch, got[s:s + 1], want, size)


def test_outputs_follow_the_stream_of_the_context(cuda, package):
    """Work queued on a side stream is in order there, whatever the current stream does."""
    torch, ops = cuda, package.operators
    stream = torch.cuda.Stream()
    context = ops.prepare_execution_context(stream.cuda_stream)
    q, k, v = normal(torch, 1, 2, 8, 128), normal(torch, 2, 2, 500, 2, 128), normal(torch, 3, 2, 500, 2, 128)
    scores = torch.rand((2, 2, 500), device="cuda")
    k2, v2 = torch.zeros((2, 100, 2, 128), dtype=torch.bfloat16, device="cuda"), torch.zeros((2, 100, 2, 128), dtype=torch.bfloat16, device="cuda")
    kept, scores2 = torch.empty((2, 2, 100), dtype=torch.int32, device="cuda"), torch.empty((2, 2, 100), device="cuda")
    new, out = torch.empty(2, dtype=torch.int32, device="cuda"), torch.empty_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        ops.evict_kv(context, k, v, scores, k2, v2, scores2, kept, new, 2, 10, length=500)
        ops.attention_window(context, q, k2, v2, out, 50, 2, lengths=new)
    stream.synchronize()
    for s in range(2):
        want, size, _, _ = attention_reference(torch, q[s:s + 1], k2[s], v2[s], window_visible(torch, 100, 1, 50, 2, 100))
        expect_attention(torch, out[s:s + 1], want, size)


def test_the_context_has_to_be_of_the_current_device(cuda, package):
    torch, ops, abi = cuda, package.operators, package.abi
    other = abi.Context()
    other.device = 1
    q, k = normal(torch, 1, 1, 2, 128), normal(torch, 2, 1, 4, 2, 128)
    with pytest.raises(ValueError):
        ops.attention_window(other, q, k, k, torch.empty_like(q), 4, length=4)
    import ctypes
    with pytest.raises(ValueError, match="another CUDA device"):
        abi.check(abi.load_library().ei_attention_window_bf16(ctypes.byref(other), abi.view3(q), abi.view4(k), abi.view4(k), abi.view3(q), None,
                                                              4, 4, 0))
