"""GPU checks of the operators for long contexts at the edges of what their documentation allows. Tolerances are those of
test_context_gpu.py."""
import math

import pytest

from test_context_gpu import attention_reference, ctx, expect_attention, normal, window_visible  # noqa: F401

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

# rows, tokens, sequences, heads, kv_heads: few rows in clusters, in one block, in two units a head, eight warps; the many-row
# kernel with one query tile, with two and loaded queries, without a cluster, in clusters.
GIVE_UP = [(1, 3000, 2, 8, 8), (1, 90, 40, 32, 8), (5, 700, 2, 28, 4), (2, 9000, 2, 8, 2), (16, 4000, 2, 32, 8), (300, 3000, 2, 28, 4),
           (700, 2000, 3, 32, 8), (130, 6000, 2, 8, 4)]


@pytest.mark.parametrize("case", GIVE_UP, ids=[str(i) for i in range(len(GIVE_UP))])
def test_window_waits_that_run_out(cuda, package, ctx, case):
    torch, ops = cuda, package.operators
    rows, tokens, sequences, heads, kv_heads = case
    q = normal(torch, 1, sequences * rows, heads, 128)
    k, v = normal(torch, 2, sequences, tokens, kv_heads, 128), normal(torch, 3, sequences, tokens, kv_heads, 128)
    want, out = torch.empty_like(q), torch.empty_like(q)
    ops.attention_window(ctx, q, k, v, want, 1 << 20, 0, length=tokens)
    for _ in range(2):
        ops.inject_wait_timeout(2000)
        ops.attention_window(ctx, q, k, v, out, 1 << 20, 0, length=tokens)
        torch.cuda.synchronize()
        assert out[:rows].isnan().all() and torch.equal(out[rows:], want[rows:])
        ops.attention_window(ctx, q, k, v, out, 1 << 20, 0, length=tokens)
        assert torch.equal(out, want)


@pytest.mark.parametrize("rows,prefix,sequences,heads,kv_heads", [(1, 900, 2, 8, 2), (1, 8192, 64, 32, 8), (40, 9001, 3, 28, 4)])
def test_prefix_waits_that_run_out(cuda, package, ctx, rows, prefix, sequences, heads, kv_heads):
    torch, ops = cuda, package.operators
    q = normal(torch, 1, sequences * rows, heads, 128)
    pk, pv = normal(torch, 2, prefix, kv_heads, 128), normal(torch, 3, prefix, kv_heads, 128)
    k, v = normal(torch, 4, sequences, 50, kv_heads, 128), normal(torch, 5, sequences, 50, kv_heads, 128)
    scratch = torch.empty(ops.attention_shared_prefix_scratch_bytes(sequences * rows, heads, kv_heads, prefix), dtype=torch.uint8, device="cuda")
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
