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
