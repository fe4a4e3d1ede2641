"""Host-side mirror of edge-infer's direct-operator API (namespace op::cuda) over the C ABI.

Same names, argument meaning and error behaviour as
operators/include/operators/cuda/execution.hpp:28-157 and direct.hpp:23-47 of the reference,
for BF16 tensors. Tensors are torch CUDA tensors used purely as device buffers; every call
launches on the context's stream and allocates nothing (scratch is passed in).
"""
from __future__ import annotations

import ctypes as C

from . import abi


def _lib():
    return abi.load_library()


def prepare_execution_context(stream_ptr: int = 0) -> abi.Context:
    ctx = abi.Context()
    abi.check(_lib().ei_prepare_execution_context(C.c_void_p(stream_ptr), C.byref(ctx)))
    return ctx


def prepare_dense(weight, bias=None) -> abi.DenseWeight:
    """weight: logical [in, out] view (either row-major or the transpose of an [out, in] matrix)."""
    out = abi.DenseWeight()
    abi.check(_lib().ei_prepare_dense_bf16(abi.view2(weight), abi.view1(bias), C.byref(out)))
    return out


def prepare_awq(qweight, scales, zeros, group_size: int, input_features: int, bias=None) -> abi.AwqWeight:
    out = abi.AwqWeight()
    abi.check(_lib().ei_prepare_awq_bf16(abi.view2(qweight), abi.view2(scales), abi.view2(zeros), group_size,
                                         input_features, abi.view1(bias), C.byref(out)))
    return out


def linear_scratch_bytes(rows: int, input_features: int, output_features: int) -> int:
    return _lib().ei_linear_scratch_bytes(rows, input_features, output_features)


def _scratch(scratch):
    if scratch is None:
        return None, 0
    return C.c_void_p(scratch.data_ptr()), scratch.numel() * scratch.element_size()


def linear(ctx, input, weight: abi.DenseWeight, output, scratch=None) -> None:
    ptr, size = _scratch(scratch)
    abi.check(_lib().ei_linear_bf16(C.byref(ctx), abi.view2(input), C.byref(weight), abi.view2(output), ptr, size))


def awq_linear(ctx, input, weight: abi.AwqWeight, output, scratch=None) -> None:
    ptr, size = _scratch(scratch)
    abi.check(_lib().ei_awq_linear_bf16(C.byref(ctx), abi.view2(input), C.byref(weight), abi.view2(output), ptr, size))


def awq_gate_up_silu(ctx, input, weight: abi.AwqWeight, output) -> None:
    """Fused SwiGLU projection over a weight whose rows are [gate; up]: output = silu(gate) * up, staged as BF16."""
    abi.check(_lib().ei_awq_gate_up_silu_bf16(C.byref(ctx), abi.view2(input), C.byref(weight), abi.view2(output)))


def add(ctx, a, b, output) -> None:
    abi.check(_lib().ei_add_bf16(C.byref(ctx), abi.array(a), abi.array(b), abi.array(output)))


def silu_multiply(ctx, gate, up, output) -> None:
    abi.check(_lib().ei_silu_multiply_bf16(C.byref(ctx), abi.array(gate), abi.array(up), abi.array(output)))


def rms_norm(ctx, input, weight, output, rows: int, features: int, epsilon: float) -> None:
    abi.check(_lib().ei_rms_norm_bf16(C.byref(ctx), abi.array(input), abi.array(weight), abi.array(output), rows,
                                      features, epsilon))


def gather(ctx, ids, table, output) -> None:
    abi.check(_lib().ei_gather_bf16(C.byref(ctx), abi.view1(ids), abi.view2(table), abi.view2(output)))


def rope_precomputed(ctx, input, cache, offset: int = 0, offsets=None, pingpong=None) -> None:
    abi.check(_lib().ei_rope_precomputed_bf16(
        C.byref(ctx), abi.view3(input), abi.view2(cache), offset,
        C.c_void_p(offsets.data_ptr()) if offsets is not None else None,
        C.c_void_p(pingpong.data_ptr()) if pingpong is not None else None))


def build_rope_table(max_positions: int, head_dim: int, theta: float):
    import numpy as np
    table = np.empty((max_positions, head_dim), dtype=np.float32)
    abi.check(_lib().ei_build_rope_table(table.ctypes.data_as(C.c_void_p), max_positions, head_dim, theta))
    return table


def store_kv(ctx, source, capacity, offset: int, device_offset=None) -> None:
    abi.check(_lib().ei_store_kv_bf16(C.byref(ctx), abi.view2(source), abi.view2(capacity), offset,
                                      C.c_void_p(device_offset.data_ptr()) if device_offset is not None else None))


def attention_scratch_bytes(q_rows: int, query_heads: int, head_dim: int, kv_length: int) -> int:
    return _lib().ei_attention_scratch_bytes(q_rows, query_heads, head_dim, kv_length)


def attention_prefill(ctx, q, k, v, output, offset: int, scratch) -> None:
    ptr, size = _scratch(scratch)
    abi.check(_lib().ei_attention_prefill_bf16(C.byref(ctx), abi.view3(q), abi.view3(k), abi.view3(v),
                                               abi.view3(output), offset, ptr, size))


STATIC_ATTENTION_SCRATCH_BYTES = 10 * 1024 * 1024


def attention_prefill_static(ctx, q, k, v, output, offset: int) -> None:
    """attention_prefill with the split partials in the library's built-in array: allocates nothing, takes no
    scratch; shapes needing more than STATIC_ATTENTION_SCRATCH_BYTES raise ValueError. Calls on one device
    share the array and must not overlap."""
    abi.check(_lib().ei_attention_prefill_static_bf16(C.byref(ctx), abi.view3(q), abi.view3(k), abi.view3(v),
                                                      abi.view3(output), offset))


def attention_verify(ctx, q, k_capacity, v_capacity, output, device_offset, scratch) -> None:
    ptr, size = _scratch(scratch)
    abi.check(_lib().ei_attention_verify_bf16(C.byref(ctx), abi.view3(q), abi.view3(k_capacity),
                                              abi.view3(v_capacity), abi.view3(output),
                                              C.c_void_p(device_offset.data_ptr()), ptr, size))


# ---- long contexts: rotation with norms, window, shared prefix, accumulated weights, eviction ------------------------
ROPE_SCALINGS = {"plain": 0, "linear": 1, "yarn": 2, "bands": 3}


_native_calls = None


def _native():
    """The calls that take tensors apart natively (csrc/python_calls.cpp); fails loudly if they are not built."""
    global _native_calls
    if _native_calls is None:
        import torch
        _lib()
        try:
            from . import _calls
        except ImportError as error:
            raise ImportError(f"{abi.HERE / '_calls'} is not built for this interpreter. Run `python edge-infer_b200/build.py` where "
                              "Python's headers are installed.") from error
        _calls.configure(torch.bfloat16, torch.float32, torch.int32)
        _native_calls = _calls
    return _native_calls


def build_rope_table_scaled(max_positions: int, rotary_dim: int, theta: float, kind: str = "plain", factor: float = 1.0,
                            original_positions: float = 0.0, fast: float = 32.0, slow: float = 1.0, length: float = 0.0):
    """Rotation table for contexts longer than a model was trained on; kinds: plain, linear, yarn, bands."""
    import numpy as np
    if kind not in ROPE_SCALINGS:
        raise ValueError(f"unknown RoPE scaling {kind!r}")
    table = np.empty((max_positions, rotary_dim), dtype=np.float32)
    scaling = abi.RopeScaling(ROPE_SCALINGS[kind], factor, original_positions, fast, slow, length)
    abi.check(_lib().ei_build_rope_table_scaled(table.ctypes.data_as(C.c_void_p), max_positions, rotary_dim, theta,
                                                C.byref(scaling)))
    return table


def qk_norm_rope(ctx, q, k, table, q_out, k_out, *, positions=None, offset: int = 0, q_weight=None, k_weight=None,
                 epsilon: float = 1e-6, interleaved: bool = False) -> None:
    """Norm of every query and key head (where a weight is given) and rotation of its first table.shape[1] values, in one
    pass with one rounding. positions: int32 [rows] on the device, else offset + row. Outputs may be the inputs."""
    abi.check(_native().qk_norm_rope(C.addressof(ctx), q, k, table, q_out, k_out, positions, offset, q_weight, k_weight, epsilon,
                                     interleaved))


def attention_window(ctx, q, k, v, output, window: int, sinks: int = 0, *, lengths=None, length: int = 0) -> None:
    """Causal attention of [sequences * rows, heads, 128] queries over caches [sequences, capacity, kv_heads, 128]: a row at
    position p sees the tokens t <= p with t > p - window or t < sinks. lengths: int32 [sequences] on the device, the rows'
    own tokens included, else `length` for all."""
    abi.check(_native().attention_window(C.addressof(ctx), q, k, v, output, window, sinks, lengths, length))


def expired_waits(ctx) -> int:
    """How many bounded waits of the operators for long contexts have run out on the context's device so far, behind all that
    its stream holds. While the count stays, nothing gave up; rows that did came out as NaN."""
    count = C.c_uint64()
    abi.check(_lib().ei_context_expired_waits(C.byref(ctx), C.byref(count)))
    return count.value


def inject_wait_timeout(polls: int) -> None:
    """Test hook: a copy of this thread's next attention for long contexts does not arrive within `polls` polls."""
    abi.check(_lib().ei_context_inject_wait_timeout(polls))


def attention_shared_prefix_scratch_bytes(q_rows: int, query_heads: int, kv_heads: int, prefix_length: int) -> int:
    return _lib().ei_attention_shared_prefix_scratch_bytes(q_rows, query_heads, kv_heads, prefix_length)


def attention_shared_prefix(ctx, q, prefix_k, prefix_v, k, v, output, scratch, *, lengths=None, length: int = 0) -> None:
    """Causal attention of sequences that share their first tokens, prefix_k / prefix_v [prefix, kv_heads, 128], read once for
    all of them; lengths and positions count each sequence's own tokens in k / v."""
    abi.check(_native().attention_shared_prefix(C.addressof(ctx), q, prefix_k, prefix_v, k, v, output, scratch, lengths, length))


def attention_accumulate_scratch_bytes(sequences: int, rows: int, query_heads: int, kv_heads: int, capacity: int) -> int:
    return _lib().ei_attention_accumulate_scratch_bytes(sequences, rows, query_heads, kv_heads, capacity)


def attention_accumulate(ctx, q, k, v, output, scores, scores_out, scratch, *, lengths=None, length: int = 0) -> None:
    """Causal attention that also adds every token's softmax weights, over rows and a KV head's query heads, to scores
    (FP32 [sequences, kv_heads, capacity]; None counts as zeros) and leaves them in scores_out (which may be scores)."""
    abi.check(_native().attention_accumulate(C.addressof(ctx), q, k, v, output, scores, scores_out, scratch, lengths, length))


def evict_kv(ctx, k, v, scores, k_out, v_out, scores_out, kept, lengths_out, sinks: int = 0, recent: int = 0, *, lengths=None,
             length: int = 0) -> None:
    """Cuts caches to the k_out.shape[1] tokens that are first, latest or heaviest, each KV head its own, in order of
    position; kept (int32) receives their positions, -1 behind them, lengths_out (int32) the new lengths."""
    abi.check(_native().evict_kv(C.addressof(ctx), k, v, scores, k_out, v_out, scores_out, kept, lengths_out, sinks, recent, lengths,
                                 length))


def sample_scratch_bytes(rows: int, vocabulary: int) -> int:
    return _lib().ei_sample_scratch_bytes(rows, vocabulary)


def sample_greedy(ctx, logits, tokens, scratch) -> None:
    """op::cuda::sample with top_k == 1: tokens[row] = argmax of logits[row] (NaN as -inf, lowest index on ties)."""
    ptr, size = _scratch(scratch)
    abi.check(_lib().ei_sample_greedy_bf16(C.byref(ctx), abi.view2(logits), abi.view1(tokens), ptr, size))


def verify_accept(ctx, inputs, targets, rows: int, context_length, pending, result) -> None:
    abi.check(_lib().ei_verify_accept(C.byref(ctx), C.c_void_p(inputs.data_ptr()), C.c_void_p(targets.data_ptr()),
                                      rows, C.c_void_p(context_length.data_ptr()), C.c_void_p(pending.data_ptr()),
                                      C.c_void_p(result.data_ptr())))
