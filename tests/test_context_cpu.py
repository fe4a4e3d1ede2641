"""CPU checks of the operators for long contexts: scaled rotation tables against their formulas, how the few-row attention is
cut, and refusals, which come before any CUDA call."""
import ctypes as C
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]


def formula(positions, rotary, theta, kind, factor, original, fast, slow, length):
    """Sines and cosines in 64 bits, pair by pair."""
    f = theta ** (-2.0 * np.arange(rotary // 2) / rotary)
    if kind == "linear":
        f = f / factor
    if kind == "bands":
        turns = original * f / (2 * math.pi)
        keep = np.clip((turns - slow) / (fast - slow), 0, 1)
        f = f * keep + f / factor * (1 - keep)
    if kind == "yarn":
        def pair(turns):
            return rotary * math.log(original / (2 * math.pi * turns)) / (2 * math.log(theta))
        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rotary - 1)
        ramp = np.clip((np.arange(rotary // 2) - low) / max(high - low, 0.001), 0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        if length == 0:
            length = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    angle = np.arange(positions)[:, None] * f
    return np.stack((np.sin(angle), np.cos(angle)), -1).reshape(positions, rotary) * (length or 1.0)


@pytest.mark.parametrize("kind", ["plain", "linear", "yarn", "bands"])
@pytest.mark.parametrize("rotary,theta,length", [(128, 1e6, 0.0), (64, 1e4, 0.0), (16, 5e5, 1.25)])
def test_scaled_rope_tables(package, kind, rotary, theta, length):
    table = package.operators.build_rope_table_scaled(3001, rotary, theta, kind, 8.0, 4096.0, 32.0, 1.0, length)
    want = formula(3001, rotary, theta, kind, 8.0, 4096.0, 32.0, 1.0, length)
    # Angles up to 3000 with a few roundings of 2^-53 each, then one rounding to FP32.
    assert np.abs(table - want).max() <= 2.0 ** -24 * 1.5 + 3000 * 8 * 2.0 ** -53


def test_plain_scaled_table_is_the_plain_table_within_its_angles(package):
    """The reference's table takes its angles in FP32: position 63 times a frequency is off by up to 63 * 2^-23."""
    ours = package.operators.build_rope_table_scaled(64, 128, 1e6)
    plain = package.operators.build_rope_table(64, 128, 1e6)
    assert np.abs(ours - plain).max() <= 63 * 2.0 ** -21


@pytest.mark.parametrize("change", [dict(kind="linear", factor=0.0), dict(kind="linear", factor=math.inf),
                                    dict(kind="yarn", factor=4.0), dict(kind="bands", factor=4.0, original_positions=100.0, fast=1.0, slow=1.0),
                                    dict(length=-1.0), dict(length=math.nan), dict(kind="spiral")])
def test_scaled_rope_table_refusals(package, change):
    with pytest.raises(ValueError):
        package.operators.build_rope_table_scaled(8, 64, 1e4, **change)


def test_scaled_rope_table_refuses_odd_widths(package):
    with pytest.raises(ValueError):
        package.operators.build_rope_table_scaled(8, 63, 1e4)


def run_choice(tmp_path, header, expression):
    source = tmp_path / "choice.cpp"
    source.write_text(f'#include "{header}"\n#include <cstdio>\n#include <cstdlib>\n'
                      f'int main(int, char** a) {{ {expression} }}\n')
    program = tmp_path / "choice"
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "edge-infer_b200" / "csrc"), "-o", str(program), str(source)], check=True)
    return lambda *values: [int(x) for x in subprocess.run([str(program), *map(str, values)], check=True, capture_output=True,
                                                           text=True).stdout.split()]


def test_step_shape(tmp_path):
    """Powers of two, at most 16, all clusters at once where a unit is split at all, no warp of a split unit without a tile."""
    four, eight = [296, 148, 71, 33, 14], [148, 74, 33, 15, 7]
    choose = run_choice(tmp_path, "step_choice.hpp", f'ei::StepCapacity c{{{{{str(four)[1:-1]}}}, {{{str(eight)[1:-1]}}}}}; '
                                                     'auto s = ei::step_shape(atoll(a[1]), atoll(a[2]), a[3][0] == 49, c); '
                                                     'std::printf("%d %d", s.splits, s.warps);')
    for units in (1, 4, 8, 40, 149, 296, 512):
        for tokens in (0, 1, 31, 300, 5000, 200000):
            for two in (0, 1):
                splits, warps = choose(units, tokens, two)
                assert splits in (1, 2, 4, 8, 16) and warps in (4, 8)
                fit = (four if warps == 4 else eight)[splits.bit_length() - 1]
                assert (splits, warps) == (1, 4) or (units <= fit and splits * warps <= max(4, (tokens + 31) // 32))
    assert choose(8, 0, 0) == [1, 4] and choose(512, 100000, 0) == [1, 4] and choose(7, 200000, 0) == [16, 8]
    assert choose(8, 200000, 0) == [8, 8] and choose(8, 200000, 1) == [16, 4]


def test_span_splits(tmp_path):
    """Rows have no more partial results than are joined, blocks have tokens, and where a prefix is cut all clusters run at once."""
    choose = run_choice(tmp_path, "span_choice.hpp", 'auto s = ei::span_splits(atoll(a[1]), atoll(a[2]), atoi(a[3])); '
                                                     'std::printf("%d %d %d %d %d", s.cluster, s.pairs, s.pair_splits, s.single_splits, '
                                                     's.partials());')
    fit = {1: 148, 2: 74, 4: 33}
    for query_tiles in (1, 2, 3, 5, 8, 50, 400):
        for tokens in (1, 63, 64, 65, 1000, 30011, 200000):
            for kv_heads in (1, 4, 8):
                cluster, pairs, pair_splits, single_splits, partials = choose(query_tiles, tokens, kv_heads)
                tiles = (tokens + 63) // 64
                assert pairs == query_tiles // 2 and (single_splits > 0) == (query_tiles % 2 == 1)
                assert 1 <= partials <= 32 and partials == max(pair_splits if pairs else 0, single_splits)
                assert (pairs * pair_splits + single_splits) * kv_heads <= fit[cluster] or (pair_splits == 1 and single_splits <= 1)
                assert pair_splits <= tiles and single_splits <= tiles


def test_span_window(tmp_path):
    """Clusters of up to eight blocks where few blocks would leave the chip idle, none where it is full."""
    choose = run_choice(tmp_path, "span_choice.hpp", 'auto s = ei::span_window(atoll(a[1]), atoll(a[2]), atoll(a[3]), atoll(a[4])); '
                                                     'std::printf("%d %d", s.cluster, int(s.microseconds));')
    assert choose(1, 8, 8192, 2200)[0] == 1
    assert choose(1, 8, 256, 8192)[0] == 8
    for sequences in (1, 3, 64):
        for stacked in (64, 128, 129, 256, 5000):
            for tokens in (1, 64, 1000, 30000):
                cluster, time = choose(sequences, 8, stacked, tokens)
                assert cluster in (1, 2, 4, 8) and time > 0


# ---- refusals: addresses are never looked at ------------------------------------------------------------------------------

BASE = 1 << 20


class Call:
    def __init__(self, package):
        self.abi, self.lib = package.abi, package.abi.load_library()
        self.ctx = package.abi.Context()
        self.views = {1: self.abi.View1, 2: self.abi.View2, 3: self.abi.View3, 4: self.abi.View4}

    def view(self, at, *shape, stride=None, offset=0):
        if stride is None:
            stride, step = [], 1
            for extent in reversed(shape):
                stride.insert(0, step)
                step *= extent
        return self.views[len(shape)](at * BASE * 64 + BASE + offset, tuple(shape), tuple(stride))


@pytest.fixture
def call(package):
    return Call(package)


def refused(call, status, what=ValueError, says=None):
    with pytest.raises(what) as caught:
        call.abi.check(status)
    if says:
        assert says in str(caught.value)


def attention_arguments(call):
    """q, k, v, out of a sound call: two sequences of three rows, eight heads over two."""
    return dict(q=call.view(1, 6, 8, 128), k=call.view(2, 2, 70, 2, 128), v=call.view(3, 2, 70, 2, 128), out=call.view(4, 6, 8, 128),
                lengths=None, length=70)


ATTENTION_FAULTS = [
    ("heads must be 128 wide", lambda c, a: a.update(q=c.view(1, 6, 8, 64), out=c.view(4, 6, 8, 64))),
    ("packed heads of 128", lambda c, a: a.update(k=c.view(2, 2, 70, 2, 64), v=c.view(3, 2, 70, 2, 64))),
    ("queries' shape", lambda c, a: a.update(out=c.view(4, 6, 4, 128))),
    ("one shape", lambda c, a: a.update(v=c.view(3, 2, 71, 2, 128))),
    ("whole multiple", lambda c, a: a.update(q=c.view(1, 6, 7, 128), out=c.view(4, 6, 7, 128))),
    ("same number for every sequence", lambda c, a: a.update(q=c.view(1, 5, 8, 128), out=c.view(4, 5, 8, 128))),
    ("capacity", lambda c, a: a.update(length=71)),
    ("16-byte aligned", lambda c, a: a.update(q=c.view(1, 6, 8, 128, offset=2))),
    ("16-byte aligned", lambda c, a: a.update(k=c.view(2, 2, 70, 2, 128, offset=8))),
    ("multiple of 16 bytes", lambda c, a: a.update(k=c.view(2, 2, 70, 2, 128, stride=(70 * 260, 260, 129, 1)))),
    ("whole head rows", lambda c, a: a.update(v=c.view(3, 2, 70, 2, 128, stride=(0, 256, 128, 1)))),
    ("packed heads", lambda c, a: a.update(v=c.view(3, 2, 70, 2, 128, stride=(70 * 512, 512, 256, 2)))),
    ("packed and adjacent", lambda c, a: a.update(q=c.view(1, 6, 8, 128, stride=(2048, 256, 1)))),
    ("disjoint rows", lambda c, a: a.update(out=c.view(4, 6, 8, 128, stride=(512, 128, 1)))),
    ("disjoint rows", lambda c, a: a.update(q=c.view(1, 6, 8, 128, stride=(1028, 128, 1)))),
    ("empty", lambda c, a: a.update(q=c.view(1, 0, 8, 128), out=c.view(4, 0, 8, 128))),
    ("empty", lambda c, a: a.update(k=c.view(2, 2, 0, 2, 128), v=c.view(3, 2, 0, 2, 128))),
]


@pytest.mark.parametrize("says,change", ATTENTION_FAULTS, ids=[f"{i}-{s}" for i, (s, _) in enumerate(ATTENTION_FAULTS)])
def test_attention_refusals(call, says, change):
    a = attention_arguments(call)
    change(call, a)
    scores = call.view(5, 2, 2, 70)
    first = [a["q"], a["k"], a["v"], a["out"], a["lengths"], a["length"]]
    refused(call, call.lib.ei_attention_window_bf16(C.byref(call.ctx), *first, 16, 0), says=says)
    refused(call, call.lib.ei_attention_accumulate_bf16(C.byref(call.ctx), *first, scores, scores, 1 << 30, 1 << 40), says=says)
    prefix = call.view(6, 33, 2, 128)
    refused(call, call.lib.ei_attention_shared_prefix_bf16(C.byref(call.ctx), a["q"], prefix, prefix, *first[1:], 1 << 30, 1 << 40), says=says)


def test_more_attention_refusals(call):
    a = list(attention_arguments(call).values())
    refused(call, call.lib.ei_attention_window_bf16(None, *a, 16, 0), says="context")
    refused(call, call.lib.ei_attention_window_bf16(C.byref(call.ctx), *a, 0, 4), says="window")
    scores, ctx = call.view(5, 2, 2, 70), C.byref(call.ctx)
    need = call.lib.ei_attention_accumulate_scratch_bytes(2, 3, 8, 2, 70)
    assert need == 2 * 2 * 12 * (96 * 4 + 8)
    accumulate = call.lib.ei_attention_accumulate_bf16
    refused(call, accumulate(ctx, *a, scores, scores, 1 << 30, need - 1), says="scratch")
    refused(call, accumulate(ctx, *a, scores, scores, (1 << 30) + 4, need), says="scratch")
    refused(call, accumulate(ctx, *a, scores, scores, None, need), says="scratch")
    refused(call, accumulate(ctx, *a, scores, call.view(5, 2, 2, 70, offset=4), 1 << 30, need), says="lie apart")
    refused(call, accumulate(ctx, *a, scores, call.view(7, 2, 2, 69), 1 << 30, need), says="[sequences, kv_heads, tokens]")
    refused(call, accumulate(ctx, *a, call.view(7, 2, 2, 70, stride=(280, 140, 2)), scores, 1 << 30, need), says="packed along")
    refused(call, accumulate(ctx, *a, scores, call.abi.View3(), 1 << 30, need), says="no storage")
    prefix, shared = call.view(6, 33, 2, 128), call.lib.ei_attention_shared_prefix_bf16
    need = call.lib.ei_attention_shared_prefix_scratch_bytes(6, 8, 2, 33)
    assert need > 0 and call.lib.ei_attention_shared_prefix_scratch_bytes(6, 8, 2, 0) == 0
    refused(call, shared(ctx, a[0], prefix, prefix, *a[1:], 1 << 30, need - 1), says="scratch")
    refused(call, shared(ctx, a[0], prefix, call.view(6, 34, 2, 128), *a[1:], 1 << 30, need), says="one shape")
    refused(call, shared(ctx, a[0], call.view(6, 33, 4, 128), prefix, *a[1:], 1 << 30, need), says="KV heads")


def test_qk_norm_rope_refusals(call):
    ctx, fn = C.byref(call.ctx), call.lib.ei_qk_norm_rope_bf16
    none = call.abi.View1()

    def go(q=call.view(1, 5, 4, 64), k=call.view(2, 5, 2, 64), table=call.view(3, 99, 64), offset=0, qw=none, kw=none, eps=1e-6,
           q_out=call.view(4, 5, 4, 64), k_out=call.view(5, 5, 2, 64)):
        return fn(ctx, q, k, table, None, offset, qw, kw, eps, 0, q_out, k_out)

    refused(call, go(k=call.view(2, 6, 2, 64), k_out=call.view(5, 6, 2, 64)), says="share rows")
    refused(call, go(q_out=call.view(4, 5, 2, 64)), says="shapes")
    refused(call, go(q=call.view(1, 5, 4, 72), k=call.view(2, 5, 2, 72), q_out=call.view(4, 5, 4, 72), k_out=call.view(5, 5, 2, 72)),
            says="multiple of 16")
    refused(call, go(table=call.view(3, 99, 24)), says="rotated width")
    refused(call, go(table=call.view(3, 99, 128)), says="rotated width")
    refused(call, go(table=call.view(3, 99, 64, offset=4)), says="aligned")
    refused(call, go(table=call.view(3, 99, 64, stride=(80, 1))), says="packed")
    refused(call, go(offset=95), what=IndexError)
    refused(call, go(offset=2 ** 64 - 2), what=IndexError)
    refused(call, go(qw=call.view(6, 32)), says="norm weight")
    refused(call, go(kw=call.view(6, 64, stride=(2,))), says="norm weight")
    refused(call, go(qw=call.view(6, 64), eps=-1.0), says="epsilon")
    refused(call, go(qw=call.view(6, 64), eps=math.nan), says="epsilon")
    refused(call, go(q_out=call.view(1, 5, 4, 64, offset=16)), says="replace their inputs")


def test_evict_refusals(call):
    ctx, fn = C.byref(call.ctx), call.lib.ei_evict_kv_bf16

    def go(k=call.view(1, 2, 90, 4, 128), v=call.view(2, 2, 90, 4, 128), scores=call.view(3, 2, 4, 90), lengths=None, length=90, sinks=4,
           recent=8, k_out=call.view(4, 2, 32, 4, 128), v_out=call.view(5, 2, 32, 4, 128), scores_out=call.view(6, 2, 4, 32),
           kept=call.view(7, 2, 4, 32), lengths_out=1 << 33):
        return fn(ctx, k, v, scores, lengths, length, sinks, recent, k_out, v_out, scores_out, kept, lengths_out)

    refused(call, go(length=91), says="capacity")
    refused(call, go(sinks=25, recent=8), says="budget")
    refused(call, go(sinks=33, recent=0), says="budget")
    refused(call, go(recent=2 ** 64 - 1), says="budget")
    refused(call, go(scores=call.view(3, 2, 4, 89)), says="accumulated weights")
    refused(call, go(kept=call.view(7, 2, 4, 31)), says="kept positions")
    refused(call, go(scores_out=call.view(6, 2, 4, 33)), says="kept weights")
    refused(call, go(v_out=call.view(5, 2, 33, 4, 128)), says="agree")
    refused(call, go(k_out=call.view(4, 2, 32, 2, 128), v_out=call.view(5, 2, 32, 2, 128)), says="agree")
    refused(call, go(k_out=call.view(1, 2, 32, 4, 128)), says="lie apart")
    refused(call, go(v_out=call.view(4, 2, 32, 4, 128)), says="share storage")
    refused(call, go(scores_out=call.view(3, 2, 4, 32)), says="lie apart")
    refused(call, go(lengths_out=None), says="lengths")
    refused(call, go(lengths=1 << 33), says="lengths")


def test_python_mirror_refuses_what_pointers_do_not_show(package):
    """Tensors of another device or type are refused before the C call."""
    import torch
    ops, ctx = package.operators, package.abi.Context()
    half, whole = torch.zeros(2, 2, 128), torch.zeros(1, 4, 2, 128)
    with pytest.raises(ValueError, match="is on cpu"):
        ops.attention_window(ctx, half.bfloat16(), whole.bfloat16(), whole.bfloat16(), half.bfloat16(), 4)
    with pytest.raises(ValueError, match="is on cpu"):
        ops.qk_norm_rope(ctx, half.bfloat16(), half.bfloat16(), torch.zeros(4, 128), half.bfloat16(), half.bfloat16())
    ctx.device = -1  # what tensors of the CPU call theirs
    with pytest.raises(ValueError, match="expected a torch.bfloat16"):
        ops.attention_window(ctx, half, whole.bfloat16(), whole.bfloat16(), half.bfloat16(), 4)
    with pytest.raises(ValueError, match="4 axes"):
        ops.attention_window(ctx, half.bfloat16(), half.bfloat16(), whole.bfloat16(), half.bfloat16(), 4)
    with pytest.raises(ValueError, match="torch.int32"):
        ops.attention_window(ctx, half.bfloat16(), whole.bfloat16(), whole.bfloat16(), half.bfloat16(), 4, lengths=torch.zeros(1))
    with pytest.raises(ValueError, match="1 packed values"):
        ops.attention_window(ctx, half.bfloat16(), whole.bfloat16(), whole.bfloat16(), half.bfloat16(), 4,
                             lengths=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(OverflowError):
        ops.attention_window(ctx, half.bfloat16(), whole.bfloat16(), whole.bfloat16(), half.bfloat16(), -1)
