"""CPU checks of what the operators for long contexts refuse: outputs that meet other arguments in memory."""
import ctypes as C
import itertools
import subprocess

import pytest

import context_cases
from test_context_cpu import ROOT, call, refused, run_choice  # noqa: F401


def accepted(call, status):
    """Nothing about the arguments is wrong: what is left to refuse is the context, of a device that no machine has."""
    with pytest.raises((RuntimeError, ValueError)) as caught:
        call.abi.check(status)
    assert isinstance(caught.value, RuntimeError) or "another CUDA device" in str(caught.value), str(caught.value)


@pytest.fixture
def elsewhere(call):  # noqa: F811
    call.ctx.device = 1 << 20
    return call


def test_views_that_may_meet(tmp_path):
    """Against the sets of bytes of small views: two that meet are always found, those that lie apart in the ways that buffers
    are shared in earnest are told apart."""
    meet = run_choice(tmp_path, "view_overlap.hpp", 'auto r = [&](int i) { ei::Region g{(uintptr_t)atoll(a[i]), (size_t)atoll(a[i + 1]), 2, '
                      '{(size_t)atoll(a[i + 2]), (size_t)atoll(a[i + 4])}, {(size_t)atoll(a[i + 3]), (size_t)atoll(a[i + 5])}}; return g; };'
                      'std::printf("%d", int(ei::may_meet(r(1), r(7))));')

    def touched(at, item, n0, s0, n1, s1):
        return {at + i * s0 + j * s1 + x for i in range(n0) for j in range(n1) for x in range(item)}

    shapes = [(4, 3, 16, 1, 4), (4, 3, 16, 2, 4), (8, 2, 48, 3, 16), (6, 1, 7, 4, 16), (4, 2, 20, 3, 8)]
    for (one, two), shift in itertools.product(itertools.product(shapes, shapes), (0, 3, 4, 8, 30, 200)):
        a, b = (64, *one), (64 + shift, *two)
        met = meet(*a, *b)[0]
        assert met == meet(*b, *a)[0]
        assert met or not touched(*a) & touched(*b)
        assert not met or min(touched(*b)) <= max(touched(*a))
    # Keys and values side by side for every token; halves of every row; one row behind the other.
    assert meet(64, 8, 5, 160, 10, 16, 72, 8, 5, 160, 10, 16) == [0]
    assert meet(64, 8, 5, 160, 10, 16, 71, 8, 5, 160, 10, 16) == [1]
    assert meet(64, 80, 5, 160, 1, 1, 144, 80, 5, 160, 1, 1) == [0]
    assert meet(64, 16, 1, 16, 1, 16, 80, 16, 1, 16, 1, 16) == [0]
    # A reach beyond 64 bits.
    assert meet(64, 1, 2 ** 40, 2 ** 40, 2 ** 40, 2 ** 40, 80, 16, 1, 16, 1, 16) == [0]
    assert meet(64, 17, 2 ** 40, 2 ** 40, 2 ** 40, 2 ** 40, 80, 16, 1, 16, 1, 16) == [1]


def test_rotated_heads_that_meet_other_arguments(elsewhere):
    call, fn, none = elsewhere, elsewhere.lib.ei_qk_norm_rope_bf16, elsewhere.abi.View1()

    def go(q=call.view(1, 5, 4, 64), k=call.view(2, 5, 2, 64), table=call.view(3, 99, 64), positions=None, qw=none, q_out=call.view(4, 5, 4, 64),
           k_out=call.view(5, 5, 2, 64)):
        return fn(C.byref(call.ctx), q, k, table, positions, 0, qw, none, 1e-6, 0, q_out, k_out)

    accepted(call, go())
    accepted(call, go(q_out=call.view(1, 5, 4, 64), k_out=call.view(2, 5, 2, 64)))
    # Slices of one projection's rows, in place and apart.
    fused = lambda first, heads: call.view(1, 5, heads, 64, stride=(14 * 64, 64, 1), offset=first * 128)
    accepted(call, go(q=fused(0, 4), k=fused(4, 2), q_out=fused(0, 4), k_out=fused(4, 2)))
    accepted(call, go(q=fused(0, 4), k=fused(4, 2), q_out=fused(8, 4), k_out=fused(12, 2)))
    for fault in (dict(q_out=call.view(2, 5, 4, 64)), dict(k_out=call.view(1, 5, 2, 64, offset=256)),
                  dict(q_out=call.view(4, 5, 4, 64), k_out=call.view(4, 5, 2, 64, offset=512)),
                  dict(q_out=call.view(1, 5, 4, 64), k_out=call.view(1, 5, 2, 64)),
                  dict(q=fused(0, 4), k=fused(4, 2), q_out=fused(1, 4)), dict(q=fused(0, 4), k=fused(4, 2), k_out=fused(3, 2)),
                  dict(q_out=call.view(3, 5, 4, 64, offset=64)), dict(k_out=call.view(3, 5, 2, 64, offset=99 * 256 - 16)),
                  dict(qw=call.view(4, 64, offset=128)), dict(positions=call.view(5, 5).data + 1264)):
        refused(call, go(**fault), says="lie apart")


def test_attention_outputs_that_meet_other_arguments(elsewhere):
    """Every attention, with everything apart, with outputs in the queries' place, and with one argument over another."""
    call, lib, ctx = elsewhere, elsewhere.lib, C.byref(elsewhere.ctx)
    view = call.view
    prefix_bytes = lib.ei_attention_shared_prefix_scratch_bytes(6, 8, 2, 33)
    scratch_bytes = lib.ei_attention_accumulate_scratch_bytes(2, 3, 8, 2, 70)

    def every(q=view(1, 6, 8, 128), k=view(2, 2, 70, 2, 128), v=view(3, 2, 70, 2, 128), out=view(4, 6, 8, 128), lengths=1 << 33,
              scores=view(5, 2, 2, 70), scores_out=view(6, 2, 2, 70), pk=view(7, 33, 2, 128), pv=view(8, 33, 2, 128), scratch=view(9, 1).data):
        first = (q, k, v, out, lengths, 0)
        return {"window": lambda: lib.ei_attention_window_bf16(ctx, *first, 16, 0),
                "prefix": lambda: lib.ei_attention_shared_prefix_bf16(ctx, q, pk, pv, k, v, out, lengths, 0, scratch, prefix_bytes),
                "accumulate": lambda: lib.ei_attention_accumulate_bf16(ctx, *first, scores, scores_out, scratch, scratch_bytes)}

    side = lambda place: view(2, 2, 70, 2, 128, stride=(70 * 512, 512, 128, 1), offset=512 * place)  # keys and values of a token adjacent
    wide = lambda first: view(4, 6, 8, 128, stride=(2048, 128, 1), offset=2048 * first)
    for fine in (dict(), dict(out=view(1, 6, 8, 128)), dict(k=side(0), v=side(1)), dict(v=view(2, 2, 70, 2, 128)), dict(q=wide(0), out=wide(1)),
                 dict(scores=view(6, 2, 2, 70)), dict(pk=view(2, 33, 2, 128)), dict(scores=call.abi.View3())):
        for go in every(**fine).values():
            accepted(call, go())
    everywhere, some = ("window", "prefix", "accumulate"), ("prefix", "accumulate")
    row, token = 2048, 512  # bytes
    for names, fault in [(everywhere, dict(out=view(1, 6, 8, 128, offset=row))), (everywhere, dict(out=view(1, 6, 8, 128, stride=(2048, 128, 1)))),
                         (everywhere, dict(q=wide(0), out=view(4, 6, 8, 128, stride=(2048, 128, 1), offset=2032))),
                         (everywhere, dict(out=view(2, 6, 8, 128, offset=140 * token - 16))), (everywhere, dict(out=view(3, 6, 8, 128))),
                         (everywhere, dict(lengths=view(4, 1).data + 6 * row - 4)), (("prefix",), dict(out=view(7, 6, 8, 128))),
                         (("prefix",), dict(out=view(8, 6, 8, 128))), (some, dict(scratch=view(4, 1).data)), (some, dict(scratch=view(1, 1).data)),
                         (some, dict(scratch=view(2, 1).data)), (some, dict(scratch=view(3, 1).data)), (some, dict(lengths=view(9, 1).data)),
                         (("prefix",), dict(scratch=view(7, 1).data)), (("prefix",), dict(scratch=view(8, 1).data)),
                         (("accumulate",), dict(scratch=view(5, 1).data)), (("accumulate",), dict(scratch=view(6, 1).data)),
                         (("accumulate",), dict(out=view(5, 6, 8, 128))), (("accumulate",), dict(out=view(6, 6, 8, 128))),
                         (("accumulate",), dict(scores_out=view(1, 2, 2, 70))), (("accumulate",), dict(scores_out=view(2, 2, 2, 70))),
                         (("accumulate",), dict(scores_out=view(3, 2, 2, 70))), (("accumulate",), dict(scores=view(6, 2, 2, 70, stride=(150, 70, 1)))),
                         (("accumulate",), dict(lengths=view(6, 1).data))]:
        for name in names:
            refused(call, every(**fault)[name](), says="lie apart")


def test_evicted_outputs_that_meet_other_arguments(elsewhere):
    call, view = elsewhere, elsewhere.view

    def go(k=view(1, 2, 90, 4, 128), v=view(2, 2, 90, 4, 128), scores=view(3, 2, 4, 90), lengths=view(8, 1).data, k_out=view(4, 2, 32, 4, 128),
           v_out=view(5, 2, 32, 4, 128), scores_out=view(6, 2, 4, 32), kept=view(7, 2, 4, 32), lengths_out=view(9, 1).data):
        return call.lib.ei_evict_kv_bf16(C.byref(call.ctx), k, v, scores, lengths, 0, 4, 8, k_out, v_out, scores_out, kept, lengths_out)

    side = lambda at, tokens, place: view(at, 2, tokens, 4, 128, stride=(tokens * 1024, 1024, 128, 1), offset=1024 * place)
    both = lambda place: view(6, 2, 4, 32, stride=(256, 64, 1), offset=128 * place)  # weights and positions of a head adjacent
    for fine in (dict(), dict(k=side(1, 90, 0), v=side(1, 90, 1), k_out=side(4, 32, 0), v_out=side(4, 32, 1)),
                 dict(scores_out=both(0), kept=both(1)), dict(lengths=view(9, 1).data + 8),
                 dict(k=view(1, 2, 90, 4, 128, stride=(200 * 512, 512, 128, 1)), k_out=view(1, 2, 32, 4, 128, stride=(200 * 512, 512, 128, 1), offset=90 * 1024))):
        accepted(call, go(**fine))
    outputs = dict(k_out=lambda *a, **o: view(a[0], 2, 32, 4, 128, **o), v_out=lambda *a, **o: view(a[0], 2, 32, 4, 128, **o),
                   scores_out=lambda *a, **o: view(a[0], 2, 4, 32, **o), kept=lambda *a, **o: view(a[0], 2, 4, 32, **o),
                   lengths_out=lambda *a, **o: view(a[0], 1, **o).data)
    own = dict(k_out=4, v_out=5, scores_out=6, kept=7, lengths_out=9)
    for name, make in outputs.items():
        for place in (1, 2, 3, 8, *(at for other, at in own.items() if other != name)):
            refused(call, go(**{name: make(place)}), says="new lengths" if (name, place) == ("lengths_out", 8) else "lie apart")
    refused(call, go(v_out=side(4, 32, 1)), says="lie apart")
    refused(call, go(lengths_out=view(8, 1).data + 4), says="lie apart")
    refused(call, go(lengths_out=view(8, 1).data - 4), says="lie apart")


def test_views_that_may_fold(tmp_path):
    fold = run_choice(tmp_path, "view_overlap.hpp", 'ei::Region g{64, (size_t)atoll(a[1]), 3, {}, {}}; for (int i = 0; i < 3; ++i) '
                      'g.count[i] = atoll(a[2 + 2 * i]), g.step[i] = atoll(a[3 + 2 * i]); std::printf("%d", int(ei::may_fold(g)));')
    for item, axes in itertools.product((1, 4), itertools.product([(1, 0), (2, 4), (3, 4), (2, 12), (3, 8), (2, 0), (4, 48)], repeat=3)):
        flat = [x for axis in axes for x in axis]
        every = [sum(i * step for i, (_, step) in zip(at, axes)) + x for at in itertools.product(*(range(n) for n, _ in axes)) for x in range(item)]
        folded = fold(item, *flat)[0]
        assert folded or len(set(every)) == len(every)
    # Packed in any order of the axes, and with gaps.
    for order in itertools.permutations([(2, 256), (3, 512), (5, 2000)]):
        assert fold(256, *(x for axis in order for x in axis)) == [0]
    assert fold(256, 2, 2 ** 63, 3, 2 ** 63, 1, 0) == [1]


def test_outputs_that_meet_themselves(elsewhere):
    """Heads or sequences of an output that share tokens' storage: two writers of one place."""
    call, view, ctx = elsewhere, elsewhere.view, C.byref(elsewhere.ctx)
    size = call.lib.ei_attention_accumulate_scratch_bytes(2, 3, 8, 2, 70)

    def accumulate(scores_out):
        return call.lib.ei_attention_accumulate_bf16(ctx, view(1, 6, 8, 128), view(2, 2, 70, 2, 128), view(3, 2, 70, 2, 128), view(4, 6, 8, 128), None, 70,
                                                     call.abi.View3(), scores_out, view(6, 1).data, size)

    accepted(call, accumulate(view(5, 2, 2, 70, stride=(72, 200, 1))))
    refused(call, accumulate(view(5, 2, 2, 70, stride=(70, 70, 1))), says="storage for every")
    refused(call, accumulate(view(5, 2, 2, 70, stride=(100, 140, 1))), says="storage for every")

    refused(call, accumulate(view(5, 2, 2, 70, stride=(2 ** 62, 70, 1))), says="too far apart")

    def evict(k_out=view(4, 2, 32, 4, 128), v_out=view(5, 2, 32, 4, 128), scores_out=view(6, 2, 4, 32), kept=view(7, 2, 4, 32)):
        return call.lib.ei_evict_kv_bf16(ctx, view(1, 2, 90, 4, 128), view(2, 2, 90, 4, 128), view(3, 2, 4, 90), None, 90, 4, 8, k_out, v_out,
                                         scores_out, kept, view(9, 1).data)

    accepted(call, evict(k_out=view(4, 2, 32, 4, 128, stride=(32 * 128, 128, 64 * 128, 1))))
    for fault in (dict(k_out=view(4, 2, 32, 4, 128, stride=(32 * 512, 128, 128, 1))), dict(v_out=view(5, 2, 32, 4, 128, stride=(512, 512, 128, 1))),
                  dict(scores_out=view(6, 2, 4, 32, stride=(32, 32, 1))), dict(kept=view(7, 2, 4, 32, stride=(64, 32, 1)))):
        refused(call, evict(**fault), says="storage for every")


def test_integers_in_device_memory_are_aligned(elsewhere):
    """A kernel that read them from an odd address would fault."""
    call, view, lib, ctx = elsewhere, elsewhere.view, elsewhere.lib, C.byref(elsewhere.ctx)
    q, k, v, out, odd = view(1, 6, 8, 128), view(2, 2, 70, 2, 128), view(3, 2, 70, 2, 128), view(4, 6, 8, 128), view(9, 1).data + 2
    prefix, scores, none = view(5, 33, 2, 128), view(6, 2, 2, 70), call.abi.View1()
    refused(call, lib.ei_attention_window_bf16(ctx, q, k, v, out, odd, 0, 16, 0), says="aligned")
    refused(call, lib.ei_attention_shared_prefix_bf16(ctx, q, prefix, prefix, k, v, out, odd, 0, 1 << 30, 1 << 26), says="aligned")
    refused(call, lib.ei_attention_accumulate_bf16(ctx, q, k, v, out, odd, 0, scores, scores, 1 << 30, 1 << 26), says="aligned")
    keys = view(1, 5, 2, 64)
    refused(call, lib.ei_qk_norm_rope_bf16(ctx, keys, keys, view(3, 99, 64), odd, 0, none, none, 1e-6, 0, view(4, 5, 2, 64), view(5, 5, 2, 64)),
            says="aligned")
    for lengths, lengths_out in ((odd, 1 << 33), (None, odd)):
        refused(call, lib.ei_evict_kv_bf16(ctx, k, v, scores, lengths, 70, 4, 8, view(10, 2, 32, 2, 128), view(11, 2, 32, 2, 128), view(12, 2, 2, 32),
                                           view(13, 2, 2, 32), lengths_out), says="aligned")


def test_set_up_once_per_device(tmp_path):
    """Threads that take devices in turn set each of them up once; a set-up that fails is tried again."""
    source = tmp_path / "devices.cpp"
    source.write_text('''#include "per_device.hpp"
#include <atomic>
#include <cstdio>
#include <stdexcept>
#include <thread>
#include <vector>
int main() {
  static ei::PerDevice<int> devices;
  std::atomic<int> made{0}, wrong{0};
  int failed = 0;
  try { devices.get(9, []() -> int { throw std::runtime_error("no"); }); } catch (const std::runtime_error&) { ++failed; }
  std::vector<std::thread> threads;
  for (int t = 0; t < 8; ++t)
    threads.emplace_back([&] {
      for (int i = 0; i < 1000; ++i) {
        const int device = i % 2 ? 3 : 9;
        if (devices.get(device, [&] { ++made; return 10 * device; }) != 10 * device) ++wrong;
      }
    });
  for (auto& t : threads) t.join();
  std::printf("%d %d %d", failed, made.load(), wrong.load());
}
''')
    program = tmp_path / "devices"
    subprocess.run(["g++", "-std=c++17", "-pthread", "-I", str(ROOT / "edge-infer_b200" / "csrc"), "-o", str(program), str(source)], check=True)
    assert subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout == "1 2 0"


def test_kernels_for_long_contexts_are_set_up_per_device_not_per_thread():
    for name in ("step_attention.cu", "span_attention.cu", "evict.cu"):
        text = (ROOT / "edge-infer_b200" / "csrc" / name).read_text()
        assert "thread_local" not in text and "PerDevice" in text


def test_kernels_trigger_their_dependents_behind_their_own_wait():
    """The rule of common.cuh, kernel by kernel: what a successor runs before its wait relies on it."""
    for path in sorted((ROOT / "edge-infer_b200" / "csrc").glob("*.cu*")):
        for kernel in path.read_text().split("__global__")[1:]:
            trigger = kernel.find("grid_launch_dependents();")
            if trigger >= 0:
                assert 0 <= kernel.find("grid_dependency_wait();") < trigger, (path.name, kernel[:80])


def test_counting_expired_waits_refuses(call):  # noqa: F811
    count = C.c_uint64(7)
    refused(call, call.lib.ei_context_expired_waits(None, C.byref(count)), says="context")
    refused(call, call.lib.ei_context_expired_waits(C.byref(call.ctx), None), says="place")
    call.ctx.device = 1 << 20
    with pytest.raises((RuntimeError, ValueError)):
        call.abi.check(call.lib.ei_context_expired_waits(C.byref(call.ctx), C.byref(count)))
    assert count.value == 7


def test_cases_run_on_the_kernels_they_are_named_for(tmp_path):
    """The GPU tests' calls against the choice that the library makes."""
    window = run_choice(tmp_path, "attention_choice.hpp", "ei::SpanWindow s{}; auto n = [&](int i) { return (size_t)atoll(a[i]); }; "
                        "bool many = ei::window_on_tensor_cores(n(1), n(2), n(3), n(4), n(5), n(6), n(7), &s); "
                        'std::printf("%d %d", int(many), many ? s.cluster : 0);')
    for cases in (context_cases.HARD, context_cases.GIVE_UP, context_cases.GRAPH):
        for name, c in cases.items():
            got = window(c.sequences, c.kv_heads, c.rows, c.heads // c.kv_heads, c.tokens, c.window, c.sinks)
            assert got == [int(c.kernel == "many"), c.cluster or 0], name
    prefix = run_choice(tmp_path, "attention_choice.hpp", "ei::SpanSplits s{}; auto n = [&](int i) { return (size_t)atoll(a[i]); }; "
                        'bool many = ei::prefix_on_tensor_cores(n(1), n(2), n(3), &s); std::printf("%d %d", int(many), many ? s.cluster : 0);')
    for cases in (context_cases.PREFIX_HARD, context_cases.PREFIX_GIVE_UP):
        for name, c in cases.items():
            got = prefix(c.sequences * c.rows * c.heads // c.kv_heads, c.prefix, c.kv_heads)
            assert got == [int(c.kernel == "many"), c.cluster or 0], name


def test_only_an_encoded_query_map_is_prefetched():
    """Groups that no box copies leave the map as it is."""
    text = (ROOT / "edge-infer_b200" / "csrc" / "span_attention.cu").read_text()
    assert text.count("prefetch_map(&p.q_map)") == text.count("if (p.copied_queries) prefetch_map(&p.q_map)") == 1
