"""CPU checks of the native Python calls of the operators for long contexts, beside stand-ins for the C entries."""
import ctypes
import importlib.machinery
import importlib.util
import subprocess
import sysconfig
import threading
import time
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

# Every entry waits for say(1), two seconds at most; 0 if it came.
STAND_INS = r"""
#include "edge_infer_b200.h"
#include <atomic>
#include <chrono>
#include <thread>
static std::atomic<int> gone{0};
static ei_status wait() {
  for (int i = 0; i < 2000 && !gone; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
  return gone.exchange(0) ? EI_OK : EI_RUNTIME;
}
extern "C" {
void say(int value) { gone = value; }
ei_status ei_qk_norm_rope_bf16(const ei_context*, ei_view3, ei_view3, ei_view2, const int32_t*, size_t, ei_view1, ei_view1, float, int32_t,
                               ei_view3, ei_view3) { return wait(); }
ei_status ei_attention_window_bf16(const ei_context*, ei_view3, ei_view4, ei_view4, ei_view3, const int32_t*, size_t, size_t, size_t) {
  return wait();
}
ei_status ei_attention_shared_prefix_bf16(const ei_context*, ei_view3, ei_view3, ei_view3, ei_view4, ei_view4, ei_view3, const int32_t*,
                                          size_t, void*, size_t) { return wait(); }
ei_status ei_attention_accumulate_bf16(const ei_context*, ei_view3, ei_view4, ei_view4, ei_view3, const int32_t*, size_t, ei_view3, ei_view3,
                                       void*, size_t) { return wait(); }
ei_status ei_evict_kv_bf16(const ei_context*, ei_view4, ei_view4, ei_view3, const int32_t*, size_t, size_t, size_t, ei_view4, ei_view4,
                           ei_view3, ei_view3, int32_t*) { return wait(); }
}
"""


@pytest.fixture(scope="module")
def beside_stand_ins(tmp_path_factory):
    import torch
    folder = tmp_path_factory.mktemp("calls")
    (folder / "stand_ins.cpp").write_text(STAND_INS)
    built = folder / "_calls.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-I" + sysconfig.get_paths()["include"],
                    "-I" + str(ROOT / "include"), str(ROOT / "edge-infer_b200" / "csrc" / "python_calls.cpp"),
                    str(folder / "stand_ins.cpp"), "-o", str(built)], check=True)
    loader = importlib.machinery.ExtensionFileLoader("_calls", str(built))
    calls = importlib.util.module_from_spec(importlib.util.spec_from_loader("_calls", loader))
    loader.exec_module(calls)
    calls.configure(torch.bfloat16, torch.float32, torch.int32)
    return calls, ctypes.CDLL(str(built))


@pytest.mark.parametrize("name", ["qk_norm_rope", "attention_window", "attention_shared_prefix", "attention_accumulate", "evict_kv"])
def test_other_threads_run_during_a_call(package, beside_stand_ins, name):
    """A call that waits for the device's queue must not stop what empties it: the entry returns when another thread says so."""
    import torch
    calls, stand_ins = beside_stand_ins
    ctx = package.abi.Context()
    ctx.device = -1  # what tensors of the CPU call theirs
    at = ctypes.addressof(ctx)
    rows, cache = torch.zeros(2, 2, 128).bfloat16(), torch.zeros(1, 4, 2, 128).bfloat16()
    scores, whole = torch.zeros(1, 2, 4), torch.zeros(1, 2, 4, dtype=torch.int32)
    arguments = {
        "qk_norm_rope": (rows, rows, torch.zeros(4, 128), rows, rows, None, 0, None, None, 1e-6, False),
        "attention_window": (rows, cache, cache, rows, 4, 0, None, 4),
        "attention_shared_prefix": (rows, rows, rows, cache, cache, rows, None, None, 4),
        "attention_accumulate": (rows, cache, cache, rows, None, scores, None, None, 4),
        "evict_kv": (cache, cache, scores, cache, cache, scores, whole, whole[0, 0, :1], 0, 0, None, 4),
    }[name]

    def soon():
        time.sleep(0.05)
        stand_ins.say(1)

    stand_ins.say(0)
    other = threading.Thread(target=soon)
    other.start()
    status = getattr(calls, name)(at, *arguments)
    other.join()
    assert status == 0
