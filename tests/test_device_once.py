"""csrc/device_once.cuh: what is done once per device is done on every device, also where threads on different devices come in
between each other. Compiled for the host against a stand-in for the two CUDA calls that it makes. No GPU."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include <thread>
#include <vector>

#include "device_once.cuh"

static thread_local int current = 0;
static thread_local bool broken = false;
extern "C" cudaError_t CUDARTAPI cudaGetDevice(int* d) { *d = current; return broken ? cudaErrorNoDevice : cudaSuccess; }
extern "C" cudaError_t CUDARTAPI cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int d) { *v = 100 + d; return cudaSuccess; }

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

int main() {
  int set[4] = {0, 0, 0, 0};
  auto mark = [&] { ++set[current]; return cudaSuccess; };
  static muse::DeviceOnce once;
  CHECK(once.run(mark) == cudaSuccess && once.run(mark) == cudaSuccess && set[0] == 1);
  // A call on device 0, done there, while device 1's first call is under way; and one on device 2, its first.
  current = 1;
  CHECK(once.run([&] { current = 0; once.run(mark); current = 2; once.run(mark); current = 1; return mark(); }) == cudaSuccess);
  CHECK(set[0] == 1 && set[1] == 1 && set[2] == 1);
  once.run(mark);
  current = 3;
  CHECK(set[1] == 1 && once.run(mark) == cudaSuccess && set[3] == 1);
  // What fails is tried again.
  static muse::DeviceOnce again;
  CHECK(again.run([] { return cudaErrorInvalidValue; }) == cudaErrorInvalidValue && again.run(mark) == cudaSuccess && set[3] == 2);
  CHECK(muse::device_sms() == 103 && muse::device_sms() == 103);
  // A device that is not known counts as new each time.
  broken = true;
  CHECK(again.run(mark) == cudaSuccess && set[3] == 3 && muse::device_sms() == 0);
  // Threads, a device each: nobody goes on before its own device is set.
  for (int round = 0; round < 200; ++round) {
    muse::DeviceOnce o;
    std::atomic<int> ready[8] = {}, late{0};
    std::vector<std::thread> threads;
    for (int t = 0; t < 8; ++t)
      threads.emplace_back([&, t] {
        current = t;
        for (int i = 0; i < 50; ++i) {
          o.run([&] { ready[t] = 1; return cudaSuccess; });
          if (!ready[t]) ++late;
        }
      });
    for (auto& t : threads) t.join();
    CHECK(late == 0);
  }
  return 0;
}
"""


def test_once_per_device_whoever_comes_between(tmp_path):
    from llm_inference_engine_b200 import build

    source, program = tmp_path / "once.cpp", tmp_path / "once"
    source.write_text(PROGRAM)
    csrc = ROOT / "llm_inference_engine_b200" / "csrc"
    cuda = Path(build._nvcc()).resolve().parent.parent / "include"
    done = subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-O1", "-pthread", "-x", "c++", str(source), f"-I{csrc}", f"-I{cuda}", "-o", str(program)],
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    ran = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert ran.returncode == 0, ran.stdout
