"""Settings that are made once per device (csrc/device_once.h), met by two host threads at once."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdlib>
#include <initializer_list>
#include <thread>
#include "device_once.h"

int main() {
  static mlpsp::DeviceOnce once;
  // a thread is inside its first setting; another one that comes meanwhile does not go on with nothing set
  std::atomic<bool> inside{false}, leave{false}, allowed{false};
  std::thread first([&] {
    once.apply(0, [&] {
      inside = true;
      while (!leave) std::this_thread::yield();
      return 0;
    });
  });
  while (!inside) std::this_thread::yield();
  std::thread second([&] {
    const int rc = once.apply(0, [&] { allowed = true; return 0; });
    if (rc != 0 || !allowed) _Exit(3);
    leave = true;
  });
  second.join();
  first.join();
  int calls = 0;
  auto count = [&] { return ++calls, 0; };
  if (once.apply(0, count) != 0 || calls != 0) return 4;         // done
  if (once.apply(1, [] { return -7; }) != -7) return 5;          // a failure is answered, and tried again
  if (once.apply(1, count) != 0 || calls != 1) return 6;
  if (once.apply(1, count) != 0 || calls != 1) return 7;
  for (int device : {-1, 64, 1000})                              // not kept: every time
    for (int i = 0; i < 2; ++i) once.apply(device, count);
  return calls == 7 ? 0 : 8;
}
"""


def test_no_thread_passes_a_setting_that_is_not_made(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no C++ compiler")
    source, program = tmp_path / "first.cpp", tmp_path / "first"
    source.write_text(PROGRAM)
    subprocess.run([compiler, "-std=c++17", "-O1", "-pthread", "-I", os.path.join(ROOT, "mlp-splatting_b200", "csrc"), str(source), "-o", str(program)],
                   check=True)
    assert subprocess.run([str(program)], timeout=60).returncode == 0


def test_no_setting_is_made_past_it():
    """Every opt-in to more shared memory goes through allow_shared_memory."""
    csrc = os.path.join(ROOT, "mlp-splatting_b200", "csrc")
    users = [f for f in sorted(os.listdir(csrc)) if f.endswith((".cu", ".cuh")) and "cudaFuncSetAttribute(" in open(os.path.join(csrc, f)).read()]
    assert users == ["frame.cuh"]
