"""The limit of dynamic shared memory that launches raise (csrc/smem_limit.cuh)
never falls below what one of them was granted, whatever the threads' order.
Host code alone: compiled here with the host compiler."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "sparseattnfunctions_b200" / "csrc"

PROGRAM = r"""
#include "smem_limit.cuh"
#include <chrono>
#include <cstdio>
#include <thread>

int main() {
  saf::SmemLimit limit;
  std::atomic<int> now{0}, calls{0};
  auto slow = [&](int n) {  // the larger request: found the limit too low, sets it late
    now = n;
    ++calls;
    std::this_thread::sleep_for(std::chrono::milliseconds(300));
    return 0;
  };
  auto quick = [&](int n) {
    now = n;
    ++calls;
    return 0;
  };
  std::thread large([&] { limit.raise(0, 200, slow); });
  while (calls == 0) std::this_thread::yield();
  std::thread small([&] { limit.raise(0, 100, quick); });
  large.join();
  small.join();
  limit.raise(0, 150, quick);
  std::printf("%d %d", now.load(), calls.load());
  limit.raise(0, 300, [](int) { return 7; });  // a failure is not remembered
  std::printf(" %d", limit.raise(0, 300, quick));
  limit.raise(1, 50, quick);  // each device has its own
  std::printf(" %d %d", now.load(), calls.load());
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_raised_by_two_threads(tmp_path):
    (tmp_path / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", str(CSRC), str(tmp_path / "main.cpp"), "-o",
                    str(tmp_path / "main")], check=True)
    said = subprocess.run([str(tmp_path / "main")], check=True, capture_output=True, text=True, timeout=60).stdout
    assert said == "200 1 0 50 3"
