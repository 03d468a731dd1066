"""4-bit storage called from several threads at once."""
import os
import shutil
import subprocess
import sys

import pytest

from conftest import PKG_ROOT

CSRC = os.path.join(PKG_ROOT, "csrc")

# csrc/smem_attr.cuh against CUDA calls of this file: thread B (60,000 bytes) has looked and is about to set the
# attribute when thread A (150,000) sets it and returns; then B sets it.
HARNESS = r"""
#include "smem_attr.cuh"
#include <chrono>
#include <cstdio>
#include <thread>

static std::atomic<int> attr{0};
static std::atomic<bool> b_inside{false}, a_done{false};
static thread_local bool is_b = false;
template <typename F> static void until(F f) {
  for (int i = 0; i < 2000 && !f(); ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
}
extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void*, enum cudaFuncAttribute, int v) {
  if (is_b) {
    b_inside = true;
    until([] { return a_done.load(); });
  }
  attr = v;
  return cudaSuccess;
}
}
int main() {
  static anima::SmemAttr s;
  bool ok_a = false, ok_b = false;
  std::thread b([&] { is_b = true; ok_b = s.raise(nullptr, 60000); });
  until([] { return b_inside.load(); });
  std::thread a([&] { ok_a = s.raise(nullptr, 150000); a_done = true; });
  a.join();
  b.join();
  const int after = attr;
  const bool again = s.raise(nullptr, 100000);
  std::printf("%d %d %d %d %d %d\n", ok_a, ok_b, after, again, attr.load(), s.raise(nullptr, 300000) ? 1 : 0);
}
"""


def test_first_calls_that_meet_keep_the_larger_limit(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
    src, exe = tmp_path / "h.cpp", tmp_path / "h"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", f"-I{CSRC}", f"-I{include}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout.split()
    ok_a, ok_b, after, again, later, too_large = map(int, out)
    assert ok_a and ok_b and again and not too_large
    assert after >= 150000 and later >= 150000


CHILD = r"""
import sys, threading
sys.path.insert(0, sys.argv[1])
import torch, anima_attn
torch.cuda.set_device(0)
failed, barrier = [], threading.Barrier(4)
def packed(N, K):
    return anima_attn.quantize4(torch.randn(N, K, device="cuda").half())
cases = [(torch.randn(M, K, device="cuda").to(dt), packed(64, K)) for K in (128, 8192) for M, dt in
         ((1, torch.float32), (4, torch.float32), (8, torch.float16), (16, torch.bfloat16))]
want = [x.float() @ anima_attn.dequantize4(w, torch.float32).t() for x, w in cases]
torch.cuda.synchronize()
def run(order):
    torch.cuda.set_device(0)
    with torch.cuda.stream(torch.cuda.Stream()):
        barrier.wait()
        for _ in range(3):
            for n in order:
                try:
                    y = anima_attn.matvec4(*cases[n])
                except Exception as e:
                    failed.append(f"{n}: {e}")
                    continue
                torch.cuda.current_stream().synchronize()
                if not torch.allclose(y, want[n], rtol=1e-2, atol=1e-1):
                    failed.append(f"{n}: result")
n = len(cases)
threads = [threading.Thread(target=run, args=(o,)) for o in (range(n), range(n - 1, -1, -1), range(n), range(n - 1, -1, -1))]
[t.start() for t in threads]; [t.join() for t in threads]
assert not failed, failed
print("done", anima_attn.status())
"""


@pytest.mark.gpu
def test_first_calls_of_long_and_short_rows_in_four_threads():
    """A fresh process whose first matvec4 calls, of K = 128 and 8192 in every kernel, meet in four threads."""
    r = subprocess.run([sys.executable, "-c", CHILD, PKG_ROOT], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["done", "0"], r.stdout + r.stderr[-2000:]


def test_lanes_exchange_under_masks_that_are_known():
    """A group's lanes exchange under the group's mask: __activemask() names whichever lanes happen to be
    together, which nothing promises to be whole groups after a branch."""
    for name in os.listdir(CSRC):
        with open(os.path.join(CSRC, name)) as f:
            assert "__activemask" not in f.read(), name
