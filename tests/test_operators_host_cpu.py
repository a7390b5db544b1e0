"""Host-side parts of the operators, compiled on their own (no device)."""

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "demucs-wgpu_b200", "csrc")


def _run(tmp_path, name, source, compile_with):
    src, exe = tmp_path / name, tmp_path / "program"
    src.write_text(source)
    subprocess.run([*compile_with, "-I", CSRC, str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)


def test_the_end_of_a_row_is_read_without_a_byte_past_it(tmp_path):
    # a heap buffer that ends with the row, under the address sanitizer: it ends
    # the program at the first byte read outside
    source = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include "row_tail.h"
int main() {
  for (int left = 1; left < 16; ++left) {
    unsigned char* row = static_cast<unsigned char*>(std::aligned_alloc(16, 64));
    row = static_cast<unsigned char*>(std::realloc(row, 32 + left));
    if (reinterpret_cast<uintptr_t>(row) % 16) return 2;
    for (int i = 0; i < 32 + left; ++i) row[i] = static_cast<unsigned char>(0x80 + 7 * i);
    uint32_t w[4];
    dmx::read_tail16(row + 32, left, w);
    unsigned char want[16] = {};
    std::memcpy(want, row + 32, left);
    if (std::memcmp(want, w, 16)) return 3;
    std::free(row);
  }
  std::puts("ok");
}
"""
    r = _run(tmp_path, "tail.cpp", source, ["g++", "-std=c++17", "-O1", "-fno-strict-aliasing",
                                            "-fsanitize=address"])
    assert r.returncode == 0 and r.stdout == "ok\n", r.stderr[:2000]


def test_settings_of_a_device_are_made_before_any_thread_goes_on(tmp_path):
    # a second thread asks while the first is still making them, and a third afterwards
    source = r"""
#include <chrono>
#include <cstdio>
#include <thread>
#include "common.cuh"
int main() {
  dmx::PerDevice configured;
  std::atomic<int> begun{0}, made{0}, early{0};
  auto set = [&] {
    if (begun++ == 0) std::this_thread::sleep_for(std::chrono::milliseconds(300));
    ++made;
  };
  std::thread first([&] { configured.once(set); });
  while (begun == 0) std::this_thread::yield();
  std::thread second([&] {
    configured.once(set);
    early = made == 0;
  });
  second.join();
  first.join();
  const int before = made;
  configured.once(set);
  std::printf("%d %d\n", early.load(), made - before);
}
"""
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    r = _run(tmp_path, "once.cu", source, [nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a"])
    assert r.returncode == 0 and r.stdout == "0 0\n", (r.stdout, r.stderr[:2000])
