"""The library's set-up store per device (csrc/per_device.cuh), compiled here as plain C++."""

import os
import shutil
import subprocess

import pytest

from conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include <thread>
#include <vector>

#include "per_device.cuh"

#define WANT(x) if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; }

int main() {
  static rf::PerDevice fit;
  int looked = 0, now = 0;
  auto find = [&] { ++looked; return now; };
  WANT(fit.get(0, find) == 0 && looked == 1);
  WANT(fit.get(0, find) == 0 && looked == 2);  // a failure is not kept
  now = 7;
  WANT(fit.get(0, find) == 7 && looked == 3);
  now = 9;
  WANT(fit.get(0, find) == 7 && looked == 3);  // what was found is
  WANT(fit.get(1, find) == 9 && looked == 4);  // each device its own
  WANT(fit.get(63, find) == 9 && fit.get(63, find) == 9 && looked == 5);
  WANT(fit.get(64, find) == 9 && fit.get(1000, find) == 9 && looked == 7);  // past the store: looked up each time
  WANT(fit.get(-1, find) == 0 && looked == 7);  // no device
  rf::PerDevice shared;
  std::vector<std::thread> threads;
  std::atomic<int> wrong{0};
  for (int i = 0; i < 8; ++i)
    threads.emplace_back([&] {
      for (int d = 0; d < 64; ++d)
        if (shared.get(d, [d] { return d + 1; }) != d + 1) ++wrong;
    });
  for (auto &t : threads) t.join();
  WANT(wrong == 0);
  return 0;
}
"""


def test_a_failed_set_up_is_tried_again(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    src, exe = tmp_path / "per_device.cpp", tmp_path / "per_device"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", "-pthread", "-I", os.path.join(ROOT, "reframework_b200", "csrc"), str(src), "-o",
                    str(exe)], check=True, capture_output=True, timeout=120)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
