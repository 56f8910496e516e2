"""What the C++ host layer's group norm refuses before it asks for device memory: a small program of its own, run without a device."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <stdexcept>
#include "am_hip_tensor.hpp"
int main() {
  am::HipTensor<float> x, w, none;                        // shapes without memory
  x.shape = {2, 4}; x.strides = {4, 1};
  w.shape = {3}; w.strides = {1};
  int refused = 0;
  auto expect = [&](auto call) { try { call(); } catch (const std::invalid_argument&) { ++refused; } catch (const std::exception& e) { std::printf("%s\n", e.what()); } };
  std::vector<am::HipTensor<float>> kept;
  for (int64_t groups : {3, 0, -1, -4}) expect([&] { am::group_norm<float>(x, nullptr, nullptr, groups, 1e-5f, AM_ACT_NONE, &kept); });
  for (int64_t groups : {3, 0, -1, -4}) expect([&] { am::group_norm_backward<float>(x, x, nullptr, nullptr, kept, groups); });
  expect([&] { am::group_norm<float>(x, &w, nullptr, 2); });
  x.shape = {2, 1}; x.strides = {1, 1};
  expect([&] { am::group_norm<float>(x, &none, nullptr, 1); });   // of rank 0: one element, and no channels
  std::printf("%d\n", refused);
  return refused == 10 ? 0 : 1;
}
"""


def test_group_norm_refuses_before_it_takes_memory(tmp_path):
    source, program = tmp_path / "refuse.cpp", tmp_path / "refuse"
    source.write_text(PROGRAM)
    lib = os.path.join(ROOT, "arraymancer_amd")
    res = subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined", "-static-libasan", "-D_GLIBCXX_ASSERTIONS", "-I", os.path.join(ROOT, "include"),
                          str(source), "-o", str(program), "-L", lib, "-lam_hip", f"-Wl,-rpath,{lib}"], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    res = subprocess.run([str(program)], capture_output=True, text=True, timeout=60, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0:protect_shadow_gap=0"))
    assert res.returncode == 0, res.stdout + res.stderr[-2000:]
