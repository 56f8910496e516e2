"""include/am_hip_tensor.hpp brings along what it uses: a program whose first and only header it is compiles."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_header_stands_alone(tmp_path):
    source = tmp_path / "alone.cpp"
    source.write_text('#include "am_hip_tensor.hpp"\ntemplate class am::HipTensor<float>;\nfloat f(const am::HipTensor<float>& t) { return am::stddev(t); }\n')
    res = subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(source)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
