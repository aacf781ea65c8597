"""Kernel attributes are set once on every device of the process (a fake of the CUDA runtime)."""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "verl_omni_b200", "csrc")

FAKE = """#pragma once
enum cudaError_t { cudaSuccess = 0, cudaErrorInvalidValue = 1, cudaErrorNoDevice = 100 };
extern int g_device, g_device_error;
inline cudaError_t cudaGetDevice(int* d) { *d = g_device; return (cudaError_t)g_device_error; }
"""

MAIN = """#include <cstdio>
#include "per_device.h"
int g_device = 0, g_device_error = 0, calls = 0, fail = 0;
template <int K> cudaError_t launch() {
  static vo::PerDevice once;
  return once([] { ++calls; return fail ? cudaErrorInvalidValue : cudaSuccess; });
}
int main() {
  auto show = [](cudaError_t e) { std::printf("%d/%d ", (int)e, calls); };
  show(launch<0>()); show(launch<0>());                 // 0/1 0/1: once
  g_device = 1; show(launch<0>()); show(launch<0>());   // 0/2 0/2: once on the second device
  g_device = 0; show(launch<0>()); show(launch<1>());   // 0/2 0/3: another kernel
  g_device = 2; fail = 1; show(launch<0>());            // 1/4: not remembered
  fail = 0; show(launch<0>()); show(launch<0>());       // 0/5 0/5
  g_device = 70; show(launch<0>()); show(launch<0>());  // 0/6 0/7: every time
  g_device_error = 100; show(launch<0>());              // 100/7
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_once_on_every_device(tmp_path):
    (tmp_path / "cuda_runtime.h").write_text(FAKE)
    (tmp_path / "main.cpp").write_text(MAIN)
    exe = tmp_path / "main"
    subprocess.run(["g++", "-std=c++17", "-I", str(tmp_path), "-I", CSRC, str(tmp_path / "main.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert out == ["0/1", "0/1", "0/2", "0/2", "0/2", "0/3", "1/4", "0/5", "0/5", "0/6", "0/7", "100/7"]


@pytest.mark.parametrize("name", ["paged8_decode_sm100.cu", "paged8_chunk_sm100.cu", "logits.cu"])
def test_launchers_use_it(name):
    with open(os.path.join(CSRC, name)) as f:
        src = f.read()
    assert src.count("cudaFuncSetAttribute(") == src.count("static PerDevice once;") == 1
