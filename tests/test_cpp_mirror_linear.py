"""The C++ mirror's wrappers of the dense products and of the whole-layer call compile and link."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

TU = r"""
#include "gx_moe.hpp"
// every wrapper once, on null buffers: compiled and linked, never run
int use_all(cudaStream_t st) {
  gx::MoeShape s{};
  gx::LayerW L{};
  gx::MoeBlock b{};
  const __nv_bfloat16* x = nullptr;
  __nv_bfloat16* out = nullptr;
  float* f = nullptr;
  void* v = nullptr;
  try {
    size_t n = gx::moe_block_ws_bytes(s) + gx::linear_bytes(64, 512) + gx::linear_bytes(64, 512, true);
    gx::moe_block_decode(s, L, x, 1, b, x, out, st);
    gx::LinearW w = gx::linear_prepare(v, nullptr, 64, 512, v, st);
    gx::linear_decode(w, x, 512, 1, x, 64, out, 64, st);
    gx::linear_decode(w, x, 512, 1, f, 64, st);
    return (int)n;
  } catch (const gx::Error& e) {
    return e.status;
  }
}
int main() { return 0; }
"""


def test_wrappers_compile_and_link(tmp_path):
    if shutil.which("nvcc") is None:
        pytest.skip("no nvcc on this machine")
    lib = os.path.join(ROOT, "dsgx10_b200", "libdsgx_moe.so")
    if not os.path.exists(lib):
        pytest.skip("libdsgx_moe.so is not built")
    src, exe = tmp_path / "tu.cu", tmp_path / "tu"
    src.write_text(TU)
    r = subprocess.run(["nvcc", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", os.path.join(ROOT, "include"),
                        "-I", os.path.join(ROOT, "dsgx10_b200", "csrc"), str(src), lib, "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
