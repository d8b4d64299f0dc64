"""An operator's set-up is its own (CPU: the library's boundary, capi.cu, linked with a fake CUDA runtime and with set-ups
that fail or count): one that fails refuses calls of that operator and stops nothing else."""

from __future__ import annotations

import subprocess

import pytest

from selas_b200 import build

from .conftest import ROOT

RUNTIME = r"""
#include <cuda_runtime_api.h>
int device = 0, mode = cudaStreamCaptureModeGlobal;
static char memory[1 << 16];
extern "C" {
cudaError_t cudaGetDeviceCount(int* n) { return *n = 2, cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { return *d = device, cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr a, int) {
  *v = a == cudaDevAttrComputeCapabilityMajor ? 10 : a == cudaDevAttrMultiProcessorCount ? 148 : 0;
  return cudaSuccess;
}
cudaError_t cudaGetDriverEntryPoint(const char*, void** f, unsigned long long, cudaDriverEntryPointQueryResult* q) {
  *f = memory;
  return *q = cudaDriverEntryPointSuccess, cudaSuccess;
}
cudaError_t cudaMalloc(void** p, size_t) { return *p = memory, cudaSuccess; }
cudaError_t cudaMemset(void*, int, size_t) { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "fake"; }
cudaError_t cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode* m) {
  const int old = mode;
  mode = *m, *m = static_cast<cudaStreamCaptureMode>(old);
  return cudaSuccess;
}
void** __cudaRegisterFatBinary(void*) { return nullptr; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
}
"""

SETUPS = r"""
#include <cstdio>
#include <new>
#include "CSRC/fb_internal.h"

extern int device, mode;
static int ran[5] = {}, broken[5] = {};
static bool throws = false;
static std::string run(int i) {
  ++ran[i];
  if (throws) throw std::bad_alloc();
  if (i >= 2 && mode != cudaStreamCaptureModeRelaxed) return "set-up without a relaxed capture mode";
  return broken[i] ? "broken set-up " + std::to_string(i) : std::string();
}
namespace fb {
std::string gemm_setup() { return run(0); }
std::string attention_setup() { return run(1); }
std::string linear_act_setup() { return run(2); }
std::string layer_norm_setup() { return run(3); }
std::string rope_axes_setup() { return run(4); }
}  // namespace fb
#define CHECK(c) do { if (!(c)) { printf("line %d: %s (%s)\n", __LINE__, #c, fb_last_error()); return 1; } } while (0)
"""

START = r"""
int main() {  // the operators' set-ups fail: the framework starts all the same, and without having run them
  broken[2] = broken[3] = broken[4] = 1;
  CHECK(fb_init() == FB_OK);
  CHECK(ran[0] == 1 && ran[1] == 1 && ran[2] + ran[3] + ran[4] == 0);
  return 0;
}
"""

CALLS = r"""
int main() {
  using fb::Operator;
  std::string err;
  broken[2] = 1;
  CHECK(fb_init() == FB_OK);
  CHECK(!fb::device_for(Operator::kLinearAct, err) && err == "broken set-up 2" && ran[0] == 1);
  CHECK(!fb::device_for(Operator::kLinearAct, err) && ran[3] + ran[4] == 0);
  CHECK(mode == cudaStreamCaptureModeGlobal);  // the caller's again, also after a failure
  fb::DeviceState* d = fb::device_for(Operator::kLayerNorm, err);
  CHECK(d && d == fb::device_for(Operator::kLayerNorm, err) && ran[3] == 1);
  CHECK(fb::device_for(Operator::kRopeAxes, err) == d && ran[4] == 1 && mode == cudaStreamCaptureModeGlobal);
  device = 1;  // each device by itself
  CHECK(fb::device_for(Operator::kLayerNorm, err) != d && ran[3] == 2 && ran[0] == 2 && ran[4] == 1);
  throws = true;
  bool thrown = false;
  try {
    fb::device_for(Operator::kRopeAxes, err);
  } catch (const std::bad_alloc&) {
    thrown = true;
  }
  CHECK(thrown && mode == cudaStreamCaptureModeGlobal);
  throws = false;
  broken[2] = 0;
  CHECK(fb::device_for(Operator::kLinearAct, err));
  return 0;
}
"""


@pytest.mark.parametrize("program", [START, CALLS], ids=["start", "calls"])
def test_a_failed_setup_stops_only_its_operator(tmp_path, program):
    nvcc = str(build.nvcc())
    src, fake, exe = tmp_path / "setups.cu", tmp_path / "runtime.cpp", tmp_path / "program"
    src.write_text(SETUPS.replace("CSRC", str(build.CSRC)) + program)
    fake.write_text(RUNTIME)
    cu = [nvcc, *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr", "-I", str(ROOT / "include"), "-c"]
    # the kernels' launchers stay unresolved: nothing here calls one
    for cmd in ([*cu, str(src), "-o", str(tmp_path / "setups.o")], [*cu, str(build.CSRC / "capi.cu"), "-o", str(tmp_path / "capi.o")],
                ["g++", "-no-pie", "-I", nvcc.rsplit("/bin/", 1)[0] + "/include", str(fake), str(tmp_path / "setups.o"), str(tmp_path / "capi.o"),
                 "-o", str(exe), "-Wl,--unresolved-symbols=ignore-all", "-Wl,-z,lazy"]):
        r = subprocess.run(cmd, capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
