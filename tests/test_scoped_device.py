"""The scope that makes a call's device current (csrc/scoped_device.h), with a stand-in for the two calls of the runtime that it makes."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include "scoped_device.h"

static int current = 0, sets = 0;
extern "C" cudaError_t CUDARTAPI cudaGetDevice(int *d) { *d = current; return cudaSuccess; }
extern "C" cudaError_t CUDARTAPI cudaSetDevice(int d) {
  ++sets;
  if (d > 7) return cudaErrorInvalidDevice;
  current = d;
  return cudaSuccess;
}

int main() {
  for (int caller = 0; caller < 3; ++caller)
    for (int device = 0; device < 3; ++device)
      for (int meanwhile = -1; meanwhile < 3; ++meanwhile) {
        current = caller, sets = 0;
        int inside;
        {
          orion::ScopedDevice scope(device);
          inside = scope.status == cudaSuccess ? current : -1;
          if (meanwhile >= 0) current = meanwhile;
        }
        const int calls = (device != caller) + ((meanwhile >= 0 ? meanwhile : device) != caller);
        if (inside != device || current != caller || sets != calls) return printf("%d %d %d: %d %d %d", caller, device, meanwhile, inside, current, sets), 1;
      }
  current = 1;
  {
    orion::ScopedDevice scope(9);
    if (scope.status == cudaSuccess) return 2;
  }
  return current == 1 ? 0 : 3;
}
"""


def test_the_callers_device_is_put_back(tmp_path):
    """Also where the work within the scope has made another device current."""
    source, program = tmp_path / "scope.cpp", tmp_path / "scope"
    source.write_text(PROGRAM)
    cuda = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "orionserve-rs_b200", "csrc"), "-I", os.path.join(cuda, "include"), str(source), "-o", str(program)], check=True)
    r = subprocess.run([str(program)], stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0, r.stdout
