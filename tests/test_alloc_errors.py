"""An allocation that fails leaves no error behind in the HIP runtime: its caller reports it, and the next
launch's check (this library's or torch's) must not find it there."""

from __future__ import annotations

import subprocess

from test_workspace_pool import CSRC, HIP

MAIN = r"""
#include "workspace.h"
#include <cstdio>
using namespace dsb;
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main() {
  device_bytes = 1 << 20;
  void* p = nullptr;
  CHECK(device_malloc(&p, 2 << 20) == hipErrorOutOfMemory);
  CHECK(hipGetLastError() == hipSuccess);
  BlockPool pool(false, 1 << 20);
  CHECK(pool.get(2 << 20).p == nullptr);
  CHECK(hipGetLastError() == hipSuccess);
  CHECK(device_malloc(&p, 1 << 10) == hipSuccess && p);
  puts("ok");
  return 0;
}
"""


def test_failed_allocations_leave_no_error_behind(tmp_path):
    hip = HIP.replace("if (device_used + n > device_bytes) return hipErrorOutOfMemory;",
                      "if (device_used + n > device_bytes) return last = hipErrorOutOfMemory;")
    hip = hip.replace("inline hipError_t hipGetLastError() { return hipSuccess; }",
                      "inline hipError_t hipGetLastError() { hipError_t e = last; last = hipSuccess; return e; }")
    hip = hip.replace("inline std::function", "inline hipError_t last = hipSuccess;\ninline std::function", 1)
    assert hip.count("last = hip") == 3
    (tmp_path / "hip").mkdir()
    (tmp_path / "hip" / "hip_runtime.h").write_text(hip)
    (tmp_path / "main.cpp").write_text(MAIN)
    exe = tmp_path / "alloc"
    subprocess.run(["g++", "-std=c++17", "-pthread", f"-I{tmp_path}", f"-I{CSRC}", str(tmp_path / "main.cpp"),
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
