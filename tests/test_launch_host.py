"""Host side of kernel launches, without a GPU: dynamic LDS is allowed on every
device that a kernel runs on."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "llm_gpu_kernels_amd" / "csrc"

# Just enough of the runtime: a current device, and the calls that set the attribute.
RUNTIME = """
#pragma once
enum hipError_t { hipSuccess = 0, hipErrorInvalidValue = 1, hipErrorNoDevice = 100 };
enum hipFuncAttribute { hipFuncAttributeMaxDynamicSharedMemorySize = 8 };
struct Runtime { int device, calls, bytes; const void *kernel; hipError_t get, set; };
extern Runtime runtime;
inline hipError_t hipGetDevice(int *d) { *d = runtime.device; return runtime.get; }
inline hipError_t hipFuncSetAttribute(const void *k, hipFuncAttribute, int bytes) {
  ++runtime.calls; runtime.kernel = k; runtime.bytes = bytes;
  return runtime.set;
}
"""

PROGRAM = r"""
#include <stdio.h>
#include "launch.h"
Runtime runtime = {};
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
  std::atomic<uint64_t> a{0}, b{0};
  int ka = 0, kb = 0;
  CHECK(moe::allow_lds(&ka, 70000, &a) == hipSuccess && runtime.calls == 1);
  CHECK(runtime.kernel == &ka && runtime.bytes == 70000);
  CHECK(moe::allow_lds(&ka, 70000, &a) == hipSuccess && runtime.calls == 1);
  runtime.device = 5;                                // each device for itself
  CHECK(moe::allow_lds(&ka, 70000, &a) == hipSuccess && runtime.calls == 2);
  runtime.device = 0;
  CHECK(moe::allow_lds(&ka, 70000, &a) == hipSuccess && runtime.calls == 2);
  CHECK(moe::allow_lds(&kb, 90000, &b) == hipSuccess && runtime.calls == 3);  // and each kernel
  runtime.device = 6;
  runtime.set = hipErrorInvalidValue;                // a failure is returned, and not kept
  CHECK(moe::allow_lds(&kb, 90000, &b) == hipErrorInvalidValue && runtime.calls == 4);
  runtime.set = hipSuccess;
  CHECK(moe::allow_lds(&kb, 90000, &b) == hipSuccess && runtime.calls == 5);
  CHECK(moe::allow_lds(&kb, 90000, &b) == hipSuccess && runtime.calls == 5);
  for (int i = 0; i < 2; ++i) {                      // past the bits: every time
    runtime.device = 64;
    CHECK(moe::allow_lds(&kb, 90000, &b) == hipSuccess && runtime.calls == 6 + i);
  }
  runtime.get = hipErrorNoDevice;
  CHECK(moe::allow_lds(&ka, 70000, &a) == hipErrorNoDevice && runtime.calls == 7);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_lds_is_allowed_on_every_device(tmp_path):
    (tmp_path / "hip").mkdir()
    (tmp_path / "hip" / "hip_runtime.h").write_text(RUNTIME)
    (tmp_path / "test.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{tmp_path}", f"-I{CSRC}", str(tmp_path / "test.cpp"),
                    "-o", str(tmp_path / "test")], check=True)
    done = subprocess.run([str(tmp_path / "test")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


def test_kernels_ask_for_lds_per_device():
    """The attribute is set by allow_lds() alone, before every launch that needs it."""
    users = []
    for path in sorted(CSRC.glob("*.h*")):
        text = path.read_text()
        if path.name != "launch.h":
            assert "hipFuncSetAttribute" not in text, path.name
        users += [path.name] * len(re.findall(r"if \(const hipError_t e = allow_lds\(\(const void \*\)k, ", text))
    assert users == ["gqa_packed.hip", "gqa_paged.hip", "gqa_prefill.hip", "moe_dma.hip", "moe_flex.hip",
                     "moe_stream.hip", "moe_tile.hip"]
