"""What the host side remembers of a device (csrc/tc_host.cuh), against a fake of the CUDA runtime: compiled by the host compiler, no GPU."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "amd_kernels_b200", "csrc")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")

FAKE = r"""
#include <cuda_runtime.h>
static int current = 0;
static cudaError_t get_device = cudaSuccess;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = current; return get_device; }
extern "C" cudaError_t cudaDeviceGetAttribute(int* v, enum cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
extern "C" cudaError_t cudaGetDriverEntryPoint(const char*, void** p, unsigned long long, enum cudaDriverEntryPointQueryResult* q) {
  *p = nullptr; *q = cudaDriverEntryPointSymbolNotFound; return cudaSuccess;
}
"""


def run(tmp_path, body):
    if shutil.which("g++") is None or not os.path.exists(os.path.join(CUDA, "include", "cuda_runtime.h")):
        pytest.skip("needs the host compiler and the CUDA headers")
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(FAKE + '#include "tc_host.cuh"\n#define EXPECT(x) if (!(x)) return __LINE__\nusing namespace b200moe;\nint main() {\n' + body + "\nreturn 0;\n}\n")
    subprocess.run(["g++", "-std=c++17", "-DB200MOE_I=768", "-I", CSRC, "-I", os.path.join(CUDA, "include"), "-o", str(exe), str(src), "-lpthread"], check=True)
    assert subprocess.run([str(exe)]).returncode == 0


def test_an_answer_is_remembered_and_a_failure_is_not(tmp_path):
    run(tmp_path, r"""
  PerDeviceAnswer<int> count;
  int asked = 0;
  const auto fails = [&](int& n) { ++asked; n = 0; return false; };
  const auto answers = [&](int& n) { ++asked; n = 70 + current; return true; };
  EXPECT(count.get(fails) == 0 && asked == 1);
  EXPECT(count.get(answers) == 70 && asked == 2);   // the failure of before is not what this device holds
  EXPECT(count.get(fails) == 70 && asked == 2);     // the answer is
  current = 1;                                      // another device has its own
  EXPECT(count.get(fails) == 0 && count.get(answers) == 71 && count.get(fails) == 71 && asked == 4);
  get_device = cudaErrorInitializationError;
  EXPECT(count.get(answers) == 0 && asked == 4);
  get_device = cudaSuccess;
  current = kMaxDevices;
  EXPECT(count.get(answers) == 0 && asked == 4);""")


def test_what_was_answered_counts_at_once(tmp_path):
    run(tmp_path, r"""
  struct Table { int of[3]; };
  PerDeviceAnswer<Table> table;
  const auto half = [&](Table& t) { t.of[0] = 5; return false; };
  const auto whole = [&](Table& t) { t.of[0] = 5, t.of[1] = 6; return true; };
  EXPECT(table.get(half).of[0] == 5 && table.get(half).of[1] == 0);
  EXPECT(table.get(whole).of[1] == 6 && table.get(half).of[1] == 6);""")
