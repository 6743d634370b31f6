"""What stands around the recurrent-block entry points, with a runtime of two pretended devices: the caller's device is current again after the
call, however the call ended, and a failure leaves its own message."""
import os
import subprocess

import pytest

from test_emu_kernels import CLANG, HERE

RUNTIME = r"""
#pragma once
typedef int hipError_t;
typedef int hipDevice_t;
typedef void *hipStream_t;
constexpr hipError_t hipSuccess = 0;
inline int &current_device() { static int d = 0; return d; }
inline hipError_t &refuse_move() { static hipError_t e = 0; return e; }
inline hipError_t hipGetDevice(int *d) { *d = current_device(); return hipSuccess; }
inline hipError_t hipSetDevice(int d) { if (refuse_move()) return refuse_move(); current_device() = d; return hipSuccess; }
inline hipError_t hipStreamGetDevice(hipStream_t s, hipDevice_t *d) { *d = (int)(long)s - 16; return hipSuccess; }
inline hipError_t hipGetLastError() { return hipSuccess; }
inline const char *hipGetErrorString(hipError_t) { return "refused"; }
"""

PROGRAM = r"""
#include <hip/hip_runtime.h>
#include <cstdio>
#include <new>
#include <stdexcept>
#include <string>
#define TCU_LAUNCH_HPP
namespace tcu { inline unsigned long launch_count() { return 0; } }
#include "stream_device.hpp"
namespace tcu {
std::string message;
int report_failure(int code, const std::string &m) { message = m; return code; }
int launch_outcome(const char *, unsigned long, int rc) { return rc; }
}
int wrong = 0;
#define EXPECT(c) do { if (!(c)) { wrong++; std::printf("line %d: %s\n", __LINE__, #c); } } while (0)
int main() {
  void *const first = (void *)16, *const second = (void *)17;
  int seen = -1;
  auto look = [&] { seen = current_device(); return 0; };
  EXPECT(tcu::on_stream_device("call", second, look) == 0 && seen == 1 && current_device() == 0);
  EXPECT(tcu::on_stream_device("call", first, look) == 0 && seen == 0 && current_device() == 0);
  EXPECT(tcu::on_stream_device("call", nullptr, look) == 0 && seen == 0);
  EXPECT(tcu::on_stream_device("call", second, [&] { return 2; }) == 2 && current_device() == 0);
  tcu::message = "of an earlier call";
  EXPECT(tcu::on_stream_device("call", second, [&]() -> int { throw std::bad_alloc(); }) == TCU_ERR_RUNTIME);
  EXPECT(current_device() == 0);
  EXPECT(tcu::message.find("call") == 0);
  EXPECT(tcu::on_stream_device("call", second, [&]() -> int { throw 7; }) == TCU_ERR_RUNTIME && current_device() == 0);
  refuse_move() = 3;
  EXPECT(tcu::on_stream_device("call", second, look) == TCU_ERR_RUNTIME && current_device() == 0 && tcu::message.find("refused") != std::string::npos);
  return wrong;
}
"""


def test_device_of_the_stream(tmp_path):
    if not os.path.exists(CLANG):
        pytest.skip("host clang++ (ROCm LLVM) not available")
    (tmp_path / "hip").mkdir()
    (tmp_path / "hip" / "hip_runtime.h").write_text(RUNTIME)
    (tmp_path / "check.cpp").write_text(PROGRAM)
    program = str(tmp_path / "check")
    subprocess.check_call([CLANG, "-x", "c++", "-std=c++17", "-I" + str(tmp_path), "-I" + os.path.join(HERE, "..", "tcu_scope_amd", "csrc"), "-o", program, str(tmp_path / "check.cpp")])
    got = subprocess.run([program], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout + got.stderr
