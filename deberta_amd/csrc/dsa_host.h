// dsa_host.h — host helpers shared by the library's translation units: the
// thread's error text, argument checks and the launch check.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/dsa.h"

namespace dsa {
namespace host {

// description of the calling thread's last error (dsa_last_error)
inline thread_local std::string g_err;

[[maybe_unused]] static int fail(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
[[maybe_unused]] static int fail(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_err = buf;
  return 1;
}

[[maybe_unused]] static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

[[maybe_unused]] static size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

[[maybe_unused]] static int round_up(int x, int a) { return (x + a - 1) / a * a; }

[[maybe_unused]] static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

[[maybe_unused]] static int elem_bytes(int dtype) { return dtype == DSA_BF16 ? 2 : 4; }

[[maybe_unused]] static bool dtype_ok(int dt) { return dt == DSA_F32 || dt == DSA_BF16; }

[[maybe_unused]] static int launch_check(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail("dsa: %s launch failed: %s", what, hipGetErrorString(e));
  return 0;
}

// Refuses a stream that is being captured into a HIP graph: capturing the
// library's launches ended in a host fault inside the runtime's capture end
// whose cause is not known, so the library does not run under capture.
[[maybe_unused]] static int refuse_capture(hipStream_t st, const char* what) {
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(st, &cs) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  if (cs != hipStreamCaptureStatusNone)
    return fail("%s: the stream is capturing a HIP graph; the library's launches are not supported under graph capture",
                what);
  return 0;
}

}  // namespace host
}  // namespace dsa
