// wfe_capi_util.h -- what the files with C entry points share.
#pragma once
#include <hip/hip_runtime.h>

struct wfe_context;

namespace wfe {

// Keeps the text for wfe_last_error (h == null: this thread's) and returns `code`.
int fail(wfe_context* h, int code, const char* fmt, ...);

struct DeviceGuard {
  int prev = -1;
  bool ok = true;
  explicit DeviceGuard(int dev) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    if (prev != dev) ok = hipSetDevice(dev) == hipSuccess;
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && hipGetDevice(&cur) == hipSuccess && cur != prev) (void)hipSetDevice(prev);
  }
};

}  // namespace wfe
