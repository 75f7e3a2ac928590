// abi.hpp -- what the entry points of the separate operators share: error returns, type codes, and the
// device copies of a host call's buffers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/t5hip.h"

#define HIP_OK(expr)                                                                   \
  do {                                                                                 \
    hipError_t e_ = (expr);                                                            \
    if (e_ != hipSuccess)                                                              \
      return fail(T5H_ERR_HIP, std::string(#expr ": ") + hipGetErrorString(e_));       \
  } while (0)

#define TRY(expr)                   \
  do {                              \
    if (int rc_ = (expr)) return rc_; \
  } while (0)

namespace t5h_detail {
int fail(int code, const std::string& msg);

inline size_t type_bytes(int32_t t) { return t == T5H_TYPE_F32 ? 4 : 2; }
inline bool known_type(int32_t t) { return t == T5H_TYPE_F32 || t == T5H_TYPE_F16 || t == T5H_TYPE_BF16; }

// Rows of `width` bytes, `stride` bytes apart.
struct Rows {
  uintptr_t at;
  uint64_t width, stride;
  const char* name;
};
// Whether some row of a shares a byte with some row of b: rows of one stride, by where the second's lie
// between the first's; otherwise by all that the rows span.
inline bool overlap(const Rows& a, const Rows& b, uint64_t rows) {
  const uintptr_t a_end = a.at + (rows - 1) * a.stride + a.width, b_end = b.at + (rows - 1) * b.stride + b.width;
  if (a_end <= b.at || b_end <= a.at) return false;
  if (rows == 1 || a.stride != b.stride) return true;
  const uint64_t d = a.at <= b.at ? (b.at - a.at) % a.stride : (a.stride - (a.at - b.at) % a.stride) % a.stride;
  return d < a.width || d + b.width > a.stride;
}


// Device copies of a host call's buffers: one allocation, parts on 256-byte boundaries, freed on every
// path.  Outputs are cleared first, so that the scales' unused rows come back as zeros.
struct HostCall {
  char* p = nullptr;
  size_t used = 0;
  HostCall() = default;
  HostCall(const HostCall&) = delete;
  HostCall& operator=(const HostCall&) = delete;
  ~HostCall() {
    if (p) (void)hipFree(p);
  }
  size_t part(size_t bytes) {
    const size_t at = used;
    used += (bytes + 255) & ~(size_t)255;
    return at;
  }
  int open(int32_t dev) {
    int ndev = 0;
    if (hipGetDeviceCount(&ndev) != hipSuccess || ndev <= 0) return fail(T5H_ERR_NODEVICE, "no HIP device");
    HIP_OK(hipSetDevice(dev < 0 ? 0 : dev));
    if (hipMalloc((void**)&p, used) != hipSuccess) {
      p = nullptr;
      return fail(T5H_ERR_NOMEM, "device buffers of a host call");
    }
    HIP_OK(hipMemset(p, 0, used));
    return T5H_OK;
  }
  int up(size_t at, const void* from, size_t bytes) {
    HIP_OK(hipMemcpy(p + at, from, bytes, hipMemcpyHostToDevice));
    return T5H_OK;
  }
  int down(void* to, size_t at, size_t bytes) {
    HIP_OK(hipMemcpy(to, p + at, bytes, hipMemcpyDeviceToHost));
    return T5H_OK;
  }
};
}  // namespace t5h_detail
