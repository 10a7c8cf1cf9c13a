// pb_host.h -- error records, overlaps of buffers and the device guard shared by the host
// side of the C ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include "pbsample.h"

namespace pb {

inline void set_error(pb_inference_error* e, uint32_t status, uint32_t domain, uint64_t needed,
               uint64_t available, uint32_t kind, uint32_t sub) {
  if (!e) return;
  e->status = status;
  e->domain = domain;
  e->layer = PB_NO_LAYER;
  e->position = 0;
  e->tensor_id = PB_NO_TENSOR;
  e->reserved = 0;
  e->needed = needed;
  e->available = available;
  e->detail = ((uint64_t)kind << 32) | sub;
}

inline void clear_error(pb_inference_error* e) {
  if (e) memset(e, 0, sizeof *e);
}

// The error is returned, so the runtime's note of it is taken back: the next launch, of any
// library in the process, would be taken for the failure.
inline uint32_t device_error(pb_inference_error* e, hipError_t code) {
  (void)hipGetLastError();
  set_error(e, PB_DEVICE, PB_DOMAIN_NONE, 0, (uint64_t)code, PB_FIELD_NONE, 0);
  return PB_DEVICE;
}

// `rows` rows of `bytes` bytes, `step` bytes from one to the next.
struct ByteRows {
  const void* at;
  int64_t rows, bytes, step;
};

// Whether two buffers share a byte.  Rows at one distance may lie between each other
// (the columns of one buffer, or every other row of it); at two distances the ranges that
// they span are compared.  Neither is empty.
inline bool share_a_byte(const ByteRows& a, const ByteRows& b) {
  const int64_t a0 = (int64_t)(uintptr_t)a.at, b0 = (int64_t)(uintptr_t)b.at;
  const int64_t last_a = a.rows - 1, last_b = b.rows - 1;
  if (a0 >= b0 + last_b * b.step + b.bytes || b0 >= a0 + last_a * a.step + a.bytes) return false;
  if (a.step != b.step) return true;
  // row i of a and row i + k of b share a byte where -b.bytes < d + k step < a.bytes
  const int64_t d = b0 - a0, step = a.step;
  auto floor_div = [](int64_t x, int64_t y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
  int64_t lo = floor_div(-b.bytes - d, step) + 1, hi = floor_div(a.bytes - 1 - d, step);
  if (lo < -last_a) lo = -last_a;
  if (hi > last_b) hi = last_b;
  return lo <= hi;
}

// Restores the caller's current device on scope exit.
struct DeviceGuard {
  int saved = -1;
  explicit DeviceGuard(int device) {
    if (hipGetDevice(&saved) != hipSuccess) saved = -1;
    if (device >= 0 && device != saved) (void)hipSetDevice(device);
  }
  ~DeviceGuard() {
    int now = -1;
    if (saved >= 0 && hipGetDevice(&now) == hipSuccess && now != saved) (void)hipSetDevice(saved);
  }
};

}  // namespace pb
