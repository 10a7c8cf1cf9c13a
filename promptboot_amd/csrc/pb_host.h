// pb_host.h -- error records and the device guard shared by the host side of the C ABI.
#pragma once

#include <hip/hip_runtime.h>
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

inline uint32_t device_error(pb_inference_error* e, hipError_t code) {
  set_error(e, PB_DEVICE, PB_DOMAIN_NONE, 0, (uint64_t)code, PB_FIELD_NONE, 0);
  return PB_DEVICE;
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
