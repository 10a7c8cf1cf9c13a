// pb_elem.h -- element types of rows (binary32, binary16, bfloat16) and their 16-byte accesses.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pb_device.h"

#pragma clang fp contract(off)

namespace pb {

// ---- element types: 16 bytes are one chunk ----

struct F32 {
  using Raw = uint32_t;
  static constexpr int kPer = 4;
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    return f_of(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ float one(Raw r) { return f_of(r); }
  static __device__ __forceinline__ Raw raw(float f) { return b_of(f); }
  static __device__ __forceinline__ uint4 pack(const float (&f)[kPer]) {
    return make_uint4(b_of(f[0]), b_of(f[1]), b_of(f[2]), b_of(f[3]));
  }
};

__device__ __forceinline__ uint32_t word_of(const uint4& v, int w) {
  return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w;
}

struct BF16 {
  using Raw = uint16_t;
  static constexpr int kPer = 8;
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    const uint32_t w = word_of(v, e >> 1);
    return f_of((e & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ float one(Raw r) { return f_of((uint32_t)r << 16); }
  static __device__ __forceinline__ Raw raw(float f) {
    return __builtin_bit_cast(uint16_t, (__bf16)f);
  }
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2));
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[kPer]) {
    return make_uint4(two(f[0], f[1]), two(f[2], f[3]), two(f[4], f[5]), two(f[6], f[7]));
  }
};

struct F16 {
  using Raw = uint16_t;
  static constexpr int kPer = 8;
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    const uint32_t w = word_of(v, e >> 1);
    return one((uint16_t)((e & 1) ? (w >> 16) : w));
  }
  static __device__ __forceinline__ float one(Raw r) {
    return (float)__builtin_bit_cast(_Float16, r);
  }
  static __device__ __forceinline__ Raw raw(float f) {
    return __builtin_bit_cast(uint16_t, (_Float16)f);
  }
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    return (uint32_t)raw(a) | ((uint32_t)raw(b) << 16);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[kPer]) {
    return make_uint4(two(f[0], f[1]), two(f[2], f[3]), two(f[4], f[5]), two(f[6], f[7]));
  }
};

// Rows start at any element: 16-byte accesses that are aligned to an element only.
typedef uint32_t Words4 __attribute__((ext_vector_type(4)));
typedef Words4 Loose4 __attribute__((aligned(2), may_alias));
template <typename E>
__device__ __forceinline__ uint4 load_chunk(const typename E::Raw* p) {
  const Words4 v = *reinterpret_cast<const Loose4*>(p);
  return make_uint4(v.x, v.y, v.z, v.w);
}
// The same for data that is not needed again.
template <typename E>
__device__ __forceinline__ uint4 stream_chunk(const typename E::Raw* p) {
  const Words4 v = __builtin_nontemporal_load(reinterpret_cast<const Loose4*>(p));
  return make_uint4(v.x, v.y, v.z, v.w);
}
// A store of what the launch does not read again: past the caches.
template <typename E>
__device__ __forceinline__ void store_chunk(typename E::Raw* p, const uint4& v) {
  __builtin_nontemporal_store(Words4{v.x, v.y, v.z, v.w}, reinterpret_cast<Loose4*>(p));
}

}  // namespace pb
