// pb_int8.hip -- product of 8-bit rows with 8-bit channels, scales for each of both.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pb_device.h"
#include "pb_elem.h"
#include "pb_hidden.h"

#pragma clang fp contract(off)

namespace pb {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef v4i Loose16 __attribute__((aligned(1), may_alias));

// 16 bytes of a row of which n are there; zeros behind them.
__device__ __forceinline__ v4i load_bytes(const int8_t* p, uint32_t n) {
  if (n >= 16u) return *reinterpret_cast<const Loose16*>(p);
  v4i v = {0, 0, 0, 0};
#pragma unroll
  for (uint32_t e = 0; e < 16; ++e)
    if (e < n) v[e / 4] |= (int)((uint32_t)(uint8_t)p[e] << (8u * (e % 4)));
  return v;
}

// 64 x 64 outputs a workgroup, 32 x 32 a wave.
template <typename Out>
__global__ __launch_bounds__(256) void int8_kernel(Int8Params p) {
  constexpr uint32_t kPitch = 80;
  __shared__ __align__(16) int8_t a[64 * kPitch], b[64 * kPitch];
  const uint32_t lane = lane_id(), wave = threadIdx.x >> 6;
  const uint32_t n0 = blockIdx.x * 64u, m0 = blockIdx.y * 64u;
  const uint32_t r = threadIdx.x >> 2, piece = (threadIdx.x & 3u) * 16u;
  const uint32_t ra = m0 + r < p.rows ? m0 + r : p.rows - 1u;
  const uint32_t rb = n0 + r < p.channels ? n0 + r : p.channels - 1u;
  const int8_t* pa = p.q + (size_t)ra * p.q_ld;
  const int8_t* pb = p.weight + (size_t)rb * p.weight_ld;
  const uint32_t wm = (wave >> 1) * 32u, wn = (wave & 1u) * 32u;
  v4i acc[2][2] = {};
  for (uint32_t k = 0; k < p.cols; k += 64u) {
    const uint32_t at = k + piece, left = at < p.cols ? p.cols - at : 0u;
    const v4i va = load_bytes(pa + at, left), vb = load_bytes(pb + at, left);
    __syncthreads();
    *reinterpret_cast<v4i*>(a + r * kPitch + piece) = va;
    *reinterpret_cast<v4i*>(b + r * kPitch + piece) = vb;
    __syncthreads();
    v4i fa[2], fb[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      fa[i] = *reinterpret_cast<const v4i*>(a + (wm + i * 16u + lane % 16u) * kPitch + lane / 16u * 16u);
      fb[i] = *reinterpret_cast<const v4i*>(b + (wn + i * 16u + lane % 16u) * kPitch + lane / 16u * 16u);
    }
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
  }
  typename Out::Raw* out = static_cast<typename Out::Raw*>(p.out);
#pragma unroll
  for (uint32_t j = 0; j < 2; ++j) {
    const uint32_t n = n0 + wn + j * 16u + lane % 16u;
    if (n >= p.channels) continue;
    const float ws = p.weight_scale[n], bias = p.bias ? p.bias[n] : 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        const uint32_t m = m0 + wm + i * 16u + lane / 16u * 4u + e;
        if (m >= p.rows) continue;
        float y = (float)acc[i][j][e] * p.scale[m] * ws;
        if (p.bias) y = y + bias;
        out[(size_t)m * p.out_ld + n] = Out::raw(y);
      }
    }
  }
}

template <typename Out>
hipError_t int8_as(const Int8Params& p, hipStream_t stream) {
  const dim3 grid((p.channels + 63u) / 64u, (p.rows + 63u) / 64u);
  int8_kernel<Out><<<grid, 256, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_int8(const Int8Params& p, uint32_t out_dtype, hipStream_t stream) {
  if (out_dtype == PB_F32) return int8_as<F32>(p, stream);
  if (out_dtype == PB_F16) return int8_as<F16>(p, stream);
  return int8_as<BF16>(p, stream);
}

}  // namespace pb
