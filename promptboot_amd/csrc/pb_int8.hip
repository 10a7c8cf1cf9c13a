// pb_int8.hip -- product of 8-bit rows with 8-bit channels, scales for each of both.
//
// out[m][n] = scale[m] weight_scale[n] sum_k q[m][k] w[n][k] (+ bias[n]).  The sums are
// exact in the matrix instructions' 32-bit whole numbers (32,768 products of at most
// 2^14), so neither the order nor the split of the contraction matters, and the lanes of
// an instruction may take any 16 of its slots as long as both operands agree.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pb_device.h"
#include "pb_elem.h"
#include "pb_hidden.h"

#pragma clang fp contract(off)

namespace pb {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef v4i Loose16 __attribute__((aligned(1), may_alias));
typedef uint32_t Loose32 __attribute__((aligned(2), may_alias));

__device__ __forceinline__ v4i load_whole(const int8_t* p) {
  return *reinterpret_cast<const Loose16*>(p);
}
// 16 bytes of a row of which n are there; zeros behind them.
__device__ __forceinline__ v4i load_bytes(const int8_t* p, uint32_t n) {
  if (n >= 16u) return load_whole(p);
  v4i v = {0, 0, 0, 0};
#pragma unroll
  for (uint32_t e = 0; e < 16; ++e)
    if (e < n) v[e / 4] |= (int)((uint32_t)(uint8_t)p[e] << (8u * (e % 4)));
  return v;
}

__device__ __forceinline__ float scaled(int sum, float s, float ws, const float* bias, float b) {
  const float y = (float)sum * s * ws;
  return bias != nullptr ? y + b : y;
}

// ---- few rows: bound by the weights' bytes ----
//
// v_mfma_i32_16x16x64_i8 on operands that come straight from memory: lane l holds row (A)
// or channel (B) l % 16 and the 16 bytes at 16 (l / 16) of the step's 64, so that a load
// takes 64 neighbouring bytes of each of 16 channels.  Result register i of the lane is
// D[4 (l / 16) + i][l % 16].  A wave takes NT x 16 channels and all rows (MT x 16), or
// the split-th part of the contraction of them; the waves of a workgroup that share their
// channels add up through LDS.
template <typename Out, int MT, int NT>
__global__ __launch_bounds__(512) void int8_few_kernel(Int8Params p, uint32_t split) {
  constexpr int U = MT <= 2 ? 4 : 2;  // steps in flight beside those in use
  extern __shared__ int partial[];    // [waves][MT][NT][4][64]
  const uint32_t lane = lane_id();
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t waves = blockDim.x >> 6, own = waves / split;
  const uint32_t group = blockIdx.x * own + wave / split, part = wave % split;
  const uint32_t n0 = group * (16u * NT);
  const uint32_t steps = (p.cols + 63u) / 64u, per = (steps + split - 1u) / split;
  const uint32_t piece = lane / 16u * 16u;
  const int8_t* pw[NT];
  const int8_t* pq[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const uint32_t n = n0 + j * 16u + lane % 16u;
    pw[j] = p.weight + (size_t)(n < p.channels ? n : p.channels - 1u) * p.weight_ld + piece;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const uint32_t m = i * 16u + lane % 16u;
    pq[i] = p.q + (size_t)(m < p.rows ? m : p.rows - 1u) * p.q_ld + piece;
  }
  v4i acc[MT][NT] = {};
  const uint32_t from = part * per, to = from + per < steps ? from + per : steps;
  const uint32_t whole = p.cols / 64u;  // steps that no row ends in
  const uint32_t stop = to < whole ? to : whole;
  uint32_t step = from;
  auto multiply = [&](const v4i (&q)[MT], const v4i (&w)[NT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[i], w[j], acc[i][j], 0, 0, 0);
  };
  v4i q[2][U][MT], w[2][U][NT];
  auto fetch = [&](int set, uint32_t at) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < NT; ++j) w[set][u][j] = load_whole(pw[j] + (size_t)(at + u) * 64u);
#pragma unroll
      for (int i = 0; i < MT; ++i) q[set][u][i] = load_whole(pq[i] + (size_t)(at + u) * 64u);
    }
  };
  auto use = [&](int set) {
#pragma unroll
    for (int u = 0; u < U; ++u) multiply(q[set][u], w[set][u]);
  };
  if (step + U <= stop) {
    fetch(0, step);
    while (true) {
      const bool second = step + 2u * U <= stop;
      if (second) fetch(1, step + U);
      use(0);
      step += U;
      if (!second) break;
      const bool third = step + 2u * U <= stop;
      if (third) fetch(0, step + U);
      use(1);
      step += U;
      if (!third) break;
    }
  }
  for (; step < to; ++step) {
    const uint32_t at = step * 64u, left = at + piece < p.cols ? p.cols - at - piece : 0u;
    v4i a[MT], b[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) b[j] = load_bytes(pw[j] + at, left);
#pragma unroll
    for (int i = 0; i < MT; ++i) a[i] = load_bytes(pq[i] + at, left);
    multiply(a, b);
  }
  if (split > 1) {
    int* to_lds = partial + (size_t)wave * (MT * NT * 256);
    if (part != 0) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) to_lds[((i * NT + j) * 4 + e) * 64 + lane] = acc[i][j][e];
    }
    __syncthreads();
    if (part != 0) return;
    for (uint32_t s = 1; s < split; ++s) {
      to_lds += MT * NT * 256;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] += to_lds[((i * NT + j) * 4 + e) * 64 + lane];
    }
  }
  typename Out::Raw* out = static_cast<typename Out::Raw*>(p.out);
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const uint32_t n = n0 + j * 16u + lane % 16u;
    if (n >= p.channels) continue;
    const float ws = p.weight_scale[n], bias = p.bias ? p.bias[n] : 0.0f;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        const uint32_t m = i * 16u + lane / 16u * 4u + e;
        if (m < p.rows)
          out[(size_t)m * p.out_ld + n] = Out::raw(scaled(acc[i][j][e], p.scale[m], ws, p.bias, bias));
      }
    }
  }
}

// ---- many rows: tiles through LDS ----
//
// Four waves, WM x WN of them, each with BM x BN blocks of v_mfma_i32_32x32x32_i8: lane
// 32 h + j holds row or channel j and the 16 bytes at 16 h of 32, result register i is
// D[8 (i / 4) + 4 h + i % 4][j].  64 bytes of every row and channel are in LDS at a time,
// twice: while one set is multiplied, the next comes through registers (rows may start at
// any byte).  A row's four pieces of 16 bytes lie swapped by the row's number, so that
// eight neighbouring lanes reach all of 128 bytes.
template <typename Out, int WM, int WN, int BM, int BN>
__global__ __launch_bounds__(256, 2) void int8_tile_kernel(Int8Params p, uint32_t m_tiles,
                                                           uint32_t n_tiles) {
  static_assert(WM * WN == 4, "four waves");
  constexpr uint32_t TM = WM * BM * 32, TN = WN * BN * 32;
  constexpr uint32_t CM = TM / 64, CN = TN / 64;  // pieces a thread brings
  __shared__ __align__(16) int8_t lds[2][(TM + TN) * 64];
  __shared__ float row_scale[TM];
  const uint32_t lane = lane_id();
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  // an XCD takes neighbouring tiles, and all row tiles of a channel tile one after the other
  const uint32_t item = xcd_contiguous_item(blockIdx.x, m_tiles * n_tiles);
  const uint32_t m0 = item % m_tiles * TM, n0 = item / m_tiles * TN;
  for (uint32_t r = threadIdx.x; r < TM; r += 256u)
    row_scale[r] = m0 + r < p.rows ? p.scale[m0 + r] : 0.0f;

  const uint32_t r0 = threadIdx.x >> 2, piece = (threadIdx.x & 3u) * 16u;
  const uint32_t swapped = r0 * 64u + (piece ^ (r0 >> 1 & 3u) * 16u);
  const int8_t* pq[CM];
  const int8_t* pw[CN];
#pragma unroll
  for (uint32_t i = 0; i < CM; ++i) {
    const uint32_t r = m0 + r0 + i * 64u;
    pq[i] = p.q + (size_t)(r < p.rows ? r : p.rows - 1u) * p.q_ld + piece;
  }
#pragma unroll
  for (uint32_t i = 0; i < CN; ++i) {
    const uint32_t r = n0 + r0 + i * 64u;
    pw[i] = p.weight + (size_t)(r < p.channels ? r : p.channels - 1u) * p.weight_ld + piece;
  }
  v4i vq[CM], vw[CN];
  auto fetch = [&](uint32_t k) {
    if (k + 64u <= p.cols) {
#pragma unroll
      for (uint32_t i = 0; i < CM; ++i) vq[i] = load_whole(pq[i] + k);
#pragma unroll
      for (uint32_t i = 0; i < CN; ++i) vw[i] = load_whole(pw[i] + k);
    } else {
      const uint32_t left = k + piece < p.cols ? p.cols - k - piece : 0u;
#pragma unroll
      for (uint32_t i = 0; i < CM; ++i) vq[i] = load_bytes(pq[i] + k, left);
#pragma unroll
      for (uint32_t i = 0; i < CN; ++i) vw[i] = load_bytes(pw[i] + k, left);
    }
  };
  auto keep = [&](int8_t* to) {
#pragma unroll
    for (uint32_t i = 0; i < CM; ++i) *reinterpret_cast<v4i*>(to + i * 4096u + swapped) = vq[i];
#pragma unroll
    for (uint32_t i = 0; i < CN; ++i)
      *reinterpret_cast<v4i*>(to + TM * 64u + i * 4096u + swapped) = vw[i];
  };
  const uint32_t wm = wave / WN * (BM * 32u), wn = wave % WN * (BN * 32u);
  const uint32_t j = lane & 31u, h = lane >> 5;
  v16i acc[BM][BN] = {};
  auto multiply = [&](const int8_t* from) {
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s) {
      const uint32_t at = j * 64u + ((2u * s + h) ^ (j >> 1 & 3u)) * 16u;
      v4i a[BM], b[BN];
#pragma unroll
      for (int i = 0; i < BM; ++i)
        a[i] = *reinterpret_cast<const v4i*>(from + (wm + i * 32u) * 64u + at);
#pragma unroll
      for (int i = 0; i < BN; ++i)
        b[i] = *reinterpret_cast<const v4i*>(from + (TM + wn + i * 32u) * 64u + at);
#pragma unroll
      for (int i = 0; i < BM; ++i)
#pragma unroll
        for (int k = 0; k < BN; ++k)
          acc[i][k] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[k], acc[i][k], 0, 0, 0);
    }
  };
  fetch(0);
  keep(lds[0]);
  __syncthreads();
  uint32_t set = 0;
  for (uint32_t k = 64; k < p.cols; k += 64u) {
    fetch(k);
    multiply(lds[set]);
    set ^= 1u;
    keep(lds[set]);
    __syncthreads();
  }
  multiply(lds[set]);

  // A lane's results are of one channel, 32 lanes' of neighbouring ones: 128 bytes of a
  // row in 32 bits.  In 16 bits, lanes of two neighbouring channels change a row's
  // value for another's, so that each stores both channels of one row.
  typename Out::Raw* out = static_cast<typename Out::Raw*>(p.out);
#pragma unroll
  for (int k = 0; k < BN; ++k) {
    const uint32_t n = n0 + wn + k * 32u + j;
    const bool real = n < p.channels;
    const float ws = real ? p.weight_scale[n] : 0.0f;
    const float bias = real && p.bias ? p.bias[n] : 0.0f;
#pragma unroll
    for (int i = 0; i < BM; ++i) {
#pragma unroll
      for (uint32_t e = 0; e < 16; e += 4) {
        const uint32_t r = wm + i * 32u + e * 2u + h * 4u;
        float y[4];
#pragma unroll
        for (uint32_t f = 0; f < 4; ++f)
          y[f] = scaled(acc[i][k][e + f], row_scale[r + f], ws, p.bias, bias);
        if constexpr (Out::kPer == 4) {
#pragma unroll
          for (uint32_t f = 0; f < 4; ++f)
            if (real && m0 + r + f < p.rows)
              out[(size_t)(m0 + r + f) * p.out_ld + n] = Out::raw(y[f]);
        } else {
          const bool odd = (lane & 1u) != 0;
#pragma unroll
          for (uint32_t f = 0; f < 4; f += 2) {
            const float give = odd ? y[f] : y[f + 1], mine = odd ? y[f + 1] : y[f];
            const float got = f_of(lane_xor(b_of(give), 1, lane));
            const uint32_t both = odd ? Out::two(got, mine) : Out::two(mine, got);
            const uint32_t m = m0 + r + f + (odd ? 1u : 0u), first = n & ~1u;
            if (m < p.rows && first < p.channels) {
              typename Out::Raw* to = out + (size_t)m * p.out_ld + first;
              if (first + 1u < p.channels) *reinterpret_cast<Loose32*>(to) = both;
              else *to = (typename Out::Raw)both;
            }
          }
        }
      }
    }
  }
}

template <typename Out, int MT, int NT>
hipError_t few_as(const Int8Params& p, hipStream_t stream) {
  const uint32_t groups = (p.channels + 16u * NT - 1u) / (16u * NT);
  const uint32_t steps = (p.cols + 63u) / 64u;
  uint32_t split = 1;
  while (split < 8 && groups * split < 4096 && steps / (2 * split) >= 4) split *= 2;
  const uint32_t waves = split > 4 ? split : 4, own = waves / split;
  const size_t lds = split > 1 ? (size_t)waves * MT * NT * 1024 : 0;
  int8_few_kernel<Out, MT, NT><<<(groups + own - 1u) / own, waves * 64u, lds, stream>>>(p, split);
  return hipGetLastError();
}

template <typename Out, int WM, int WN, int BM, int BN>
hipError_t tile_as(const Int8Params& p, hipStream_t stream) {
  const uint32_t m_tiles = (p.rows + WM * BM * 32u - 1u) / (WM * BM * 32u);
  const uint32_t n_tiles = (p.channels + WN * BN * 32u - 1u) / (WN * BN * 32u);
  int8_tile_kernel<Out, WM, WN, BM, BN><<<m_tiles * n_tiles, 256, 0, stream>>>(p, m_tiles, n_tiles);
  return hipGetLastError();
}

template <typename Out>
hipError_t int8_as(const Int8Params& p, hipStream_t stream) {
  if (p.rows <= 16) return few_as<Out, 1, 1>(p, stream);
  if (p.rows <= 32) return few_as<Out, 2, 1>(p, stream);
  if (p.rows <= 48) return few_as<Out, 3, 2>(p, stream);
  if (p.rows <= 64) return few_as<Out, 4, 2>(p, stream);
  const uint64_t outputs = (uint64_t)p.rows * p.channels;
  if (outputs >= (uint64_t)512 * 256 * 128) return tile_as<Out, 2, 2, 4, 2>(p, stream);
  if (outputs >= (uint64_t)512 * 128 * 128) return tile_as<Out, 2, 2, 2, 2>(p, stream);
  return tile_as<Out, 2, 2, 1, 1>(p, stream);
}

}  // namespace

hipError_t launch_int8(const Int8Params& p, uint32_t out_dtype, hipStream_t stream) {
  if (out_dtype == PB_F32) return int8_as<F32>(p, stream);
  if (out_dtype == PB_F16) return int8_as<F16>(p, stream);
  return int8_as<BF16>(p, stream);
}

}  // namespace pb
