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

__device__ __forceinline__ v4i load_whole(const int8_t* p) {
  return *reinterpret_cast<const Loose16*>(p);
}
// The 16 bytes at `at` of a row of `cols` bytes, zeros behind its end.  A row's last piece is
// taken from the row's last 16 bytes and shifted: byte by byte it cost 333 rows of 1,001
// bytes 11 of 59 us.
__device__ __forceinline__ v4i load_piece(const int8_t* row, uint32_t at, uint32_t cols) {
  if (at + 16u <= cols) return load_whole(row + at);
  v4i v = {0, 0, 0, 0};
  if (at >= cols) return v;
  if (cols < 16u) {
    for (uint32_t e = 0; e < cols; ++e)
      v[e / 4] |= (int)((uint32_t)(uint8_t)row[e] << (8u * (e % 4)));
    return v;
  }
  const uint32_t out = at + 16u - cols;  // bytes that another piece has
  v = load_whole(row + cols - 16u);
  if (out & 8u) v = v4i{v[2], v[3], 0, 0};
  if (out & 4u) v = v4i{v[1], v[2], v[3], 0};
  const uint32_t shift = out & 3u;
  return v4i{(int)__builtin_amdgcn_alignbyte((uint32_t)v[1], (uint32_t)v[0], shift),
             (int)__builtin_amdgcn_alignbyte((uint32_t)v[2], (uint32_t)v[1], shift),
             (int)__builtin_amdgcn_alignbyte((uint32_t)v[3], (uint32_t)v[2], shift),
             (int)__builtin_amdgcn_alignbyte(0u, (uint32_t)v[3], shift)};
}

// A channel without a bias has -0, which leaves every number as it is.
constexpr float kNoBias = -0.0f;
__device__ __forceinline__ float scaled(int sum, float s, float ws, float bias) {
  return (float)sum * s * ws + bias;
}

// ---- few rows of short products ----
//
// v_mfma_i32_16x16x64_i8 on operands that come straight from memory: lane l holds row (A)
// or channel (B) l % 16 and the 16 bytes at 16 (l / 16) of the step's 64, so that a load
// takes 64 neighbouring bytes of each of 16 channels.  Result register i of the lane is
// D[4 (l / 16) + i][l % 16].  A wave takes 16 channels and all rows, or the split-th part
// of the contraction of them; the waves of a workgroup that share their channels add up
// through LDS.  No barrier stands between a load and its use, so that a short product is
// little more than a launch and two round trips.  1 x 151,936 x 896: 25.7 us, 5.3 TB/s of
// weights; 1 x 4,096 x 4,096: 5.5 us; 16 x 1,000 x 4,096: 6.2.
constexpr uint32_t kFewWaves = 4;
template <typename Out>
__global__ __launch_bounds__(64 * kFewWaves) void int8_few_kernel(Int8Params p, uint32_t split) {
  constexpr uint32_t U = 4;  // steps on their way beside those in use
  __shared__ int sums[kFewWaves][4][64];
  const uint32_t lane = lane_id();
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t part = wave % split;
  const uint32_t n = (blockIdx.x * (kFewWaves / split) + wave / split) * 16u + lane % 16u;
  const uint32_t m = lane % 16u, piece = lane / 16u * 16u;
  const int8_t* pw = p.weight + (size_t)(n < p.channels ? n : p.channels - 1u) * p.weight_ld;
  const int8_t* pq = p.q + (size_t)(m < p.rows ? m : p.rows - 1u) * p.q_ld;
  const uint32_t steps = (p.cols + 63u) / 64u, per = (steps + split - 1u) / split;
  const uint32_t from = part * per, to = from + per < steps ? from + per : steps;
  v4i acc = {};
  v4i q[2][U], w[2][U];
  auto fetch = [&](int set, uint32_t step) {
    if (step + U <= to && (step + U) * 64u <= p.cols) {
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        w[set][u] = load_whole(pw + (step + u) * 64u + piece);
        q[set][u] = load_whole(pq + (step + u) * 64u + piece);
      }
    } else {
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        const uint32_t at = step + u < to ? (step + u) * 64u + piece : p.cols;
        w[set][u] = load_piece(pw, at, p.cols);
        q[set][u] = load_piece(pq, at, p.cols);
      }
    }
  };
  auto use = [&](int set) {
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[set][u], w[set][u], acc, 0, 0, 0);
  };
  if (from < to) fetch(0, from);
  for (uint32_t step = from; step < to; step += 2u * U) {
    if (step + U < to) fetch(1, step + U);
    use(0);
    if (step + U < to) {
      if (step + 2u * U < to) fetch(0, step + 2u * U);
      use(1);
    }
  }
  if (split > 1) {
    if (part != 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[wave][e][lane] = acc[e];
    }
    __syncthreads();
    if (part != 0) return;
    for (uint32_t s = 1; s < split; ++s) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += sums[wave + s][e][lane];
    }
  }
  if (n >= p.channels) return;
  const float ws = p.weight_scale[n], bias = p.bias ? p.bias[n] : kNoBias;
  typename Out::Raw* out = static_cast<typename Out::Raw*>(p.out) + n;
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) {
    const uint32_t r = lane / 16u * 4u + e;
    if (r < p.rows)
      out[(size_t)r * p.out_ld] = Out::raw(scaled(acc[e], p.scale[r], ws, bias));
  }
}

// ---- many rows: tiles through LDS ----
//
// v_mfma_i32_32x32x32_i8 with the channels as A and the rows as B: lane 32 h + j holds
// channel or row j and the 16 bytes at 16 h of 32, and result register i is the sum of
// channel 8 (i / 4) + 4 h + i % 4 and row j: four neighbouring channels of one row.
// KB bytes of every row and channel of a tile are in LDS at a time, twice: while one set
// is multiplied the next is on its way.  The pieces of 16 bytes of a row lie swapped by
// the row's number, so that the 16 rows that 16 lanes read together lie in 16 different
// places of 256 bytes (with one swap for two rows, half of the LDS cycles were conflicts).
template <int WM, int WN, int BM, int BN>
struct Tile {
  static constexpr uint32_t kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr uint32_t kRows = WM * BM * 32, kChannels = WN * BN * 32;
};

// Where piece `piece` of row `row` lies in a set whose rows are KB bytes.
template <uint32_t KB>
__device__ __forceinline__ uint32_t piece_at(uint32_t row, uint32_t piece) {
  static_assert(KB == 64 || KB == 128 || KB == 256, "four, eight or sixteen pieces");
  constexpr uint32_t kPieces = KB / 16u;
  return row * KB + (piece ^ (row / (16u / kPieces) & (kPieces - 1u))) * 16u;
}

// The tile of a workgroup.  An XCD takes neighbouring tiles, and the row tiles of a group
// one after the other for each channel tile, so that a group's rows stay in its L2: about
// 1 MB, or four tiles (4,096 x 151,936 x 896 by groups of 1, 2, 4, 8 and 16 tiles of 256
// rows: 743, 727, 717, 717 and 731 us).
struct TilePlan {
  uint32_t m_tiles, n_tiles, group;
};
__device__ __forceinline__ void tile_of(const TilePlan& t, uint32_t linear, uint32_t* m,
                                        uint32_t* n) {
  const uint32_t item = xcd_contiguous_item(linear, t.m_tiles * t.n_tiles);
  const uint32_t whole = t.group * t.n_tiles, g = item / whole, in_group = item - g * whole;
  const uint32_t left = t.m_tiles - g * t.group, rows = left < t.group ? left : t.group;
  *m = g * t.group + in_group % rows;
  *n = in_group / rows;
}

// A wave's part of one set's products: blocks of its rows and channels, and the part `wk` of
// WK of the set's bytes.
template <uint32_t KB, uint32_t TM, int WK, int BM, int BN>
__device__ __forceinline__ void multiply_set(const int8_t* set, uint32_t wm, uint32_t wn,
                                             uint32_t wk, v16i (&acc)[BM][BN]) {
  constexpr uint32_t kSteps = KB / 32u / WK;
  const uint32_t j = lane_id() & 31u, h = lane_id() >> 5;
#pragma unroll
  for (uint32_t s = 0; s < kSteps; ++s) {
    const uint32_t at = piece_at<KB>(j, 2u * (wk * kSteps + s) + h);
    v4i a[BM], b[BN];
#pragma unroll
    for (int i = 0; i < BM; ++i)
      a[i] = *reinterpret_cast<const v4i*>(set + (wm + i * 32u) * KB + at);
#pragma unroll
    for (int k = 0; k < BN; ++k)
      b[k] = *reinterpret_cast<const v4i*>(set + (TM + wn + k * 32u) * KB + at);
#pragma unroll
    for (int i = 0; i < BM; ++i)
#pragma unroll
      for (int k = 0; k < BN; ++k)
        acc[i][k] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[k], a[i], acc[i][k], 0, 0, 0);
  }
}

// Scales and stores a wave's sums.  They go through LDS (kSliceBytes a wave), 128 bytes of
// 32 rows at a time, so that eight lanes store 128 neighbouring bytes: with one element a
// lane (64 bytes of a row together) 4,096 x 151,936 bf16 logits alone took 594 us, so 356.
// They go past the caches (262 us) where those 128 bytes are whole lines of 64, and through
// them where they are not: there a line is put together from two stores, and memory takes
// half lines badly.  With the product, past and through the caches:
//   4,096 x 512 by 100,032 channels, rows of lines    bf16  322 / 350 us   fp32  399 /  465
//              by 100,016 (32 bytes left / lines)           347 / 378            433 /  535
//              by 100,008 (16 bytes left / 32)              430 / 390            916 /  624
//              by 100,001 (2 bytes left / 4)                516 / 394          1,390 /  667
//   333 x 1,001 by 50,304                                  44.6 / 46.9          46.5 / 65.4
//              by 50,257                                   54.4 / 46.5          76.4 / 65.7
constexpr uint32_t kLine = 64;
constexpr uint32_t kSlicePitch = 144, kSliceBytes = 32 * kSlicePitch;
template <typename Out, bool kPast, int BM, int BN>
__device__ __forceinline__ void store_by(const Int8Params& p, int8_t* slice,
                                         const float* chan_scale, const float* chan_bias,
                                         uint32_t m0, uint32_t n0, uint32_t wn,
                                         const float (&row_scale)[BM],
                                         const v16i (&acc)[BM][BN]) {
  constexpr uint32_t kSize = 16 / Out::kPer;           // bytes of an element
  constexpr int kWhole = 128 / (32 * (int)kSize);
  constexpr int kBlocks = BN < kWhole ? BN : kWhole;  // blocks of channels of a slice
  static_assert(BN % kBlocks == 0, "whole slices");
  constexpr uint32_t kLanes = kBlocks * 2u * kSize, kAtOnce = 64u / kLanes;  // a row's, and rows
  const uint32_t lane = lane_id(), j = lane & 31u, h = lane >> 5;
  typename Out::Raw* out = static_cast<typename Out::Raw*>(p.out);
  // the lane's channels: 32 k + 2 e + 4 h and the three next to it, from register e on (with
  // four blocks of rows the registers hold no biases too)
  constexpr bool kHold = BM < 4;
  float4 ws[BN][4], bs[kHold ? BN : 1][4];
#pragma unroll
  for (int k = 0; k < BN; ++k) {
#pragma unroll
    for (uint32_t e = 0; e < 16; e += 4) {
      const uint32_t c = wn + k * 32u + 2u * e + 4u * h;
      ws[k][e / 4] = *reinterpret_cast<const float4*>(chan_scale + c);
      if constexpr (kHold) bs[k][e / 4] = *reinterpret_cast<const float4*>(chan_bias + c);
    }
  }
#pragma unroll
  for (int i = 0; i < BM; ++i) {
#pragma unroll
    for (int k0 = 0; k0 < BN; k0 += kBlocks) {
#pragma unroll
      for (int k = k0; k < k0 + kBlocks; ++k) {
#pragma unroll
        for (uint32_t e = 0; e < 16; e += 4) {
          const float4 w = ws[k][e / 4];
          float4 b;
          if constexpr (kHold)
            b = bs[k][e / 4];
          else
            b = *reinterpret_cast<const float4*>(chan_bias + wn + k * 32u + 2u * e + 4u * h);
          const float y0 = scaled(acc[i][k][e], row_scale[i], w.x, b.x);
          const float y1 = scaled(acc[i][k][e + 1], row_scale[i], w.y, b.y);
          const float y2 = scaled(acc[i][k][e + 2], row_scale[i], w.z, b.z);
          const float y3 = scaled(acc[i][k][e + 3], row_scale[i], w.w, b.w);
          int8_t* to = slice + j * kSlicePitch + ((k - k0) * 32u + 2u * e + 4u * h) * kSize;
          if constexpr (kSize == 4)
            *reinterpret_cast<float4*>(to) = make_float4(y0, y1, y2, y3);
          else
            *reinterpret_cast<uint2*>(to) = make_uint2(Out::two(y0, y1), Out::two(y2, y3));
        }
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (uint32_t s = 0; s < 32u / kAtOnce; ++s) {
        const uint32_t r = s * kAtOnce + lane / kLanes, piece = lane % kLanes;
        const uint4 v = *reinterpret_cast<const uint4*>(slice + r * kSlicePitch + piece * 16u);
        const uint32_t m = m0 + i * 32u + r, n = n0 + wn + k0 * 32u + piece * Out::kPer;
        if (m < p.rows && n < p.channels) {
          typename Out::Raw* to = out + (size_t)m * p.out_ld + n;
          if (n + Out::kPer <= p.channels) {
            if constexpr (kPast)
              store_chunk<Out>(to, v);
            else
              *reinterpret_cast<Loose4*>(to) = Words4{v.x, v.y, v.z, v.w};
          } else {
#pragma unroll
            for (uint32_t e = 0; e + 1u < (uint32_t)Out::kPer; ++e)
              if (n + e < p.channels) to[e] = Out::raw(Out::get(v, e));
          }
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

template <typename Out, int BM, int BN>
__device__ __forceinline__ void store_sums(const Int8Params& p, int8_t* slice,
                                           const float* chan_scale, const float* chan_bias,
                                           uint32_t m0, uint32_t n0, uint32_t wn,
                                           const float (&row_scale)[BM],
                                           const v16i (&acc)[BM][BN]) {
  if (((uintptr_t)p.out | p.out_ld * (16 / Out::kPer)) % kLine == 0)
    store_by<Out, true>(p, slice, chan_scale, chan_bias, m0, n0, wn, row_scale, acc);
  else
    store_by<Out, false>(p, slice, chan_scale, chan_bias, m0, n0, wn, row_scale, acc);
}

// The channels' scales and biases of a tile, in LDS.
template <uint32_t kThreads, uint32_t TN>
__device__ __forceinline__ void load_channels(const Int8Params& p, uint32_t n0, float* scale,
                                              float* bias) {
  for (uint32_t c = threadIdx.x; c < TN; c += kThreads) {
    const bool real = n0 + c < p.channels;
    scale[c] = real ? p.weight_scale[n0 + c] : 0.0f;
    bias[c] = real && p.bias ? p.bias[n0 + c] : kNoBias;
  }
}

// The sums of the WK parts of a tile's contraction, in its first kWaves waves.
template <uint32_t kWaves, int WK, int BM, int BN>
__device__ __forceinline__ void join_parts(int8_t* lds, uint32_t wave, v16i (&acc)[BM][BN]) {
  constexpr uint32_t kSums = BM * BN * 16 * 64;  // of a wave
  int* sums = reinterpret_cast<int*>(lds) + lane_id();
  if (wave >= kWaves) {
#pragma unroll
    for (int i = 0; i < BM; ++i)
#pragma unroll
      for (int k = 0; k < BN; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          sums[(wave - kWaves) * kSums + ((i * BN + k) * 16 + e) * 64] = acc[i][k][e];
  }
  __syncthreads();
  if (wave < kWaves) {
#pragma unroll
    for (int g = 0; g < WK - 1; ++g)
#pragma unroll
      for (int i = 0; i < BM; ++i)
#pragma unroll
        for (int k = 0; k < BN; ++k)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            acc[i][k][e] += sums[(g * kWaves + wave) * kSums + ((i * BN + k) * 16 + e) * 64];
  }
  __syncthreads();
}

// Rows that start at any byte and end anywhere: pieces come through registers.
template <typename Out, int WM, int WN, int BM, int BN, uint32_t KB, int WK>
__global__ __launch_bounds__(64 * WM * WN * WK, 2) void int8_tile_kernel(Int8Params p,
                                                                         TilePlan plan) {
  using T = Tile<WM, WN, BM, BN>;
  constexpr uint32_t TM = T::kRows, TN = T::kChannels, kThreads = T::kThreads * WK;
  constexpr uint32_t kPieces = KB / 16u, kAtOnce = kThreads / kPieces;  // rows at a time
  constexpr uint32_t CM = TM / kAtOnce, CN = TN / kAtOnce;  // pieces a thread brings
  static_assert(TM % kAtOnce == 0 && TN % kAtOnce == 0 && kAtOnce % 16 == 0, "whole turns");
  constexpr uint32_t kSet = (TM + TN) * KB, kSlices = T::kWaves * kSliceBytes;
  static_assert(T::kWaves * (WK - 1) * BM * BN * 4096 <= 2 * kSet, "the sums fit");
  __shared__ __align__(16) int8_t lds[2 * kSet > kSlices ? 2 * kSet : kSlices];
  __shared__ __align__(16) float chan_scale[TN], chan_bias[TN];
  const uint32_t lane = lane_id();
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  uint32_t m0, n0;
  tile_of(plan, blockIdx.x, &m0, &n0);
  m0 *= TM;
  n0 *= TN;
  load_channels<kThreads, TN>(p, n0, chan_scale, chan_bias);
  const uint32_t r0 = threadIdx.x / kPieces, piece = threadIdx.x % kPieces * 16u;
  const uint32_t at = piece_at<KB>(r0, threadIdx.x % kPieces);  // kAtOnce rows on, the same swap
  const int8_t* pq[CM];
  const int8_t* pw[CN];
#pragma unroll
  for (uint32_t i = 0; i < CM; ++i) {
    const uint32_t r = m0 + r0 + i * kAtOnce;
    pq[i] = p.q + (size_t)(r < p.rows ? r : p.rows - 1u) * p.q_ld;
  }
#pragma unroll
  for (uint32_t i = 0; i < CN; ++i) {
    const uint32_t r = n0 + r0 + i * kAtOnce;
    pw[i] = p.weight + (size_t)(r < p.channels ? r : p.channels - 1u) * p.weight_ld;
  }
  v4i vq[CM], vw[CN];
  auto fetch = [&](uint32_t k) {
    if (k + KB <= p.cols) {
#pragma unroll
      for (uint32_t i = 0; i < CM; ++i) vq[i] = load_whole(pq[i] + k + piece);
#pragma unroll
      for (uint32_t i = 0; i < CN; ++i) vw[i] = load_whole(pw[i] + k + piece);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < CM; ++i) vq[i] = load_piece(pq[i], k + piece, p.cols);
#pragma unroll
      for (uint32_t i = 0; i < CN; ++i) vw[i] = load_piece(pw[i], k + piece, p.cols);
    }
  };
  auto keep = [&](int8_t* to) {
#pragma unroll
    for (uint32_t i = 0; i < CM; ++i) *reinterpret_cast<v4i*>(to + i * kAtOnce * KB + at) = vq[i];
#pragma unroll
    for (uint32_t i = 0; i < CN; ++i)
      *reinterpret_cast<v4i*>(to + (TM + i * kAtOnce) * KB + at) = vw[i];
  };
  const uint32_t wk = wave / T::kWaves, place = wave % T::kWaves;
  const uint32_t wm = place / WN * (BM * 32u), wn = place % WN * (BN * 32u);
  float row_scale[BM];
#pragma unroll
  for (int i = 0; i < BM; ++i) {
    const uint32_t m = m0 + wm + i * 32u + (lane & 31u);
    row_scale[i] = m < p.rows ? p.scale[m] : 0.0f;
  }
  v16i acc[BM][BN] = {};
  fetch(0);
  keep(lds);
  __syncthreads();
  uint32_t set = 0;
  for (uint32_t k = KB; k < p.cols; k += KB) {
    fetch(k);
    multiply_set<KB, TM, WK>(lds + set, wm, wn, wk, acc);
    set ^= kSet;
    keep(lds + set);
    __syncthreads();
  }
  multiply_set<KB, TM, WK>(lds + set, wm, wn, wk, acc);
  __syncthreads();
  if constexpr (WK > 1) {
    join_parts<T::kWaves, WK>(lds, wave, acc);
    if (wk != 0) return;
  }
  store_sums<Out>(p, lds + wave * kSliceBytes, chan_scale, chan_bias, m0 + wm, n0, wn, row_scale,
                  acc);
}

// Rows of whole, aligned pieces: they go from memory to LDS by themselves, a wave 1 KB at a
// time, lane l to the 16 bytes at 16 l.  Those loads are written in assembly, since the
// compiler would wait for all of them before each read of LDS; every wait for them stands
// here, before the barrier behind which their set is read.
__device__ const v4i kZeroPiece = {0, 0, 0, 0};  // what stands behind a row's end
__device__ __forceinline__ void to_lds(const int8_t* from, int8_t* wave_to) {
  const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)wave_to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to),
               "v"(from)
               : "memory", "m0");
}

template <typename Out, int WM, int WN, int BM, int BN, uint32_t KB, uint32_t kSets, int WK>
__global__ __launch_bounds__(64 * WM * WN * WK) void int8_pieces_kernel(Int8Params p, TilePlan plan) {
  using T = Tile<WM, WN, BM, BN>;
  constexpr uint32_t TM = T::kRows, TN = T::kChannels, kWaves = T::kWaves * WK;
  constexpr uint32_t kPieces = KB / 16u;  // of a row
  constexpr uint32_t kLoads = (TM + TN) * KB / 1024u / kWaves;  // a wave's of a set
  static_assert((TM + TN) * KB % (1024u * kWaves) == 0, "as many for every wave");
  constexpr uint32_t kSet = (TM + TN) * KB;
  static_assert(T::kWaves * kSliceBytes <= kSets * kSet, "the slices fit");
  __shared__ __align__(16) int8_t lds[kSets * kSet];
  __shared__ __align__(16) float chan_scale[TN], chan_bias[TN];
  const uint32_t lane = lane_id();
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  uint32_t m0, n0;
  tile_of(plan, blockIdx.x, &m0, &n0);
  m0 *= TM;
  n0 *= TN;
  // load i of the wave brings 1 KB of rows, a lane the piece whose place it has
  const int8_t* from[kLoads];
  uint32_t offset[kLoads];
#pragma unroll
  for (uint32_t i = 0; i < kLoads; ++i) {
    const uint32_t row = (wave * kLoads + i) * (64u / kPieces) + lane / kPieces;  // of the tile's rows, then channels
    offset[i] = piece_at<KB>(row, lane % kPieces) - row * KB;
    if (row < TM) {
      const uint32_t r = m0 + row;
      from[i] = p.q + (size_t)(r < p.rows ? r : p.rows - 1u) * p.q_ld + offset[i];
    } else {
      const uint32_t r = n0 + row - TM;
      from[i] = p.weight + (size_t)(r < p.channels ? r : p.channels - 1u) * p.weight_ld + offset[i];
    }
  }
  auto bring = [&](int8_t* set, uint32_t step) {
    const uint32_t k = step * KB;
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const int8_t* at = from[i] + k;
      if (k + KB > p.cols && k + offset[i] >= p.cols)
        at = reinterpret_cast<const int8_t*>(&kZeroPiece);
      to_lds(at, set + (wave * kLoads + i) * 1024u);
    }
  };
  const uint32_t steps = (p.cols + KB - 1u) / KB;
#pragma unroll
  for (uint32_t i = 0; i + 1u < kSets; ++i)
    if (i < steps) bring(lds + i * kSet, i);
  load_channels<64 * kWaves, TN>(p, n0, chan_scale, chan_bias);
  const uint32_t wk = wave / T::kWaves, place = wave % T::kWaves;
  const uint32_t wm = place / WN * (BM * 32u), wn = place % WN * (BN * 32u);
  float row_scale[BM];
#pragma unroll
  for (int i = 0; i < BM; ++i) {
    const uint32_t m = m0 + wm + i * 32u + (lane & 31u);
    row_scale[i] = m < p.rows ? p.scale[m] : 0.0f;
  }
  v16i acc[BM][BN] = {};
  uint32_t use = 0, next = (kSets - 1u) * kSet;
  for (uint32_t step = 0; step < steps; ++step) {
    // This wave's loads of the set are there and its reads of the one before are done; then
    // everyone's are.  Loads end in their order: those of the kSets - 2 sets behind may go on.
    if (step + kSets - 1u <= steps)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kSets - 2u) * kLoads)
                   : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (step + kSets - 1u < steps) bring(lds + next, step + kSets - 1u);
    multiply_set<KB, TM, WK>(lds + use, wm, wn, wk, acc);
    next = use;
    use = use + kSet == kSets * kSet ? 0u : use + kSet;
  }
  __syncthreads();
  if constexpr (WK > 1) {
    static_assert(T::kWaves * (WK - 1) * BM * BN * 4096 <= kSets * kSet, "the sums fit");
    join_parts<T::kWaves, WK>(lds, wave, acc);
    if (wk != 0) return;
  }
  store_sums<Out>(p, lds + wave * kSliceBytes, chan_scale, chan_bias, m0 + wm, n0, wn, row_scale,
                  acc);
}

// The same for many large tiles: a workgroup takes one after the other, and the first set of
// the next is on its way while the last of this one is multiplied and its sums are stored.
// Tiles of 256 x 256: 4,096 x 151,936 x 896 to bf16 716 us, 1,560 TOP/s (a workgroup a tile
// 742); 4,096 x 8,192 x 8,192 245 us, 2,240 TOP/s (252).  Without the stores the first takes
// 631: they end before the next tile's second set, for loads wait behind them.  Of 128 x 256:
// 1,024 x 8,192 x 8,192 73 us (128 x 128, two workgroups a unit, a tile each: 86), 700 x 6,144
// x 4,096 32.8 (36.3), 3,000 x 8,192 x 1,024 35.3 (39.3), 384 x 50,304 x 896 30.3 (30.7),
// 1,500 x 12,000 x 2,048 55.1 (52.3).
constexpr uint32_t kLargeGroups = 256;  // one a compute unit
template <typename Out, int WM, int WN, int BM, int BN>
__global__ __launch_bounds__(64 * WM * WN) void int8_large_kernel(Int8Params p, TilePlan plan) {
  using T = Tile<WM, WN, BM, BN>;
  constexpr uint32_t TM = T::kRows, TN = T::kChannels, KB = 128, kPieces = KB / 16u;
  constexpr uint32_t kLoads = (TM + TN) * KB / 1024u / T::kWaves;
  constexpr uint32_t kSet = (TM + TN) * KB;
  // stores of a wave of a whole tile, none of which is left out
  constexpr uint32_t kStores = BM * BN * 32u * 32u / (64u * Out::kPer);
  __shared__ __align__(16) int8_t lds[2 * kSet];
  __shared__ __align__(16) float chan_scale[2][TN], chan_bias[2][TN];
  const uint32_t lane = lane_id();
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t wm = wave / WN * (BM * 32u), wn = wave % WN * (BN * 32u);
  const uint32_t tiles = plan.m_tiles * plan.n_tiles, steps = (p.cols + KB - 1u) / KB;
  const int8_t* from[kLoads];
  uint32_t offset[kLoads];
#pragma unroll
  for (uint32_t i = 0; i < kLoads; ++i) {
    const uint32_t row = (wave * kLoads + i) * (64u / kPieces) + lane / kPieces;
    offset[i] = piece_at<KB>(row, lane % kPieces) - row * KB;
  }
  uint32_t m0, n0;
  auto go_to = [&](uint32_t linear) {
    tile_of(plan, linear, &m0, &n0);
    m0 *= TM;
    n0 *= TN;
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const uint32_t row = (wave * kLoads + i) * (64u / kPieces) + lane / kPieces;
      if (row < TM) {
        const uint32_t r = m0 + row;
        from[i] = p.q + (size_t)(r < p.rows ? r : p.rows - 1u) * p.q_ld + offset[i];
      } else {
        const uint32_t r = n0 + row - TM;
        from[i] = p.weight + (size_t)(r < p.channels ? r : p.channels - 1u) * p.weight_ld + offset[i];
      }
    }
  };
  auto bring = [&](int8_t* set, uint32_t step) {
    const uint32_t k = step * KB;
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const int8_t* at = from[i] + k;
      if (k + KB > p.cols && k + offset[i] >= p.cols)
        at = reinterpret_cast<const int8_t*>(&kZeroPiece);
      to_lds(at, set + (wave * kLoads + i) * 1024u);
    }
  };
  // a tile's scales and biases, in registers
  struct Scales {
    float row[BM], chan, bias;
  };
  auto scales_of = [&]() {
    Scales s;
#pragma unroll
    for (int i = 0; i < BM; ++i) {
      const uint32_t m = m0 + wm + i * 32u + (lane & 31u);
      s.row[i] = m < p.rows ? p.scale[m] : 0.0f;
    }
    const uint32_t n = n0 + threadIdx.x;
    const bool real = threadIdx.x < TN && n < p.channels;
    s.chan = real ? p.weight_scale[n] : 0.0f;
    s.bias = real && p.bias ? p.bias[n] : kNoBias;
    return s;
  };
  uint32_t item = blockIdx.x, use = 0, turn = 0;
  bool stored = false;  // kStores stores are behind the loads of the first set
  go_to(item);
  Scales scales = scales_of();
  bring(lds, 0);
  while (true) {
    if (threadIdx.x < TN) {  // the other pair may still be read by waves that store
      chan_scale[turn][threadIdx.x] = scales.chan;
      chan_bias[turn][threadIdx.x] = scales.bias;
    }
    const uint32_t my_m0 = m0, my_n0 = n0, next = item + kLargeGroups;
    float row_scale[BM];
#pragma unroll
    for (int i = 0; i < BM; ++i) row_scale[i] = scales.row[i];
    v16i acc[BM][BN] = {};
    // As above; loads and stores end in their order, so with the tile's stores behind the loads
    // all but the newest of those may go on.
    if (stored)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kStores - 4u) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    for (uint32_t step = 1; step < steps; ++step) {
      bring(lds + (use ^ kSet), step);
      multiply_set<KB, TM, 1>(lds + use, wm, wn, 0, acc);
      use ^= kSet;
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    if (next < tiles) {
      go_to(next);
      scales = scales_of();
      bring(lds + (use ^ kSet), 0);
    }
    multiply_set<KB, TM, 1>(lds + use, wm, wn, 0, acc);
    use ^= kSet;
    // the set that was multiplied last takes the slices
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    store_sums<Out>(p, lds + (use ^ kSet) + wave * kSliceBytes, chan_scale[turn], chan_bias[turn],
                    my_m0 + wm, my_n0, wn, row_scale, acc);
    if (next >= tiles) return;
    stored = my_m0 + TM <= p.rows && my_n0 + TN <= p.channels;
    item = next;
    turn ^= 1u;
  }
}

template <typename Out>
hipError_t few_as(const Int8Params& p, hipStream_t stream) {
  const uint32_t groups = (p.channels + 15u) / 16u, steps = (p.cols + 63u) / 64u;
  uint32_t split = 1;
  while (split < kFewWaves && groups * split < 4096 && steps / (2 * split) >= 4) split *= 2;
  const uint32_t own = kFewWaves / split;
  int8_few_kernel<Out><<<(groups + own - 1u) / own, 64u * kFewWaves, 0, stream>>>(p, split);
  return hipGetLastError();
}

template <typename T>
TilePlan plan_tiles(const Int8Params& p) {
  TilePlan t;
  t.m_tiles = (p.rows + T::kRows - 1u) / T::kRows;
  t.n_tiles = (p.channels + T::kChannels - 1u) / T::kChannels;
  const uint32_t fit = (1u << 20) / (T::kRows * p.cols);
  t.group = fit > 4u ? fit : 4u;
  if (t.group > t.m_tiles) t.group = t.m_tiles;
  return t;
}
template <typename Out, int WM, int WN, int BM, int BN, uint32_t KB, int WK>
hipError_t tile_as(const Int8Params& p, hipStream_t stream) {
  using T = Tile<WM, WN, BM, BN>;
  const TilePlan t = plan_tiles<T>(p);
  int8_tile_kernel<Out, WM, WN, BM, BN, KB, WK>
      <<<t.m_tiles * t.n_tiles, T::kThreads * WK, 0, stream>>>(p, t);
  return hipGetLastError();
}
template <typename Out, int WM, int WN, int BM, int BN, uint32_t KB, uint32_t kSets, int WK>
hipError_t pieces_as(const Int8Params& p, hipStream_t stream) {
  using T = Tile<WM, WN, BM, BN>;
  const TilePlan t = plan_tiles<T>(p);
  int8_pieces_kernel<Out, WM, WN, BM, BN, KB, kSets, WK>
      <<<t.m_tiles * t.n_tiles, T::kThreads * WK, 0, stream>>>(p, t);
  return hipGetLastError();
}

template <typename Out, int WM, int WN, int BM, int BN>
hipError_t large_as(const Int8Params& p, hipStream_t stream) {
  using T = Tile<WM, WN, BM, BN>;
  const TilePlan t = plan_tiles<T>(p);
  const uint32_t all = t.m_tiles * t.n_tiles;
  int8_large_kernel<Out, WM, WN, BM, BN>
      <<<all < kLargeGroups ? all : kLargeGroups, T::kThreads, 0, stream>>>(p, t);
  return hipGetLastError();
}

// Whole pieces: 16 bytes divide the columns, the addresses and the distances of rows.
bool whole_pieces(const Int8Params& p) {
  return ((p.cols | p.q_ld | p.weight_ld | (uintptr_t)p.q | (uintptr_t)p.weight) & 15u) == 0;
}

uint32_t tiles(const Int8Params& p, uint32_t rows, uint32_t channels) {
  return (p.rows + rows - 1u) / rows * ((p.channels + channels - 1u) / channels);
}

// Which kernel takes a product (us, both sides of each line; rows x channels x columns).
//
// Up to 16 rows of up to 4,096 channels go without LDS tiles, and one or two rows of whole
// pieces of any channels; few / the tiles that take it otherwise:
//   16 x 4,096 x 4,096  6.9 / 7.4     8 x 8,192 x 8,192  14.6 / 12.5     1 x 8,192 x 8,192  13.4 / 12.4
//   8 x 1,024 x 8,192   8.8 / 10.1    16 x 8,192 x 896    4.4 / 4.0      1 x 32,000 x 4,096  24 / 32
//   16 x 4,001 x 4,001  13.2 / 15.5   1 x 8,192 x 8,001  24.4 / 23.4     1 x 151,936 x 896   26 / 28
//   16 x 2,048 x 2,048  4.4 / 4.8     16 x 32,000 x 2,001  34 / 16       4 x 151,936 x 896   28.4 / 28.3
//
// Tiles by how many there are for 256 compute units: where the small ones do not fill them,
// eight waves take one, the contraction cut by eight or four.  32 x 32; 32 x 64, which up
// to 64 rows run two a unit (their weights are read once, and wait for memory); 64 x 64;
// then 64 x 128 tiles, one and two a unit; 128 x 256; and 256 x 256 where their rounds are
// few enough: one takes 1.4 to 1.8 times as long.  Of whole pieces:
//                       32 x 32   32 x 64   64 x 64   64 x 128   64 x 128   128 x 256   256 x 256
//                        K by 8    K by 4    K by 4     K by 2
//   24 x 8,192 x 8,192     12.6      14.5      17.3          -          -           -           -
//   64 x 1,000 x 8,192     11.6      14.1      17.2          -          -           -           -
//   300 x 1,024 x 4,096     8.9       8.6      10.6       14.1       17.8           -           -
//   48 x 8,192 x 8,192     16.0      14.2      17.9       24.7       32.5           -           -
//   32 x 16,384 x 4,096    12.7      12.4      13.8       14.4       17.9           -           -
//   32 x 32,000 x 4,096    33.9      31.6      35.2       32.5       33.3           -           -
//   32 x 50,304 x 896      12.7      11.7      21.2       14.1       10.6           -           -
//   64 x 16,384 x 4,096    17.6      13.5      15.2       15.0       18.0           -           -
//   64 x 32,000 x 4,096    42.9      38.1      36.1       32.8       33.6           -           -
//   96 x 8,192 x 8,192     21.1      20.2      18.3       24.0       31.8           -           -
//   256 x 4,096 x 4,096    15.9      11.9      11.0       14.4       17.8           -           -
//   200 x 5,000 x 2,048    11.8      10.9      13.7        9.5       10.8           -           -
//   256 x 8,192 x 8,192       -         -      37.8       29.3       35.5           -        97.3
//   500 x 5,000 x 896         -         -      14.9       12.3        8.8           -        17.6
//   2,048 x 2,048 x 2,048     -         -      26.9       19.0       15.3        18.8        29.1
//   64 x 151,936 x 896     60.1      50.2      59.9       42.1       31.8           -           -
//   700 x 6,144 x 4,096       -         -         -          -       42.4        32.8        52.3
//   1,024 x 8,192 x 8,192     -         -         -          -       97.8        72.9        98.5
//   333 x 50,304 x 1,008      -         -         -          -       46.8        36.6        38.0
//   1,000 x 10,000 x 896      -         -         -          -       23.1        20.8        19.2
//   3,000 x 8,192 x 1,024     -         -         -          -       48.5        35.3        38.1
//   256 x 151,936 x 896       -         -         -          -          -        68.9        59.4
//   4,096 x 4,096 x 4,096     -         -         -          -          -        75.0        65.9
//   8,192 x 8,192 x 512       -         -         -          -          -        58.9        63.5
// Through registers, 64 x 128 with K by 2 and without, 128 x 128 two a unit, and 256 x 256 by
// the same rule (for a round of 128 x 128, 1.2 to 1.9):
//   24 x 8,192 x 8,001     27.5      33.2      41.8       64.1       87.2           -           -
//   128 x 4,096 x 4,001    16.9      18.7      23.1       33.8       45.3           -           -
//   32 x 32,000 x 2,001    18.7      15.9      20.1       21.8       27.1           -           -
//   256 x 4,096 x 4,001    30.1      22.7      23.4       33.7       44.9           -           -
//   200 x 5,000 x 2,001    22.6      19.7      19.2       19.5       24.6           -           -
//   32 x 50,257 x 1,001    18.2      18.1      24.1       16.1       17.6           -           -
//   2,000 x 2,000 x 2,001     -         -      35.6       23.9       27.0        31.9           -
//   8 x 151,936 x 896         -         -      44.6       32.1       28.7           -           -
//   300 x 20,001 x 2,001      -         -         -          -          -        34.6        44.1
//   1,500 x 12,000 x 1,001    -         -         -          -          -        44.0        53.4
//   333 x 50,257 x 1,001      -         -      85.3       56.4       56.6        54.9        53.4
//   2,000 x 20,000 x 2,001    -         -         -          -          -       165.5       137.0
//   4,096 x 4,096 x 4,001     -         -         -          -          -       140.4        83.3
//   4,096 x 30,001 x 897      -         -         -          -          -       262.3       239.2
template <typename Out>
hipError_t int8_as(const Int8Params& p, hipStream_t stream) {
  const bool whole = whole_pieces(p);
  if (p.rows <= 16 && (p.channels <= 4096 || (p.rows <= 2 && whole)))
    return few_as<Out>(p, stream);
  const uint32_t of32 = tiles(p, 32, 32), of64 = tiles(p, 32, 64), of128 = tiles(p, 64, 128);
  const uint32_t large = (tiles(p, 256, 256) + kLargeGroups - 1u) / kLargeGroups;
  if (!whole) {
    if (of32 <= 512) return tile_as<Out, 1, 1, 1, 1, 256, 8>(p, stream);
    if (of64 <= 512) return tile_as<Out, 1, 2, 1, 1, 256, 4>(p, stream);
    if (of128 <= 512) return tile_as<Out, 2, 2, 1, 2, 128, 2>(p, stream);
    if (p.rows <= 64) return tile_as<Out, 2, 2, 1, 2, 64, 1>(p, stream);
    const uint32_t rounds = (tiles(p, 128, 128) + 511u) / 512u;
    if (8u * large < 5u * rounds) return tile_as<Out, 2, 4, 4, 2, 128, 1>(p, stream);
    return tile_as<Out, 2, 2, 2, 2, 64, 1>(p, stream);
  }
  if (of32 <= 256) return pieces_as<Out, 1, 1, 1, 1, 256, 3, 8>(p, stream);
  if (of64 <= (p.rows <= 64 ? 512u : 256u)) return pieces_as<Out, 1, 2, 1, 1, 256, 3, 4>(p, stream);
  if (tiles(p, 64, 64) <= 256) return pieces_as<Out, 2, 1, 1, 2, 256, 4, 4>(p, stream);
  if (of128 <= 256) return pieces_as<Out, 2, 2, 1, 2, 256, 3, 2>(p, stream);
  if (of128 <= 512 || p.rows <= 64) return pieces_as<Out, 2, 2, 1, 2, 128, 3, 1>(p, stream);
  const uint32_t rounds = (tiles(p, 128, 256) + kLargeGroups - 1u) / kLargeGroups;
  if (8u * large < 5u * rounds) return large_as<Out, 2, 4, 4, 2>(p, stream);
  return large_as<Out, 2, 4, 2, 2>(p, stream);
}

}  // namespace

hipError_t launch_int8(const Int8Params& p, uint32_t out_dtype, hipStream_t stream) {
  if (out_dtype == PB_F32) return int8_as<F32>(p, stream);
  if (out_dtype == PB_F16) return int8_as<F16>(p, stream);
  return int8_as<BF16>(p, stream);
}

}  // namespace pb
