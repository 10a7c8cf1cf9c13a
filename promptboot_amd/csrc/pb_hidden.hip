// pb_hidden.hip -- table rows of tokens, norms with 8-bit outputs, and their gradients.
//
// All of it is bound by the bytes of its rows.  A thread takes chunks of eight
// elements, so that 16-bit rows are read and written 16 bytes at a time; rows may start
// at any element, and a row's last chunk goes element by element where it is short.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pb_device.h"
#include "pb_elem.h"
#include "pb_hidden.h"
#include "pb_internal.h"

#pragma clang fp contract(off)

namespace pb {

namespace {

constexpr uint32_t kChunk = 8;

// ---- chunks of N elements of a row, of which the first n are there ----

typedef uint32_t Words2 __attribute__((ext_vector_type(2)));
typedef Words2 Loose2 __attribute__((aligned(2), may_alias));
typedef Words2 Bytes8 __attribute__((aligned(1), may_alias));

template <typename E, int N>
__device__ __forceinline__ void load_row(const typename E::Raw* p, uint32_t n, float (&x)[N]) {
  static_assert(N % E::kPer == 0 || (N == 4 && E::kPer == 8), "whole chunks");
  if (n >= (uint32_t)N) {
    if constexpr (N == 4 && E::kPer == 8) {
      const Words2 v = *reinterpret_cast<const Loose2*>(p);
      const uint4 c = make_uint4(v.x, v.y, 0u, 0u);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = E::get(c, e);
    } else {
#pragma unroll
      for (int k = 0; k < N / E::kPer; ++k) {
        const uint4 c = load_chunk<E>(p + k * E::kPer);
#pragma unroll
        for (int e = 0; e < E::kPer; ++e) x[k * E::kPer + e] = E::get(c, e);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = (uint32_t)e < n ? E::one(p[e]) : 0.0f;
  }
}

template <typename E, int N>
__device__ __forceinline__ void store_row(typename E::Raw* p, uint32_t n, const float (&x)[N]) {
  if (n >= (uint32_t)N) {
    if constexpr (N == 4 && E::kPer == 8) {
      *reinterpret_cast<Loose2*>(p) = Words2{E::two(x[0], x[1]), E::two(x[2], x[3])};
    } else {
#pragma unroll
      for (int k = 0; k < N / E::kPer; ++k) {
        float y[E::kPer];
#pragma unroll
        for (int e = 0; e < E::kPer; ++e) y[e] = x[k * E::kPer + e];
        const uint4 v = E::pack(y);
        *reinterpret_cast<Loose4*>(p + k * E::kPer) = Words4{v.x, v.y, v.z, v.w};
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if ((uint32_t)e < n) p[e] = E::raw(x[e]);
  }
}

// The same for a type that is known at the launch only.
template <int N>
__device__ __forceinline__ void load_any(const void* base, uint32_t dtype, size_t at, uint32_t n,
                                         float (&x)[N]) {
  if (dtype == PB_F32)
    load_row<F32, N>(static_cast<const uint32_t*>(base) + at, n, x);
  else if (dtype == PB_F16)
    load_row<F16, N>(static_cast<const uint16_t*>(base) + at, n, x);
  else
    load_row<BF16, N>(static_cast<const uint16_t*>(base) + at, n, x);
}
template <int N>
__device__ __forceinline__ void store_any(void* base, uint32_t dtype, size_t at, uint32_t n,
                                          const float (&x)[N]) {
  if (dtype == PB_F32)
    store_row<F32, N>(static_cast<uint32_t*>(base) + at, n, x);
  else if (dtype == PB_F16)
    store_row<F16, N>(static_cast<uint16_t*>(base) + at, n, x);
  else
    store_row<BF16, N>(static_cast<uint16_t*>(base) + at, n, x);
}

__device__ __forceinline__ uint32_t chunk_left(uint32_t cols, uint32_t j) {
  return j < cols ? cols - j : 0u;
}

// A row's record: zeros, or what failed.
__device__ __forceinline__ void put_record(pb_inference_error* err, uint32_t row, uint32_t status,
                                           uint64_t needed, uint64_t available, uint64_t detail) {
  pb_inference_error e{};
  if (status != PB_OK) {
    e.status = status;
    e.domain = PB_DOMAIN_NONE;
    e.layer = PB_NO_LAYER;
    e.position = row;
    e.tensor_id = PB_NO_TENSOR;
    e.needed = needed;
    e.available = available;
    e.detail = detail;
  }
  err[row] = e;
}

__device__ __forceinline__ double wave_add(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1)
    v = v + __builtin_bit_cast(double, shfl_xor64(__builtin_bit_cast(uint64_t, v), m));
  return v;
}

// ---- table rows of tokens ----

// 2^shift threads take a row.  40 rows of 896 bf16: 2.4 us, a launch; 16,384 of them: 11.4 us
// (5.1 TB/s read and written).
// A product goes to its type by way of binary32: in one rounding 16,384 rows of 896 bf16 by
// 31.6 took 17.4 us in place of 10.2.  (31.6 is 158 / 5 but for 4e-17, so many of its products
// with 8 bits are next to the middle of two numbers, and what decides is behind the 53rd digit.)
template <typename In, typename Out>
__global__ __launch_bounds__(256) void embed_kernel(EmbedParams p, uint32_t shift) {
  const uint32_t row = blockIdx.x * (256u >> shift) + (threadIdx.x >> shift);
  if (row >= p.rows) return;
  const uint32_t t = threadIdx.x & ((1u << shift) - 1u);
  const uint32_t id = p.token[row];
  if (t == 0 && p.err != nullptr) {
    const bool bad = id != kNone && id >= p.vocab;
    put_record(p.err, row, bad ? PB_TOKEN_ID : PB_OK, p.vocab, id, (uint64_t)PB_FIELD_TOKEN << 32);
  }
  const bool live = id < p.vocab;
  const float other = id == kNone ? 0.0f : __builtin_nanf("");
  const typename In::Raw* from =
      static_cast<const typename In::Raw*>(p.table) + (live ? (size_t)id * p.table_ld : 0);
  typename Out::Raw* to = static_cast<typename Out::Raw*>(p.out) + (size_t)row * p.out_ld;
  for (uint32_t j = t * kChunk; j < p.cols; j += kChunk << shift) {
    const uint32_t n = p.cols - j;
    float x[kChunk];
    if (live) {
      load_row<In>(from + j, n, x);
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) x[e] = (float)((double)x[e] * p.scale);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) x[e] = other;
    }
    store_row<Out>(to + j, n, x);
  }
}

// ---- the table's gradient ----
//
// The rows are sorted by token (a stable radix sort of (id, row) pairs, kSortBits at a
// time), so a token's rows come next to each other and in order.  Then the sorted rows are
// cut into parts of kSumRows: a wave adds up its part's rows token by token, and what lies
// whole within a part is written at once.  What crosses parts is left in the workspace and
// joined in 64 bits.  No atomics touch the sums, so they repeat.
//
// Where the whole table is written, its zeros go out beside the sort, from the same
// launches: the sort keeps one compute unit busy, or a few, and the zeros the others.

constexpr uint32_t kDigits = 1u << kSortBits;
constexpr uint32_t sum_parts(uint32_t rows) { return (rows + kSumRows - 1u) / kSumRows; }
// Parts behind its first up to which a token's sum is joined by one wave.
constexpr uint32_t kLongParts = 32;

// Rows that add nothing sort behind every token.
__device__ __forceinline__ uint32_t token_key(const EmbedGradParams& p, uint32_t i) {
  const uint32_t id = p.token[i];
  return id < p.vocab ? id : p.vocab;
}
__device__ __forceinline__ uint32_t digit_of(uint32_t key, uint32_t pass) {
  return key >> (pass * kSortBits) & (kDigits - 1u);
}

// The lanes of the wave whose digit is this lane's, among those that are `real`.
__device__ __forceinline__ uint64_t same_digit(uint32_t d, bool real) {
  uint64_t same = __ballot(real);
#pragma unroll
  for (uint32_t b = 0; b < kSortBits; ++b) {
    const uint64_t set = __ballot(d >> b & 1u);
    same &= (d >> b & 1u) ? set : ~set;
  }
  return same;
}

// Zeros for the `part`-th of `parts` runs of a table, by kThreads threads.  They go past the
// caches, which hold the gradient's rows that a training step has just written: 16,384 rows
// into 32,000 x 4,096 bf16 91 us (120 through the caches), 65,536 into 151,936 x 896 148 (181),
// 700 into 50,257 x 1,001 47 (48).
template <typename T, uint32_t kThreads>
__device__ __forceinline__ void zero_part(const EmbedGradParams& p, uint32_t part,
                                          uint32_t parts) {
  typename T::Raw* table = static_cast<typename T::Raw*>(p.table);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  if (p.table_ld == p.cols) {  // one run of elements, from 16 aligned bytes on
    const size_t all = (size_t)p.vocab * p.cols;
    const size_t odd = (16u - ((uintptr_t)table & 15u)) % 16u / sizeof(typename T::Raw);
    const size_t head = odd < all ? odd : all, chunks = (all - head) / T::kPer;
    // workgroups next to each other write next to each other: one window that moves on (the
    // sort with 545 MB of zeros by 1, 2, 4, 8, 16, 32 stores a turn 111, 103, 101, 96, 99, 113 us;
    // a run of its own for each workgroup 131)
    constexpr uint32_t kTurn = 8u * kThreads;
    for (size_t c0 = (size_t)part * kTurn; c0 < chunks; c0 += (size_t)parts * kTurn) {
#pragma unroll
      for (uint32_t k = 0; k < 8; ++k) {
        const size_t c = c0 + k * kThreads + threadIdx.x;
        if (c < chunks)
          store_chunk<T>(table + head + c * T::kPer, zero);
      }
    }
    if (part == 0) {
      const size_t tail = head + chunks * T::kPer;
      if (threadIdx.x < head) table[threadIdx.x] = 0;
      if (tail + threadIdx.x < all) table[tail + threadIdx.x] = 0;
    }
    return;
  }
  const uint32_t from = (uint32_t)((uint64_t)p.vocab * part / parts);
  const uint32_t to = (uint32_t)((uint64_t)p.vocab * (part + 1u) / parts);
  const uint32_t wave = threadIdx.x >> 6, lane = lane_id();
  for (uint32_t v = from + wave; v < to; v += kThreads / 64u) {
    typename T::Raw* row = table + (size_t)v * p.table_ld;
    for (uint32_t j = lane * T::kPer; j < p.cols; j += 64u * T::kPer) {
      if (j + T::kPer <= p.cols) {
        store_chunk<T>(row + j, zero);
      } else {
        for (uint32_t e = j; e < p.cols; ++e) row[e] = 0;
      }
    }
  }
}

// Up to kSortRows rows: one workgroup sorts them in LDS, the others write zeros.  A pass
// gives every wave a run of the rows: a row's rank among its wave's rows of its digit, then
// the prefix over digits and waves.  (By launches over tiles, as more rows take, 16,384 rows
// took 53 us, all of them behind the zeros.)  Up to kSortFew rows leave LDS for a second
// workgroup that writes zeros on the same unit.
constexpr uint32_t kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr uint32_t kSortFew = 4096;
template <typename T, uint32_t kRows>
__global__ __launch_bounds__(kSortThreads) void sort_rows_kernel(EmbedGradParams p,
                                                                 uint32_t passes) {
  constexpr uint32_t kSortSteps = kRows / kSortThreads;
  __shared__ uint32_t key[kRows];
  __shared__ uint16_t order[2][kRows];
  __shared__ uint16_t place[kSortWaves][kDigits];
  __shared__ uint32_t run[kSortWaves];
  if (blockIdx.x != 0) {
    zero_part<T, kSortThreads>(p, blockIdx.x - 1u, gridDim.x - 1u);
    return;
  }
  const uint32_t lane = lane_id(), wave = threadIdx.x >> 6;
  if (threadIdx.x < 2) p.cross[threadIdx.x] = 0;
  for (uint32_t i = threadIdx.x; i < p.rows; i += kSortThreads) {
    key[i] = token_key(p, i);
    order[0][i] = (uint16_t)i;
  }
  // the rows in kSortWaves runs of whole steps
  const uint32_t steps = (p.rows + kSortThreads - 1u) / kSortThreads;
  const uint32_t first = wave * steps * 64u;
  for (uint32_t pass = 0; pass < passes; ++pass) {
    const uint16_t* from = order[pass & 1u];
    for (uint32_t d = lane; d < kDigits; d += 64u) place[wave][d] = 0;
    __syncthreads();
    uint32_t digit[kSortSteps], rank[kSortSteps];
#pragma unroll
    for (uint32_t k = 0; k < kSortSteps; ++k) {
      if (k >= steps) break;
      const uint32_t i = first + k * 64u + lane;
      const bool real = i < p.rows;
      digit[k] = real ? digit_of(key[from[i]], pass) : 0u;
      const uint64_t same = same_digit(digit[k], real);
      // a wave's reads and writes of LDS keep their order; other waves have other rows
      volatile uint16_t* seen = &place[wave][digit[k]];
      const uint32_t before = real ? *seen : 0u;
      rank[k] = before + lanes_below(same);
      if (real && lanes_below(same) == 0)
        *seen = (uint16_t)(before + (uint32_t)__popcll((unsigned long long)same));
    }
    __syncthreads();
    // exclusive prefix over digits, within a digit over waves
    uint32_t sum = 0;
    if (threadIdx.x < kDigits) {
#pragma unroll
      for (uint32_t w = 0; w < kSortWaves; ++w) sum += place[w][threadIdx.x];
    }
    uint32_t upto = sum;
#pragma unroll
    for (uint32_t m = 1; m < 64; m <<= 1) {
      const uint32_t o = (uint32_t)__shfl_up((int)upto, m, 64);
      if (lane >= m) upto += o;
    }
    if (lane == 63) run[wave] = upto;
    __syncthreads();
    if (threadIdx.x < kDigits) {
      uint32_t base = upto - sum;
      for (uint32_t w = 0; w < wave; ++w) base += run[w];
#pragma unroll
      for (uint32_t w = 0; w < kSortWaves; ++w) {
        const uint32_t n = place[w][threadIdx.x];
        place[w][threadIdx.x] = (uint16_t)base;
        base += n;
      }
    }
    __syncthreads();
    uint16_t* to = order[(pass + 1u) & 1u];
#pragma unroll
    for (uint32_t k = 0; k < kSortSteps; ++k) {
      if (k >= steps) break;
      const uint32_t i = first + k * 64u + lane;
      if (i < p.rows) to[place[wave][digit[k]] + rank[k]] = from[i];
    }
    __syncthreads();
  }
  for (uint32_t i = threadIdx.x; i < p.rows; i += kSortThreads) {
    const uint32_t r = order[passes & 1u][i];
    p.id[passes & 1u][i] = key[r];
    p.row[passes & 1u][i] = r;
  }
}

// More rows: two launches a pass, the rows in tiles of kSortTile: counts of a tile's digits,
// then the pairs' places, for which every tile adds up all counts.  The workgroups behind the
// tiles' write the launch's share of the zeros.
__device__ __forceinline__ uint32_t sort_key(const EmbedGradParams& p, uint32_t pass, uint32_t i) {
  return pass != 0 ? p.id[pass & 1u][i] : token_key(p, i);
}
struct ZeroShare {
  uint32_t part, parts;  // of all launches' workgroups: this launch's first, and how many
};

template <typename T>
__global__ __launch_bounds__(256) void sort_count_kernel(EmbedGradParams p, uint32_t pass,
                                                         uint32_t tiles, ZeroShare zero) {
  __shared__ uint32_t hist[kDigits];
  const uint32_t tile = blockIdx.x;
  if (tile >= tiles) {
    zero_part<T, 256>(p, zero.part + tile - tiles, zero.parts);
    return;
  }
  for (uint32_t d = threadIdx.x; d < kDigits; d += 256u) hist[d] = 0;
  if (pass == 0 && tile == 0 && threadIdx.x < 2) p.cross[threadIdx.x] = 0;
  __syncthreads();
  for (uint32_t k = 0; k < kSortTile / 256u; ++k) {
    const uint32_t i = tile * kSortTile + k * 256u + threadIdx.x;
    if (i < p.rows) atomicAdd(&hist[digit_of(sort_key(p, pass, i), pass)], 1u);
  }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < kDigits; d += 256u)
    p.count[(size_t)tile * kDigits + d] = hist[d];
}

template <typename T>
__global__ __launch_bounds__(256) void sort_place_kernel(EmbedGradParams p, uint32_t pass,
                                                         uint32_t tiles, ZeroShare zero) {
  constexpr uint32_t kSteps = kSortTile / 256u;
  __shared__ uint32_t place[4][kDigits];
  const uint32_t tile = blockIdx.x, lane = lane_id(), wave = threadIdx.x >> 6;
  if (tile >= tiles) {
    zero_part<T, 256>(p, zero.part + tile - tiles, zero.parts);
    return;
  }
  for (uint32_t d = threadIdx.x; d < 4u * kDigits; d += 256u) (&place[0][0])[d] = 0;
  __syncthreads();
  // a wave's rows in order, 64 at a time; a row's rank among the wave's rows of its digit
  const uint32_t first = tile * kSortTile + wave * (kSortTile / 4u);
  uint32_t key[kSteps], rank[kSteps];
#pragma unroll
  for (uint32_t k = 0; k < kSteps; ++k) {
    const uint32_t i = first + k * 64u + lane;
    key[k] = i < p.rows ? sort_key(p, pass, i) : 0u;
  }
#pragma unroll
  for (uint32_t k = 0; k < kSteps; ++k) {
    const bool real = first + k * 64u + lane < p.rows;
    const uint64_t same = same_digit(digit_of(key[k], pass), real);
    // a wave's reads and writes of LDS keep their order; other waves have other rows
    volatile uint32_t* seen = &place[wave][digit_of(key[k], pass)];
    const uint32_t before = real ? *seen : 0u;
    rank[k] = before + lanes_below(same);
    if (real && lanes_below(same) == 0)
      *seen = before + (uint32_t)__popcll((unsigned long long)same);
  }
  __syncthreads();
  // where the tile's rows of a digit go: behind all rows of lower digits and those of the
  // digit in earlier tiles.  A thread has two neighbouring digits.
  static_assert(kDigits == 512, "two digits a thread");
  const uint32_t d0 = 2u * threadIdx.x;
  uint2 all = make_uint2(0, 0), before = make_uint2(0, 0);
#pragma unroll 8
  for (uint32_t t = 0; t < tiles; ++t) {
    const uint2 c = *reinterpret_cast<const uint2*>(p.count + (size_t)t * kDigits + d0);
    all.x += c.x;
    all.y += c.y;
    if (t < tile) {
      before.x += c.x;
      before.y += c.y;
    }
  }
  uint32_t upto = all.x + all.y;  // inclusive over the wave's lanes
#pragma unroll
  for (uint32_t m = 1; m < 64; m <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)upto, m, 64);
    if (lane >= m) upto += o;
  }
  __shared__ uint32_t run[4];
  if (lane == 63) run[wave] = upto;
  __syncthreads();
  uint32_t base[2] = {upto - all.x - all.y, upto - all.y};
#pragma unroll
  for (uint32_t w = 0; w < 3; ++w) {
    base[0] += w < wave ? run[w] : 0u;
    base[1] += w < wave ? run[w] : 0u;
  }
  base[0] += before.x;
  base[1] += before.y;
#pragma unroll
  for (uint32_t k = 0; k < 2; ++k) {
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
      const uint32_t n = place[w][d0 + k];
      place[w][d0 + k] = base[k];
      base[k] += n;
    }
  }
  __syncthreads();
  uint32_t* id = p.id[(pass + 1u) & 1u];
  uint32_t* row = p.row[(pass + 1u) & 1u];
#pragma unroll
  for (uint32_t k = 0; k < kSteps; ++k) {
    const uint32_t i = first + k * 64u + lane;
    if (i < p.rows) {
      const uint32_t at = place[wave][digit_of(key[k], pass)] + rank[k];
      id[at] = key[k];
      row[at] = pass == 0 ? i : p.row[pass & 1u][i];
    }
  }
}

// Zeros alone: a gradient without rows.
template <typename T>
__global__ __launch_bounds__(256) void zero_table_kernel(EmbedGradParams p) {
  zero_part<T, 256>(p, blockIdx.x, gridDim.x);
}

// A token's sum times the factor, as the table holds it.
template <typename T, int N>
__device__ __forceinline__ void put_product(const EmbedGradParams& p, uint32_t id, uint32_t j,
                                            uint32_t n, float (&y)[N]) {
  typename T::Raw* to = static_cast<typename T::Raw*>(p.table) + (size_t)id * p.table_ld + j;
  if (p.accumulate) {
    float old[N];
    load_row<T>(to, n, old);
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = old[e] + y[e];
  }
  store_row<T>(to, n, y);
}

// One wave: the sorted rows [part kSumRows, + kSumRows) and 64 chunks of columns.  All of the
// part's rows are requested before the first is added, which bounds a part by the registers.
// 16,384 rows of 896 bf16 14 us, 700 of 1,001 in 32 bits 8.5: one round trip for the ids, one
// for the rows.
template <typename G, typename T>
__global__ __launch_bounds__(256) void sum_rows_kernel(EmbedGradParams p, uint32_t last,
                                                       uint32_t col_tiles, uint32_t units) {
  constexpr int N = G::kPer;
  const uint32_t unit =
      (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4u + (threadIdx.x >> 6)));
  if (unit >= units) return;
  const uint32_t part = unit / col_tiles, tile = unit - part * col_tiles, lane = lane_id();
  const uint32_t j = (tile * 64u + lane) * N, n = chunk_left(p.cols, j);
  const uint32_t lo = part * kSumRows;
  const uint32_t hi = lo + kSumRows < p.rows ? lo + kSumRows : p.rows;
  // the part's ids, with the one before and the one behind it: lane k has sorted row lo - 1 + k
  static_assert(kSumRows + 2 <= 64, "a lane each");
  const uint32_t at = lo + lane;  // + 1
  const bool inside = at >= 1u && at <= p.rows && lane < kSumRows + 2u;
  const uint32_t my_id = inside ? p.id[last][at - 1u] : kNone;
  const uint32_t my_row = inside ? p.row[last][at - 1u] : 0u;
  const typename G::Raw* grad = static_cast<const typename G::Raw*>(p.grad) + j;
  uint4 x[kSumRows];
#pragma unroll
  for (uint32_t k = 0; k < kSumRows; ++k) {
    const uint32_t row = bcast32(my_row, k + 1u);
    x[k] = make_uint4(0, 0, 0, 0);
    if (lo + k < hi && bcast32(my_id, k + 1u) < p.vocab) {
      const typename G::Raw* from = grad + (size_t)row * p.grad_ld;
      if (n >= (uint32_t)N) {
        x[k] = load_chunk<G>(from);
      } else if (n != 0) {
        float y[N];
        load_row<G>(from, n, y);
        x[k] = G::pack(y);
      }
    }
  }
  uint32_t cur = bcast32(my_id, 1u);
  if (cur >= p.vocab) return;
  bool from_before = lo > 0 && bcast32(my_id, 0u) == cur;  // the sum goes on from the part before
  float sum[N] = {};
  auto leave = [&](bool goes_on) {
    if (!from_before && !goes_on) {
      // the factor is a binary32 number: one of 64 bits, in two words or in binary64, took 16,384 rows
      // added to a table from 68.5 to 70 us (this stands here sixteen times)
      float y[N];
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = sum[e] * p.scale;
      put_product<T>(p, cur, j, n, y);
    } else {
      float* to = p.part + ((size_t)part * 2u + (from_before ? 0u : 1u)) * p.cols + j;
      store_row<F32>(reinterpret_cast<uint32_t*>(to), n, sum);
      if (!from_before && tile == 0 && lane == 0) {
        // in whose place of which list does not matter: each is joined by itself
        const uint32_t far = hi - 1u + kLongParts * kSumRows;
        if (far < p.rows && p.id[last][far] == cur)
          p.cross[1u + sum_parts(p.rows) - atomicAdd(p.cross + 1, 1u)] = part;
        else
          p.cross[2u + atomicAdd(p.cross, 1u)] = part;
      }
    }
  };
#pragma clang loop unroll(full)
  for (uint32_t k = 0; k < kSumRows; ++k) {
    const uint32_t id = bcast32(my_id, k + 1u);
    if (lo + k < hi && cur < p.vocab) {
      if (id != cur) {
        leave(false);
        cur = id;
        from_before = false;
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] = sum[e] + G::get(x[k], e);
    }
  }
  if (cur < p.vocab) leave(hi < p.rows && bcast32(my_id, kSumRows + 1u) == cur);
}

// The first sorted row from `lo` on whose token is another: 64 places at a time.
__device__ __forceinline__ uint32_t token_end(const uint32_t* id, uint32_t own, uint32_t lo,
                                              uint32_t hi) {
  while (lo < hi) {
    const uint32_t step = (hi - lo + 63u) / 64u, at = lo + lane_id() * step;
    const uint64_t not_own = __ballot(at >= hi || id[at] != own);
    const uint32_t k = not_own ? (uint32_t)__ffsll((unsigned long long)not_own) - 1u : 64u;
    const uint32_t end = lo + k * step;  // its place is behind the token's rows, or at hi
    lo = k == 0 ? lo : end - step + 1u;
    hi = end < hi ? end : hi;
  }
  return lo;
}

// The sums that cross parts, 5 to 11 us.  A wave takes 256 columns of a token of up to kLongParts more
// parts; a workgroup 64 columns of a longer one, its waves a run of parts each.
constexpr uint32_t kJoinWaves = 16;
template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void join_rows_kernel(EmbedGradParams p,
                                                                    uint32_t last) {
  __shared__ double waves[kJoinWaves][64];
  const uint32_t lane = lane_id();
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t* id = p.id[last];
  const uint32_t few = p.cross[0], many = p.cross[1];
  const uint32_t wide = (p.cols + 255u) / 256u, narrow = (p.cols + 63u) / 64u;
  for (size_t unit = (size_t)blockIdx.x * kJoinWaves + wave; unit < (size_t)few * wide;
       unit += (size_t)gridDim.x * kJoinWaves) {
    const uint32_t part = p.cross[2u + unit / wide];
    const uint32_t j = ((uint32_t)(unit % wide) * 64u + lane) * 4u, n = chunk_left(p.cols, j);
    const uint32_t next = (part + 1u) * kSumRows, own = id[next - 1u];
    const uint32_t most = next + kLongParts * kSumRows;
    const uint32_t to = (token_end(id, own, next, most < p.rows ? most : p.rows) - 1u) / kSumRows;
    float x[4];
    load_row<F32, 4>(reinterpret_cast<const uint32_t*>(p.part + ((size_t)part * 2u + 1u) * p.cols + j),
                     n, x);
    double sum[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll 8
    for (uint32_t k = part + 1u; k <= to; ++k) {
      load_row<F32, 4>(reinterpret_cast<const uint32_t*>(p.part + (size_t)k * 2u * p.cols + j), n,
                       x);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = sum[e] + (double)x[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (float)(sum[e] * (double)p.scale);
    put_product<T>(p, own, j, n, x);
  }
  for (size_t unit = blockIdx.x; unit < (size_t)many * narrow; unit += gridDim.x) {
    const uint32_t part = p.cross[1u + sum_parts(p.rows) - (uint32_t)(unit / narrow)];
    const uint32_t j = (uint32_t)(unit % narrow) * 64u + lane;
    const uint32_t next = (part + 1u) * kSumRows, own = id[next - 1u];
    const uint32_t n = (token_end(id, own, next, p.rows) - 1u) / kSumRows - part + 1u;
    const uint32_t from = (uint32_t)((uint64_t)n * wave / kJoinWaves);
    const uint32_t to = (uint32_t)((uint64_t)n * (wave + 1u) / kJoinWaves);
    double sum = 0.0;
    if (j < p.cols) {
#pragma unroll 8
      for (uint32_t k = from; k < to; ++k)
        sum = sum + (double)p.part[((size_t)(part + k) * 2u + (k == 0 ? 1u : 0u)) * p.cols + j];
    }
    waves[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && j < p.cols) {
#pragma unroll
      for (uint32_t w = 1; w < kJoinWaves; ++w) sum = sum + waves[w][lane];
      const float y = (float)(sum * (double)p.scale);
      typename T::Raw* at = static_cast<typename T::Raw*>(p.table) + (size_t)own * p.table_ld + j;
      *at = T::raw(p.accumulate ? T::one(*at) + y : y);
    }
    __syncthreads();
  }
}

// ---- norms ----
//
// A row is held in registers between its statistics and its outputs, as it is in memory: T
// threads take C chunks of eight elements each.  mean(h^2) is summed in 64 bits: no
// binary32 row overflows there, and a 64-bit multiply-add issues as fast as a 32-bit
// product and its addition would.  1 / sqrt(mean + eps) is used as binary32: for rows next to the
// largest numbers (a root mean square past 2^126) that is below the normal range, where it has
// 22 digits or more.  All 24, by a power of two, cost every gradient of a norm 1 to 2 %.

// Eight elements as they are in memory.
template <typename E>
struct Chunk {
  static constexpr int kWords = kChunk / E::kPer;
  uint4 v[kWords];
  __device__ __forceinline__ float get(uint32_t e) const {
    return E::get(v[e / E::kPer], (int)(e % E::kPer));
  }
  __device__ __forceinline__ void set(const float (&x)[kChunk]) {
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      float y[E::kPer];
#pragma unroll
      for (int e = 0; e < E::kPer; ++e) y[e] = x[k * E::kPer + e];
      v[k] = E::pack(y);
    }
  }
  // The first n from `p`, zeros behind them.
  __device__ __forceinline__ void load(const typename E::Raw* p, uint32_t n) {
    if (n >= kChunk) {
#pragma unroll
      for (int k = 0; k < kWords; ++k) v[k] = load_chunk<E>(p + k * E::kPer);
    } else {
      float x[kChunk];
      load_row<E>(p, n, x);
      set(x);
    }
  }
  __device__ __forceinline__ void store(typename E::Raw* p, uint32_t n) const {
    if (n >= kChunk) {
#pragma unroll
      for (int k = 0; k < kWords; ++k)
        *reinterpret_cast<Loose4*>(p + k * E::kPer) = Words4{v[k].x, v[k].y, v[k].z, v[k].w};
    } else {
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e)
        if (e < n) p[e] = E::raw(get(e));
    }
  }
};

// w of a chunk, ones without a weight.
__device__ __forceinline__ void load_weight(const void* weight, uint32_t dtype, uint32_t j,
                                            uint32_t n, float (&w)[kChunk]) {
  if (weight == nullptr) {
#pragma unroll
    for (uint32_t e = 0; e < kChunk; ++e) w[e] = 1.0f;
  } else {
    load_any(weight, dtype, j, n, w);
  }
}
template <typename E>
__device__ __forceinline__ void load_weight(const void* weight, uint32_t j, uint32_t n,
                                            Chunk<E>& w) {
  if (weight == nullptr) {
    const float ones[kChunk] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
    w.set(ones);
  } else {
    w.load(static_cast<const typename E::Raw*>(weight) + j, n);
  }
}

// What is reduced over a row's T threads, in every one of them.
template <int T, typename V, typename Join>
__device__ __forceinline__ V row_join(V v, Join join) {
  if constexpr (T > 64) {
    __shared__ V waves[T / 64];
    __syncthreads();
    if (lane_id() == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = waves[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) v = join(v, waves[w]);
  }
  return v;
}
struct Stats {
  double sum;
  uint64_t top;
};
template <int T>
__device__ __forceinline__ Stats row_stats(double sum, uint64_t top) {
  return row_join<T>(Stats{wave_add(sum), wave_max64(top)}, [](const Stats& a, const Stats& b) {
    return Stats{a.sum + b.sum, a.top > b.top ? a.top : b.top};
  });
}
struct Stats32 {
  double sum;
  uint32_t top;
};
template <int T>
__device__ __forceinline__ Stats32 row_stats(double sum, uint32_t top) {
  const uint32_t lane = lane_id();
  auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  top = larger(top, lane_xor(top, 32, lane));
  top = larger(top, lane_xor(top, 16, lane));
  top = larger(top, lane_xor(top, 8, lane));
  top = larger(top, lane_xor(top, 4, lane));
  top = larger(top, lane_xor(top, 2, lane));
  top = larger(top, lane_xor(top, 1, lane));
  return row_join<T>(Stats32{wave_add(sum), top}, [](const Stats32& a, const Stats32& b) {
    return Stats32{a.sum + b.sum, a.top > b.top ? a.top : b.top};
  });
}

__device__ __forceinline__ uint64_t abs_bits(double v) {
  return __builtin_bit_cast(uint64_t, v) & 0x7fffffffffffffffull;
}
constexpr uint64_t kInfBits = 0x7ff0000000000000ull;

// The whole number nearest to 127 p / top, ties to even.  v = p (127 / top) is off by less
// than 2^-50 relatively, so it decides unless it is that near to a half; there 254 |p| is
// compared with (2 k + 1) top, k = floor |v|, without rounding: the product is s + r
// exactly, and 254 |p| - s is exact too, since p and top are products of two binary32 numbers (48
// bits, so 55 with the factor) and what cancellation leaves has fewer than 53.
__device__ __forceinline__ int nearest_step(double p, double top, double step) {
  const double v = fabs(p) * step;
  double t = __builtin_rint(v);
  if (__builtin_expect(fabs(v - t) > 0.5 - 0x1p-30, 0)) {
    const double k = __builtin_floor(v), odd = 2.0 * k + 1.0;
    const double s = odd * top, r = fma(odd, top, -s), d = fma(254.0, fabs(p), -s);
    const bool up = d > r || (d == r && ((int)k & 1));
    t = up ? k + 1.0 : k;
  }
  const int whole = (int)t;
  return p < 0.0 ? -whole : whole;
}
__device__ __forceinline__ uint32_t four_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t low = __builtin_amdgcn_perm(b, a, 0x0c0c0400u);
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), low, 0x05040100u);
}

// A row's norm and its 8-bit rounding, from one read of the row: 16,384 rows of 4,096 bf16 with
// a residual, the sum kept, 88 us (470 MB, 5.3 TB/s: no byte more than the formulas need by
// the counters).  A single row of 896: 3.5 us, a launch and its chain of read, join over the
// waves, quotient, store.
//
// kNarrow: rows and weight of one 16-bit type, or no weight.  Their products h w are exact in
// binary32, so the largest is, and all but values near a half are rounded in 32 bits:
// p (127 / top) is off by 2^-24 of 127 there, and those that come nearer than 2^-15 to a half
// go the exact way.  Rows whose largest product binary32 does not hold well (2^-60 to 2^120)
// go it as a whole, and so do all others, in 64 bits: 16,384 rows of 4,096 bf16 under an f32
// weight 110 us.
template <typename E, bool kNarrow, int T, int C>
__global__ __launch_bounds__(T < 128 ? 256 : T) void norm_kernel(NormParams p) {
  constexpr uint32_t kRows = T < 128 ? 256 / T : 1;
  const uint32_t t = threadIdx.x % T;
  const uint32_t row = blockIdx.x * kRows + threadIdx.x / T;
  if (row >= p.rows) return;  // whole waves, and with T > 64 never
  const typename E::Raw* x = static_cast<const typename E::Raw*>(p.x) + (size_t)row * p.x_ld;
  Chunk<E> h[C], w[kNarrow ? C : 1];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const uint32_t j = (i * T + t) * kChunk, n = chunk_left(p.cols, j);
    h[i].load(x + j, n);
    if constexpr (kNarrow) load_weight<E>(p.weight, j, n, w[i]);
  }
  if (p.residual != nullptr) {
    const typename E::Raw* r =
        static_cast<const typename E::Raw*>(p.residual) + (size_t)row * p.residual_ld;
    Chunk<E> more[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t j = (i * T + t) * kChunk;
      more[i].load(r + j, chunk_left(p.cols, j));
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float y[kChunk];
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) y[e] = h[i].get(e) + more[i].get(e);
      h[i].set(y);
    }
  }
  if (p.sum != nullptr) {
    typename E::Raw* to = static_cast<typename E::Raw*>(p.sum) + (size_t)row * p.sum_ld;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t j = (i * T + t) * kChunk;
      h[i].store(to + j, chunk_left(p.cols, j));
    }
  }
  auto weights = [&](int i, float (&y)[kChunk]) {
    if constexpr (kNarrow) {
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) y[e] = w[i].get(e);
    } else {
      const uint32_t j = (i * T + t) * kChunk;
      load_weight(p.weight, p.weight_dtype, j, chunk_left(p.cols, j), y);
    }
  };

  // statistics: the squares' sum, and the bits of the largest |h w| (a NaN's are larger still)
  const bool eight = p.q != nullptr;
  double squares = 0.0, most = 0.0;
  bool narrow = false, bad = false;
  if constexpr (kNarrow) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < C; ++i) {
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) {
        const float v = h[i].get(e);
        squares = fma((double)v, (double)v, squares);
        const uint32_t b = b_of(v * w[i].get(e)) & 0x7fffffffu;  // 0 behind the row's end
        top = b > top ? b : top;
      }
    }
    const Stats32 s = row_stats<T>(squares, top);
    squares = s.sum;
    most = (double)f_of(s.top);
    narrow = s.top >= 0x21800000u && s.top <= 0x7b800000u;  // 2^-60 to 2^120
  }
  if (!kNarrow || (eight && !narrow)) {
    squares = 0.0;
    uint64_t top = 0;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float y[kChunk];
      if (eight) weights(i, y);
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) {
        const double v = (double)h[i].get(e);
        squares = fma(v, v, squares);
        if (eight) {
          const uint64_t b = abs_bits(v * (double)y[e]);
          top = b > top ? b : top;
        }
      }
    }
    const Stats s = row_stats<T>(squares, top);
    squares = s.sum;
    most = __builtin_bit_cast(double, s.top);
    bad = s.top >= kInfBits;
  }
  const double rstd = p.norm ? 1.0 / sqrt(squares / (double)p.cols + p.eps) : 1.0;
  const float scale = (float)(rstd * (most / 127.0));
  bad = !isfinite(squares) || (eight && (bad || !isfinite(scale)));

  if (p.out != nullptr) {
    const float r = bad ? __builtin_nanf("") : (float)rstd;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t j = (i * T + t) * kChunk, n = chunk_left(p.cols, j);
      float y[kChunk];
      weights(i, y);
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) y[e] = h[i].get(e) * r * y[e];
      store_any(p.out, p.out_dtype, (size_t)row * p.out_ld + j, n, y);
    }
  }
  if (eight) {
    const double step = most > 0.0 ? 127.0 / most : 0.0;
    const float step32 = (float)step;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t j = (i * T + t) * kChunk, n = chunk_left(p.cols, j);
      float y[kChunk];
      weights(i, y);
      uint32_t q[kChunk];
      bool exact = true;
      if (kNarrow && narrow) {
        // added to 1.5 2^23, a number is rounded to a whole one, whose low byte is the byte
        float off = 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < kChunk; ++e) {
          const float v = h[i].get(e) * y[e], whole = fmaf(v, step32, 0x1.8p23f);
          q[e] = b_of(whole);
          off = fmaxf(off, fabsf(fmaf(v, step32, -(whole - 0x1.8p23f))));
        }
        exact = off > 0.5f - 0x1p-15f;
      }
      if (__builtin_expect(exact, !kNarrow)) {
#pragma unroll
        for (uint32_t e = 0; e < kChunk; ++e)
          q[e] = (uint32_t)nearest_step((double)h[i].get(e) * (double)y[e], most, step);
      }
      uint32_t lo = four_bytes(q[0], q[1], q[2], q[3]), hi = four_bytes(q[4], q[5], q[6], q[7]);
      if (bad) lo = hi = 0;
      int8_t* to = p.q + (size_t)row * p.q_ld + j;
      if (n >= kChunk) {
        *reinterpret_cast<Bytes8*>(to) = Words2{lo, hi};
      } else {
#pragma unroll
        for (uint32_t e = 0; e < kChunk; ++e)
          if (e < n) to[e] = (int8_t)((e < 4 ? lo : hi) >> (8u * (e % 4)));
      }
    }
    if (t == 0) p.scale[row] = bad ? __builtin_nanf("") : scale;
  }
  if (p.err != nullptr) {
    if (!bad) {
      if (t == 0) put_record(p.err, row, PB_OK, 0, 0, 0);
      return;
    }
    // the first column that failed, with its bits of h: the smallest (column, bits)
    uint64_t at = ~0ull;
#pragma unroll
    for (int i = C - 1; i >= 0; --i) {
      float y[kChunk];
      weights(i, y);
#pragma unroll
      for (int e = (int)kChunk - 1; e >= 0; --e) {
        const uint32_t j = (i * T + t) * kChunk + e;
        const float v = h[i].get(e);
        const bool failed =
            !isfinite(v) || (eight && !isfinite((double)v * (double)y[e]));
        if (j < p.cols && failed) at = (uint64_t)j << 32 | b_of(v);
      }
    }
    at = ~row_stats<T>(0.0, ~at).top;
    if (t == 0) {
      if (at == ~0ull) at = (uint64_t)p.cols << 32;  // the scale
      put_record(p.err, row, PB_NONFINITE_INPUT, 0, at & 0xffffffffu,
                 (uint64_t)PB_FIELD_FINITE << 32 | at >> 32);
    }
  }
}

// The gradient, bound by its rows' bytes: 8,192 rows of 2,048 bf16 25.9 us (5.5 TB/s
// with the parts' sums).  With m = rstd and c = mean(g w h): dh = gh + m (g w - h m^2 c), and
// the weight's is the sum of g h m over the rows.  The statistics are taken anew from h,
// which is read anyway.  A workgroup goes over rows, the next one requested before the one at
// hand is worked out, and holds its sums of the weight's gradient in registers; they are
// joined over the workgroups in 64 bits.  Rows of more than 8,192 columns do not fit the
// registers: their second pass reads them again, and the sums are in LDS.  kSame: gradients, weight
// and rows of one type, held as they are in memory.
template <typename E, bool kSame, int T, int C>
__global__ __launch_bounds__(T < 128 ? 256 : T) void norm_grad_kernel(NormGradParams p) {
  constexpr uint32_t kRows = T < 128 ? 256 / T : 1;
  constexpr bool kHold = T < 1024, kHoldAll = kHold && kSame;
  const uint32_t t = threadIdx.x % T;
  auto column = [&](int i) { return (i * T + t) * kChunk; };
  constexpr int kUnroll = kHold ? C : 1;
  Chunk<E> w[kHoldAll ? C : 1];
  // the sums of the weight's gradient
  float held[kHold ? C : 1][kChunk];
  __shared__ float kept[kHold ? 1 : C * kChunk][kHold ? 1 : T];
  auto dw = [&](int i, uint32_t e) -> float& {
    if constexpr (kHold) return held[i][e];
    else return kept[i * kChunk + e][t];
  };
#pragma unroll
  for (int i = 0; i < C; ++i) {
    if constexpr (kHoldAll) load_weight<E>(p.weight, column(i), chunk_left(p.cols, column(i)), w[i]);
#pragma unroll
    for (uint32_t e = 0; e < kChunk; ++e) dw(i, e) = 0.0f;
  }
  struct Row {
    Chunk<E> h[kHold ? C : 1], g[kHoldAll ? C : 1], more[kHold ? C : 1];
  };
  auto load_rows = [&](Chunk<E>& c, const void* base, size_t ld, uint32_t row, int i) {
    c.load(static_cast<const typename E::Raw*>(base) + (size_t)row * ld + column(i),
           chunk_left(p.cols, column(i)));
  };
  auto request = [&](Row& r, uint32_t row) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      load_rows(r.h[i], p.h, p.h_ld, row, i);
      if constexpr (kSame) load_rows(r.g[i], p.grad, p.grad_ld, row, i);
      if (p.grad_sum != nullptr) load_rows(r.more[i], p.grad_sum, p.grad_sum_ld, row, i);
    }
  };
  const uint32_t turn = p.groups * kRows;
  uint32_t row = blockIdx.x * kRows + threadIdx.x / T;
  Row next{};
  if (kHold && row < p.rows) request(next, row);
  for (; row < p.rows; row += turn) {
    const Row r = next;
    if (kHold && row + turn < p.rows) request(next, row + turn);
    // h, g and g w of a chunk
    auto take = [&](int i, float (&h)[kChunk], float (&g)[kChunk], float (&gw)[kChunk]) {
      const uint32_t j = column(i), n = chunk_left(p.cols, j);
      if constexpr (kHold) {
#pragma unroll
        for (uint32_t e = 0; e < kChunk; ++e) h[e] = r.h[i].get(e);
      } else {
        load_row<E>(static_cast<const typename E::Raw*>(p.h) + (size_t)row * p.h_ld + j, n, h);
      }
      if constexpr (kHoldAll) {
#pragma unroll
        for (uint32_t e = 0; e < kChunk; ++e) {
          g[e] = r.g[i].get(e);
          gw[e] = g[e] * w[i].get(e);
        }
      } else {
        load_any(p.grad, p.grad_dtype, (size_t)row * p.grad_ld + j, n, g);
        load_weight(p.weight, p.weight_dtype, j, n, gw);
#pragma unroll
        for (uint32_t e = 0; e < kChunk; ++e) gw[e] = g[e] * gw[e];
      }
    };
    double squares = 0.0, along = 0.0;
#pragma unroll kUnroll
    for (int i = 0; i < C; ++i) {
      float h[kChunk], g[kChunk], gw[kChunk];
      take(i, h, g, gw);
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) {
        const double v = (double)h[e];
        squares = fma(v, v, squares);
        along = fma((double)gw[e], v, along);
      }
    }
    struct Two {
      double a, b;
    };
    const Two s = row_join<T>(Two{wave_add(squares), wave_add(along)}, [](Two x, Two y) {
      return Two{x.a + y.a, x.b + y.b};
    });
    const double rstd = 1.0 / sqrt(s.a / (double)p.cols + p.eps);
    const float m = (float)rstd, k = (float)(rstd * rstd * (s.b / (double)p.cols));
#pragma unroll kUnroll
    for (int i = 0; i < C; ++i) {
      const uint32_t j = column(i), n = chunk_left(p.cols, j);
      float h[kChunk], g[kChunk], gw[kChunk];
      take(i, h, g, gw);
      if (p.grad_h != nullptr) {
        float y[kChunk];
#pragma unroll
        for (uint32_t e = 0; e < kChunk; ++e) y[e] = m * (gw[e] - h[e] * k);
        if (p.grad_sum != nullptr) {
          float more[kChunk];
          if constexpr (kHold) {
#pragma unroll
            for (uint32_t e = 0; e < kChunk; ++e) more[e] = r.more[i].get(e);
          } else {
            load_row<E>(static_cast<const typename E::Raw*>(p.grad_sum) +
                            (size_t)row * p.grad_sum_ld + j, n, more);
          }
#pragma unroll
          for (uint32_t e = 0; e < kChunk; ++e) y[e] = y[e] + more[e];
        }
        store_row<E>(static_cast<typename E::Raw*>(p.grad_h) + (size_t)row * p.grad_h_ld + j, n,
                     y);
      }
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) dw(i, e) = dw(i, e) + g[e] * (h[e] * m);
    }
  }
  if (p.grad_weight == nullptr) return;
  float* part = p.part + (size_t)blockIdx.x * p.cols;
  if constexpr (T == 64) {
    __shared__ float waves[3][C * 64 * kChunk];  // of all waves but the first
    const uint32_t wave = threadIdx.x >> 6;
    if (wave != 0) {
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (uint32_t e = 0; e < kChunk; ++e) waves[wave - 1u][(i * kChunk + e) * 64u + t] = dw(i, e);
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) {
        const uint32_t at = (i * kChunk + e) * 64u + t;
        dw(i, e) = ((dw(i, e) + waves[0][at]) + waves[1][at]) + waves[2][at];
      }
  }
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const uint32_t j = column(i);
    float y[kChunk];
#pragma unroll
    for (uint32_t e = 0; e < kChunk; ++e) y[e] = dw(i, e);
    store_row<F32>(reinterpret_cast<uint32_t*>(part + j), chunk_left(p.cols, j), y);
  }
}

// The workgroups' sums of the weight's gradient: 16 columns a workgroup, 64 of the sums at a
// time.  A launch of its own, 4 to 5 us: joined by the last workgroup to come instead, one
// compute unit would read them all (1,024 x 2,048 sums: 8 MB).
__global__ __launch_bounds__(1024) void norm_weight_kernel(NormGradParams p) {
  __shared__ double parts[64][16];
  const uint32_t c = threadIdx.x % 16u, k0 = threadIdx.x / 16u;
  const uint32_t j = blockIdx.x * 16u + c;
  double sum = 0.0;
  if (j < p.cols) {
#pragma unroll 8
    for (uint32_t k = k0; k < p.groups; k += 64u) sum = sum + (double)p.part[(size_t)k * p.cols + j];
  }
  parts[k0][c] = sum;
  __syncthreads();
  if (k0 != 0 || j >= p.cols) return;
#pragma unroll
  for (uint32_t k = 1; k < 64; ++k) sum = sum + parts[k][c];
  p.grad_weight[j] = p.accumulate ? (float)((double)p.grad_weight[j] + sum) : (float)sum;
}

// ---- plans ----

// log2 of the threads of a row of `cols` elements, up to a workgroup.
uint32_t row_shift(uint32_t cols) {
  const uint32_t chunks = (cols + kChunk - 1u) / kChunk;
  uint32_t shift = 0;
  while (shift < 8 && (1u << shift) < chunks) ++shift;
  return shift;
}

uint32_t sort_tiles(uint32_t rows) { return (rows + kSortTile - 1u) / kSortTile; }

// Chunks of a row's plan below: its threads times theirs.
uint32_t row_span(uint32_t cols) {
  uint32_t span = 64;
  while (span * kChunk < cols) span *= 2;
  return span;
}

// Workgroups of the norm's gradient.  More have more rows on their way, fewer leave fewer sums
// to join: as many as hold kGradChunks chunks at once, 512 or more, and none with more than
// kGradTerms rows, whose sum it has in 32 bits.  512 / 1,024 / 2,048 of them, us:
//   65,536 x 512 (256 chunks)     58 /  57 /  59     16,384 x 4,096 (512)  103 / 119 / 118
//   65,536 x 896 (128)           215 / 126 / 100     8,192 x 8,192 (1,024) 109 / 117 / 134
//   8,192 x 2,048 (256)         33.1 / 32.8 / 37.8
constexpr uint32_t kGradChunks = 1u << 18;
constexpr uint32_t kGradTerms = 768;
uint32_t grad_groups(uint32_t rows, uint32_t cols) {
  const uint32_t span = row_span(cols), at_once = span < 128 ? 256 / span : 1;
  const uint32_t all = (rows + at_once - 1u) / at_once;
  const uint32_t held = kGradChunks / (span * at_once), turns = kGradTerms / at_once;
  const uint32_t least = (all + turns - 1u) / turns;
  uint32_t most = held > 512 ? held : 512;
  if (most < least) most = least;
  return all < most ? all : most;
}

size_t round_up(size_t bytes) { return (bytes + 255u) & ~(size_t)255u; }

// A row's threads and their chunks.  One chunk a thread, and two where the statistics' join
// over the waves then weighs more; but two as well where there are rows enough to keep the
// memory busy, so that more of them are on their way.  Norms of bf16 rows to 8 bits, us (threads,
// chunks):
//                  1 row                                70 rows                65,536 to 8,192 rows
//   512   (64, 1)  2.6 (128, 1) 2.9                      3.6 / 3.8               56 / 77
//   896   (64, 2)  3.7 (128, 1) 3.1 (256, 1) 3.2         5.3 / 3.9 / 4.1         96 / 91 / 159
//   2,048 (128, 2) 3.1 (256, 1) 3.0 (512, 1) 3.5         4.8 / 4.1 / 4.2         93 / 90 / 159
//   4,096 (128, 4) 4.2 (256, 2) 3.6 (512, 1) 3.2         7.2 / 5.3 / 4.4        104 / 91 / 95
//   8,192 (256, 4) 4.6 (512, 2) 3.8 (1024, 1) 4.2        8.0 / 6.0 / 5.9        109 / 99 / 136
//   16,384 (512, 4) 5.3 (1024, 2) 5.4                    9.2 / 8.7              123 / 122
constexpr uint32_t kManyRows = 1024;  // 512 rows of 4,096: (256, 2) 6.6, (512, 1) 6.3; 8,192: 48.8, 49.8
template <typename E, bool kOne, template <typename, bool, int, int> class Launch, typename P>
hipError_t by_width(const P& p, hipStream_t stream) {
  switch (row_span(p.cols)) {
    case 64: return Launch<E, kOne, 64, 1>::run(p, stream);
    case 128: return Launch<E, kOne, 128, 1>::run(p, stream);
    case 256: return Launch<E, kOne, 256, 1>::run(p, stream);
    case 512:
      return p.rows < kManyRows ? Launch<E, kOne, 512, 1>::run(p, stream)
                                : Launch<E, kOne, 256, 2>::run(p, stream);
    case 1024: return Launch<E, kOne, 512, 2>::run(p, stream);
    case 2048: return Launch<E, kOne, 1024, 2>::run(p, stream);
    default: return Launch<E, kOne, 1024, 4>::run(p, stream);
  }
}

template <typename E, bool kNarrow, int T, int C>
struct NormLaunch {
  static hipError_t run(const NormParams& p, hipStream_t stream) {
    constexpr uint32_t kRows = T < 128 ? 256 / T : 1;
    norm_kernel<E, kNarrow, T, C><<<(p.rows + kRows - 1u) / kRows, T * kRows, 0, stream>>>(p);
    return hipGetLastError();
  }
};

template <typename E, bool kSame, int T, int C>
struct NormGradLaunch {
  static hipError_t run(const NormGradParams& in, hipStream_t stream) {
    constexpr uint32_t kRows = T < 128 ? 256 / T : 1;  // as grad_groups has it
    NormGradParams p = in;
    p.groups = grad_groups(p.rows, p.cols);
    hipError_t e = hipSuccess;
    if (p.groups != 0) {  // without rows the weight's gradient is zeros
      norm_grad_kernel<E, kSame, T, C><<<p.groups, T * kRows, 0, stream>>>(p);
      e = hipGetLastError();
    }
    if (e != hipSuccess || p.grad_weight == nullptr) return e;
    norm_weight_kernel<<<(p.cols + 15u) / 16u, 1024, 0, stream>>>(p);
    return hipGetLastError();
  }
};

template <typename In, typename Out>
hipError_t embed_as(const EmbedParams& p, hipStream_t stream) {
  const uint32_t shift = row_shift(p.cols), at_once = 256u >> shift;
  embed_kernel<In, Out><<<(p.rows + at_once - 1u) / at_once, 256, 0, stream>>>(p, shift);
  return hipGetLastError();
}
template <typename In>
hipError_t embed_from(const EmbedParams& p, uint32_t out_dtype, hipStream_t stream) {
  if (out_dtype == PB_F32) return embed_as<In, F32>(p, stream);
  if (out_dtype == PB_F16) return embed_as<In, F16>(p, stream);
  return embed_as<In, BF16>(p, stream);
}

// Workgroups that write zeros beside a sort: four a compute unit, of 256 threads.
constexpr uint32_t kZeroGroups = 1024;

template <typename G, typename T>
hipError_t embed_grad_as(const EmbedGradParams& p, hipStream_t stream) {
  hipError_t e = hipSuccess;
  if (p.rows == 0) {
    if (!p.accumulate) {
      zero_table_kernel<T><<<kZeroGroups, 256, 0, stream>>>(p);
      e = hipGetLastError();
    }
    return e;
  }
  uint32_t bits = 0;
  while (p.vocab >> bits) ++bits;
  const uint32_t passes = (bits + kSortBits - 1u) / kSortBits;
  if (p.rows <= kSortFew) {
    sort_rows_kernel<T, kSortFew><<<p.accumulate ? 1 : 512, kSortThreads, 0, stream>>>(p, passes);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  } else if (p.rows <= kSortRows) {
    sort_rows_kernel<T, kSortRows><<<p.accumulate ? 1 : 256, kSortThreads, 0, stream>>>(p, passes);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  } else {
    const uint32_t tiles = sort_tiles(p.rows), groups = p.accumulate ? 0 : kZeroGroups;
    ZeroShare zero{0, 2u * passes * groups};
    for (uint32_t pass = 0; pass < passes; ++pass) {
      sort_count_kernel<T><<<tiles + groups, 256, 0, stream>>>(p, pass, tiles, zero);
      zero.part += groups;
      if ((e = hipGetLastError()) != hipSuccess) return e;
      sort_place_kernel<T><<<tiles + groups, 256, 0, stream>>>(p, pass, tiles, zero);
      zero.part += groups;
      if ((e = hipGetLastError()) != hipSuccess) return e;
    }
  }
  const uint32_t last = passes & 1u;
  const uint32_t col_tiles = (p.cols + 64u * G::kPer - 1u) / (64u * G::kPer);
  const uint32_t units = sum_parts(p.rows) * col_tiles;
  sum_rows_kernel<G, T><<<(units + 3u) / 4u, 256, 0, stream>>>(p, last, col_tiles, units);
  if ((e = hipGetLastError()) != hipSuccess || p.rows <= kSumRows) return e;
  // as many as the most there can be to do, waves for short tokens or workgroups for long ones
  const size_t parts = sum_parts(p.rows) - 1u;
  const size_t short_groups = (parts * ((p.cols + 255u) / 256u) + kJoinWaves - 1u) / kJoinWaves;
  const size_t long_groups = parts / (kLongParts + 1u) * ((p.cols + 63u) / 64u);
  const size_t most = short_groups > long_groups ? short_groups : long_groups;
  join_rows_kernel<T>
      <<<(uint32_t)(most < 512 ? most : 512), 64 * kJoinWaves, 0, stream>>>(p, last);
  return hipGetLastError();
}
template <typename G>
hipError_t embed_grad_from(const EmbedGradParams& p, uint32_t table_dtype, hipStream_t stream) {
  if (table_dtype == PB_F32) return embed_grad_as<G, F32>(p, stream);
  if (table_dtype == PB_F16) return embed_grad_as<G, F16>(p, stream);
  return embed_grad_as<G, BF16>(p, stream);
}

}  // namespace

size_t embed_grad_bytes(uint32_t rows, size_t cols) {
  const size_t tiles = sort_tiles(rows), parts = sum_parts(rows);
  return 4 * round_up((size_t)rows * 4) + round_up((tiles << kSortBits) * 4) +
         round_up((parts + 2) * 4) + round_up(parts * 2 * cols * 4);
}

size_t norm_grad_bytes(uint32_t rows, size_t cols) {
  return (size_t)grad_groups(rows, (uint32_t)cols) * cols * 4;
}

size_t hidden_workspace_bytes(uint32_t rows, size_t cols) {
  size_t most = embed_grad_bytes(rows, cols);
  auto hold = [&](size_t c) {
    const size_t b = norm_grad_bytes(rows, c);
    if (b > most) most = b;
  };
  hold(cols);
  // narrower rows may have more workgroups: the widest of each plan
  for (size_t c = 64 * kChunk; c < cols; c *= 2) hold(c);
  return most;
}

void place_embed_grad(void* work, EmbedGradParams* p) {
  char* at = static_cast<char*>(work);
  auto take = [&](size_t bytes) {
    char* here = at;
    at += round_up(bytes);
    return here;
  };
  const size_t words = (size_t)p->rows * 4;
  for (uint32_t k = 0; k < 2; ++k) {
    p->id[k] = reinterpret_cast<uint32_t*>(take(words));
    p->row[k] = reinterpret_cast<uint32_t*>(take(words));
  }
  p->count = reinterpret_cast<uint32_t*>(take(((size_t)sort_tiles(p->rows) << kSortBits) * 4));
  p->cross = reinterpret_cast<uint32_t*>(take(((size_t)sum_parts(p->rows) + 2) * 4));
  p->part = reinterpret_cast<float*>(at);
}

void place_norm_grad(void* work, NormGradParams* p) { p->part = static_cast<float*>(work); }

hipError_t launch_embed(const EmbedParams& p, uint32_t dtype, uint32_t out_dtype,
                        hipStream_t stream) {
  if (dtype == PB_F32) return embed_from<F32>(p, out_dtype, stream);
  if (dtype == PB_F16) return embed_from<F16>(p, out_dtype, stream);
  return embed_from<BF16>(p, out_dtype, stream);
}

hipError_t launch_embed_grad(const EmbedGradParams& p, uint32_t dtype, uint32_t table_dtype,
                             hipStream_t stream) {
  if (dtype == PB_F32) return embed_grad_from<F32>(p, table_dtype, stream);
  if (dtype == PB_F16) return embed_grad_from<F16>(p, table_dtype, stream);
  return embed_grad_from<BF16>(p, table_dtype, stream);
}

hipError_t launch_norm(const NormParams& p, uint32_t dtype, hipStream_t stream) {
  const bool one = p.weight == nullptr || p.weight_dtype == dtype;
  if (dtype == PB_F32) return by_width<F32, false, NormLaunch>(p, stream);
  if (dtype == PB_F16)
    return one ? by_width<F16, true, NormLaunch>(p, stream)
               : by_width<F16, false, NormLaunch>(p, stream);
  return one ? by_width<BF16, true, NormLaunch>(p, stream)
             : by_width<BF16, false, NormLaunch>(p, stream);
}

template <typename E>
hipError_t norm_grad_as(const NormGradParams& p, uint32_t dtype, hipStream_t stream) {
  if (p.grad_dtype == dtype && (p.weight == nullptr || p.weight_dtype == dtype))
    return by_width<E, true, NormGradLaunch>(p, stream);
  return by_width<E, false, NormGradLaunch>(p, stream);
}
hipError_t launch_norm_grad(const NormGradParams& p, uint32_t dtype, hipStream_t stream) {
  if (dtype == PB_F32) return norm_grad_as<F32>(p, dtype, stream);
  if (dtype == PB_F16) return norm_grad_as<F16>(p, dtype, stream);
  return norm_grad_as<BF16>(p, dtype, stream);
}

}  // namespace pb
