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
__device__ __forceinline__ uint64_t wave_max_word(uint64_t v) { return wave_max64(v); }

// ---- table rows of tokens ----

// 2^kShift threads take a row.
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
// time: counts of a tile's digits, their prefix over digits and tiles, and the pairs'
// places), so a token's rows come next to each other and in order.  Then the sorted rows
// are cut into parts of kSumRows: a wave adds up its part's rows token by token, and
// what lies whole within a part is written at once.  What crosses parts is left in the
// workspace and joined in 64 bits.  No atomics touch the sums, so they repeat.

// Rows that add nothing sort behind every token.
__device__ __forceinline__ uint32_t sort_key(const EmbedGradParams& p, uint32_t pass, uint32_t i) {
  if (pass != 0) return p.id[pass & 1u][i];
  const uint32_t id = p.token[i];
  return id < p.vocab ? id : p.vocab;
}

__global__ __launch_bounds__(256) void sort_count_kernel(EmbedGradParams p, uint32_t pass,
                                                         uint32_t tiles) {
  __shared__ uint32_t hist[1u << kSortBits];
  const uint32_t tile = blockIdx.x;
  for (uint32_t d = threadIdx.x; d < (1u << kSortBits); d += 256u) hist[d] = 0;
  if (pass == 0 && tile == 0 && threadIdx.x == 0) p.cross[0] = 0;
  __syncthreads();
  for (uint32_t k = 0; k < kSortTile / 256u; ++k) {
    const uint32_t i = tile * kSortTile + k * 256u + threadIdx.x;
    if (i < p.rows) {
      const uint32_t d = sort_key(p, pass, i) >> (pass * kSortBits) & ((1u << kSortBits) - 1u);
      atomicAdd(&hist[d], 1u);
    }
  }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < (1u << kSortBits); d += 256u)
    p.count[(size_t)d * tiles + tile] = hist[d];
}

// Exclusive prefix of the counts, digit by digit and tile by tile, by one workgroup.
__global__ __launch_bounds__(1024) void sort_prefix_kernel(uint32_t* count, uint32_t n) {
  __shared__ uint32_t waves[16];
  const uint32_t lane = lane_id(), wave = threadIdx.x >> 6;
  const uint32_t per = (n + 1023u) / 1024u;
  const uint32_t lo = threadIdx.x * per < n ? threadIdx.x * per : n;
  const uint32_t hi = lo + per < n ? lo + per : n;
  uint32_t sum = 0;
  for (uint32_t i = lo; i < hi; ++i) sum += count[i];
  uint32_t upto = sum;  // inclusive over the wave's lanes
#pragma unroll
  for (uint32_t m = 1; m < 64; m <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)upto, m, 64);
    if (lane >= m) upto += o;
  }
  if (lane == 63) waves[wave] = upto;
  __syncthreads();
  uint32_t base = upto - sum;
  for (uint32_t w = 0; w < wave; ++w) base += waves[w];
  for (uint32_t i = lo; i < hi; ++i) {
    const uint32_t c = count[i];
    count[i] = base;
    base += c;
  }
}

__global__ __launch_bounds__(256) void sort_place_kernel(EmbedGradParams p, uint32_t pass,
                                                         uint32_t tiles) {
  constexpr uint32_t kSteps = kSortTile / 256u;
  __shared__ uint32_t place[4][1u << kSortBits];
  const uint32_t tile = blockIdx.x, lane = lane_id(), wave = threadIdx.x >> 6;
  for (uint32_t d = threadIdx.x; d < 4u << kSortBits; d += 256u) (&place[0][0])[d] = 0;
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
    const uint32_t d = key[k] >> (pass * kSortBits) & ((1u << kSortBits) - 1u);
    uint64_t same = __ballot(real);
#pragma unroll
    for (uint32_t b = 0; b < kSortBits; ++b) {
      const uint64_t set = __ballot(d >> b & 1u);
      same &= (d >> b & 1u) ? set : ~set;
    }
    rank[k] = 0;
    if (real) {
      const uint32_t below = lanes_below(same);
      uint32_t before = 0;
      if (below == 0)
        before = atomicAdd(&place[wave][d], (uint32_t)__popcll((unsigned long long)same));
      const int leader = __ffsll((unsigned long long)same) - 1;
      rank[k] = (uint32_t)__shfl((int)before, leader, 64) + below;
    }
  }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < (1u << kSortBits); d += 256u) {
    uint32_t base = p.count[(size_t)d * tiles + tile];
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
      const uint32_t n = place[w][d];
      place[w][d] = base;
      base += n;
    }
  }
  __syncthreads();
  uint32_t* id = p.id[(pass + 1u) & 1u];
  uint32_t* row = p.row[(pass + 1u) & 1u];
#pragma unroll
  for (uint32_t k = 0; k < kSteps; ++k) {
    const uint32_t i = first + k * 64u + lane;
    if (i < p.rows) {
      const uint32_t d = key[k] >> (pass * kSortBits) & ((1u << kSortBits) - 1u);
      const uint32_t at = place[wave][d] + rank[k];
      id[at] = key[k];
      row[at] = pass == 0 ? i : p.row[pass & 1u][i];
    }
  }
}

// Zeros for a whole table, 2^shift threads a row.
template <typename T>
__global__ __launch_bounds__(256) void zero_rows_kernel(typename T::Raw* table, size_t ld,
                                                        uint32_t rows, uint32_t cols,
                                                        uint32_t shift) {
  const uint32_t row = blockIdx.x * (256u >> shift) + (threadIdx.x >> shift);
  if (row >= rows) return;
  typename T::Raw* to = table + (size_t)row * ld;
  const float zero[kChunk] = {};
  for (uint32_t j = (threadIdx.x & ((1u << shift) - 1u)) * kChunk; j < cols; j += kChunk << shift)
    store_row<T>(to + j, cols - j, zero);
}

template <typename T, int N>
__device__ __forceinline__ void put_table(const EmbedGradParams& p, uint32_t id, uint32_t j,
                                          uint32_t n, const float (&sum)[N]) {
  typename T::Raw* to = static_cast<typename T::Raw*>(p.table) + (size_t)id * p.table_ld + j;
  float y[N];
#pragma unroll
  for (int e = 0; e < N; ++e) y[e] = sum[e] * p.scale;
  if (p.accumulate) {
    float old[N];
    load_row<T>(to, n, old);
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = old[e] + y[e];
  }
  store_row<T>(to, n, y);
}

// One wave: the sorted rows [part kSumRows, + kSumRows) and 64 chunks of columns.
template <typename G, typename T>
__global__ __launch_bounds__(256) void sum_rows_kernel(EmbedGradParams p, uint32_t last,
                                                       uint32_t col_tiles, uint32_t units) {
  constexpr int N = G::kPer;
  constexpr uint32_t kAhead = 8;
  static_assert(kSumRows % kAhead == 0, "whole groups");
  const uint32_t unit =
      (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4u + (threadIdx.x >> 6)));
  if (unit >= units) return;
  const uint32_t part = unit / col_tiles, tile = unit - part * col_tiles;
  const uint32_t j = (tile * 64u + lane_id()) * N;
  const uint32_t n = chunk_left(p.cols, j);
  const uint32_t* id = p.id[last];
  const uint32_t* row = p.row[last];
  const typename G::Raw* grad = static_cast<const typename G::Raw*>(p.grad) + j;
  const uint32_t lo = part * kSumRows;
  const uint32_t hi = lo + kSumRows < p.rows ? lo + kSumRows : p.rows;
  uint32_t cur = id[lo];
  if (cur >= p.vocab) return;
  bool from_before = lo > 0 && id[lo - 1] == cur;  // the sum goes on from the part before
  float sum[N] = {};
  auto leave = [&](bool goes_on) {
    if (!from_before && !goes_on) {
      put_table<T>(p, cur, j, n, sum);
    } else {
      float* to = p.part + ((size_t)part * 2u + (from_before ? 0u : 1u)) * p.cols + j;
      store_row<F32>(reinterpret_cast<uint32_t*>(to), n, sum);
      if (!from_before && tile == 0 && lane_id() == 0) p.cross[1u + atomicAdd(p.cross, 1u)] = part;
    }
  };
  for (uint32_t i = lo; i < hi; i += kAhead) {
    uint32_t ids[kAhead], rows[kAhead];
    float x[kAhead][N];
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) {
      const uint32_t at = i + k < hi ? i + k : hi - 1u;
      ids[k] = (uint32_t)__builtin_amdgcn_readfirstlane((int)id[at]);
      rows[k] = (uint32_t)__builtin_amdgcn_readfirstlane((int)row[at]);
    }
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) load_row<G>(grad + (size_t)rows[k] * p.grad_ld, n, x[k]);
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) {
      if (i + k >= hi) break;
      if (ids[k] != cur) {
        leave(false);
        cur = ids[k];
        from_before = false;
        if (cur >= p.vocab) return;
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] = sum[e] + x[k][e];
    }
  }
  leave(hi < p.rows && id[hi] == cur);
}

// The sums that cross parts, 64 columns a workgroup: its waves take a run of parts each.
template <typename T>
__global__ __launch_bounds__(256) void join_rows_kernel(EmbedGradParams p, uint32_t last,
                                                        uint32_t col_tiles) {
  __shared__ double waves[4][64];
  const uint32_t lane = lane_id(), wave = threadIdx.x >> 6;
  const uint32_t* id = p.id[last];
  const uint32_t crossing = p.cross[0];
  for (size_t unit = blockIdx.x; unit < (size_t)crossing * col_tiles; unit += gridDim.x) {
    const uint32_t part = p.cross[1u + unit / col_tiles];
    const uint32_t j = (uint32_t)(unit % col_tiles) * 64u + lane;
    const uint32_t own = id[(part + 1u) * kSumRows - 1u];
    // the first sorted row behind the token's last
    uint32_t lo = (part + 1u) * kSumRows, hi = p.rows;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2u;
      if (id[mid] == own) lo = mid + 1u;
      else hi = mid;
    }
    const uint32_t n = (lo - 1u) / kSumRows - part + 1u;  // parts, the first one's tail included
    const uint32_t from = (uint32_t)((uint64_t)n * wave / 4u);
    const uint32_t to = (uint32_t)((uint64_t)n * (wave + 1u) / 4u);
    double sum = 0.0;
    if (j < p.cols)
      for (uint32_t k = from; k < to; ++k)
        sum = sum + (double)p.part[((size_t)(part + k) * 2u + (k == 0 ? 1u : 0u)) * p.cols + j];
    waves[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && j < p.cols) {
      const float all[1] = {
          (float)(((waves[0][lane] + waves[1][lane]) + waves[2][lane]) + waves[3][lane])};
      typename T::Raw* at = static_cast<typename T::Raw*>(p.table) + (size_t)own * p.table_ld + j;
      const float y = all[0] * p.scale;
      *at = T::raw(p.accumulate ? T::one(*at) + y : y);
    }
    __syncthreads();
  }
}

// ---- norms ----
//
// A row is held in registers between its statistics and its outputs: T threads take C
// chunks of eight elements each.  mean(h^2) is summed in 64 bits: no binary32 row
// overflows there, and 64-bit multiply-adds issue as often as 32-bit ones here.

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

// Sums of `a` and maxima of `m` over a row's T threads, in every one of them.
template <int T>
__device__ __forceinline__ void row_reduce(double& a, uint64_t& m) {
  a = wave_add(a);
  m = wave_max_word(m);
  if constexpr (T > 64) {
    __shared__ double as[T / 64];
    __shared__ uint64_t ms[T / 64];
    __syncthreads();
    if (lane_id() == 0) {
      as[threadIdx.x >> 6] = a;
      ms[threadIdx.x >> 6] = m;
    }
    __syncthreads();
    a = as[0];
    m = ms[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) {
      a = a + as[w];
      m = ms[w] > m ? ms[w] : m;
    }
  }
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

template <typename E, int T, int C>
__global__ __launch_bounds__(T < 256 ? 256 : T) void norm_kernel(NormParams p) {
  constexpr uint32_t kRows = T < 256 ? 256 / T : 1;
  const uint32_t t = threadIdx.x % T;
  const uint32_t row = blockIdx.x * kRows + threadIdx.x / T;
  if (row >= p.rows) return;  // whole waves, and with T > 64 never
  const typename E::Raw* x = static_cast<const typename E::Raw*>(p.x) + (size_t)row * p.x_ld;
  float h[C][kChunk], w[C][kChunk];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const uint32_t j = (i * T + t) * kChunk, n = chunk_left(p.cols, j);
    load_row<E>(x + j, n, h[i]);
    load_weight(p.weight, p.weight_dtype, j, n, w[i]);
  }
  if (p.residual != nullptr) {
    const typename E::Raw* r =
        static_cast<const typename E::Raw*>(p.residual) + (size_t)row * p.residual_ld;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t j = (i * T + t) * kChunk, n = chunk_left(p.cols, j);
      float y[kChunk];
      load_row<E>(r + j, n, y);
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) h[i][e] = E::one(E::raw(h[i][e] + y[e]));
    }
  }
  if (p.sum != nullptr) {
    typename E::Raw* to = static_cast<typename E::Raw*>(p.sum) + (size_t)row * p.sum_ld;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t j = (i * T + t) * kChunk, n = chunk_left(p.cols, j);
      store_row<E>(to + j, n, h[i]);
    }
  }

  // statistics: the squares' sum, and the bits of the largest |h w| (a NaN's are larger still)
  double squares = 0.0;
  uint64_t top = 0;
#pragma unroll
  for (int i = 0; i < C; ++i) {
#pragma unroll
    for (uint32_t e = 0; e < kChunk; ++e) {
      const double v = (double)h[i][e];
      squares = fma(v, v, squares);
      if (p.q != nullptr) {
        const uint32_t j = (i * T + t) * kChunk + e;
        const uint64_t b = j < p.cols ? abs_bits(v * (double)w[i][e]) : 0;
        top = b > top ? b : top;
      }
    }
  }
  row_reduce<T>(squares, top);
  const double rstd = p.norm ? 1.0 / sqrt(squares / (double)p.cols + p.eps) : 1.0;
  const double most = __builtin_bit_cast(double, top);
  const float scale = (float)(rstd * (most / 127.0));
  const bool bad = !isfinite(squares) || (p.q != nullptr && (top >= kInfBits || !isfinite(scale)));

  if (p.out != nullptr) {
    const float r = bad ? __builtin_nanf("") : (float)rstd;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t j = (i * T + t) * kChunk, n = chunk_left(p.cols, j);
      float y[kChunk];
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) y[e] = h[i][e] * r * w[i][e];
      store_any(p.out, p.out_dtype, (size_t)row * p.out_ld + j, n, y);
    }
  }
  if (p.q != nullptr) {
    const double step = most > 0.0 ? 127.0 / most : 0.0;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t j = (i * T + t) * kChunk, n = chunk_left(p.cols, j);
      uint32_t word[2] = {};
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) {
        const int v = bad ? 0 : nearest_step((double)h[i][e] * (double)w[i][e], most, step);
        word[e / 4] |= ((uint32_t)v & 0xffu) << (8u * (e % 4));
      }
      int8_t* to = p.q + (size_t)row * p.q_ld + j;
      if (n >= kChunk) {
        *reinterpret_cast<Bytes8*>(to) = Words2{word[0], word[1]};
      } else {
#pragma unroll
        for (uint32_t e = 0; e < kChunk; ++e)
          if (e < n) to[e] = (int8_t)(word[e / 4] >> (8u * (e % 4)));
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
#pragma unroll
      for (int e = (int)kChunk - 1; e >= 0; --e) {
        const uint32_t j = (i * T + t) * kChunk + e;
        const bool failed = !isfinite(h[i][e]) ||
                            (p.q != nullptr && !isfinite((double)h[i][e] * (double)w[i][e]));
        if (j < p.cols && failed) at = (uint64_t)j << 32 | b_of(h[i][e]);
      }
    }
    double none = 0.0;
    at = ~at;
    row_reduce<T>(none, at);
    at = ~at;
    if (t == 0) {
      if (at == ~0ull) at = (uint64_t)p.cols << 32;  // the scale
      put_record(p.err, row, PB_NONFINITE_INPUT, 0, at & 0xffffffffu,
                 (uint64_t)PB_FIELD_FINITE << 32 | at >> 32);
    }
  }
}

// The gradient.  With m = rstd and c = mean(g w h): dh = gh + m (g w - h m^2 c), and
// the weight's is the sum of g h m over the rows.  The statistics are taken anew from h,
// which is read anyway.  A workgroup goes over rows and holds its sums of the weight's
// gradient in registers; they are joined over the workgroups in 64 bits.
template <typename E, int T, int C>
__global__ __launch_bounds__(T < 256 ? 256 : T) void norm_grad_kernel(NormGradParams p) {
  constexpr uint32_t kRows = T < 256 ? 256 / T : 1;
  const uint32_t t = threadIdx.x % T;
  float w[C][kChunk], dw[C][kChunk];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const uint32_t j = (i * T + t) * kChunk, n = chunk_left(p.cols, j);
    load_weight(p.weight, p.weight_dtype, j, n, w[i]);
#pragma unroll
    for (uint32_t e = 0; e < kChunk; ++e) dw[i][e] = 0.0f;
  }
  for (uint32_t row = blockIdx.x * kRows + threadIdx.x / T; row < p.rows;
       row += p.groups * kRows) {
    float h[C][kChunk], g[C][kChunk];
    const typename E::Raw* hp = static_cast<const typename E::Raw*>(p.h) + (size_t)row * p.h_ld;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t j = (i * T + t) * kChunk, n = chunk_left(p.cols, j);
      load_row<E>(hp + j, n, h[i]);
      load_any(p.grad, p.grad_dtype, (size_t)row * p.grad_ld + j, n, g[i]);
    }
    double squares = 0.0, along = 0.0;
#pragma unroll
    for (int i = 0; i < C; ++i) {
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) {
        const double v = (double)h[i][e];
        squares = fma(v, v, squares);
        along = fma((double)(g[i][e] * w[i][e]), v, along);
      }
    }
    uint64_t none = 0;
    row_reduce<T>(squares, none);
    row_reduce<T>(along, none);
    const double rstd = 1.0 / sqrt(squares / (double)p.cols + p.eps);
    const float m = (float)rstd, k = (float)(rstd * rstd * (along / (double)p.cols));
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t j = (i * T + t) * kChunk, n = chunk_left(p.cols, j);
      float y[kChunk];
      if (p.grad_h != nullptr) {
#pragma unroll
        for (uint32_t e = 0; e < kChunk; ++e) y[e] = m * (g[i][e] * w[i][e] - h[i][e] * k);
        if (p.grad_sum != nullptr) {
          float more[kChunk];
          load_row<E>(static_cast<const typename E::Raw*>(p.grad_sum) +
                          (size_t)row * p.grad_sum_ld + j, n, more);
#pragma unroll
          for (uint32_t e = 0; e < kChunk; ++e) y[e] = y[e] + more[e];
        }
        store_row<E>(static_cast<typename E::Raw*>(p.grad_h) + (size_t)row * p.grad_h_ld + j, n,
                     y);
      }
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) dw[i][e] = dw[i][e] + g[i][e] * (h[i][e] * m);
    }
  }
  if (p.grad_weight == nullptr) return;
  float* part = p.part + (size_t)blockIdx.x * p.cols;
  if constexpr (T == 64) {
    extern __shared__ float waves[];  // [3][cols]: of all waves but the first
    const uint32_t wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < C; ++i) {
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) {
        const uint32_t j = (i * T + t) * kChunk + e;
        if (wave != 0 && j < p.cols) waves[(wave - 1u) * p.cols + j] = dw[i][e];
      }
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < C; ++i) {
#pragma unroll
      for (uint32_t e = 0; e < kChunk; ++e) {
        const uint32_t j = (i * T + t) * kChunk + e;
        if (j < p.cols)
          dw[i][e] = ((dw[i][e] + waves[j]) + waves[p.cols + j]) + waves[2u * p.cols + j];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const uint32_t j = (i * T + t) * kChunk;
    store_row<F32>(reinterpret_cast<uint32_t*>(part + j), chunk_left(p.cols, j), dw[i]);
  }
}

// The workgroups' sums of the weight's gradient, 64 columns a workgroup.
__global__ __launch_bounds__(1024) void norm_weight_kernel(NormGradParams p) {
  __shared__ double waves[16][64];
  const uint32_t lane = lane_id(), wave = threadIdx.x >> 6;
  const uint32_t j = blockIdx.x * 64u + lane;
  double sum = 0.0;
  if (j < p.cols)
    for (uint32_t k = wave; k < p.groups; k += 16u) sum = sum + (double)p.part[(size_t)k * p.cols + j];
  waves[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || j >= p.cols) return;
  for (uint32_t w = 1; w < 16; ++w) sum = sum + waves[w][lane];
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
uint32_t sum_parts(uint32_t rows) { return (rows + kSumRows - 1u) / kSumRows; }

// Workgroups of the norm's gradient, each with at most kMaxTerms rows a thread.
constexpr uint32_t kGradGroups = 512;
constexpr uint32_t kGradTerms = 768;
uint32_t grad_groups(uint32_t rows, uint32_t rows_at_once) {
  const uint32_t all = (rows + rows_at_once - 1u) / rows_at_once;
  const uint32_t least = (all + kGradTerms - 1u) / kGradTerms;
  const uint32_t most = least > kGradGroups ? least : kGradGroups;
  return all < most ? all : most;
}

size_t round_up(size_t bytes) { return (bytes + 255u) & ~(size_t)255u; }

template <typename E, template <typename, int, int> class Launch, typename P>
hipError_t by_width(const P& p, hipStream_t stream) {
  const uint32_t chunks = (p.cols + kChunk - 1u) / kChunk;
  if (chunks <= 64) return Launch<E, 64, 1>::run(p, stream);
  if (chunks <= 128) return Launch<E, 64, 2>::run(p, stream);
  if (chunks <= 256) return Launch<E, 64, 4>::run(p, stream);
  if (chunks <= 512) return Launch<E, 256, 2>::run(p, stream);
  if (chunks <= 1024) return Launch<E, 256, 4>::run(p, stream);
  if (chunks <= 2048) return Launch<E, 1024, 2>::run(p, stream);
  return Launch<E, 1024, 4>::run(p, stream);
}

template <typename E, int T, int C>
struct NormLaunch {
  static hipError_t run(const NormParams& p, hipStream_t stream) {
    constexpr uint32_t kRows = T < 256 ? 256 / T : 1;
    norm_kernel<E, T, C><<<(p.rows + kRows - 1u) / kRows, T < 256 ? 256 : T, 0, stream>>>(p);
    return hipGetLastError();
  }
};

template <typename E, int T, int C>
struct NormGradLaunch {
  static hipError_t run(const NormGradParams& in, hipStream_t stream) {
    constexpr uint32_t kRows = T < 256 ? 256 / T : 1;
    NormGradParams p = in;
    p.groups = grad_groups(p.rows, kRows);
    const size_t lds = T == 64 && p.grad_weight != nullptr ? (size_t)3 * p.cols * 4 : 0;
    hipError_t e = hipSuccess;
    if (p.groups != 0) {  // without rows the weight's gradient is zeros
      norm_grad_kernel<E, T, C><<<p.groups, T < 256 ? 256 : T, lds, stream>>>(p);
      e = hipGetLastError();
    }
    if (e != hipSuccess || p.grad_weight == nullptr) return e;
    norm_weight_kernel<<<(p.cols + 63u) / 64u, 1024, 0, stream>>>(p);
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

template <typename T>
hipError_t zero_table(const EmbedGradParams& p, hipStream_t stream) {
  const uint32_t shift = row_shift(p.cols), at_once = 256u >> shift;
  zero_rows_kernel<T><<<(p.vocab + at_once - 1u) / at_once, 256, 0, stream>>>(
      static_cast<typename T::Raw*>(p.table), p.table_ld, p.vocab, p.cols, shift);
  return hipGetLastError();
}

template <typename G, typename T>
hipError_t embed_grad_as(const EmbedGradParams& p, hipStream_t stream) {
  hipError_t e = hipSuccess;
  if (!p.accumulate && (e = zero_table<T>(p, stream)) != hipSuccess) return e;
  if (p.rows == 0) return e;
  const uint32_t tiles = sort_tiles(p.rows);
  uint32_t bits = 0;
  while (p.vocab >> bits) ++bits;
  const uint32_t passes = (bits + kSortBits - 1u) / kSortBits;
  for (uint32_t pass = 0; pass < passes; ++pass) {
    sort_count_kernel<<<tiles, 256, 0, stream>>>(p, pass, tiles);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    sort_prefix_kernel<<<1, 1024, 0, stream>>>(p.count, tiles << kSortBits);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    sort_place_kernel<<<tiles, 256, 0, stream>>>(p, pass, tiles);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  const uint32_t last = passes & 1u;
  const uint32_t col_tiles = (p.cols + 64u * G::kPer - 1u) / (64u * G::kPer);
  const uint32_t units = sum_parts(p.rows) * col_tiles;
  sum_rows_kernel<G, T><<<(units + 3u) / 4u, 256, 0, stream>>>(p, last, col_tiles, units);
  if ((e = hipGetLastError()) != hipSuccess || p.rows <= kSumRows) return e;
  const uint32_t join_tiles = (p.cols + 63u) / 64u;
  const size_t most = (size_t)(sum_parts(p.rows) - 1u) * join_tiles;
  join_rows_kernel<T><<<(uint32_t)(most < 1024 ? most : 1024), 256, 0, stream>>>(p, last, join_tiles);
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
         round_up((parts + 1) * 4) + round_up(parts * 2 * cols * 4);
}

size_t norm_grad_bytes(uint32_t rows, size_t cols) {
  return (size_t)grad_groups(rows, 1) * cols * 4;
}

size_t hidden_workspace_bytes(uint32_t rows, size_t cols) {
  const size_t a = embed_grad_bytes(rows, cols), b = norm_grad_bytes(rows, cols);
  return a > b ? a : b;
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
  p->cross = reinterpret_cast<uint32_t*>(take(((size_t)sum_parts(p->rows) + 1) * 4));
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
  if (dtype == PB_F32) return by_width<F32, NormLaunch>(p, stream);
  if (dtype == PB_F16) return by_width<F16, NormLaunch>(p, stream);
  return by_width<BF16, NormLaunch>(p, stream);
}

hipError_t launch_norm_grad(const NormGradParams& p, uint32_t dtype, hipStream_t stream) {
  if (dtype == PB_F32) return by_width<F32, NormGradLaunch>(p, stream);
  if (dtype == PB_F16) return by_width<F16, NormGradLaunch>(p, stream);
  return by_width<BF16, NormGradLaunch>(p, stream);
}

}  // namespace pb
