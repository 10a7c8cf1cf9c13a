// pb_scores.hip -- scores and losses of logits rows and their gradients.
//
// Mathematics.  With c = log2(e) / T, u = x c and a = u - shift for a shift near
// the row's largest u, a row's softmax is q = 2^a / sum 2^a, its log-sum-exp
// ln 2 (shift + log2 sum 2^a), and its entropy ln 2 (log2 sum - moment / sum) with
// moment = sum 2^a a.  Every gradient here is 2^a (alpha + beta a) for all
// elements but the row's token or the teacher's listed ids, which are written
// from scalars worked out in 64 bits.  So a row needs one pass for its
// statistics, a few scalars, and one pass for its gradient.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pb_device.h"
#include "pb_internal.h"
#include "pb_scores.h"

#pragma clang fp contract(off)

namespace pb {

namespace {

constexpr double kLn2 = 0.693147180559945309417232121458;
constexpr uint32_t kStatsThreads = 256;
static_assert(kMaxSpan == kStatsThreads * kMaxTerms, "a part's threads take kMaxTerms each");
constexpr uint32_t kStatsUnroll = 4;
constexpr uint32_t kGradThreads = 256;
constexpr uint32_t kTopThreads = 256;
static_assert(kTopThreads == kStatsThreads, "both passes have the same parts");
// Logits count while |u| is below 2^31.  A shift is a rounded u, and what that leaves out,
// up to 64 there, is in every exponent about it; further on 2^128 would be.  (With a
// limit of 3e38, a mask of the type's lowest value at T = 2 made its thread's sum infinite
// or 0, as the rounding fell.)
constexpr float kTooBig = 0x1p31f;

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
// Gradients pass the caches by: kept there, they push out the logits that are
// still to be read (4,096 x 151,936 bf16 distillation 548 us, so 504).
template <typename E>
__device__ __forceinline__ void store_chunk(typename E::Raw* p, const uint4& v) {
  __builtin_nontemporal_store(Words4{v.x, v.y, v.z, v.w}, reinterpret_cast<Loose4*>(p));
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- wave reductions in a fixed order ----

// step(v, lane ^ m) for m = 32 .. 1; written out, since lane_xor needs constants.
template <typename Step>
__device__ __forceinline__ uint32_t wave_fold(uint32_t v, Step step) {
  const uint32_t lane = lane_id();
  v = step(v, lane_xor(v, 32, lane));
  v = step(v, lane_xor(v, 16, lane));
  v = step(v, lane_xor(v, 8, lane));
  v = step(v, lane_xor(v, 4, lane));
  v = step(v, lane_xor(v, 2, lane));
  return step(v, lane_xor(v, 1, lane));
}
__device__ __forceinline__ float wave_max_f32(float v) {
  return f_of(wave_fold(
      b_of(v), [](uint32_t a, uint32_t b) { return b_of(fmaxf(f_of(a), f_of(b))); }));
}
__device__ __forceinline__ uint32_t wave_min_word(uint32_t v) {
  return wave_fold(v, [](uint32_t a, uint32_t b) { return b < a ? b : a; });
}
__device__ __forceinline__ uint32_t wave_sum_word(uint32_t v) {
  return wave_fold(v, [](uint32_t a, uint32_t b) { return a + b; });
}
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1)
    v = v + __builtin_bit_cast(double, shfl_xor64(__builtin_bit_cast(uint64_t, v), m));
  return v;
}

// ---- rows ----

// A per-row word by a scalar load (the same row in every lane; nothing in the
// launch writes it): counted apart from the rows' loads.
__device__ __forceinline__ uint32_t uniform_word(const uint32_t* at) {
  return *(const __attribute__((address_space(4))) uint32_t*)at;
}
__device__ __forceinline__ float uniform_float(const float* at) {
  return f_of(uniform_word(reinterpret_cast<const uint32_t*>(at)));
}

// Whether the statistics pass leaves a row out: it is masked, or its id is bad
// (which the finishing pass reports).
__device__ __forceinline__ bool row_unread(const ScoreParams& p, uint32_t row) {
  if (p.mode == kModeTop) return false;
  if (p.mode == kModeDistill)
    return p.weight != nullptr && uniform_float(p.weight + row) == 0.0f;
  if (p.mode == kModePreference) {
    if (row < uniform_word(p.seq_start) || row >= uniform_word(p.seq_start + 2 * p.pairs))
      return true;
  }
  if (p.mode == kModePolicy && p.weight != nullptr && uniform_float(p.weight + row) == 0.0f)
    return true;
  return uniform_word(p.token + row) >= p.vocab;
}

template <typename E>
__device__ __forceinline__ const typename E::Raw* row_ptr(const ScoreParams& p, uint32_t row) {
  return static_cast<const typename E::Raw*>(p.logits) + (size_t)row * p.ld;
}

struct Acc {
  float shift = 0.0f;
  float sum = 0.0f;
  float moment = 0.0f;
};

// The shift of a thread whose first chunk's largest u is `u`: that, or 0 where the
// chunk is masked out.  Past kTooBig it is one that fails the fast sums.
__device__ __forceinline__ float first_shift(float u) {
  return u < kTooBig ? (u > -kTooBig ? u : 0.0f) : -__builtin_inff();
}

// Bits of the marks of the elements j .. j + kPer - 1 of a part that starts at lo.
template <typename E>
__device__ __forceinline__ uint32_t chunk_marks(const uint32_t* marks, uint32_t at) {
  return (marks[at >> 5] >> (at & 31u)) & ((1u << E::kPer) - 1u);
}

// The largest of three without the compiler's quieting of signalling NaNs (a row
// that holds a NaN fails by its sum).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
template <typename E>
__device__ __forceinline__ float chunk_max(const float (&x)[E::kPer]) {
  float m = max3(x[0], x[1], x[2]);
  if constexpr (E::kPer == 8) {
    m = max3(m, x[3], x[4]);
    return max3(m, x[5], max3(x[6], x[7], x[7]));
  } else {
    return max3(m, x[3], x[3]);
  }
}
// A thread's shift moves up where a chunk's largest value m passes it by more than 16:
// a then keeps 19 bits behind the point for whatever weighs.  (By steps of more than 8,
// which ordinary rows take too, 240 rows' 32-bit statistics took 19.9 us, so 16.7, and
// 16.4 without any.)  A step past 2^60 is left to the second scan, and a sum that has
// failed stays failed (inf 0 is NaN).
template <bool kEntropy>
__device__ __forceinline__ void follow(Acc& s, float m, float c) {
  const float over = fmaf(m, c, -s.shift);
  if (__builtin_expect(over > 16.0f, 0)) {
    if (over < 0x1p60f) {
      const float u = m * c, rise = u - s.shift, f = exp2_hw(-rise);
      if (kEntropy) s.moment = f * fmaf(-rise, s.sum, s.moment);
      s.sum = f * s.sum;
      s.shift = u;
    }
  }
}

// Whether a thread's sum stands.  It is 1 and more about a first chunk's largest u (up
// to the rounding of a large one); a shift of 0, under a masked first chunk, has to be
// as near to what weighs.  A sum of NaN or out of range, or one about a shift that is,
// holds something that has failed.
__device__ __forceinline__ bool sum_holds(const Acc& s) {
  return s.sum >= 0x1p-16f && s.sum <= 0x1p100f && s.shift < kTooBig;
}

template <typename E, bool kEntropy>
__device__ __forceinline__ void add_chunk(Acc& s, const float (&x)[E::kPer], float c) {
  float e[E::kPer], m = 0.0f;
#pragma unroll
  for (int i = 0; i < E::kPer; ++i) {
    float a = fmaf(x[i], c, -s.shift);
    e[i] = exp2_hw(a);
    if (kEntropy) {
      a = fmaxf(a, -1000.0f);  // 0 for a weight of 0, where a is -inf
      m = fmaf(e[i], a, m);
    }
  }
  float sum;
  if constexpr (E::kPer == 8)
    sum = ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
  else
    sum = (e[0] + e[1]) + (e[2] + e[3]);
  s.sum = s.sum + sum;
  if (kEntropy) s.moment = s.moment + m;
}
// The same for kCount chunks that are at hand, take(q, x) giving chunk q: where one of
// their logits passes the shift by more than 16 their own sum shows it, and they are
// summed again about the shift that follows.
template <typename E, bool kEntropy, uint32_t kCount, typename Take>
__device__ __forceinline__ void add_group(Acc& s, float c, Take take) {
  float x[E::kPer];
  Acc t{s.shift};
#pragma unroll
  for (uint32_t q = 0; q < kCount; ++q) {
    take(q, x);
    add_chunk<E, kEntropy>(t, x, c);
  }
  if (__builtin_expect(t.sum > 0x1p16f, 0)) {
    float m = -__builtin_inff();
#pragma unroll
    for (uint32_t q = 0; q < kCount; ++q) {
      take(q, x);
      m = fmaxf(m, chunk_max<E>(x));
    }
    follow<kEntropy>(s, m, c);
    t = Acc{s.shift};
#pragma unroll
    for (uint32_t q = 0; q < kCount; ++q) {
      take(q, x);
      add_chunk<E, kEntropy>(t, x, c);
    }
  }
  s.sum = s.sum + t.sum;
  if (kEntropy) s.moment = s.moment + t.moment;
}

template <typename E, bool kTail>
__device__ __forceinline__ void unpack(const uint4& v, uint32_t marks, float (&x)[E::kPer]) {
#pragma unroll
  for (int i = 0; i < E::kPer; ++i) {
    x[i] = E::get(v, i);
    if (kTail && (marks >> i & 1u)) x[i] = -__builtin_inff();
  }
}

// A thread's sums over its chunks of [lo, hi), chunk i of thread t being
// element lo + (i kThreads + t) kPer.  The shift starts as the thread's first
// chunk's largest u and follows what passes it: nothing then underflows that weighs.
// Where the first chunk is masked out, or something in the row is out of range, the
// sum shows it (too large, too small or none) and the thread goes over its chunks
// again with their true maximum.
template <typename E, uint32_t kThreads, bool kEntropy, bool kTail, bool kKeep>
struct PartScan {
  template <typename T>
  static __device__ __forceinline__ uint4 load(const typename T::Raw* p) {
    return kKeep ? load_chunk<T>(p) : stream_chunk<T>(p);
  }
  const typename E::Raw* row;
  const uint32_t* marks;
  uint32_t lo, hi;
  float c;

  template <typename Fn>
  __device__ __forceinline__ void each(Fn fn) const {
    each(fn, [&](const uint4 (&v)[kStatsUnroll], uint32_t i) {
#pragma unroll
      for (uint32_t q = 0; q < kStatsUnroll; ++q) chunk(v[q], (i + q * kThreads) * E::kPer, fn);
    });
  }
  // many(chunks, index of the first) where there are kStatsUnroll of them.
  template <typename Fn, typename Many>
  __device__ __forceinline__ void each(Fn fn, Many many) const {
    constexpr uint32_t kPer = E::kPer;
    const uint32_t whole = (hi - lo) / kPer;
    uint32_t i = threadIdx.x;
    for (; i + (kStatsUnroll - 1) * kThreads < whole; i += kStatsUnroll * kThreads) {
      uint4 v[kStatsUnroll];
#pragma unroll
      for (uint32_t q = 0; q < kStatsUnroll; ++q)
        v[q] = load<E>(row + lo + (size_t)(i + q * kThreads) * kPer);
      many(v, i);
    }
    for (; i < whole; i += kThreads)
      chunk(load<E>(row + lo + (size_t)i * kPer), i * kPer, fn);
    const uint32_t rest = (hi - lo) - whole * kPer;
    if (rest != 0 && i == whole) {
      float x[E::kPer];
#pragma unroll
      for (uint32_t e = 0; e < kPer; ++e) {
        x[e] = -__builtin_inff();
        if (e < rest) {
          const uint32_t at = whole * kPer + e;
          if (!(kTail && (marks[at >> 5] >> (at & 31u) & 1u))) x[e] = E::one(row[lo + at]);
        }
      }
      fn(x, whole * kPer);
    }
  }

  template <typename Fn>
  __device__ __forceinline__ void chunk(const uint4& v, uint32_t at, Fn& fn) const {
    float x[E::kPer];
    unpack<E, kTail>(v, kTail ? chunk_marks<E>(marks, at) : 0u, x);
    fn(x, at);
  }

  __device__ __forceinline__ Acc run(uint32_t* bad) const {
    Acc s;
    bool first = true;
    auto one = [&](const float (&x)[E::kPer], uint32_t) {
      if (first) {
        first = false;
        s.shift = first_shift(chunk_max<E>(x) * c);
      } else {
        follow<kEntropy>(s, chunk_max<E>(x), c);
      }
      add_chunk<E, kEntropy>(s, x, c);
    };
    if constexpr (E::kPer == 4) {
      each(one);
    } else {
      // twice the elements to compare for the same bytes: by groups (1,023 of 2,563 bf16
      // rows 74 us, 79 with a comparison a chunk, 74 without any)
      each(one, [&](const uint4 (&v)[kStatsUnroll], uint32_t i) {
        auto take = [&](uint32_t q, float (&x)[E::kPer]) {
          const uint32_t at = (i + q * kThreads) * E::kPer;
          unpack<E, kTail>(v[q], kTail ? chunk_marks<E>(marks, at) : 0u, x);
        };
        if (first) {
          float x[E::kPer];
          take(0, x);
          first = false;
          s.shift = first_shift(chunk_max<E>(x) * c);
        }
        add_group<E, kEntropy, kStatsUnroll>(s, c, take);
      });
    }
    *bad = kNone;
    if (first || sum_holds(s)) return s;
    return again(bad);
  }

  // The sums about the largest u of all.
  __device__ __forceinline__ Acc again(uint32_t* bad) const {
    float top = -__builtin_inff();
    uint32_t at_bad = kNone;
    each([&](const float (&x)[E::kPer], uint32_t at) {
#pragma unroll
      for (int e = 0; e < E::kPer; ++e) {
        const float u = x[e] * c;
        if (!(u < kTooBig) && at_bad == kNone) at_bad = lo + at + e;
        top = fmaxf(top, u);
      }
    });
    Acc s;
    if (at_bad != kNone) {
      *bad = at_bad;
      return s;
    }
    if (!(top > -kTooBig)) return s;
    s.shift = top;
    each([&](const float (&x)[E::kPer], uint32_t) { add_chunk<E, kEntropy>(s, x, c); });
    return s;
  }
};

// A row's sums (or a part's): sum 2^(u - shift), its moment, the first bad element.
struct RowSum {
  double shift, sum, moment;
  uint32_t bad;
};

// One RowSum per lane into one, the same in every lane.  The factors between
// parts come from the 32-bit exp2: the part that holds the largest u has 1.
template <bool kMoment>
__device__ __forceinline__ RowSum wave_join(float shift, double sum, double moment, uint32_t bad) {
  const bool live = sum > 0.0;
  const float top = wave_max_f32(live ? shift : -__builtin_inff());
  const float off = live ? shift - top : 0.0f;
  const double f = live ? (double)exp2_hw(off) : 0.0;
  RowSum r;
  r.sum = wave_sum_f64(f * sum);
  r.moment = kMoment ? wave_sum_f64(f * (moment + (double)off * sum)) : 0.0;
  r.bad = wave_min_word(bad);
  r.shift = r.sum > 0.0 ? (double)top : 0.0;
  return r;
}

// The workgroup's sums, valid in every lane of wave 0; one barrier.
struct BlockSum {
  float shift[16];
  uint32_t bad[16];
  double sum[16];
  double moment[16];
};
template <uint32_t kThreads, bool kMoment>
__device__ __forceinline__ RowSum block_sum(const Acc& s, uint32_t bad, BlockSum& l) {
  const uint32_t lane = lane_id(), wave = threadIdx.x >> 6;
  const RowSum w = wave_join<kMoment>(s.shift, (double)s.sum, (double)s.moment, bad);
  if (lane == 0 && wave < kThreads / 64) {
    l.shift[wave] = (float)w.shift;
    l.sum[wave] = w.sum;
    l.moment[wave] = w.moment;
    l.bad[wave] = w.bad;
  }
  __syncthreads();
  if (wave != 0) return w;
  const bool on = lane < kThreads / 64;
  return wave_join<kMoment>(on ? l.shift[lane] : 0.0f, on ? l.sum[lane] : 0.0,
                            on ? l.moment[lane] : 0.0, on ? l.bad[lane] : kNone);
}

// Marks the teacher's ids that lie in [lo, hi); every thread, then a barrier.
__device__ __forceinline__ void mark_ids(const ScoreParams& p, uint32_t row, uint32_t lo,
                                         uint32_t hi, uint32_t* marks) {
  for (uint32_t i = threadIdx.x; i < (hi - lo + 31u) / 32u + 1u; i += blockDim.x) marks[i] = 0;
  __syncthreads();
  if (threadIdx.x < p.k) {
    const uint32_t id = p.teacher_id[(size_t)row * p.k + threadIdx.x];
    if (id >= lo && id < hi) atomicOr(&marks[(id - lo) >> 5], 1u << ((id - lo) & 31u));
  }
  __syncthreads();
}

// ---- a row's scalars, by one wave ----

__device__ __forceinline__ void write_error(pb_inference_error* at, uint32_t status,
                                            uint32_t position, uint64_t needed,
                                            uint64_t available, uint32_t kind, uint32_t sub) {
  if (at == nullptr) return;
  pb_inference_error e;
  e.status = status;
  e.domain = PB_DOMAIN_LOGITS;
  e.layer = PB_NO_LAYER;
  e.position = position;
  e.tensor_id = PB_NO_TENSOR;
  e.reserved = 0;
  e.needed = needed;
  e.available = available;
  e.detail = ((uint64_t)kind << 32) | sub;
  *at = e;
}
__device__ __forceinline__ void no_error(pb_inference_error* at) {
  if (at == nullptr) return;
  *at = pb_inference_error{0, 0, 0, 0, 0, 0, 0, 0, 0};
}

__device__ __forceinline__ float nan32() { return f_of(0x7fc00000u); }

// A gradient's shift is the row's log-sum, to the nearest binary32: the elements
// that weigh then have small a, where a's own rounding is small too.  (About the
// sums' shift, 40 below an outlier, gradients of 32-bit logits were off by 1e-6.)
// What that rounding leaves out goes into the factors.  log2_own: log2 of the sum
// about `shift`; the two stay apart, since together they lose it under large logits.
struct GradShift {
  float at;
  double factor;  // q = factor 2^(u - at)
};
__device__ __forceinline__ GradShift grad_shift(double shift, double log2_own) {
  const float at = (float)(shift + log2_own);
  return {at, exp2(((double)at - shift) - log2_own)};
}

// Gradient slope (delta - q) of a row with one token; rise = q[token] - 1.
__device__ __forceinline__ RowCoef token_coef(double shift, double log2_own, double slope,
                                              double rise, uint32_t token) {
  RowCoef r{};
  r.state = slope == 0.0 ? kRowZero : slope == slope ? kRowNormal : kRowNan;
  const GradShift g = grad_shift(shift, log2_own);
  r.shift = g.at;
  r.alpha = (float)(-slope * g.factor);
  r.token = token;
  r.patch = (float)(slope * -rise);
  return r;
}

// ln q[token] in 64 bits; x the token's logit.
__device__ __forceinline__ double token_logprob(const ScoreParams& p, float x, double shift,
                                                double log2_own) {
  return kLn2 * (((double)x * (double)p.c - shift) - log2_own);
}

// Whether a row that was read has failed, and the record of it.
__device__ __forceinline__ bool bad_row(uint32_t bad, double sum) {
  return bad != kNone || !(sum > 0.0);
}
template <typename E>
__device__ __forceinline__ void report_row(const ScoreParams& p, uint32_t row, uint32_t bad,
                                           pb_inference_error* at) {
  const uint32_t index = bad == kNone ? 0u : bad;
  write_error(at, PB_NONFINITE_OUTPUT, row, 0, b_of(E::one(row_ptr<E>(p, row)[index])),
              PB_FIELD_FINITE, index);
}

// What a row with one token needs beside its sums, requested before them.
struct TokenRow {
  uint32_t token;
  float x;       // the token's logit
  float weight;
  float old_logprob, advantage, ref_logprob;
};
__device__ __forceinline__ TokenRow token_row(const ScoreParams& p, uint32_t row) {
  TokenRow t{uniform_word(p.token + row), 0.0f, 1.0f, 0.0f, 0.0f, 0.0f};
  if (p.mode == kModePolicy) {
    if (p.weight != nullptr) t.weight = uniform_float(p.weight + row);
    t.old_logprob = uniform_float(p.old_logprob + row);
    t.advantage = uniform_float(p.advantage + row);
    if (p.ref_logprob != nullptr) t.ref_logprob = uniform_float(p.ref_logprob + row);
  }
  return t;
}

// A row's scalars are worked out in two steps: what its gradient needs, and then
// the outputs, which no other wave waits for.

// One wave; the three exponentials are one call over three lanes.  Lane 0's
// result counts.
struct PolicyRow {
  RowCoef coef;
  double loss, logprob, kl;
};
template <typename E>
__device__ __forceinline__ PolicyRow policy_row(const ScoreParams& p, uint32_t row,
                                                const RowSum& r, const TokenRow& t) {
  PolicyRow o{};
  o.coef.state = kRowZero;
  pb_inference_error* at = p.err ? p.err + row : nullptr;
  if (t.token == PB_NO_TOKEN || t.weight == 0.0f) {
    if (lane_id() == 0) no_error(at);
    return o;
  }
  bool failed = t.token >= p.vocab;
  if (failed) {
    if (lane_id() == 0) write_error(at, PB_TOKEN_ID, row, p.vocab, t.token, PB_FIELD_TOKEN, 0);
  } else {
    failed = bad_row(r.bad, r.sum);
    if (failed && lane_id() == 0) report_row<E>(p, row, r.bad, at);
  }
  if (failed) {
    o.loss = o.logprob = o.kl = (double)nan32();
    o.coef.state = kRowNan;
    return o;
  }
  if (lane_id() == 0) no_error(at);
  const double log2_own = log2(r.sum);
  const double lp = token_logprob(p, t.x, r.shift, log2_own), gap = (double)t.ref_logprob - lp;
  const uint32_t lane = lane_id();
  const double rise = expm1(lane == 0 ? lp - (double)t.old_logprob : lane == 1 ? gap : lp);
  const double ratio = 1.0 + bcast_f64(rise, 0), away = bcast_f64(rise, 1);
  const double adv = (double)t.advantage;
  const double low = 1.0 - p.clip_low, high = 1.0 + p.clip_high;
  const double kept = ratio < low ? low : ratio > high ? high : ratio;
  const double open = ratio * adv, shut = kept * adv;
  double slope = open <= shut ? -open : 0.0;
  o.logprob = lp;
  o.loss = open <= shut ? -open : -shut;
  if (open != open) o.loss = slope = open;
  if (p.ref_logprob != nullptr) {
    o.kl = gap == __builtin_inf() ? gap : away - gap;  // e^d outgrows d
    if (p.kl_coef != 0.0) {
      o.loss += p.kl_coef * o.kl;
      slope -= p.kl_coef * away;
    }
  }
  slope = slope * (double)t.weight * p.inv_t;
  o.coef = token_coef(r.shift, log2_own, slope, bcast_f64(rise, 2), t.token);
  return o;
}
__device__ __forceinline__ void write_policy(const ScoreParams& p, uint32_t row,
                                             const PolicyRow& o) {
  if (lane_id() != 0) return;
  p.loss[row] = (float)o.loss;
  if (p.logprob) p.logprob[row] = (float)o.logprob;
  if (p.kl) p.kl[row] = (float)o.kl;
}

template <typename E>
__device__ __forceinline__ void finish_logprobs(const ScoreParams& p, uint32_t row,
                                                const RowSum& r, const TokenRow& t) {
  if (lane_id() != 0) return;
  pb_inference_error* at = p.err ? p.err + row : nullptr;
  float logprob = 0.0f, lse = 0.0f, low = 0.0f, entropy = 0.0f;
  if (t.token == PB_NO_TOKEN) {
    no_error(at);
  } else {
    bool failed = t.token >= p.vocab;
    if (failed) {
      write_error(at, PB_TOKEN_ID, row, p.vocab, t.token, PB_FIELD_TOKEN, 0);
    } else {
      failed = bad_row(r.bad, r.sum);
      if (failed) report_row<E>(p, row, r.bad, at);
    }
    if (failed) {
      logprob = lse = low = entropy = nan32();
    } else {
      no_error(at);
      const double log2_own = log2(r.sum);
      logprob = (float)token_logprob(p, t.x, r.shift, log2_own);
      const double whole = kLn2 * (r.shift + log2_own);
      lse = (float)whole;
      low = (float)(whole - (double)lse);
      entropy = (float)(kLn2 * (log2_own - r.moment / r.sum));
    }
  }
  p.logprob[row] = logprob;
  if (p.lse) p.lse[row] = lse;
  if (p.lse_low) p.lse_low[row] = low;
  if (p.entropy) p.entropy[row] = entropy;
}

// The last sequence that starts at or before a row, by one wave: one look at every
// 64th part of what is left.  Where offsets decrease, sequences may share rows; the
// row then still has one owner, and the pairs that find another's fail.  The second
// wave of a row's first part does it beside the first's scalars.
__device__ __forceinline__ void note_sequence(const ScoreParams& p, uint32_t row) {
  uint32_t at = 0, n = 2u * p.pairs + 1u;
  while (n > 1u) {
    const uint32_t step = (n + 63u) / 64u, i = lane_id() * step;
    const uint64_t before = __ballot(i < n && p.seq_start[at + i] <= row);
    const uint32_t k = before ? 63u - (uint32_t)__builtin_clzll(before) : 0u;
    at += k * step;
    n = n - k * step < step ? n - k * step : step;
  }
  if (lane_id() == 0) p.sequence[row] = at;
}

// The preference loss' rows, for the pairs' pass.
__device__ __forceinline__ void finish_pair_row(const ScoreParams& p, uint32_t row,
                                                const RowSum& r, const TokenRow& t) {
  if (lane_id() != 0) return;
  PairRow* v = reinterpret_cast<PairRow*>(p.coef + row);
  const bool failed = bad_row(r.bad, r.sum);
  v->state = kRowUntouched;
  v->bad = r.bad;
  v->failed = failed ? 1u : 0u;
  v->shift = (float)r.shift;
  v->log2_own = failed ? 0.0 : log2(r.sum);
  v->logprob = failed ? 0.0 : token_logprob(p, t.x, r.shift, v->log2_own);
}

// A row's list, two entries a lane (i = lane, lane + 64); kNone past its end.
struct ListLanes {
  uint32_t id[2];
  float logit[2];
  float lse;
};
__device__ __forceinline__ ListLanes load_list(const ScoreParams& p, uint32_t row, uint32_t lane) {
  ListLanes l;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t i = lane + 64u * h;
    const size_t at = (size_t)row * p.k + i;
    l.id[h] = i < p.k ? p.teacher_id[at] : kNone;
    l.logit[h] = i < p.k ? p.teacher_logit[at] : 0.0f;
  }
  l.lse = p.teacher_lse != nullptr ? p.teacher_lse[row] : 0.0f;
  return l;
}

// The first entry whose id another entry has too, or kNone.
__device__ __forceinline__ uint32_t first_repeat(const ScoreParams& p, const ListLanes& l,
                                                 uint32_t lane) {
  uint32_t seen[2] = {0, 0};  // entries of the same id, the entry itself included
#pragma unroll
  for (uint32_t j = 0; j < 64; ++j) {
    const uint32_t a = bcast32(l.id[0], j);
    seen[0] += a == l.id[0] ? 1u : 0u;
    seen[1] += a == l.id[1] ? 1u : 0u;
  }
  if (p.k > 64) {
#pragma unroll
    for (uint32_t j = 0; j < 64; ++j) {
      const uint32_t a = bcast32(l.id[1], j);
      seen[0] += a == l.id[0] ? 1u : 0u;
      seen[1] += a == l.id[1] ? 1u : 0u;
    }
  }
  const bool second = l.id[1] != kNone && seen[1] > 1u;
  return wave_min_word(l.id[0] != kNone && seen[0] > 1u ? lane : second ? lane + 64u : kNone);
}

// What the teacher's list says by itself, the same in every lane: its
// log-sum-exp, its mass sum p, sum p ln p, the first bad entries, and whether
// anything in it weighs.
struct ListSum {
  double norm, mass, plogp;
  uint32_t bad_id, bad_logit;
  uint32_t any;
};

// pr: the lane's p.
__device__ __forceinline__ ListSum sum_teacher(const ScoreParams& p, const ListLanes& l,
                                               uint32_t lane, uint32_t repeat, double (&pr)[2]) {
  ListSum s{};
  s.bad_id = s.bad_logit = kNone;
  float top = -__builtin_inff();
  bool on[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t i = lane + 64u * h;
    on[h] = l.id[h] < p.vocab;
    if (l.id[h] != kNone && !on[h]) s.bad_id = i < s.bad_id ? i : s.bad_id;
    if (on[h] && !(l.logit[h] < __builtin_inff())) s.bad_logit = i < s.bad_logit ? i : s.bad_logit;
    if (on[h]) top = fmaxf(top, l.logit[h]);
  }
  s.bad_id = wave_min_word(s.bad_id);
  s.bad_id = repeat < s.bad_id ? repeat : s.bad_id;
  s.bad_logit = wave_min_word(s.bad_logit);
  const bool lse_given = p.teacher_lse != nullptr;
  if (lse_given && !__builtin_isfinite(l.lse)) s.bad_logit = p.k < s.bad_logit ? p.k : s.bad_logit;
  top = wave_max_f32(top);
  s.any = top > -__builtin_inff() && s.bad_logit == kNone;
  pr[0] = pr[1] = 0.0;
  if (!s.any) return s;
  // e = 2^.. of each entry by the teacher's lse, or by its largest logit
  const double base = lse_given ? (double)l.lse : (double)top * p.inv_t;
  double sum = 0.0, moment = 0.0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h == 1 && p.k <= 64) break;
    const double d = (double)l.logit[h] * p.inv_t - base;
    pr[h] = on[h] ? exp(d) : 0.0;
    sum += pr[h];
    if (pr[h] > 0.0) moment += pr[h] * d;
  }
  sum = wave_sum_f64(sum);
  moment = wave_sum_f64(moment);
  if (lse_given) {
    s.norm = base;
    s.mass = sum;
    s.plogp = moment;
    return s;
  }
  const double own = log(sum), inv = 1.0 / sum;
  s.norm = base + own;
  s.mass = 1.0;
  s.plogp = moment * inv - own;
  pr[0] *= inv;
  pr[1] *= inv;
  return s;
}

// A listed id's gradient; pr: its p.
__device__ __forceinline__ float listed_grad(const ScoreParams& p, const RowCoef& r, float x,
                                             double pr) {
  const double q = exp2((double)x * (double)p.c - (double)r.own_shift) * r.inv;
  return (float)(r.weight * (r.mass * q - pr));
}

// One wave: the row's sums joined with those of its listed ids (x, the lane's
// logits of them), and what its gradient needs.  The student's mass off the list,
// qr, is kept by its log2: finite logits may lie thousands below the listed ones, and
// what off-list elements get, q (mass - left / qr), adds up to about -left all the same.
struct DistillRow {
  RowCoef coef;
  double shift, log2_own;  // the row's log2 sum 2^u is their sum
  double log2_rest;        // log2 qr
  double left;             // the teacher's mass in the rest bucket
  bool skipped, failed;
};
template <typename E>
__device__ __forceinline__ DistillRow distill_row(const ScoreParams& p, uint32_t row, float weight,
                                                  const RowSum& r, const ListSum& s,
                                                  const uint32_t (&id)[2], const float (&x)[2]) {
  DistillRow o{};
  o.coef.state = kRowZero;
  pb_inference_error* at = p.err ? p.err + row : nullptr;
  const bool writer = lane_id() == 0;
  o.skipped = weight == 0.0f;
  if (o.skipped) {
    if (writer) no_error(at);
    return o;
  }
  uint32_t bad = r.bad;
  o.shift = r.shift;
  double whole = r.sum;  // sum 2^(u - o.shift) of the row
  if (p.teacher_lse != nullptr) {
    // the listed ids were left out of the row's sums: their logits are looked at here
    float top = -__builtin_inff();
    uint32_t bad_x = kNone;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (id[h] >= p.vocab) continue;
      if (!(x[h] * p.c < kTooBig)) bad_x = id[h] < bad_x ? id[h] : bad_x;
      top = fmaxf(top, x[h]);
    }
    bad_x = wave_min_word(bad_x);
    bad = bad_x < bad ? bad_x : bad;
    top = wave_max_f32(top) * p.c;
    if (top > -kTooBig) {
      o.shift = r.sum > 0.0 && r.shift > (double)top ? r.shift : (double)top;
      double listed = 0.0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && p.k <= 64) break;
        if (id[h] < p.vocab) listed += exp2((double)x[h] * (double)p.c - o.shift);
      }
      whole = (r.sum > 0.0 ? r.sum * exp2(r.shift - o.shift) : 0.0) + wave_sum_f64(listed);
    }
  }
  o.failed = true;
  if (s.bad_id != kNone) {
    if (writer)
      write_error(at, PB_TOKEN_ID, row, p.vocab, p.teacher_id[(size_t)row * p.k + s.bad_id],
                  PB_FIELD_TOKEN, s.bad_id);
  } else if (s.bad_logit != kNone) {
    if (writer)
      write_error(at, PB_NONFINITE_INPUT, row, 0,
                  b_of(s.bad_logit == p.k ? p.teacher_lse[row]
                                          : p.teacher_logit[(size_t)row * p.k + s.bad_logit]),
                  PB_FIELD_FINITE, s.bad_logit);
  } else if (bad_row(bad, whole)) {
    if (writer) report_row<E>(p, row, bad, at);
  } else {
    o.failed = false;
    if (writer) no_error(at);
  }
  if (o.failed) o.coef.state = kRowNan;
  if (!o.failed) o.log2_own = log2(whole);
  if (o.failed || !s.any) return o;
  double mass = s.mass;
  o.coef.weight = (double)weight * p.inv_t;
  o.coef.state = weight == weight ? kRowNormal : kRowNan;
  GradShift g = grad_shift(o.shift, o.log2_own);
  o.coef.own_shift = g.at;
  o.coef.inv = g.factor;
  double off = mass;  // what 2^(u - log-sum) is multiplied by off the list
  if (p.teacher_lse != nullptr && r.sum > 0.0) {
    // q (mass - left / qr) = (q / qr) (mass qr - left), and q / qr is taken about the
    // rest's own log-sum: about the row's, 2^a underflows and 1 / qr leaves binary32
    // from 87 below the listed ids on.  (A listed element may then be inf before its
    // own gradient is stored over it.)
    const double log2_sum = log2(r.sum);
    o.log2_rest = (r.shift - o.shift) + (log2_sum - o.log2_own);
    if (mass < 1.0) {
      o.left = 1.0 - mass;
      mass += o.left;
    }
    g = grad_shift(r.shift, log2_sum);
    off = mass * exp2(o.log2_rest) - o.left;
  }
  o.coef.shift = g.at;
  o.coef.alpha = (float)(o.coef.weight * off * g.factor);
  o.coef.norm = s.norm;
  o.coef.mass = mass;
  o.coef.token = kNone;
  return o;
}
__device__ __forceinline__ void write_distill(const ScoreParams& p, uint32_t row,
                                              const DistillRow& o, const ListSum& s,
                                              const float (&x)[2], const double (&pr)[2]) {
  double loss = 0.0, lse = 0.0;
  if (o.failed) {
    loss = lse = (double)nan32();
  } else if (!o.skipped) {
    const double log2_sum = o.shift + o.log2_own;
    lse = kLn2 * log2_sum;
    if (s.any) {
      double pu = 0.0;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (pr[h] > 0.0) pu += pr[h] * ((double)x[h] * (double)p.c);
      loss = s.plogp - kLn2 * (wave_sum_f64(pu) - s.mass * log2_sum);
      if (o.left > 0.0) loss += o.left * (log(o.left) - kLn2 * o.log2_rest);
    }
  }
  if (lane_id() != 0) return;
  p.loss[row] = (float)loss;
  if (p.lse) p.lse[row] = (float)lse;
}

// What a wave of its own has made of a row's list while the others scan the row.
struct ListShared {
  ListSum sum;
  uint32_t id[PB_TOP_LOGITS_MAX];
  float x[PB_TOP_LOGITS_MAX];
  double pr[PB_TOP_LOGITS_MAX];
};
template <typename E>
__device__ __forceinline__ void prepare_list(const ScoreParams& p, uint32_t row, ListShared& l) {
  const uint32_t lane = lane_id();
  const ListLanes list = load_list(p, row, lane);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l.id[lane + 64 * h] = list.id[h];
    l.x[lane + 64 * h] = list.id[h] < p.vocab ? E::one(row_ptr<E>(p, row)[list.id[h]]) : 0.0f;
  }
  double pr[2];
  const ListSum s = sum_teacher(p, list, lane, first_repeat(p, list, lane), pr);
#pragma unroll
  for (int h = 0; h < 2; ++h) l.pr[lane + 64 * h] = pr[h];
  if (lane == 0) l.sum = s;
}

// A row's scalars from its sums; one wave.
template <typename E>
__device__ __forceinline__ void finish_row(const ScoreParams& p, uint32_t row, const RowSum& r) {
  TokenRow t = token_row(p, row);
  if (t.token < p.vocab) t.x = E::one(row_ptr<E>(p, row)[t.token]);
  if (p.mode == kModePolicy) {
    const PolicyRow o = policy_row<E>(p, row, r, t);
    if (lane_id() == 0 && p.grad) p.coef[row] = o.coef;
    write_policy(p, row, o);
  } else if (p.mode == kModePreference) {
    finish_pair_row(p, row, r, t);
  } else {
    finish_logprobs<E>(p, row, r, t);
  }
}
template <typename E>
__device__ __forceinline__ void finish_list_row(const ScoreParams& p, uint32_t row,
                                                const RowSum& r, const ListShared& l) {
  const uint32_t lane = lane_id();
  const float weight = p.weight ? uniform_float(p.weight + row) : 1.0f;
  ListSum s{};
  uint32_t id[2] = {kNone, kNone};
  float x[2] = {0.0f, 0.0f};
  double pr[2] = {0.0, 0.0};
  if (weight != 0.0f) {
    s = l.sum;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      id[h] = l.id[lane + 64 * h];
      x[h] = l.x[lane + 64 * h];
      pr[h] = l.pr[lane + 64 * h];
    }
  }
  const DistillRow o = distill_row<E>(p, row, weight, r, s, id, x);
  if (lane == 0 && p.grad) p.coef[row] = o.coef;
  write_distill(p, row, o, s, x, pr);
}

// Parts of a row pass between workgroups of one launch, which may run on XCDs
// with an L2 each: every word goes and comes at the device's scope, past those
// caches, and a part's words are acknowledged (vmcnt 0) before its ticket is
// taken.  A device-wide fence instead writes back and drops the whole L2: the
// 70 rows x 13 parts of 50,257 ids took 21.9 us with it.
__device__ __forceinline__ void publish_part(RowPart* at, const RowSum& r) {
  uint64_t* w = reinterpret_cast<uint64_t*>(at);
  const uint64_t head = (uint64_t)b_of((float)r.shift) | ((uint64_t)r.bad << 32);
  __hip_atomic_store(w, head, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(w + 1, __builtin_bit_cast(uint64_t, r.sum), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(w + 2, __builtin_bit_cast(uint64_t, r.moment), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void acknowledged() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ RowPart collect_part(const RowPart* at) {
  const uint64_t* w = reinterpret_cast<const uint64_t*>(at);
  const uint64_t head = __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const uint64_t sum = __hip_atomic_load(w + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const uint64_t moment = __hip_atomic_load(w + 2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return RowPart{f_of((uint32_t)head), (uint32_t)(head >> 32), __builtin_bit_cast(double, sum),
                 __builtin_bit_cast(double, moment)};
}
// Takes the ticket of a part whose words are acknowledged; true in the wave whose
// part was the row's last.
__device__ __forceinline__ bool last_part(const ScoreParams& p, uint32_t row) {
  uint32_t before = 0;
  if (lane_id() == 0)
    before = __hip_atomic_fetch_add(&p.ticket[row], 1u, __ATOMIC_RELAXED,
                                    __HIP_MEMORY_SCOPE_AGENT);
  if (bcast32(before, 0) != p.splits - 1u) return false;
  if (lane_id() == 0) p.ticket[row] = 0;
  return true;
}
// The row's parts joined, by one wave.
template <bool kMoment>
__device__ __forceinline__ RowSum join_parts(const ScoreParams& p, uint32_t row) {
  RowPart v{0.0f, kNone, 0.0, 0.0};
  if (lane_id() < p.splits) v = collect_part(p.part + (size_t)row * p.splits + lane_id());
  return wave_join<kMoment>(v.shift, v.sum, v.moment, v.bad);
}

// The statistics pass; large batches read at 6.3 TB/s (4,096 rows of 151,936 bf16
// logits in 197 us, 188 without the check of each group; a plain read reaches 7.0).
// A row's parts leave their sums in the workspace, and the workgroup that comes last
// (by the row's ticket, which it sets back to 0) joins them and works out the row's
// scalars, so that they need no launch of their own.
// kKeep: the row is read again soon, and what the call reads may stay in the caches.
// kList: the distillation; a fifth wave takes the teacher's list (at the end of
// the row's last part instead, 12 rows took 1.8 us longer).
constexpr uint32_t kNoList = 0, kListOnly = 1, kListWithRest = 2;
template <typename E, bool kEntropy, uint32_t kList, bool kKeep>
__global__ __launch_bounds__(kStatsThreads + (kList ? 64 : 0)) void stats_kernel(
    const ScoreParams p) {
  constexpr bool kTail = kList == kListWithRest;
  __shared__ BlockSum l;
  __shared__ ListShared list;
  extern __shared__ uint32_t marks[];
  const uint32_t row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits;
  const bool notes =
      !kList && p.mode == kModePreference && split == 0 && threadIdx.x / 64u == 1u;
  if (row_unread(p, row)) {
    if (notes) note_sequence(p, row);
    if (split != 0 || threadIdx.x >= 64) return;
    const RowSum none{0.0, 0.0, 0.0, kNone};
    if (kList)
      finish_list_row<E>(p, row, none, list);
    else
      finish_row<E>(p, row, none);
    return;
  }
  const uint32_t lo = split * p.span;
  const uint32_t hi = p.vocab - lo < p.span ? p.vocab : lo + p.span;
  if (kTail) mark_ids(p, row, lo, hi, marks);
  uint32_t bad = kNone;
  Acc s;
  if (!kList || threadIdx.x < kStatsThreads) {
    const PartScan<E, kStatsThreads, kEntropy, kTail, kKeep> scan{row_ptr<E>(p, row), marks, lo,
                                                                 hi, p.c};
    s = scan.run(&bad);
  } else {
    prepare_list<E>(p, row, list);
  }
  RowSum r = block_sum<kStatsThreads, kEntropy>(s, bad, l);
  if (notes) note_sequence(p, row);
  if (threadIdx.x >= 64) return;
  if (p.splits > 1) {
    if (lane_id() == 0) publish_part(p.part + (size_t)row * p.splits + split, r);
    acknowledged();
    if (!last_part(p, row)) return;
    r = join_parts<kEntropy>(p, row);
  }
  if (kList)
    finish_list_row<E>(p, row, r, list);
  else
    finish_row<E>(p, row, r);
}

// ---- preference loss: one workgroup a pair ----

__device__ __forceinline__ PairRow pair_row(const ScoreParams& p, uint32_t row) {
  return *reinterpret_cast<const PairRow*>(p.coef + row);
}

template <typename E>
__global__ __launch_bounds__(256) void pair_kernel(const ScoreParams p) {
  __shared__ double sums[2][4];
  __shared__ uint32_t worst[4], foreign[4];
  __shared__ double slope_at;
  const uint32_t pair = blockIdx.x, lane = lane_id(), wave = threadIdx.x >> 6;
  pb_inference_error* at = p.err ? p.err + pair : nullptr;
  const uint32_t a = p.seq_start[2 * pair], b = p.seq_start[2 * pair + 1],
                 e = p.seq_start[2 * pair + 2];
  auto refuse = [&](uint32_t offset) {
    if (threadIdx.x != 0) return;
    write_error(at, PB_CAPACITY, pair, p.rows, offset, PB_FIELD_BYTES, 10);
    p.loss[pair] = nan32();
    if (p.logprob) p.logprob[2 * pair] = p.logprob[2 * pair + 1] = nan32();
  };
  // rows outside the first and the last offset have no statistics
  if (a > b || b > e || e > p.rows || a < p.seq_start[0] || e > p.seq_start[2 * p.pairs])
    return refuse(e > p.rows ? e : b);
  const float w = p.weight ? p.weight[pair] : 1.0f;
  double mine[2] = {0.0, 0.0};
  uint32_t failed = kNone, stray = 0;
  for (uint32_t row = a + threadIdx.x; row < e; row += 256u) {
    const uint32_t token = p.token[row];
    const PairRow v = pair_row(p, row);
    // every row has to be this pair's before any coefficient is written
    stray |= p.sequence[row] ^ (2u * pair + (row < b ? 0u : 1u));
    if (w == 0.0f || token == PB_NO_TOKEN) continue;
    if (token >= p.vocab || v.failed)
      failed = row < failed ? row : failed;
    else
      mine[row < b ? 0 : 1] += v.logprob;
  }
  const double c = wave_sum_f64(mine[0]), d = wave_sum_f64(mine[1]);
  const uint32_t f = wave_min_word(failed);
  const bool strays = __ballot(stray != 0) != 0;
  if (lane == 0) {
    foreign[wave] = strays ? 1u : 0u;
    sums[0][wave] = c;
    sums[1][wave] = d;
    worst[wave] = f;
  }
  __syncthreads();
  if (foreign[0] | foreign[1] | foreign[2] | foreign[3]) return refuse(a);
  if (threadIdx.x == 0) {
    double l[2] = {0.0, 0.0};
    uint32_t first = kNone;
    for (int i = 0; i < 4; ++i) {
      l[0] += sums[0][i];
      l[1] += sums[1][i];
      first = worst[i] < first ? worst[i] : first;
    }
    double loss = 0.0, slope = 0.0;
    if (first != kNone) {
      const uint32_t token = p.token[first];
      if (token >= p.vocab) {
        write_error(at, PB_TOKEN_ID, first, p.vocab, token, PB_FIELD_TOKEN, 0);
      } else {
        report_row<E>(p, first, pair_row(p, first).bad, at);
      }
      loss = slope = l[0] = l[1] = (double)nan32();
    } else {
      no_error(at);
      if (w != 0.0f) {
        const double rc = p.ref_logprob ? (double)p.ref_logprob[2 * pair] : 0.0;
        const double rr = p.ref_logprob ? (double)p.ref_logprob[2 * pair + 1] : 0.0;
        const double h = p.beta * ((l[0] - rc) - (l[1] - rr));
        // -ln sigma(h) = max(-h, 0) + ln(1 + e^-|h|); a token without weight makes h
        // infinite, and a term whose factor is 0 then counts 0
        const double soft = log1p(exp(-fabs(h)));
        if (p.smoothing < 1.0) loss += (1.0 - p.smoothing) * ((h < 0.0 ? -h : 0.0) + soft);
        if (p.smoothing > 0.0) loss += p.smoothing * ((h > 0.0 ? h : 0.0) + soft);
        if (h != h) loss = h;
        const double up = 1.0 / (1.0 + exp(-h)), down = 1.0 / (1.0 + exp(h));
        slope = (p.smoothing * up - (1.0 - p.smoothing) * down) * p.beta * (double)w * p.inv_t;
      }
    }
    p.loss[pair] = (float)loss;
    if (p.logprob) {
      p.logprob[2 * pair] = (float)l[0];
      p.logprob[2 * pair + 1] = (float)l[1];
    }
    slope_at = slope;
  }
  __syncthreads();
  if (p.grad == nullptr) return;
  const double slope = slope_at;
  for (uint32_t row = a + threadIdx.x; row < e; row += 256u) {
    const uint32_t token = p.token[row];
    RowCoef coef{};
    coef.state = kRowZero;
    if (slope != slope) {
      coef.state = kRowNan;
    } else if (token != PB_NO_TOKEN && w != 0.0f) {
      const PairRow v = pair_row(p, row);
      coef = token_coef(v.shift, v.log2_own, row < b ? slope : -slope, expm1(v.logprob), token);
    }
    p.coef[row] = coef;
  }
}

// ---- gradient pass ----

template <typename E, bool kBeta>
__device__ __forceinline__ float grad_of(float x, float c, const RowCoef& r) {
  const float a = fmaf(x, c, -r.shift);
  const float e = exp2_hw(a);
  if (!kBeta) return e * r.alpha;
  return e * fmaf(fmaxf(a, -1000.0f), r.beta, r.alpha);
}

// A gradient row's elements lo .. hi - 1 (out: its first) of a row that has none, or that failed.
template <typename E, uint32_t kThreads>
__device__ __forceinline__ void fill_row(typename E::Raw* out, uint32_t lo, uint32_t hi,
                                         uint32_t state) {
  constexpr uint32_t kPer = E::kPer;
  const float f = state == kRowZero ? 0.0f : nan32();
  float fill[kPer];
#pragma unroll
  for (uint32_t e = 0; e < kPer; ++e) fill[e] = f;
  const uint4 v = E::pack(fill);
  const uint32_t whole = (hi - lo) / kPer;
  for (uint32_t i = threadIdx.x; i < whole; i += kThreads)
    store_chunk<E>(out + lo + (size_t)i * kPer, v);
  for (uint32_t j = lo + whole * kPer + threadIdx.x; j < hi; j += kThreads) out[j] = E::raw(f);
}

// token_logprobs_grad: what the gradient needs, from the forward pass' outputs:
// g (delta - q) - ge q (ln q + H), about the log-sum's nearest binary32 as above (d
// is what that leaves out).  `patch` is left to the thread that holds the token.
struct TokenGrad {
  double log2_sum, g, ge, entropy;
};
__device__ __forceinline__ RowCoef token_grad(const ScoreParams& p, uint32_t row, TokenGrad* o) {
  RowCoef r{};
  r.state = kRowZero;
  r.token = uniform_word(p.token + row);
  if (r.token == PB_NO_TOKEN) return r;
  double lse = (double)uniform_float(p.in_lse + row);
  if (p.in_lse_low) lse += (double)uniform_float(p.in_lse_low + row);
  o->g = p.grad_logprob ? (double)uniform_float(p.grad_logprob + row) : 0.0;
  o->ge = p.grad_entropy ? (double)uniform_float(p.grad_entropy + row) : 0.0;
  o->entropy = p.grad_entropy ? (double)uniform_float(p.in_entropy + row) : 0.0;
  o->log2_sum = lse * (1.0 / kLn2);
  if (r.token >= p.vocab || !__builtin_isfinite(lse) || o->g != o->g || o->ge != o->ge ||
      o->entropy != o->entropy) {
    r.state = kRowNan;
  } else if (o->g != 0.0 || o->ge != 0.0) {
    r.state = kRowNormal;
    r.shift = (float)o->log2_sum;
    const double d = ((double)r.shift - o->log2_sum) * kLn2;
    // e^d; d, half a step of the log-sum, is small unless the logits are very large
    const double f = (fabs(d) < 0x1p-9 ? 1.0 + d * (1.0 + 0.5 * d) : exp(d)) * p.inv_t;
    r.alpha = (float)(f * ((-o->g - o->ge * o->entropy) - o->ge * d));
    r.beta = (float)(f * -o->ge * kLn2);
  }
  return r;
}
__device__ __forceinline__ float token_patch(const ScoreParams& p, const TokenGrad& o, float x) {
  const double lp = kLn2 * ((double)x * (double)p.c - o.log2_sum), q = exp(lp);
  return (float)((o.g * -expm1(lp) - (q > 0.0 ? o.ge * q * (lp + o.entropy) : 0.0)) * p.inv_t);
}

// The gradient pass, by parts of a row of about 4,096 elements: 1,000 rows of
// 151,936 bf16 logits took 114 us by 151,936 elements a workgroup, 93 by 9,536, 88
// by 4,032 and 98 by 2,368.
constexpr uint32_t kFromToken = 0, kFromList = 1, kFromForward = 2;
template <typename E, uint32_t kFrom, bool kBeta>
__global__ __launch_bounds__(kGradThreads) void grad_kernel(const ScoreParams p) {
  using Raw = typename E::Raw;
  constexpr uint32_t kPer = E::kPer;
  const uint32_t row = blockIdx.x / p.grad_splits, split = blockIdx.x - row * p.grad_splits;
  const uint32_t lo = split * p.grad_span;
  const uint32_t hi = p.vocab - lo < p.grad_span ? p.vocab : lo + p.grad_span;
  const Raw* in = row_ptr<E>(p, row) + lo;
  Raw* out = static_cast<Raw*>(p.grad) + (size_t)row * p.grad_ld + lo;
  const uint32_t n = hi - lo, whole = n / kPer;
  TokenGrad token{};
  RowCoef r;
  if (kFrom == kFromForward)
    r = token_grad(p, row, &token);
  else
    r = p.coef[row];
  if (r.state == kRowUntouched) return;
  if (r.state != kRowNormal) {
    fill_row<E, kGradThreads>(out, 0, n, r.state);
    return;
  }
  // The special elements' gradients come from scalars in 64 bits, and their
  // logits are read before anything is written, since the gradient may go in
  // their place.  A token's is stored by the thread that stores its chunk, after
  // it; the listed ids' behind a barrier.
  uint32_t at = kNone;
  float patch = 0.0f;
  if (kFrom == kFromList) {
    if (threadIdx.x < p.k) {
      const size_t entry = (size_t)row * p.k + threadIdx.x;
      const uint32_t id = p.teacher_id[entry];
      if (id >= lo && id < hi) {
        at = id - lo;
        const double pr = exp((double)p.teacher_logit[entry] * p.inv_t - r.norm);
        patch = listed_grad(p, r, E::one(in[at]), pr);
      }
    }
    __syncthreads();
  } else if (r.token >= lo && r.token < hi) {
    const uint32_t place = r.token - lo;
    const uint32_t owner = place < whole * kPer ? place / kPer % kGradThreads
                                                : (place - whole * kPer) % kGradThreads;
    if (threadIdx.x == owner) {
      at = place;
      patch = kFrom == kFromForward ? token_patch(p, token, E::one(in[at])) : r.patch;
    }
  }
#pragma unroll 1
  for (uint32_t i = threadIdx.x; i < whole; i += kGradThreads) {
    const uint4 v = stream_chunk<E>(in + (size_t)i * kPer);
    float g[kPer];
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e) g[e] = grad_of<E, kBeta>(E::get(v, e), p.c, r);
    store_chunk<E>(out + (size_t)i * kPer, E::pack(g));
  }
  for (uint32_t j = whole * kPer + threadIdx.x; j < n; j += kGradThreads)
    out[j] = E::raw(grad_of<E, kBeta>(E::one(in[j]), p.c, r));
  if (kFrom == kFromList) __syncthreads();
  if (at != kNone) out[at] = E::raw(patch);
}

// ---- a row's loss and gradient in one launch ----
// One workgroup takes a whole row and holds on to it between the statistics and
// the gradient: its first kHeld chunks a thread in registers, with 512 threads
// kShelved more in LDS.  512 threads hold 114,688 16-bit logits and leave room for
// a second workgroup, whose loads run under the first one's scalars and stores;
// what lies beyond is read again.  Of 4,096 rows of 151,936 bf16 logits a quarter
// is, and they take 494 us: 2.5 GB at 5.0 TB/s, a large copy's rate.
// While gradients still went through the caches the same rows took 548 us, 566 by
// 1,024 threads that hold the whole row alone on their compute unit, and 590 with
// the next row's loads run into the gradient's stores; requesting the chunks that
// are read again ahead of their turn costs registers and took 525 instead of 495.
// The row's special elements (its token, or the teacher's list) hang in chains on
// the threads that hold them: the owner leaves their logits for the row's scalars,
// takes them out of the sums where the list has a rest bucket, and stores their
// gradients over its own chunks', so that no store waits for another thread's.

constexpr uint32_t kHeld = 19;
// With a rest bucket the row's scalars need more registers of their own.
constexpr uint32_t kHeldTail = 16;
// Chunks a thread in LDS behind them, so that two workgroups of 512 threads share a compute unit.
constexpr uint32_t kShelved = 9;

struct FusedShared {
  BlockSum sums;
  ListSum list;
  RowCoef coef;
  double pr[PB_TOP_LOGITS_MAX];
  uint32_t id[PB_TOP_LOGITS_MAX];
  uint32_t next[PB_TOP_LOGITS_MAX];
  float x[PB_TOP_LOGITS_MAX];
};

template <typename E, uint32_t kThreads, uint32_t kShelf, bool kTail>
struct FusedRow {
  static constexpr uint32_t kHeld = kTail ? kHeldTail : pb::kHeld;
  static constexpr uint32_t kPer = E::kPer;
  using Raw = typename E::Raw;
  const ScoreParams& p;
  FusedShared& l;
  const Raw* in;
  uint32_t whole;
  uint4* shelf;  // the kShelf chunks a thread behind the held ones
  uint32_t first_entry;

  // The special elements of the thread's chunk i out of x.
  __device__ __forceinline__ void take_out(float (&x)[E::kPer], uint32_t i) const {
    for (uint32_t e = first_entry; e != kNone; e = l.next[e]) {
      const uint32_t j = l.id[e] - i * kPer;
#pragma unroll
      for (uint32_t q = 0; q < kPer; ++q)
        if (q == j) x[q] = -__builtin_inff();
    }
  }
  // The partial chunk behind the whole ones, by the thread whose turn it is.
  __device__ __forceinline__ uint32_t rest() const { return p.vocab - whole * kPer; }
  __device__ __forceinline__ bool has_rest() const {
    return rest() != 0 && threadIdx.x == whole % kThreads;
  }
  __device__ __forceinline__ void load_rest(float (&x)[E::kPer]) const {
#pragma unroll
    for (uint32_t q = 0; q < kPer; ++q)
      x[q] = q < rest() ? E::one(in[(size_t)whole * kPer + q]) : -__builtin_inff();
  }
  // fn(chunk, i) for the thread's whole chunks from index `from` on, from memory, four loads at
  // once.
  template <typename Fn>
  __device__ __forceinline__ void each_chunk(uint32_t from, Fn fn) const {
    uint32_t i = from + threadIdx.x;
#pragma unroll 1
    for (; i + 3 * kThreads < whole; i += 4 * kThreads) {
      uint4 w[4];
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) w[q] = load_chunk<E>(in + (size_t)(i + q * kThreads) * kPer);
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) fn(w[q], i + q * kThreads);
    }
#pragma unroll 1
    for (; i < whole; i += kThreads) fn(load_chunk<E>(in + (size_t)i * kPer), i);
  }
  // fn(x, i), the partial chunk included and the special elements left out; keep(chunk, i) before
  // it.
  template <typename Keep, typename Fn>
  __device__ __forceinline__ void each_read(uint32_t from, Keep keep, Fn fn) const {
    float x[E::kPer];
    each_chunk(from, [&](const uint4& w, uint32_t i) {
      keep(w, i);
      unpack<E, false>(w, 0, x);
      if (kTail) take_out(x, i);
      fn(x, i);
    });
    if (has_rest()) {
      load_rest(x);
      if (kTail) take_out(x, whole);
      fn(x, whole);
    }
  }
  __device__ __forceinline__ void start(Acc& s, const float (&x)[E::kPer]) const {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < E::kPer; ++e) m = fmaxf(m, x[e]);
    const float u = m * p.c;
    s.shift = first_shift(u);
  }

  // special: bit c is set where the thread's chunk c holds a special element.
  __device__ __forceinline__ Acc sums(const uint4 (&v)[kHeld], uint32_t special,
                                      uint32_t* bad) const {
    const float c = p.c;
    Acc s;
    float x[E::kPer];
#pragma unroll
    for (uint32_t n = 0; n < kHeld; ++n) {
      const uint32_t i = n * kThreads + threadIdx.x;
      if (i < whole) {
        unpack<E, false>(v[n], 0, x);
        if (kTail && (special >> n & 1u)) take_out(x, i);
        if (n == 0) start(s, x);
        follow<false>(s, chunk_max<E>(x), c);
        add_chunk<E, false>(s, x, c);
      }
    }
    each_read(
        kHeld * kThreads,
        [&](const uint4& w, uint32_t i) {
          if (i < (kHeld + kShelf) * kThreads) shelf[i - kHeld * kThreads] = w;
        },
        [&](const float (&y)[E::kPer], uint32_t i) {
          if (i < kThreads) start(s, y);
          follow<false>(s, chunk_max<E>(y), c);
          add_chunk<E, false>(s, y, c);
        });
    *bad = kNone;
    if (sum_holds(s)) return s;
    // PartScan's second scan, from memory
    float top = -__builtin_inff();
    uint32_t at_bad = kNone;
    auto forget = [](const uint4&, uint32_t) {};
    each_read(0, forget, [&](const float (&y)[E::kPer], uint32_t i) {
#pragma unroll
      for (int e = 0; e < E::kPer; ++e) {
        const float u = y[e] * c;
        if (!(u < kTooBig) && at_bad == kNone) at_bad = i * kPer + e;
        top = fmaxf(top, u);
      }
    });
    s = Acc();
    *bad = at_bad;
    if (at_bad != kNone || !(top > -kTooBig)) return s;
    s.shift = top;
    each_read(0, forget,
              [&](const float (&y)[E::kPer], uint32_t) { add_chunk<E, false>(s, y, c); });
    return s;
  }
};

template <typename E, uint32_t kThreads, uint32_t kShelf, bool kTail>
__global__ __launch_bounds__(kThreads, 4) void fused_kernel(const ScoreParams p) {
  using Raw = typename E::Raw;
  constexpr uint32_t kPer = E::kPer, kHeld = kTail ? kHeldTail : pb::kHeld;
  __shared__ FusedShared l;
  __shared__ uint32_t head[kThreads];
  __shared__ uint4 shelf[kShelf * kThreads + 1];
  const uint32_t row = blockIdx.x, lane = lane_id(), wave = threadIdx.x >> 6;
  const uint32_t mine = threadIdx.x * kPer;  // the thread's place in a round of chunks
  const bool distill = p.mode == kModeDistill;
  const Raw* in = row_ptr<E>(p, row);
  Raw* out = static_cast<Raw*>(p.grad) + (size_t)row * p.grad_ld;
  const uint32_t whole = p.vocab / kPer;
  FusedRow<E, kThreads, kShelf, kTail> f{p, l, in, whole, shelf, kNone};
  uint4 v[kHeld];
  RowSum r{0.0, 0.0, 0.0, kNone};
  TokenRow token{};
  float weight = 1.0f;
  if (distill)
    weight = p.weight ? uniform_float(p.weight + row) : 1.0f;
  else
    token = token_row(p, row);
  const bool unread = row_unread(p, row);
  if (!unread) {
    // the list first: its loads come back before the row's
    ListLanes list{};
    if (wave == 0) {
      if (distill) {
        list = load_list(p, row, lane);
      } else {
        list.id[0] = lane == 0 ? token.token : kNone;
        list.id[1] = kNone;
      }
    }
#pragma unroll
    for (uint32_t n = 0; n < kHeld; ++n)
      if (n * kThreads + threadIdx.x < whole)
        v[n] = stream_chunk<E>(in + (size_t)n * (kThreads * kPer) + mine);
    head[threadIdx.x] = kNone;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t e = lane + 64u * h;
        l.id[e] = list.id[h];
        l.x[e] = 0.0f;
        if (list.id[h] < p.vocab)
          l.next[e] = atomicExch(&head[list.id[h] / kPer % kThreads], e);
      }
    }
    __syncthreads();
    f.first_entry = head[threadIdx.x];
    uint32_t special = 0;
    for (uint32_t e = f.first_entry; e != kNone; e = l.next[e]) {
      const uint32_t id = l.id[e];
      l.x[e] = E::one(in[id]);
      if (kTail && id / kPer < kHeld * kThreads) special |= 1u << (id / kPer / kThreads);
    }
    if (wave == 0 && distill) {
      double pr[2];
      const ListSum s = sum_teacher(p, list, lane, first_repeat(p, list, lane), pr);
      l.pr[lane] = pr[0];
      l.pr[lane + 64] = pr[1];
      if (lane == 0) l.list = s;
    }
    uint32_t bad;
    const Acc s = f.sums(v, special, &bad);
    r = block_sum<kThreads, false>(s, bad, l.sums);
  }
  DistillRow student;
  PolicyRow policy;
  ListSum list_sum{};
  uint32_t id[2] = {kNone, kNone};
  float x[2] = {0.0f, 0.0f};
  double pr[2] = {0.0, 0.0};
  if (wave == 0) {
    if (distill) {
      if (!unread) {
        list_sum = l.list;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          id[h] = l.id[lane + 64 * h];
          x[h] = l.x[lane + 64 * h];
          pr[h] = l.pr[lane + 64 * h];
        }
      }
      student = distill_row<E>(p, row, weight, r, list_sum, id, x);
      if (lane == 0) l.coef = student.coef;
      write_distill(p, row, student, list_sum, x, pr);
    } else {
      if (!unread) token.x = l.x[0];
      policy = policy_row<E>(p, row, r, token);
      if (lane == 0) l.coef = policy.coef;
      write_policy(p, row, policy);
    }
  }
  __syncthreads();
  const RowCoef& k = l.coef;
  if (k.state != kRowNormal) {
    fill_row<E, kThreads>(out, 0, p.vocab, k.state);
    return;
  }
  const RowCoef near{k.shift, k.alpha};  // what most elements need
  float g[kPer];
#pragma unroll
  for (uint32_t n = 0; n < kHeld; ++n) {
    if (n * kThreads + threadIdx.x < whole) {
#pragma unroll
      for (uint32_t e = 0; e < kPer; ++e) g[e] = grad_of<E, false>(E::get(v[n], e), p.c, near);
      store_chunk<E>(out + (size_t)n * (kThreads * kPer) + mine, E::pack(g));
    }
  }
  auto gradient = [&](const uint4& w) {
    float h[kPer];
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e) h[e] = grad_of<E, false>(E::get(w, e), p.c, near);
    return E::pack(h);
  };
#pragma unroll 1
  for (uint32_t n = 0; n < kShelf; ++n) {
    const uint32_t i = (kHeld + n) * kThreads + threadIdx.x;
    if (i < whole)
      store_chunk<E>(out + (size_t)i * kPer, gradient(shelf[n * kThreads + threadIdx.x]));
  }
  f.each_chunk((kHeld + kShelf) * kThreads, [&](const uint4& w, uint32_t i) {
    store_chunk<E>(out + (size_t)i * kPer, gradient(w));
  });
  if (f.has_rest()) {
    float x[kPer];
    f.load_rest(x);
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e)
      if (e < f.rest()) out[(size_t)whole * kPer + e] = E::raw(grad_of<E, false>(x[e], p.c, near));
  }
  // the thread's own special elements, over what it has just stored
  for (uint32_t e = f.first_entry; e != kNone; e = l.next[e])
    out[l.id[e]] = E::raw(distill ? listed_grad(p, k, l.x[e], l.pr[e]) : k.patch);
}

// ---- top logits ----
// A row's tiles of 2^tile_shift consecutive logits: the k largest logits lie in
// the k tiles of the largest maxima (the lower tile first among equal ones),
// since each of those holds a logit that ranks before any logit of another tile.
// So one pass over the row leaves its sums and a word a tile, and only k to
// k + kSlack tiles are read again: 2,048 rows of 151,936 bf16 logits in 104 us, 6.0
// TB/s, with the vector units busy two thirds of the time (109 us with quieting
// maxima and separate lane moves, 163 by halving the words' range for the k-th).

constexpr uint32_t kSlack = 64;            // tiles more than k that may be read
constexpr uint32_t kMaxList = PB_TOP_LOGITS_MAX + kSlack;
constexpr uint32_t kMaxCandidates = 512;
constexpr uint32_t kRounds = 32;           // of the search for the k-th largest word

struct TopShared {
  BlockSum sums;
  uint64_t keys[kMaxCandidates];
  uint64_t best[kTopThreads / 64];
  uint32_t list[kMaxList];
  uint32_t largest[kTopThreads];
  uint32_t counts[kRounds];
  uint32_t n_list, n_keys, low;
  uint32_t state;  // of the row: whether this workgroup selects, and whether it failed
};

// Larger key: larger value, then lower id.
__device__ __forceinline__ uint64_t value_key(float x, uint32_t id) {
  return ((uint64_t)ord_of(b_of(x)) << 32) | (0xffffffffu - id);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t ord = (uint32_t)(key >> 32);
  return f_of((ord & 0x80000000u) ? (ord & 0x7fffffffu) : ~ord);
}

// A chunk's largest value as an order word (-0 as 0), over the lanes that share
// its 64 elements: the four of a quad, mirrored halves of 8 and, for 32-bit rows,
// mirrored 16.
template <typename E>
__device__ __forceinline__ uint32_t tile_word(float m) {
  const uint32_t bits = b_of(m + 0.0f);
  uint32_t w = bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u);
  w = max(w, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xB1, 0xF, 0xF, true));
  w = max(w, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x4E, 0xF, 0xF, true));
  w = max(w, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x141, 0xF, 0xF, true));
  if (E::kPer == 4)
    w = max(w, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x140, 0xF, 0xF, true));
  return w;
}

// The part's sums, and its tiles' words; every lane of a wave takes part in
// every round, with -inf where the part has ended.  `words` has room for the
// last round's whole wave.  kWide: tiles of more than 64 elements.
template <typename E, bool kWide>
__device__ __forceinline__ Acc scan_tiles(const ScoreParams& p, const typename E::Raw* in,
                                          uint32_t n, uint32_t* words) {
  constexpr uint32_t kPer = E::kPer, kGroup = 64u / kPer;
  const uint32_t whole = n / kPer, rest = n - whole * kPer;
  Acc s;
  bool first = true;
  auto take = [&](const float (&x)[E::kPer], uint32_t i) {
    const float m = chunk_max<E>(x);
    if (first) {
      first = false;
      s.shift = first_shift(m * p.c);
    }
    follow<false>(s, m, p.c);
    add_chunk<E, false>(s, x, p.c);
    const uint32_t word = tile_word<E>(m);
    // the lanes of a tile write the same word
    if (kWide)
      atomicMax(&words[(i * kPer) >> p.tile_shift], word);
    else
      words[i / kGroup] = word;
  };
  float x[E::kPer];
  uint32_t base = 0;
  for (; base + 4u * kTopThreads <= whole; base += 4u * kTopThreads) {
    uint4 v[4];
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q)
      v[q] = stream_chunk<E>(in + (size_t)(base + q * kTopThreads + threadIdx.x) * kPer);
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q) {
      unpack<E, false>(v[q], 0, x);
      take(x, base + q * kTopThreads + threadIdx.x);
    }
  }
  for (; base < whole + (rest ? 1u : 0u); base += kTopThreads) {
    const uint32_t i = base + threadIdx.x;
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e) x[e] = -__builtin_inff();
    if (i < whole) {
      unpack<E, false>(stream_chunk<E>(in + (size_t)i * kPer), 0, x);
    } else if (i == whole) {
#pragma unroll
      for (uint32_t e = 0; e < kPer; ++e)
        if (e < rest) x[e] = E::one(in[(size_t)whole * kPer + e]);
    }
    take(x, i);
  }
  return s;
}

// Lists `want` tiles by one wave: those whose words are above `low`, then the
// first of those at it.
__device__ __forceinline__ void list_words(const uint32_t* words, uint32_t tiles, uint32_t low,
                                           uint32_t want, TopShared& l) {
  const uint32_t lane = lane_id();
  uint32_t above = 0;
  for (uint32_t i = lane; i < tiles; i += 64u) above += words[i] > low ? 1u : 0u;
  uint32_t n = 0, equal = want - wave_sum_word(above);
  for (uint32_t base = 0; base < tiles; base += 64u) {
    const uint32_t i = base + lane;
    const uint32_t v = i < tiles ? words[i] : 0u;
    const bool at = i < tiles && v == low;
    const uint64_t same = __ballot(at);
    const bool take = (i < tiles && v > low) || (at && lanes_below(same) < equal);
    const uint64_t taken = __ballot(take);
    if (take) l.list[n + lanes_below(taken)] = i;
    n += (uint32_t)__popcll((unsigned long long)taken);
    const uint32_t got = (uint32_t)__popcll((unsigned long long)same);
    equal -= got < equal ? got : equal;
  }
  if (lane == 0) l.n_list = n;
}

// The k best of a row from its tiles' words in LDS; every thread.
template <typename E>
__device__ void select_top(const ScoreParams& p, uint32_t row, uint32_t tiles,
                           const uint32_t* words, TopShared& l) {
  constexpr uint32_t kPer = E::kPer, kWaves = kTopThreads / 64;
  const uint32_t lane = lane_id(), wave = threadIdx.x >> 6;
  const uint32_t want = p.k < tiles ? p.k : tiles;
  // The want-th largest of some groups' largest words is reached by `want` words
  // at least, and rarely by many more: of 2,374 words of normal logits, 24 for 20
  // of 64 groups, 72 for 64 of 256.  (Halving the words' range took 10 rounds.)
  uint32_t mine = 0;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < tiles; i += kTopThreads) mine = max(mine, words[i]);
  // distinct among the threads; their low bits only lower the word that is found
  mine = (mine & ~(kTopThreads - 1u)) | threadIdx.x;
  l.largest[threadIdx.x] = mine;
  if (threadIdx.x < kRounds) l.counts[threadIdx.x] = 0;
  if (threadIdx.x == 0) l.n_list = l.n_keys = 0;
  __syncthreads();
  if (want <= 48u) {
    if (wave == 0) {
      for (uint32_t w = 1; w < kWaves; ++w) mine = max(mine, l.largest[64u * w + lane]);
      mine = bcast32(wave_sort_desc_u32(mine, lane), want - 1u);
      if (lane == 0) l.low = mine & ~(kTopThreads - 1u);
    }
  } else {
    uint32_t rank = 0;
    const uint4* others = reinterpret_cast<const uint4*>(l.largest);
#pragma unroll 8
    for (uint32_t q = 0; q < kTopThreads / 4; ++q) {
      const uint4 o = others[q];
      rank += (o.x > mine ? 1u : 0u) + (o.y > mine ? 1u : 0u) + (o.z > mine ? 1u : 0u) +
              (o.w > mine ? 1u : 0u);
    }
    if (rank == want - 1u) l.low = mine & ~(kTopThreads - 1u);
  }
  __syncthreads();
  uint32_t low = l.low;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < tiles; i += kTopThreads) {
    if (words[i] >= low) {
      const uint32_t at = atomicAdd(&l.n_list, 1u);
      if (at < kMaxList) l.list[at] = i;
    }
  }
  __syncthreads();
  uint32_t reach = l.n_list;  // words >= low
  if (reach > kMaxList) {
    // A word that want to want + kSlack words reach, by halving; failing that
    // (many equal words) the want-th largest, and the first tiles that reach it.
    uint32_t high = ~0u;
    for (uint32_t round = 0; round < kRounds && reach > want + kSlack; ++round) {
      const uint32_t middle = low + (high - low) / 2u + 1u;
      uint32_t n = 0;
      for (uint32_t i = threadIdx.x; i < ((tiles + 63u) & ~63u); i += kTopThreads)
        n += (uint32_t)__popcll((unsigned long long)__ballot(i < tiles && words[i] >= middle));
      if (lane == 0) atomicAdd(&l.counts[round], n);
      __syncthreads();
      n = l.counts[round];
      if (n >= want) {
        low = middle;
        reach = n;
      } else {
        high = middle - 1u;
      }
    }
    if (wave == 0) list_words(words, tiles, low, reach <= want + kSlack ? reach : want, l);
    __syncthreads();
  }
  // the listed tiles' logits that reach the word: all of the k largest, and few others
  const typename E::Raw* in = row_ptr<E>(p, row);
  const uint32_t per_tile = 1u << p.tile_shift, total = l.n_list << p.tile_shift;
  auto offer = [&](float x, uint32_t id) {
    const uint64_t key = value_key(x, id);
    if ((uint32_t)(key >> 32) >= low) {
      const uint32_t at = atomicAdd(&l.n_keys, 1u);
      if (at < kMaxCandidates) l.keys[at] = key;
    }
  };
#pragma unroll 1
  for (uint32_t i = threadIdx.x * kPer; i < total; i += kTopThreads * kPer) {
    const uint32_t id = (l.list[i >> p.tile_shift] << p.tile_shift) + (i & (per_tile - 1u));
    if (id + kPer <= p.vocab) {
      const uint4 v = load_chunk<E>(in + id);
#pragma unroll
      for (uint32_t e = 0; e < kPer; ++e) offer(E::get(v, e), id + e);
    } else {
      for (uint32_t e = 0; e < kPer; ++e)
        if (id + e < p.vocab) offer(E::one(in[id + e]), id + e);
    }
  }
  __syncthreads();
  uint32_t* out_id = p.top_id + (size_t)row * p.k;
  float* out_value = p.top_value + (size_t)row * p.k;
  const uint32_t n = l.n_keys;
  if (n >= p.k && n <= kMaxCandidates) {
    // a key's rank is the number of keys above it (no two are equal)
    for (uint32_t i = threadIdx.x; i < n; i += kTopThreads) {
      const uint64_t key = l.keys[i];
      uint32_t rank = 0;
#pragma unroll 8
      for (uint32_t j = 0; j < n; ++j) rank += l.keys[j] > key ? 1u : 0u;
      if (rank < p.k) {
        out_id[rank] = 0xffffffffu - (uint32_t)key;
        out_value[rank] = key_value(key);
      }
    }
    return;
  }
  // Many equal values, or fewer tiles than k: one largest key after the other.
  uint64_t last = ~0ull;
  for (uint32_t rank = 0; rank < p.k; ++rank) {
    uint64_t best = 0;
    for (uint32_t i = threadIdx.x; i < total; i += kTopThreads) {
      const uint32_t id = (l.list[i >> p.tile_shift] << p.tile_shift) + (i & (per_tile - 1u));
      if (id >= p.vocab) continue;
      const uint64_t key = value_key(E::one(in[id]), id);
      if (key < last && key > best) best = key;
    }
    best = wave_max64(best);
    if (lane == 0) l.best[wave] = best;
    __syncthreads();
    for (uint32_t w = 0; w < kWaves; ++w) best = l.best[w] > best ? l.best[w] : best;
    if (threadIdx.x == 0) {
      out_id[rank] = 0xffffffffu - (uint32_t)best;
      out_value[rank] = key_value(best);
    }
    last = best;
    __syncthreads();
  }
}

constexpr uint32_t kTopWaits = 0, kTopSelects = 1, kTopFailed = 2;

// A part's pass, and by the row's last part its selection.  The words of a row
// in parts go through the workspace at the device's scope, as RowPart does.
template <typename E>
__global__ __launch_bounds__(kTopThreads, 8) void top_kernel(const ScoreParams p) {
  __shared__ TopShared l;
  extern __shared__ uint32_t words[];  // the row's
  const uint32_t row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits;
  const uint32_t lo = split * p.span;
  const uint32_t hi = p.vocab - lo < p.span ? p.vocab : lo + p.span;
  const uint32_t round_up = (1u << p.tile_shift) - 1u;
  const uint32_t own = (hi - lo + round_up) >> p.tile_shift;
  const uint32_t tiles = (p.vocab + round_up) >> p.tile_shift;
  if (p.tile_shift > 6) {
    for (uint32_t i = threadIdx.x; i < own; i += kTopThreads) words[i] = 0;
    __syncthreads();
  }
  const typename E::Raw* in = row_ptr<E>(p, row) + lo;
  Acc s = p.tile_shift > 6 ? scan_tiles<E, true>(p, in, hi - lo, words)
                           : scan_tiles<E, false>(p, in, hi - lo, words);
  uint32_t bad = kNone;
  if (!sum_holds(s)) {
    const PartScan<E, kTopThreads, false, false, false> scan{row_ptr<E>(p, row), nullptr, lo, hi,
                                                              p.c};
    s = scan.again(&bad);
  }
  RowSum r = block_sum<kTopThreads, false>(s, bad, l.sums);  // its barrier: the words are there
  uint32_t* shared_words = p.tiles + (size_t)row * tiles;
  if (p.splits > 1) {
    if (threadIdx.x == 0) publish_part(p.part + (size_t)row * p.splits + split, r);
    for (uint32_t i = threadIdx.x; i < own; i += kTopThreads)
      __hip_atomic_store(shared_words + (lo >> p.tile_shift) + i, words[i], __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    acknowledged();
    __syncthreads();
    if (threadIdx.x < 64) {
      const bool last = last_part(p, row);
      if (threadIdx.x == 0) l.state = last ? kTopSelects : kTopWaits;
    }
    __syncthreads();
    if (l.state == kTopWaits) return;
    for (uint32_t i = threadIdx.x; i < tiles; i += kTopThreads)
      words[i] = __hip_atomic_load(shared_words + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();  // l.state is written again
  }
  if (threadIdx.x < 64) {
    if (p.splits > 1) r = join_parts<false>(p, row);
    if (threadIdx.x == 0) {
      pb_inference_error* at = p.err ? p.err + row : nullptr;
      const bool failed = bad_row(r.bad, r.sum);
      if (failed)
        report_row<E>(p, row, r.bad, at);
      else
        no_error(at);
      if (p.lse) p.lse[row] = failed ? nan32() : (float)(kLn2 * (r.shift + log2(r.sum)));
      l.state = failed ? kTopFailed : kTopSelects;
    }
  }
  __syncthreads();
  if (l.state == kTopFailed) {
    for (uint32_t i = threadIdx.x; i < p.k; i += kTopThreads) {
      p.top_id[(size_t)row * p.k + i] = PB_NO_TOKEN;
      p.top_value[(size_t)row * p.k + i] = nan32();
    }
    return;
  }
  select_top<E>(p, row, tiles, words, l);
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1u) / b; }

// Workgroups that the statistics of few rows are cut into: four of the eight that a
// compute unit takes.  More parts lengthen the join, and rows that then come in two
// parts are read no faster; fewer leave units idle.  Log-probabilities of rows of
// 151,936 bf16 logits, us with a target of 512 / 1,024 / 2,048 / 4,096:
//   4 rows 7.2 / 7.1 / 6.9 / 7.0   33 rows 9.3 / 14.6 / 16.8 / 16.8   150 rows 12.7 / 13.7 / 16.7 / 26.7
//   400 rows 34 / 27 / 30 / 34     1,000 rows 56 / 56 / 64 / 63       2,000 rows 106 / 107 / 106 / 101
constexpr uint32_t kTargetGroups = 1024;
// The same for the top logits, whose parts publish their tiles' words too; f32, k = 64,
// us with 256 / 512 / 1,024:
//   4 rows 17.8 / 17.8 / 18.4   33 rows 22.8 / 23.1 / 29.0   70 rows 29.0 / 25.6 / 29.0
//   150 rows 45 / 33 / 34       300 rows 51 / 50 / 48
constexpr uint32_t kTopGroups = 512;
// Of the gradient pass, never in parts of less than 4,096 elements; us with 8,192 /
// 65,536, bf16: 40 rows 7.2 / 7.2, 300 rows 32 / 31, 1,000 rows 110 / 95, 3,000 rows
// 348 / 290.
constexpr uint32_t kGradGroups = 65536;
// Logits that may stay in the caches between the two passes (plan_scores).
constexpr uint64_t kCacheBytes = 400000000;
// A loss and its gradient take one launch, a workgroup a row, for rows of up to
// kShortRow bytes and from kFusedRows longer ones on.
constexpr uint32_t kShortRow = 160 * 1024;
constexpr uint32_t kFusedRows = 64;
constexpr uint32_t kFewChunks = 4;  // a thread, below which more threads share a row

uint32_t tile_shift_of(uint32_t vocab) {
  uint32_t shift = 6;
  while (((vocab + (1u << shift) - 1u) >> shift) > kMaxTiles) ++shift;
  return shift;
}

uint32_t max_slots(uint32_t rows, uint32_t vocab) {
  // rows x splits: at most the target and one part a row more, or the parts
  // that the largest span asks for
  const uint32_t by_span = rows * ceil_div(vocab, kMaxSpan);
  const uint32_t by_target = kTargetGroups + rows;
  return by_span > by_target ? by_span : by_target;
}

struct ScoresLayout {
  size_t part, coef, tiles, total;
};
ScoresLayout scores_layout(uint32_t rows, uint32_t vocab) {
  ScoresLayout l;
  const uint32_t by_64 = ceil_div(vocab, 64u);  // never fewer than the tiles in use
  l.part = 0;
  l.coef = l.part + align256((size_t)max_slots(rows, vocab) * sizeof(RowPart));
  l.tiles = l.coef + align256((size_t)rows * sizeof(RowCoef));
  l.total = l.tiles + align256((size_t)rows * (by_64 < kMaxTiles ? by_64 : kMaxTiles) * 4);
  return l;
}

}  // namespace

void plan_scores(uint32_t dtype, ScoreParams* p) {
  p->fused = 0;
  // Forward and gradient of rows of 304 KB, us with the first read kept in the
  // caches and without: 900 rows 128 / 132, 1,300 rows 189 / 191, 2,000 rows 287 /
  // 283, 3,000 rows 431 / 426.  The preference loss keeps twice that: many of a batch's
  // rows are prompts or padding, which are not read.  With none, 30 % and 60 % of the
  // rows left out: 1,400 rows 200 / 203, 164 / 176, 124 / 146; 2,000 rows 290 / 297,
  // 229 / 245, 177 / 198; 2,600 rows 379 / 377, 312 / 331, 229 / 257.
  const uint64_t logit_bytes = (uint64_t)p->rows * p->vocab * (dtype == PB_F32 ? 4u : 2u);
  p->keep = logit_bytes <= (p->mode == kModePreference ? 2u : 1u) * kCacheBytes;
  if (p->grad != nullptr && (p->mode == kModeDistill || p->mode == kModePolicy)) {
    const uint32_t chunks = ceil_div(p->vocab, dtype == PB_F32 ? 4u : 8u);
    // threads a row: as few as hold it, or more where rows do not fill the compute
    // units (64 rows of 8,000 bf16 logits: 7.2 us by 256 threads, 7.8 by 64)
    uint32_t threads = chunks <= 64 * kHeld ? 64 : chunks <= 256 * kHeld ? 256 : 512;
    if (p->rows <= 1024 && threads < 256 && chunks > 64 * kFewChunks) threads = 256;
    if (p->rows <= 512 && threads < 512 && chunks > 256 * kFewChunks) threads = 512;
    if (p->rows <= 256 && threads < 1024 && chunks > 512 * kFewChunks) threads = 1024;
    // One launch or two passes, us by rows (policy loss with gradient):
    //   rows              1           12          64          256         1,000
    //   1,000 bf16    4.7 / 7.7   5.8 / 10.8  5.9 / 11.2  6.1 / 10.3  6.6 / 8.4
    //   32,000 f32    8.5 / 11.5  9.2 / 9.8  10.0 / 12.9   14 / 22     48 / 51
    //   100,003 f16    15 / 10     18 / 13     20 / 20     24 / 32     87 / 95
    //   151,936 f32    21 / 9.8    21 / 15     23 / 26     54 / 61    247 / 253
    // A long row takes one workgroup longer than many, and past kMaxTerms logits a
    // thread its sums would need more bits (64 rows of 1,048,576 took one launch 282 us
    // in f32 and 144 in bf16, and two passes 138 and 75).
    const uint64_t row_bytes = (uint64_t)p->vocab * (dtype == PB_F32 ? 4u : 2u);
    if ((row_bytes <= kShortRow || p->rows >= kFusedRows) && p->vocab <= kMaxTerms * threads)
      p->fused = threads;
  }
  p->tile_shift = tile_shift_of(p->vocab);
  const uint32_t tile = 1u << p->tile_shift;
  if (p->rows == 0) return;
  uint32_t splits = (p->mode == kModeTop ? kTopGroups : kTargetGroups) / p->rows;
  const uint32_t most = ceil_div(p->vocab, 4096u);
  if (splits > most) splits = most;
  if (splits > kMaxSplits) splits = kMaxSplits;
  if (splits < 1) splits = 1;
  const uint32_t least = ceil_div(p->vocab, kMaxSpan);
  if (splits < least) splits = least;
  p->span = ceil_div(ceil_div(p->vocab, splits), tile) * tile;
  p->splits = ceil_div(p->vocab, p->span);
  uint32_t grad_splits = ceil_div(kGradGroups, p->rows);
  if (grad_splits > most) grad_splits = most;
  p->grad_span = ceil_div(ceil_div(p->vocab, grad_splits), 64u) * 64u;
  p->grad_splits = ceil_div(p->vocab, p->grad_span);
}

size_t scores_workspace_bytes(uint32_t rows, size_t vocab) {
  return rows == 0 || vocab == 0 ? 0 : scores_layout(rows, (uint32_t)vocab).total;
}

void place_scores(void* work, ScoreParams* p) {
  const ScoresLayout l = scores_layout(p->rows, p->vocab);
  char* base = static_cast<char*>(work);
  p->part = reinterpret_cast<RowPart*>(base + l.part);
  p->coef = reinterpret_cast<RowCoef*>(base + l.coef);
  p->tiles = p->sequence = reinterpret_cast<uint32_t*>(base + l.tiles);
}

namespace {

template <typename E, bool kEntropy, uint32_t kList>
void launch_stats(const ScoreParams& p, hipStream_t stream) {
  const size_t marks = kList == kListWithRest ? ((size_t)p.span / 32 + 2) * 4 : 0;
  const uint32_t groups = p.rows * p.splits, threads = kStatsThreads + (kList ? 64u : 0u);
  if (p.keep)
    stats_kernel<E, kEntropy, kList, true><<<groups, threads, marks, stream>>>(p);
  else
    stats_kernel<E, kEntropy, kList, false><<<groups, threads, marks, stream>>>(p);
}

template <typename E>
struct Launch {
  static void logprobs(const ScoreParams& p, hipStream_t s) {
    if (p.entropy)
      launch_stats<E, true, kNoList>(p, s);
    else
      launch_stats<E, false, kNoList>(p, s);
  }
  template <uint32_t kFrom, bool kBeta>
  static void grad(const ScoreParams& p, hipStream_t s) {
    grad_kernel<E, kFrom, kBeta><<<p.rows * p.grad_splits, kGradThreads, 0, s>>>(p);
  }
  static void logprobs_grad(const ScoreParams& p, hipStream_t s) {
    if (p.grad_entropy)
      grad<kFromForward, true>(p, s);
    else
      grad<kFromForward, false>(p, s);
  }
  static void top(const ScoreParams& p, hipStream_t s) {
    // and what the last round of threads writes past the row's end
    const size_t words =
        (size_t)(ceil_div(p.vocab, 1u << p.tile_shift) + kTopThreads * E::kPer / 64u) * 4;
    top_kernel<E><<<p.rows * p.splits, kTopThreads, words, s>>>(p);
  }
  template <uint32_t kThreads, uint32_t kShelf>
  static void fused(const ScoreParams& p, hipStream_t s) {
    if (p.teacher_lse)
      fused_kernel<E, kThreads, kShelf, true><<<p.rows, kThreads, 0, s>>>(p);
    else
      fused_kernel<E, kThreads, kShelf, false><<<p.rows, kThreads, 0, s>>>(p);
  }
  static void row_loss(const ScoreParams& p, hipStream_t s) {
    switch (p.fused) {
      case 64: return fused<64, 0>(p, s);
      case 256: return fused<256, 0>(p, s);
      case 512: return fused<512, kShelved>(p, s);
      case 1024: return fused<1024, 0>(p, s);
    }
    if (p.mode != kModeDistill)
      launch_stats<E, false, kNoList>(p, s);
    else if (p.teacher_lse)
      launch_stats<E, false, kListWithRest>(p, s);
    else
      launch_stats<E, false, kListOnly>(p, s);
    if (p.grad == nullptr) return;
    if (p.mode == kModeDistill)
      grad<kFromList, false>(p, s);
    else
      grad<kFromToken, false>(p, s);
  }
  static void preference(const ScoreParams& p, hipStream_t s) {
    if (p.rows == 0) {  // pairs of empty sequences
      pair_kernel<E><<<p.pairs, 256, 0, s>>>(p);
      return;
    }
    launch_stats<E, false, kNoList>(p, s);
    pair_kernel<E><<<p.pairs, 256, 0, s>>>(p);
    if (p.grad) grad<kFromToken, false>(p, s);
  }
};

}  // namespace

#define PB_SCORE_LAUNCH(name, call)                                                    \
  hipError_t name(const ScoreParams& p, uint32_t dtype, hipStream_t stream) {          \
    (void)hipGetLastError();                                                           \
    if (dtype == PB_F32)                                                               \
      Launch<F32>::call(p, stream);                                                    \
    else if (dtype == PB_F16)                                                          \
      Launch<F16>::call(p, stream);                                                    \
    else                                                                               \
      Launch<BF16>::call(p, stream);                                                   \
    return hipGetLastError();                                                          \
  }
PB_SCORE_LAUNCH(launch_token_logprobs, logprobs)
PB_SCORE_LAUNCH(launch_token_logprobs_grad, logprobs_grad)
PB_SCORE_LAUNCH(launch_top_logits, top)
PB_SCORE_LAUNCH(launch_row_loss, row_loss)
PB_SCORE_LAUNCH(launch_preference, preference)
#undef PB_SCORE_LAUNCH

}  // namespace pb
