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
constexpr uint32_t kStatsThreads = 512;
constexpr uint32_t kGradThreads = 256;
constexpr uint32_t kSelectThreads = 512;
constexpr float kTooBig = 3.0e38f;  // |u| past this has left binary32's range

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
typedef Words4 Loose4 __attribute__((aligned(2)));
template <typename E>
__device__ __forceinline__ uint4 load_chunk(const typename E::Raw* p) {
  const Words4 v = *reinterpret_cast<const Loose4*>(p);
  return make_uint4(v.x, v.y, v.z, v.w);
}
template <typename E>
__device__ __forceinline__ void store_chunk(typename E::Raw* p, const uint4& v) {
  *reinterpret_cast<Loose4*>(p) = Words4{v.x, v.y, v.z, v.w};
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
  return f_of(wave_fold(b_of(v), [](uint32_t a, uint32_t b) { return b_of(fmaxf(f_of(a), f_of(b))); }));
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
__device__ __forceinline__ double wave_max_f64(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    const double o = __builtin_bit_cast(double, shfl_xor64(__builtin_bit_cast(uint64_t, v), m));
    v = o > v ? o : v;
  }
  return v;
}

// ---- rows ----

// Whether the statistics pass leaves a row out: it is masked, or its id is bad
// (which the finishing pass reports).
__device__ __forceinline__ bool row_unread(const ScoreParams& p, uint32_t row) {
  if (p.mode == kModeTop) return false;
  if (p.mode == kModeDistill) return p.weight != nullptr && p.weight[row] == 0.0f;
  if (p.mode == kModePreference) {
    const uint32_t end = p.seq_start[2 * p.pairs];
    if (row < p.seq_start[0] || row >= end) return true;
  }
  if (p.mode == kModePolicy && p.weight != nullptr && p.weight[row] == 0.0f) return true;
  return p.token[row] >= p.vocab;
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

// Bits of the marks of the elements j .. j + kPer - 1 of a part that starts at lo.
template <typename E>
__device__ __forceinline__ uint32_t chunk_marks(const uint32_t* marks, uint32_t at) {
  return (marks[at >> 5] >> (at & 31u)) & ((1u << E::kPer) - 1u);
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

template <typename E, bool kTail>
__device__ __forceinline__ void unpack(const uint4& v, uint32_t marks, float (&x)[E::kPer]) {
#pragma unroll
  for (int i = 0; i < E::kPer; ++i) {
    x[i] = E::get(v, i);
    if (kTail && (marks >> i & 1u)) x[i] = -__builtin_inff();
  }
}

// A thread's sums over its chunks of [lo, hi), chunk i of thread t being
// element lo + (i kStatsThreads + t) kPer.  The shift is the thread's first
// chunk's largest u: nothing then underflows that weighs, and where a later u
// passes it by over 2^127, or the first chunk is masked out, the sum shows it
// (infinite, or too small) and the thread goes over its chunks again with their
// true maximum.  So the pass does no comparison per element.
template <typename E, bool kEntropy, bool kTail>
struct PartScan {
  const typename E::Raw* row;
  const uint32_t* marks;
  uint32_t lo, hi;
  float c;

  template <typename Fn>
  __device__ __forceinline__ void each(Fn fn) const {
    constexpr uint32_t kPer = E::kPer;
    const uint32_t whole = (hi - lo) / kPer;
    uint32_t i = threadIdx.x;
    for (; i + 3 * kStatsThreads < whole; i += 4 * kStatsThreads) {
      uint4 v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        v[q] = load_chunk<E>(row + lo + (size_t)(i + q * kStatsThreads) * kPer);
#pragma unroll
      for (int q = 0; q < 4; ++q) chunk(v[q], (i + q * kStatsThreads) * kPer, fn);
    }
    for (; i < whole; i += kStatsThreads)
      chunk(load_chunk<E>(row + lo + (size_t)i * kPer), i * kPer, fn);
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
    each([&](const float (&x)[E::kPer], uint32_t) {
      if (first) {
        first = false;
        float m = x[0];
#pragma unroll
        for (int e = 1; e < E::kPer; ++e) m = fmaxf(m, x[e]);
        const float u = m * c;
        s.shift = u > -kTooBig ? u : 0.0f;
      }
      add_chunk<E, kEntropy>(s, x, c);
    });
    *bad = kNone;
    if (first || (s.sum >= 0x1p-60f && s.sum <= 3.4e38f)) return s;
    // again, with the largest u of all
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
    s = Acc();
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

// The workgroup's sums, valid in thread 0.
struct BlockSum {
  float shift[16];
  double sum[16];
  double moment[16];
  uint32_t bad[16];
};
template <uint32_t kThreads>
__device__ __forceinline__ RowPart block_sum(const Acc& s, uint32_t bad, BlockSum& l) {
  const uint32_t lane = lane_id(), wave = threadIdx.x >> 6;
  const float top = wave_max_f32(s.sum > 0.0f ? s.shift : -__builtin_inff());
  const float off = s.shift - top;
  const double f = s.sum > 0.0f ? (double)exp2_hw(off) : 0.0;
  const double sum = wave_sum_f64(f * (double)s.sum);
  const double moment =
      wave_sum_f64(f == 0.0 ? 0.0 : f * ((double)s.moment + (double)off * (double)s.sum));
  const uint32_t b = wave_min_word(bad);
  if (lane == 0) {
    l.shift[wave] = top;
    l.sum[wave] = sum;
    l.moment[wave] = moment;
    l.bad[wave] = b;
  }
  __syncthreads();
  RowPart out{0.0f, kNone, 0.0, 0.0};
  if (threadIdx.x == 0) {
    float best = l.shift[0];
    for (uint32_t w = 1; w < kThreads / 64; ++w) best = fmaxf(best, l.shift[w]);
    for (uint32_t w = 0; w < kThreads / 64; ++w) {
      out.bad = l.bad[w] < out.bad ? l.bad[w] : out.bad;
      if (!(l.sum[w] > 0.0)) continue;
      const double d = (double)l.shift[w] - (double)best;
      const double g = exp2(d);
      out.sum += g * l.sum[w];
      out.moment += g * (l.moment[w] + d * l.sum[w]);
    }
    out.shift = out.sum > 0.0 ? best : 0.0f;
  }
  return out;
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

template <typename E, bool kEntropy, bool kTail>
__global__ __launch_bounds__(kStatsThreads) void stats_kernel(const ScoreParams p) {
  __shared__ BlockSum l;
  extern __shared__ uint32_t marks[];
  const uint32_t row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits;
  if (row_unread(p, row)) return;
  const uint32_t lo = split * p.span;
  const uint32_t hi = p.vocab - lo < p.span ? p.vocab : lo + p.span;
  if (kTail) mark_ids(p, row, lo, hi, marks);
  const PartScan<E, kEntropy, kTail> scan{row_ptr<E>(p, row), marks, lo, hi, p.c};
  uint32_t bad;
  const Acc s = scan.run(&bad);
  const RowPart out = block_sum<kStatsThreads>(s, bad, l);
  if (threadIdx.x == 0) p.part[(size_t)row * p.splits + split] = out;
}

// ---- a row's scalars, one wave a row ----

struct RowSum {
  double shift, sum, moment;  // sum 2^(u - shift)
  uint32_t bad;
};

__device__ __forceinline__ RowSum join_parts(const ScoreParams& p, uint32_t row, uint32_t lane) {
  RowPart v{0.0f, kNone, 0.0, 0.0};
  if (lane < p.splits) v = p.part[(size_t)row * p.splits + lane];
  const bool live = v.sum > 0.0;
  RowSum r;
  const float top = wave_max_f32(live ? v.shift : -__builtin_inff());
  r.bad = wave_min_word(v.bad);
  const double d = live ? (double)v.shift - (double)top : 0.0;
  const double f = live ? exp2(d) : 0.0;
  r.sum = wave_sum_f64(f * v.sum);
  r.moment = wave_sum_f64(f * (v.moment + d * v.sum));
  r.shift = r.sum > 0.0 ? (double)top : 0.0;
  return r;
}

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

// The binary32 bits of a logit, for an error record.
template <typename E>
__device__ __forceinline__ uint32_t logit_bits(const ScoreParams& p, uint32_t row, uint32_t id) {
  return b_of(E::one(row_ptr<E>(p, row)[id]));
}

__device__ __forceinline__ float nan32() { return f_of(0x7fc00000u); }

// alpha, beta and shift of a row whose gradient is q (A + B ln q) for most
// elements: the shift is log2_sum's nearest binary32, and what that rounding
// leaves out goes into the factors.
__device__ __forceinline__ void set_factors(RowCoef& r, double log2_sum, double a, double b) {
  const float shift = (float)log2_sum;
  const double d = (double)shift - log2_sum;
  const double f = exp2(d);
  r.shift = shift;
  r.alpha = (float)(f * (a + b * kLn2 * d));
  r.beta = (float)(f * b * kLn2);
  r.log2_sum = log2_sum;
}

// Gradient w / T (delta - q) slope of a row with one token; lp = ln q[token].
__device__ __forceinline__ RowCoef token_coef(double log2_sum, double slope, double lp,
                                              uint32_t token) {
  RowCoef r{};
  if (slope == 0.0) {
    r.state = kRowZero;
    return r;
  }
  r.state = slope == slope ? kRowNormal : kRowNan;
  set_factors(r, log2_sum, -slope, 0.0);
  r.token = token;
  r.patch = (float)(slope * -expm1(lp));
  return r;
}

// ln q[token] in 64 bits.
template <typename E>
__device__ __forceinline__ double token_logprob(const ScoreParams& p, uint32_t row, uint32_t token,
                                                double log2_sum) {
  const double u = (double)E::one(row_ptr<E>(p, row)[token]) * (double)p.c;
  return kLn2 * (u - log2_sum);
}

// Reports what is wrong with a row that was read; true if anything is.
template <typename E>
__device__ __forceinline__ bool row_failed(const ScoreParams& p, uint32_t row, uint32_t bad,
                                           double sum, pb_inference_error* at) {
  if (bad == kNone && sum > 0.0) return false;
  const uint32_t index = bad == kNone ? 0u : bad;
  write_error(at, PB_NONFINITE_OUTPUT, row, 0, logit_bits<E>(p, row, index), PB_FIELD_FINITE,
              index);
  return true;
}

template <typename E>
__device__ void finish_policy(const ScoreParams& p, uint32_t row, const RowSum& r, uint32_t lane) {
  if (lane != 0) return;
  const uint32_t token = p.token[row];
  const float w = p.weight ? p.weight[row] : 1.0f;
  pb_inference_error* at = p.err ? p.err + row : nullptr;
  float loss = 0.0f, logprob = 0.0f, kl_out = 0.0f;
  RowCoef coef{};
  coef.state = kRowZero;
  if (token == PB_NO_TOKEN || w == 0.0f) {
    no_error(at);
  } else {
    bool failed = token >= p.vocab;
    if (failed)
      write_error(at, PB_TOKEN_ID, row, p.vocab, token, PB_FIELD_TOKEN, 0);
    else
      failed = row_failed<E>(p, row, r.bad, r.sum, at);
    if (failed) {
      loss = logprob = kl_out = nan32();
      coef.state = kRowNan;
    } else {
      no_error(at);
      const double log2_sum = r.shift + log2(r.sum);
      const double lp = token_logprob<E>(p, row, token, log2_sum);
      const double ratio = exp(lp - (double)p.old_logprob[row]), adv = (double)p.advantage[row];
      const double low = 1.0 - p.clip_low, high = 1.0 + p.clip_high;
      const double kept = ratio < low ? low : ratio > high ? high : ratio;
      const double open = ratio * adv, shut = kept * adv;
      double l = open <= shut ? -open : -shut;
      double slope = open <= shut ? -open : 0.0;
      if (open != open) l = slope = open;
      double kl = 0.0;
      if (p.ref_logprob != nullptr) {
        const double gap = (double)p.ref_logprob[row] - lp;
        const double rise = expm1(gap);
        kl = rise - gap;
        if (p.kl_coef != 0.0) {
          l += p.kl_coef * kl;
          slope -= p.kl_coef * rise;
        }
      }
      loss = (float)l;
      logprob = (float)lp;
      kl_out = (float)kl;
      coef = token_coef(log2_sum, slope * (double)w * p.inv_t, lp, token);
    }
  }
  p.loss[row] = loss;
  if (p.logprob) p.logprob[row] = logprob;
  if (p.kl) p.kl[row] = kl_out;
  if (p.grad) p.coef[row] = coef;
}

template <typename E>
__device__ void finish_logprobs(const ScoreParams& p, uint32_t row, const RowSum& r,
                                uint32_t lane) {
  if (lane != 0) return;
  const uint32_t token = p.token[row];
  pb_inference_error* at = p.err ? p.err + row : nullptr;
  float logprob = 0.0f, lse = 0.0f, entropy = 0.0f;
  if (token == PB_NO_TOKEN) {
    no_error(at);
  } else {
    bool failed = token >= p.vocab;
    if (failed)
      write_error(at, PB_TOKEN_ID, row, p.vocab, token, PB_FIELD_TOKEN, 0);
    else
      failed = row_failed<E>(p, row, r.bad, r.sum, at);
    if (failed) {
      logprob = lse = entropy = nan32();
    } else {
      no_error(at);
      const double log2_sum = r.shift + log2(r.sum);
      logprob = (float)token_logprob<E>(p, row, token, log2_sum);
      lse = (float)(kLn2 * log2_sum);
      entropy = (float)(kLn2 * (log2(r.sum) - r.moment / r.sum));
    }
  }
  p.logprob[row] = logprob;
  if (p.lse) p.lse[row] = lse;
  if (p.entropy) p.entropy[row] = entropy;
}

template <typename E>
__device__ void finish_distill(const ScoreParams& p, uint32_t row, RowSum r, uint32_t lane) {
  pb_inference_error* at = p.err ? p.err + row : nullptr;
  const float w = p.weight ? p.weight[row] : 1.0f;
  RowCoef coef{};
  coef.state = kRowZero;
  float loss = 0.0f, lse = 0.0f;
  if (w == 0.0f) {
    if (lane == 0) no_error(at);
  } else {
    const bool rest_bucket = p.teacher_lse != nullptr;
    const uint32_t* ids = p.teacher_id + (size_t)row * p.k;
    const float* logits = p.teacher_logit + (size_t)row * p.k;
    // two list entries a lane
    uint32_t id[2];
    double t[2], u[2], pr[2];
    uint32_t bad_id = kNone, bad_logit = kNone, bad_x = kNone;
    double top_t = -__builtin_inf(), top_u = r.sum > 0.0 ? r.shift : -__builtin_inf();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t i = lane + 64u * h;
      id[h] = i < p.k ? ids[i] : kNone;
      t[h] = u[h] = -__builtin_inf();
      if (id[h] == kNone) continue;
      bool bad = id[h] >= p.vocab;
      for (uint32_t j = 0; j < p.k; ++j) bad |= j != i && ids[j] == id[h];
      if (bad) {
        bad_id = i < bad_id ? i : bad_id;
        continue;
      }
      const float tf = logits[i];
      if (!(tf < __builtin_inff())) bad_logit = i < bad_logit ? i : bad_logit;
      t[h] = (double)tf * p.inv_t;
      const float x = E::one(row_ptr<E>(p, row)[id[h]]);
      if (!(x * p.c < kTooBig)) bad_x = id[h] < bad_x ? id[h] : bad_x;
      u[h] = (double)x * (double)p.c;
      top_t = t[h] > top_t ? t[h] : top_t;
      top_u = u[h] > top_u ? u[h] : top_u;
    }
    bad_id = wave_min_word(bad_id);
    bad_logit = wave_min_word(bad_logit);
    bad_x = wave_min_word(bad_x);
    if (rest_bucket && !__builtin_isfinite(p.teacher_lse[row]))
      bad_logit = p.k < bad_logit ? p.k : bad_logit;
    top_t = wave_max_f64(top_t);
    top_u = wave_max_f64(top_u);
    // the student's sum over the listed ids joins the rest's
    double rest = r.sum, whole = r.sum, shift = r.shift;
    if (rest_bucket && top_u > -__builtin_inf()) {
      const double f = r.sum > 0.0 ? exp2(r.shift - top_u) : 0.0;
      double listed = 0.0;
#pragma unroll
      for (int h = 0; h < 2; ++h) listed += u[h] > -__builtin_inf() ? exp2(u[h] - top_u) : 0.0;
      rest = f * r.sum;
      whole = rest + wave_sum_f64(listed);
      shift = top_u;
    }
    const uint32_t bad = bad_x < r.bad ? bad_x : r.bad;
    bool failed = false;
    if (bad_id != kNone) {
      failed = true;
      if (lane == 0)
        write_error(at, PB_TOKEN_ID, row, p.vocab, ids[bad_id], PB_FIELD_TOKEN, bad_id);
    } else if (bad_logit != kNone) {
      failed = true;
      if (lane == 0)
        write_error(at, PB_NONFINITE_INPUT, row, 0,
                    b_of(bad_logit == p.k ? p.teacher_lse[row] : logits[bad_logit]),
                    PB_FIELD_FINITE, bad_logit);
    } else if (bad != kNone || !(whole > 0.0)) {
      failed = true;
      if (lane == 0) row_failed<E>(p, row, bad, whole, at);
    }
    if (failed) {
      loss = lse = nan32();
      coef.state = kRowNan;
    } else {
      if (lane == 0) no_error(at);
      const double log2_sum = shift + log2(whole);
      lse = (float)(kLn2 * log2_sum);
      const bool any = top_t > -__builtin_inf();
      double norm = 0.0, mass = 0.0, l = 0.0;
      if (rest_bucket) {
        norm = (double)p.teacher_lse[row];
      } else if (any) {
        double sum = 0.0;
#pragma unroll
        for (int h = 0; h < 2; ++h) sum += id[h] != kNone ? exp(t[h] - top_t) : 0.0;
        norm = top_t + log(wave_sum_f64(sum));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pr[h] = any && id[h] != kNone ? exp(t[h] - norm) : 0.0;
        mass += pr[h];
        if (pr[h] > 0.0) l += pr[h] * ((t[h] - norm) - kLn2 * (u[h] - log2_sum));
      }
      mass = wave_sum_f64(mass);
      l = wave_sum_f64(l);
      double off = mass;  // what q is multiplied by off the list
      if (rest_bucket && any) {
        const double left = mass < 1.0 ? 1.0 - mass : 0.0;
        if (left > 0.0 && rest > 0.0) {
          l += left * (log(left) - log(rest / whole));
          mass += left;
          off = mass - left * (whole / rest);
        }
      }
      if (any) {
        loss = (float)l;
        const double weight = (double)w * p.inv_t;
        coef.state = weight == weight ? kRowNormal : kRowNan;
        set_factors(coef, log2_sum, weight * off, 0.0);
        coef.norm = norm;
        coef.mass = mass;
        coef.weight = weight;
        coef.token = kNone;
      }
    }
  }
  if (lane == 0) {
    p.loss[row] = loss;
    if (p.lse) p.lse[row] = lse;
    if (p.grad) p.coef[row] = coef;
  }
}

template <typename E>
__global__ __launch_bounds__(256) void finish_kernel(const ScoreParams p) {
  const uint32_t row = blockIdx.x * 4u + (threadIdx.x >> 6), lane = lane_id();
  if (row >= p.rows) return;
  RowSum r{0.0, 0.0, 0.0, kNone};
  if (!row_unread(p, row)) r = join_parts(p, row, lane);
  if (p.mode == kModePolicy)
    finish_policy<E>(p, row, r, lane);
  else if (p.mode == kModeDistill)
    finish_distill<E>(p, row, r, lane);
  else
    finish_logprobs<E>(p, row, r, lane);
}

// ---- preference loss: one workgroup a pair ----

__global__ __launch_bounds__(256) void clear_coef_kernel(const ScoreParams p) {
  const uint32_t row = blockIdx.x * 256u + threadIdx.x;
  if (row < p.rows) p.coef[row].state = kRowUntouched;
}

// A row's log2 sum by one thread.
__device__ __forceinline__ double join_parts_serial(const ScoreParams& p, uint32_t row,
                                                    uint32_t* bad, double* sum) {
  const RowPart* v = p.part + (size_t)row * p.splits;
  float top = -__builtin_inff();
  for (uint32_t i = 0; i < p.splits; ++i)
    if (v[i].sum > 0.0) top = fmaxf(top, v[i].shift);
  double s = 0.0;
  uint32_t b = kNone;
  for (uint32_t i = 0; i < p.splits; ++i) {
    b = v[i].bad < b ? v[i].bad : b;
    if (v[i].sum > 0.0) s += v[i].sum * exp2((double)v[i].shift - (double)top);
  }
  *bad = b;
  *sum = s;
  return (double)top + log2(s);
}

template <typename E>
__global__ __launch_bounds__(256) void pair_kernel(const ScoreParams p) {
  __shared__ double sums[2][4];
  __shared__ uint32_t worst[4];
  __shared__ double slope_at;
  const uint32_t pair = blockIdx.x, lane = lane_id(), wave = threadIdx.x >> 6;
  pb_inference_error* at = p.err ? p.err + pair : nullptr;
  const uint32_t a = p.seq_start[2 * pair], b = p.seq_start[2 * pair + 1],
                 e = p.seq_start[2 * pair + 2];
  // rows outside the first and the last offset have no statistics
  if (a > b || b > e || e > p.rows || a < p.seq_start[0] || e > p.seq_start[2 * p.pairs]) {
    if (threadIdx.x == 0) {
      write_error(at, PB_CAPACITY, pair, p.rows, e > p.rows ? e : b, PB_FIELD_BYTES, 10);
      p.loss[pair] = nan32();
      if (p.logprob) p.logprob[2 * pair] = p.logprob[2 * pair + 1] = nan32();
    }
    return;
  }
  const float w = p.weight ? p.weight[pair] : 1.0f;
  double mine[2] = {0.0, 0.0};
  uint32_t failed = kNone;
  if (w != 0.0f) {
    for (uint32_t row = a + threadIdx.x; row < e; row += 256u) {
      const uint32_t token = p.token[row];
      if (token == PB_NO_TOKEN) continue;
      double lp = 0.0, sum = 0.0;
      uint32_t bad = kNone;
      bool wrong = token >= p.vocab;
      if (!wrong) {
        const double log2_sum = join_parts_serial(p, row, &bad, &sum);
        wrong = bad != kNone || !(sum > 0.0);
        if (!wrong) lp = token_logprob<E>(p, row, token, log2_sum);
      }
      if (wrong) failed = row < failed ? row : failed;
      mine[row < b ? 0 : 1] += lp;
    }
  }
  const double c = wave_sum_f64(mine[0]), d = wave_sum_f64(mine[1]);
  const uint32_t f = wave_min_word(failed);
  if (lane == 0) {
    sums[0][wave] = c;
    sums[1][wave] = d;
    worst[wave] = f;
  }
  __syncthreads();
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
        uint32_t bad = kNone;
        double sum = 0.0;
        (void)join_parts_serial(p, first, &bad, &sum);
        row_failed<E>(p, first, bad, sum, at);
      }
      loss = slope = l[0] = l[1] = (double)nan32();
    } else {
      no_error(at);
      if (w != 0.0f) {
        const double rc = p.ref_logprob ? (double)p.ref_logprob[2 * pair] : 0.0;
        const double rr = p.ref_logprob ? (double)p.ref_logprob[2 * pair + 1] : 0.0;
        const double h = p.beta * ((l[0] - rc) - (l[1] - rr));
        // -ln sigma(h) = max(-h, 0) + ln(1 + e^-|h|)
        const double soft = log1p(exp(-fabs(h)));
        loss = (1.0 - p.smoothing) * ((h < 0.0 ? -h : 0.0) + soft) +
               p.smoothing * ((h > 0.0 ? h : 0.0) + soft);
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
      uint32_t bad;
      double sum;
      const double log2_sum = join_parts_serial(p, row, &bad, &sum);
      coef = token_coef(log2_sum, row < b ? slope : -slope,
                        token_logprob<E>(p, row, token, log2_sum), token);
    }
    p.coef[row] = coef;
  }
}

// ---- token_logprobs_grad: coefficients from the forward pass' outputs ----

template <typename E>
__global__ __launch_bounds__(256) void logprobs_coef_kernel(const ScoreParams p) {
  const uint32_t row = blockIdx.x * 256u + threadIdx.x;
  if (row >= p.rows) return;
  const uint32_t token = p.token[row];
  RowCoef r{};
  r.state = kRowZero;
  if (token != PB_NO_TOKEN) {
    const double lse = (double)p.in_lse[row], g = p.grad_logprob ? (double)p.grad_logprob[row] : 0.0,
                 ge = p.grad_entropy ? (double)p.grad_entropy[row] : 0.0;
    const double log2_sum = lse / kLn2, h = p.grad_entropy ? (double)p.in_entropy[row] : 0.0;
    if (token >= p.vocab || !__builtin_isfinite(lse) || g != g || ge != ge || h != h) {
      r.state = kRowNan;
    } else if (g != 0.0 || ge != 0.0) {
      r.state = kRowNormal;
      // g (delta - q) - ge q (ln q + H)
      set_factors(r, log2_sum, (-g - ge * h) * p.inv_t, -ge * p.inv_t);
      const double lp = token_logprob<E>(p, row, token, log2_sum), q = exp(lp);
      r.token = token;
      r.patch = (float)((g * -expm1(lp) - (q > 0.0 ? ge * q * (lp + h) : 0.0)) * p.inv_t);
    }
  }
  p.coef[row] = r;
}

// ---- gradient pass ----

template <typename E, bool kBeta>
__device__ __forceinline__ float grad_of(float x, float c, const RowCoef& r) {
  const float a = fmaf(x, c, -r.shift);
  const float e = exp2_hw(a);
  if (!kBeta) return e * r.alpha;
  return e * fmaf(fmaxf(a, -1000.0f), r.beta, r.alpha);
}

template <typename E, bool kBeta>
__global__ __launch_bounds__(kGradThreads) void grad_kernel(const ScoreParams p) {
  using Raw = typename E::Raw;
  constexpr uint32_t kPer = E::kPer;
  const uint32_t row = blockIdx.x / p.grad_splits, split = blockIdx.x - row * p.grad_splits;
  const RowCoef r = p.coef[row];
  if (r.state == kRowUntouched) return;
  const uint32_t lo = split * p.grad_span;
  const uint32_t hi = p.vocab - lo < p.grad_span ? p.vocab : lo + p.grad_span;
  const Raw* in = row_ptr<E>(p, row) + lo;
  Raw* out = static_cast<Raw*>(p.grad) + (size_t)row * p.grad_ld + lo;
  const uint32_t n = hi - lo, whole = n / kPer;
  if (r.state != kRowNormal) {
    const float f = r.state == kRowZero ? 0.0f : nan32();
    float fill[kPer];
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e) fill[e] = f;
    const uint4 v = E::pack(fill);
    for (uint32_t i = threadIdx.x; i < whole; i += kGradThreads)
      store_chunk<E>(out + (size_t)i * kPer, v);
    for (uint32_t j = whole * kPer + threadIdx.x; j < n; j += kGradThreads) out[j] = E::raw(f);
    return;
  }
  // The listed ids' gradients come from scalars in 64 bits; their logits are
  // read before anything is written, since the gradient may go in their place.
  uint32_t at = kNone;
  float patch = 0.0f;
  if (p.mode == kModeDistill) {
    if (threadIdx.x < p.k) {
      const size_t entry = (size_t)row * p.k + threadIdx.x;
      const uint32_t id = p.teacher_id[entry];
      if (id >= lo && id < hi) {
        at = id - lo;
        const double u = (double)E::one(in[at]) * (double)p.c;
        const double q = exp2(u - r.log2_sum);
        const double t = exp((double)p.teacher_logit[entry] * p.inv_t - r.norm);
        patch = (float)(r.weight * (r.mass * q - t));
      }
    }
    __syncthreads();
  } else if (threadIdx.x == 0 && r.token >= lo && r.token < hi) {
    at = r.token - lo;
    patch = r.patch;
  }
  for (uint32_t i = threadIdx.x; i < whole; i += kGradThreads) {
    const uint4 v = load_chunk<E>(in + (size_t)i * kPer);
    float g[kPer];
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e) g[e] = grad_of<E, kBeta>(E::get(v, e), p.c, r);
    store_chunk<E>(out + (size_t)i * kPer, E::pack(g));
  }
  for (uint32_t j = whole * kPer + threadIdx.x; j < n; j += kGradThreads)
    out[j] = E::raw(grad_of<E, kBeta>(E::one(in[j]), p.c, r));
  __syncthreads();  // the patches come after the stores they replace
  if (at != kNone) out[at] = E::raw(patch);
}

// ---- top logits ----
// A row's tiles of 2^tile_shift consecutive logits: the k largest logits lie in
// the k tiles of the largest maxima (the lower tile first among equal ones),
// since each of those holds a logit that ranks before any logit of another tile.

template <typename E>
__global__ __launch_bounds__(kStatsThreads) void top_tiles_kernel(const ScoreParams p) {
  __shared__ BlockSum l;
  __shared__ uint32_t words[kMaxTiles];
  const uint32_t row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits;
  const uint32_t lo = split * p.span;
  const uint32_t hi = p.vocab - lo < p.span ? p.vocab : lo + p.span;
  const uint32_t tiles = (hi - lo + (1u << p.tile_shift) - 1u) >> p.tile_shift;
  for (uint32_t i = threadIdx.x; i < tiles; i += kStatsThreads) words[i] = 0;
  __syncthreads();
  const PartScan<E, false, false> scan{row_ptr<E>(p, row), nullptr, lo, hi, p.c};
  uint32_t bad;
  const Acc s = scan.run(&bad);
  scan.each([&](const float (&x)[E::kPer], uint32_t at) {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < E::kPer; ++e) m = fmaxf(m, x[e]);
    atomicMax(&words[at >> p.tile_shift], ord_of(b_of(m)));
  });
  const RowPart out = block_sum<kStatsThreads>(s, bad, l);
  if (threadIdx.x == 0) p.part[(size_t)row * p.splits + split] = out;
  const uint32_t all = (p.vocab + (1u << p.tile_shift) - 1u) >> p.tile_shift;
  uint32_t* to = p.tiles + (size_t)row * all + (lo >> p.tile_shift);
  for (uint32_t i = threadIdx.x; i < tiles; i += kStatsThreads) to[i] = words[i];
}

constexpr uint32_t kMaxCandidates = 1024;

struct SelectShared {
  uint32_t words[kMaxTiles];
  uint64_t keys[kMaxCandidates];
  uint32_t list[PB_TOP_LOGITS_MAX];
  uint32_t counts[kSelectThreads / 64];
  uint32_t n_list, n_keys;
  uint64_t best[kSelectThreads / 64];
};

// Larger key: larger value, then lower id.
__device__ __forceinline__ uint64_t value_key(float x, uint32_t id) {
  return ((uint64_t)ord_of(b_of(x)) << 32) | (0xffffffffu - id);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t ord = (uint32_t)(key >> 32);
  return f_of((ord & 0x80000000u) ? (ord & 0x7fffffffu) : ~ord);
}

// The k best of a row from its tiles' words in LDS; every thread.
template <typename E>
__device__ void select_top(const ScoreParams& p, uint32_t row, uint32_t tiles, SelectShared& l) {
  const uint32_t lane = lane_id(), wave = threadIdx.x >> 6;
  const uint32_t want = p.k < tiles ? p.k : tiles;
  constexpr uint32_t kWaves = kSelectThreads / 64;
  // the want-th largest word, bit by bit
  uint32_t level = 0;
  for (uint32_t bit = 0x80000000u; bit != 0; bit >>= 1) {
    const uint32_t trial = level | bit;
    uint32_t n = 0;
    for (uint32_t i = threadIdx.x; i < tiles; i += kSelectThreads) n += l.words[i] >= trial ? 1u : 0u;
    const uint32_t sum = wave_sum_word(n);
    if (lane == 0) l.counts[wave] = sum;
    __syncthreads();
    uint32_t total = 0;
    for (uint32_t w = 0; w < kWaves; ++w) total += l.counts[w];
    if (total >= want) level = trial;
    __syncthreads();
  }
  // the tiles above it, and the first of those at it
  if (threadIdx.x == 0) l.n_keys = 0;
  if (wave == 0) {
    uint32_t above = 0;
    for (uint32_t i = lane; i < tiles; i += 64u) above += l.words[i] > level ? 1u : 0u;
    above = wave_sum_word(above);
    uint32_t n = 0, equal = want - above;
    for (uint32_t base = 0; base < tiles; base += 64u) {
      const uint32_t i = base + lane;
      const uint32_t v = i < tiles ? l.words[i] : 0u;
      const bool at = i < tiles && v == level;
      const uint64_t same = __ballot(at);
      const bool take = (i < tiles && v > level) || (at && lanes_below(same) < equal);
      const uint64_t taken = __ballot(take);
      if (take) l.list[n + lanes_below(taken)] = i;
      n += (uint32_t)__popcll((unsigned long long)taken);
      const uint32_t got = (uint32_t)__popcll((unsigned long long)same);
      equal -= got < equal ? got : equal;
    }
    if (lane == 0) l.n_list = n;
  }
  __syncthreads();
  const typename E::Raw* x = row_ptr<E>(p, row);
  const uint32_t size = 1u << p.tile_shift, n_list = l.n_list;
  const uint32_t total = n_list << p.tile_shift;
  uint32_t* out_id = p.top_id + (size_t)row * p.k;
  float* out_value = p.top_value + (size_t)row * p.k;
  for (uint32_t i = threadIdx.x; i < total; i += kSelectThreads) {
    const uint32_t id = (l.list[i >> p.tile_shift] << p.tile_shift) + (i & (size - 1u));
    if (id >= p.vocab) continue;
    const uint64_t key = value_key(E::one(x[id]), id);
    if ((uint32_t)(key >> 32) >= level) {
      const uint32_t at = atomicAdd(&l.n_keys, 1u);
      if (at < kMaxCandidates) l.keys[at] = key;
    }
  }
  __syncthreads();
  const uint32_t n = l.n_keys;
  if (tiles > p.k && n <= kMaxCandidates) {
    // a key's rank is the number of keys above it (no two are equal)
    for (uint32_t i = threadIdx.x; i < n; i += kSelectThreads) {
      const uint64_t key = l.keys[i];
      uint32_t rank = 0;
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
    for (uint32_t i = threadIdx.x; i < total; i += kSelectThreads) {
      const uint32_t id = (l.list[i >> p.tile_shift] << p.tile_shift) + (i & (size - 1u));
      if (id >= p.vocab) continue;
      const uint64_t key = value_key(E::one(x[id]), id);
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

template <typename E>
__global__ __launch_bounds__(kSelectThreads) void top_select_kernel(const ScoreParams p) {
  __shared__ SelectShared l;
  __shared__ bool failed;
  const uint32_t row = blockIdx.x;
  const uint32_t tiles = (p.vocab + (1u << p.tile_shift) - 1u) >> p.tile_shift;
  for (uint32_t i = threadIdx.x; i < tiles; i += kSelectThreads)
    l.words[i] = p.tiles[(size_t)row * tiles + i];
  if (threadIdx.x < 64) {
    const RowSum r = join_parts(p, row, threadIdx.x);
    if (threadIdx.x == 0) {
      pb_inference_error* at = p.err ? p.err + row : nullptr;
      failed = row_failed<E>(p, row, r.bad, r.sum, at);
      if (!failed) no_error(at);
      if (p.lse) p.lse[row] = failed ? nan32() : (float)(kLn2 * (r.shift + log2(r.sum)));
    }
  }
  __syncthreads();
  if (failed) {
    for (uint32_t i = threadIdx.x; i < p.k; i += kSelectThreads) {
      p.top_id[(size_t)row * p.k + i] = PB_NO_TOKEN;
      p.top_value[(size_t)row * p.k + i] = nan32();
    }
    return;
  }
  select_top<E>(p, row, tiles, l);
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1u) / b; }

// Workgroups that a pass over few rows is cut into.
constexpr uint32_t kTargetGroups = 1024;

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
  (void)dtype;
  p->tile_shift = tile_shift_of(p->vocab);
  const uint32_t tile = 1u << p->tile_shift;
  if (p->rows == 0) return;
  uint32_t splits = kTargetGroups / p->rows;
  const uint32_t most = ceil_div(p->vocab, 4096u);
  if (splits > most) splits = most;
  if (splits > kMaxSplits) splits = kMaxSplits;
  if (splits < 1) splits = 1;
  const uint32_t least = ceil_div(p->vocab, kMaxSpan);
  if (splits < least) splits = least;
  p->span = ceil_div(ceil_div(p->vocab, splits), tile) * tile;
  p->splits = ceil_div(p->vocab, p->span);
  uint32_t grad_splits = ceil_div(2u * kTargetGroups, p->rows);
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
  p->tiles = reinterpret_cast<uint32_t*>(base + l.tiles);
}

namespace {

template <typename E, bool kEntropy, bool kTail>
void launch_stats(const ScoreParams& p, hipStream_t stream) {
  const size_t marks = kTail ? ((size_t)p.span / 32 + 2) * 4 : 0;
  stats_kernel<E, kEntropy, kTail><<<p.rows * p.splits, kStatsThreads, marks, stream>>>(p);
}

template <typename E>
struct Launch {
  static void logprobs(const ScoreParams& p, hipStream_t s) {
    if (p.entropy)
      launch_stats<E, true, false>(p, s);
    else
      launch_stats<E, false, false>(p, s);
    finish_kernel<E><<<ceil_div(p.rows, 4), 256, 0, s>>>(p);
  }
  static void grad(const ScoreParams& p, bool beta, hipStream_t s) {
    const uint32_t groups = p.rows * p.grad_splits;
    if (beta)
      grad_kernel<E, true><<<groups, kGradThreads, 0, s>>>(p);
    else
      grad_kernel<E, false><<<groups, kGradThreads, 0, s>>>(p);
  }
  static void logprobs_grad(const ScoreParams& p, hipStream_t s) {
    logprobs_coef_kernel<E><<<ceil_div(p.rows, 256), 256, 0, s>>>(p);
    grad(p, p.grad_entropy != nullptr, s);
  }
  static void top(const ScoreParams& p, hipStream_t s) {
    top_tiles_kernel<E><<<p.rows * p.splits, kStatsThreads, 0, s>>>(p);
    top_select_kernel<E><<<p.rows, kSelectThreads, 0, s>>>(p);
  }
  static void row_loss(const ScoreParams& p, hipStream_t s) {
    if (p.teacher_lse)
      launch_stats<E, false, true>(p, s);
    else
      launch_stats<E, false, false>(p, s);
    finish_kernel<E><<<ceil_div(p.rows, 4), 256, 0, s>>>(p);
    if (p.grad) grad(p, false, s);
  }
  static void preference(const ScoreParams& p, hipStream_t s) {
    if (p.rows == 0) {  // pairs of empty sequences
      pair_kernel<E><<<p.pairs, 256, 0, s>>>(p);
      return;
    }
    launch_stats<E, false, false>(p, s);
    if (p.grad) clear_coef_kernel<<<ceil_div(p.rows, 256), 256, 0, s>>>(p);
    pair_kernel<E><<<p.pairs, 256, 0, s>>>(p);
    if (p.grad) grad(p, false, s);
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
