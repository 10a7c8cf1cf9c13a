// pb_scores_api.cpp -- C ABI of the scores and losses of logits rows
// (include/pbsample.h): argument checks, the plan of a call and its workspace.
// Nothing here allocates but pb_context_reserve_scores.
#include <hip/hip_runtime.h>
#include <math.h>

#include <initializer_list>

#include "pb_host.h"
#include "pb_internal.h"
#include "pb_scores.h"
#include "pbsample.h"

using pb::clear_error;
using pb::device_error;
using pb::DeviceGuard;
using pb::ScoreParams;
using pb::set_error;

namespace {

uint32_t refuse(pb_inference_error* err, uint32_t status, uint64_t needed, uint64_t available,
                uint32_t kind, uint32_t sub) {
  set_error(err, status, PB_DOMAIN_LOGITS, needed, available, kind, sub);
  return status;
}

// Limits of rows and ids, shared with the reservation.
uint32_t check_sizes(size_t vocab, uint32_t rows, pb_inference_error* err) {
  if (vocab == 0 || vocab > PB_SCORE_MAX_VOCAB)
    return refuse(err, PB_CAPACITY, PB_SCORE_MAX_VOCAB, vocab, PB_FIELD_LOGITS, 2);
  if (rows > PB_SCORE_MAX_ROWS)
    return refuse(err, PB_CAPACITY, PB_SCORE_MAX_ROWS, rows, PB_FIELD_BYTES, 8);
  return PB_OK;
}

struct Rows {
  const void* logits;
  uint32_t dtype;
  size_t vocab, ld;
  uint32_t rows;
  double temperature;
  const void* grad;  // or null
  size_t grad_ld;
};

bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// Whether a gradient that is not in place of the logits shares an element with
// them.  Rows of one stride may lie between each other (the columns of one buffer,
// or every other row of it); of two strides the ranges they span are compared.
bool overlap(const Rows& r, size_t size) {
  const uintptr_t a = (uintptr_t)r.logits, b = (uintptr_t)r.grad;
  const uintptr_t a_end = a + ((size_t)(r.rows - 1) * r.ld + r.vocab) * size;
  const uintptr_t b_end = b + ((size_t)(r.rows - 1) * r.grad_ld + r.vocab) * size;
  if (a >= b_end || b >= a_end) return false;
  if (r.ld != r.grad_ld) return true;
  // row i of the logits and row i - k of the gradient start `m` elements apart, row i
  // and row i - k - 1 ld - m
  const int64_t d = ((int64_t)b - (int64_t)a) / (int64_t)size, ld = (int64_t)r.ld;
  const int64_t k = d >= 0 ? d / ld : -((-d + ld - 1) / ld), m = d - k * ld;
  const int64_t rows = r.rows, vocab = (int64_t)r.vocab;
  return (k < rows && -k < rows && m < vocab) ||
         (k + 1 < rows && -(k + 1) < rows && ld - m < vocab);
}

// The checks that every call makes of its rows.  `missing`: a required
// pointer is null.
uint32_t check_rows(const Rows& r, bool missing, pb_inference_error* err) {
  clear_error(err);
  const uint32_t st = check_sizes(r.vocab, r.rows, err);
  if (st != PB_OK) return st;
  if (r.dtype > PB_BF16) return refuse(err, PB_STATE, PB_BF16, r.dtype, PB_FIELD_NONE, 1);
  if (r.ld < r.vocab) return refuse(err, PB_CAPACITY, r.vocab, r.ld, PB_FIELD_LOGITS, 1);
  if (r.grad != nullptr && r.grad_ld < r.vocab)
    return refuse(err, PB_CAPACITY, r.vocab, r.grad_ld, PB_FIELD_LOGITS, 3);
  if (!(r.temperature >= 0.01 && r.temperature <= 100.0))
    return refuse(err, PB_ARITHMETIC, 0, 0, PB_FIELD_FINITE, 0);
  const size_t size = r.dtype == PB_F32 ? 4 : 2;
  if (!aligned(r.logits, size) || !aligned(r.grad, size))
    return refuse(err, PB_ALIGNMENT, size, 0, PB_FIELD_ALIGNMENT, 0);
  // addresses of a row's end stay below 2^62 bytes
  if (r.ld >> 40 || r.grad_ld >> 40)
    return refuse(err, PB_CAPACITY, (uint64_t)1 << 40, r.ld, PB_FIELD_LOGITS, 4);
  if (r.rows != 0 && missing) return refuse(err, PB_CAPACITY, 1, 0, PB_FIELD_BYTES, 3);
  if (r.rows != 0 && r.grad != nullptr && !(r.grad == r.logits && r.grad_ld == r.ld) &&
      overlap(r, size))
    return refuse(err, PB_STATE, 0, 0, PB_FIELD_BYTES, 9);
  return PB_OK;
}

ScoreParams params_of(const Rows& r, uint32_t mode) {
  ScoreParams p{};
  p.logits = r.logits;
  p.ld = r.ld;
  p.vocab = (uint32_t)r.vocab;
  p.rows = r.rows;
  p.mode = mode;
  p.c = (float)(1.4426950408889634073599246810019 / r.temperature);
  p.inv_t = 1.0 / r.temperature;
  p.grad = const_cast<void*>(r.grad);
  p.grad_ld = r.grad_ld;
  return p;
}

using Launch = hipError_t (*)(const ScoreParams&, uint32_t, hipStream_t);

uint32_t enqueue(pb_context* ctx, ScoreParams& p, uint32_t dtype, Launch launch, void* stream,
                 pb_inference_error* err) {
  if (ctx == nullptr) {
    set_error(err, PB_STATE, PB_DOMAIN_NONE, 1, 0, PB_FIELD_NONE, 0);
    return PB_STATE;
  }
  pb::ScoresAccess work = pb::scores_access(ctx);
  const size_t need = pb::scores_workspace_bytes(p.rows, p.vocab);
  if (need > work.bytes) {
    set_error(err, PB_CAPACITY, PB_DOMAIN_NONE, need, work.bytes, PB_FIELD_BYTES, 6);
    return PB_CAPACITY;
  }
  if (p.rows > work.rows) {
    set_error(err, PB_CAPACITY, PB_DOMAIN_NONE, p.rows, work.rows, PB_FIELD_BYTES, 6);
    return PB_CAPACITY;
  }
  pb::plan_scores(dtype, &p);
  pb::place_scores(work.work, &p);
  p.ticket = work.ticket;
  DeviceGuard guard(work.device);
  const hipError_t e = launch(p, dtype, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? PB_OK : device_error(err, e);
}

bool words(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (!aligned(p, 4)) return false;
  return true;
}

}  // namespace

extern "C" {

uint32_t pb_context_reserve_scores(pb_context* ctx, uint32_t rows, size_t vocab,
                                   pb_inference_error* err) {
  clear_error(err);
  const uint32_t st = check_sizes(vocab, rows, err);
  if (st != PB_OK) return st;
  if (ctx == nullptr) {
    set_error(err, PB_STATE, PB_DOMAIN_NONE, 1, 0, PB_FIELD_NONE, 0);
    return PB_STATE;
  }
  const hipError_t e = pb::scores_reserve(ctx, rows, pb::scores_workspace_bytes(rows, vocab));
  return e == hipSuccess ? PB_OK : device_error(err, e);
}

uint32_t pb_token_logprobs_wide(pb_context* ctx, const void* d_logits, uint32_t dtype,
                                size_t vocab, size_t ld, uint32_t rows, double temperature,
                                const uint32_t* d_token, float* d_logprob, float* d_lse,
                                float* d_lse_low, float* d_entropy, pb_inference_error* d_err,
                                void* stream, pb_inference_error* err) {
  const Rows r{d_logits, dtype, vocab, ld, rows, temperature, nullptr, 0};
  const uint32_t st =
      check_rows(r, !d_logits || !d_token || !d_logprob || (d_lse_low && !d_lse), err);
  if (st != PB_OK || rows == 0) return st;
  if (!words({d_token, d_logprob, d_lse, d_lse_low, d_entropy}) || !aligned(d_err, 8))
    return refuse(err, PB_ALIGNMENT, 8, 0, PB_FIELD_ALIGNMENT, 1);
  ScoreParams p = params_of(r, pb::kModeLogprobs);
  p.token = d_token;
  p.logprob = d_logprob;
  p.lse = d_lse;
  p.lse_low = d_lse_low;
  p.entropy = d_entropy;
  p.err = d_err;
  return enqueue(ctx, p, dtype, pb::launch_token_logprobs, stream, err);
}

uint32_t pb_token_logprobs(pb_context* ctx, const void* d_logits, uint32_t dtype, size_t vocab,
                           size_t ld, uint32_t rows, double temperature, const uint32_t* d_token,
                           float* d_logprob, float* d_lse, float* d_entropy,
                           pb_inference_error* d_err, void* stream, pb_inference_error* err) {
  return pb_token_logprobs_wide(ctx, d_logits, dtype, vocab, ld, rows, temperature, d_token,
                                d_logprob, d_lse, nullptr, d_entropy, d_err, stream, err);
}

uint32_t pb_token_logprobs_wide_grad(pb_context* ctx, const void* d_logits, uint32_t dtype,
                                     size_t vocab, size_t ld, uint32_t rows, double temperature,
                                     const uint32_t* d_token, const float* d_lse,
                                     const float* d_lse_low, const float* d_entropy,
                                     const float* d_grad_logprob, const float* d_grad_entropy,
                                     void* d_grad, size_t grad_ld, void* stream,
                                     pb_inference_error* err) {
  const Rows r{d_logits, dtype, vocab, ld, rows, temperature, d_grad, grad_ld};
  const uint32_t st = check_rows(
      r, !d_logits || !d_token || !d_lse || !d_grad || (d_grad_entropy && !d_entropy), err);
  if (st != PB_OK || rows == 0) return st;
  if (!words({d_token, d_lse, d_lse_low, d_entropy, d_grad_logprob, d_grad_entropy}))
    return refuse(err, PB_ALIGNMENT, 4, 0, PB_FIELD_ALIGNMENT, 1);
  ScoreParams p = params_of(r, pb::kModeLogprobs);
  p.token = d_token;
  p.in_lse = d_lse;
  p.in_lse_low = d_lse_low;
  p.in_entropy = d_entropy;
  p.grad_logprob = d_grad_logprob;
  p.grad_entropy = d_grad_entropy;
  return enqueue(ctx, p, dtype, pb::launch_token_logprobs_grad, stream, err);
}

uint32_t pb_token_logprobs_grad(pb_context* ctx, const void* d_logits, uint32_t dtype,
                                size_t vocab, size_t ld, uint32_t rows, double temperature,
                                const uint32_t* d_token, const float* d_lse,
                                const float* d_entropy, const float* d_grad_logprob,
                                const float* d_grad_entropy, void* d_grad, size_t grad_ld,
                                void* stream, pb_inference_error* err) {
  return pb_token_logprobs_wide_grad(ctx, d_logits, dtype, vocab, ld, rows, temperature, d_token,
                                     d_lse, nullptr, d_entropy, d_grad_logprob, d_grad_entropy,
                                     d_grad, grad_ld, stream, err);
}

uint32_t pb_top_logits(pb_context* ctx, const void* d_logits, uint32_t dtype, size_t vocab,
                       size_t ld, uint32_t rows, uint32_t k, double temperature, uint32_t* d_token,
                       float* d_value, float* d_lse, pb_inference_error* d_err, void* stream,
                       pb_inference_error* err) {
  const Rows r{d_logits, dtype, vocab, ld, rows, temperature, nullptr, 0};
  const uint32_t st = check_rows(r, !d_logits || !d_token || !d_value, err);
  if (st != PB_OK) return st;
  const size_t most = vocab < PB_TOP_LOGITS_MAX ? vocab : PB_TOP_LOGITS_MAX;
  if (k == 0 || k > most) return refuse(err, PB_CAPACITY, most, k, PB_FIELD_TOKEN, 1);
  if (rows == 0) return PB_OK;
  if (!words({d_token, d_value, d_lse}) || !aligned(d_err, 8))
    return refuse(err, PB_ALIGNMENT, 8, 0, PB_FIELD_ALIGNMENT, 1);
  ScoreParams p = params_of(r, pb::kModeTop);
  p.k = k;
  p.top_id = d_token;
  p.top_value = d_value;
  p.lse = d_lse;
  p.err = d_err;
  return enqueue(ctx, p, dtype, pb::launch_top_logits, stream, err);
}

uint32_t pb_distill_loss(pb_context* ctx, const void* d_logits, uint32_t dtype, size_t vocab,
                         size_t ld, uint32_t rows, double temperature, uint32_t k,
                         const uint32_t* d_teacher_id, const float* d_teacher_logit,
                         const float* d_teacher_lse, const float* d_weight, float* d_loss,
                         float* d_lse, void* d_grad, size_t grad_ld, pb_inference_error* d_err,
                         void* stream, pb_inference_error* err) {
  const Rows r{d_logits, dtype, vocab, ld, rows, temperature, d_grad, grad_ld};
  const uint32_t st =
      check_rows(r, !d_logits || !d_teacher_id || !d_teacher_logit || !d_loss, err);
  if (st != PB_OK) return st;
  if (k == 0 || k > PB_TOP_LOGITS_MAX)
    return refuse(err, PB_CAPACITY, PB_TOP_LOGITS_MAX, k, PB_FIELD_TOKEN, 1);
  if (rows == 0) return PB_OK;
  if (!words({d_teacher_id, d_teacher_logit, d_teacher_lse, d_weight, d_loss, d_lse}) ||
      !aligned(d_err, 8))
    return refuse(err, PB_ALIGNMENT, 8, 0, PB_FIELD_ALIGNMENT, 1);
  ScoreParams p = params_of(r, pb::kModeDistill);
  p.k = k;
  p.teacher_id = d_teacher_id;
  p.teacher_logit = d_teacher_logit;
  p.teacher_lse = d_teacher_lse;
  p.weight = d_weight;
  p.loss = d_loss;
  p.lse = d_lse;
  p.err = d_err;
  return enqueue(ctx, p, dtype, pb::launch_row_loss, stream, err);
}

uint32_t pb_policy_loss(pb_context* ctx, const void* d_logits, uint32_t dtype, size_t vocab,
                        size_t ld, uint32_t rows, double temperature, const uint32_t* d_token,
                        const float* d_old_logprob, const float* d_advantage,
                        const float* d_ref_logprob, const float* d_weight, double clip_low,
                        double clip_high, double kl_coef, float* d_loss, float* d_logprob,
                        float* d_kl, void* d_grad, size_t grad_ld, pb_inference_error* d_err,
                        void* stream, pb_inference_error* err) {
  const Rows r{d_logits, dtype, vocab, ld, rows, temperature, d_grad, grad_ld};
  const uint32_t st = check_rows(
      r, !d_logits || !d_token || !d_old_logprob || !d_advantage || !d_loss, err);
  if (st != PB_OK) return st;
  if (!(clip_low >= 0.0 && clip_low <= 1.0) || !(clip_high >= 0.0) || !isfinite(kl_coef))
    return refuse(err, PB_ARITHMETIC, 0, 0, PB_FIELD_FINITE, 1);
  if (kl_coef != 0.0 && d_ref_logprob == nullptr)
    return refuse(err, PB_CAPACITY, 1, 0, PB_FIELD_BYTES, 3);
  if (rows == 0) return PB_OK;
  if (!words({d_token, d_old_logprob, d_advantage, d_ref_logprob, d_weight, d_loss, d_logprob,
              d_kl}) ||
      !aligned(d_err, 8))
    return refuse(err, PB_ALIGNMENT, 8, 0, PB_FIELD_ALIGNMENT, 1);
  ScoreParams p = params_of(r, pb::kModePolicy);
  p.token = d_token;
  p.old_logprob = d_old_logprob;
  p.advantage = d_advantage;
  p.ref_logprob = d_ref_logprob;
  p.weight = d_weight;
  p.clip_low = clip_low;
  p.clip_high = clip_high;
  p.kl_coef = kl_coef;
  p.loss = d_loss;
  p.logprob = d_logprob;
  p.kl = d_kl;
  p.err = d_err;
  return enqueue(ctx, p, dtype, pb::launch_row_loss, stream, err);
}

uint32_t pb_preference_loss(pb_context* ctx, const void* d_logits, uint32_t dtype, size_t vocab,
                            size_t ld, uint32_t rows, double temperature, const uint32_t* d_token,
                            const uint32_t* d_seq_start, uint32_t pairs,
                            const float* d_ref_logprob, const float* d_weight, double beta,
                            double label_smoothing, float* d_loss, float* d_logprob, void* d_grad,
                            size_t grad_ld, pb_inference_error* d_err, void* stream,
                            pb_inference_error* err) {
  const Rows r{d_logits, dtype, vocab, ld, rows, temperature, d_grad, grad_ld};
  const uint32_t st = check_rows(r, !d_logits || !d_token, err);
  if (st != PB_OK) return st;
  if (pairs > PB_SCORE_MAX_ROWS)
    return refuse(err, PB_CAPACITY, PB_SCORE_MAX_ROWS, pairs, PB_FIELD_BYTES, 8);
  if (pairs != 0 && (!d_seq_start || !d_loss))
    return refuse(err, PB_CAPACITY, 1, 0, PB_FIELD_BYTES, 3);
  if (!isfinite(beta) || !(label_smoothing >= 0.0 && label_smoothing <= 1.0))
    return refuse(err, PB_ARITHMETIC, 0, 0, PB_FIELD_FINITE, 1);
  if (!words({d_token, d_seq_start, d_ref_logprob, d_weight, d_loss, d_logprob}) ||
      !aligned(d_err, 8))
    return refuse(err, PB_ALIGNMENT, 8, 0, PB_FIELD_ALIGNMENT, 1);
  if (pairs == 0) return PB_OK;
  // no rows: pairs of empty sequences still have their losses
  ScoreParams p = params_of(r, pb::kModePreference);
  p.token = d_token;
  p.seq_start = d_seq_start;
  p.pairs = pairs;
  p.ref_logprob = d_ref_logprob;
  p.weight = d_weight;
  p.beta = beta;
  p.smoothing = label_smoothing;
  p.loss = d_loss;
  p.logprob = d_logprob;
  p.err = d_err;
  return enqueue(ctx, p, dtype, pb::launch_preference, stream, err);
}

}  // extern "C"
