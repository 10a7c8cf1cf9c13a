// pb_scores.h -- launch parameters of the scores and losses of logits rows.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "pbsample.h"

namespace pb {

enum ScoreMode : uint32_t {
  kModeLogprobs = 0,
  kModeTop = 1,
  kModeDistill = 2,
  kModePolicy = 3,
  kModePreference = 4,
};

// What one workgroup of the statistics pass leaves about its part of a row:
// sum 2^(x c - shift) = sum (over the ids off the teacher's list, for the
// distillation with a rest bucket) and sum 2^(x c - shift) (x c - shift) =
// moment (entropy only).  bad: the first NaN or +inf of the part, or kNone.
struct RowPart {
  float shift;
  uint32_t bad;
  double sum;
  double moment;
};

// What the gradient pass needs of a row: with a = x c - shift, element j gets
// 2^a (alpha + beta a), the token's element `patch`, and a listed id of the
// distillation weight (mass q - p).
enum CoefState : uint32_t { kRowUntouched = 0, kRowZero = 1, kRowNormal = 2, kRowNan = 3 };
struct RowCoef {
  float shift, alpha, beta;
  uint32_t state;
  uint32_t token;
  float patch;
  float own_shift;  // of a listed id's q; off the list `shift` is the rest's
  double inv;       // q = inv 2^(x c - own_shift)
  double norm;      // the teacher's log-sum-exp
  double mass;      // the teacher's mass, its rest bucket included
  double weight;    // weight / T
};
// The same room between the preference loss' statistics and its pairs' pass: a
// row's log-sum, what is wrong with it (bad as in RowPart) and ln q[token].  A row
// that no pair takes stays untouched.
struct PairRow {
  float shift;
  uint32_t bad;
  uint32_t failed;
  uint32_t state;   // kRowUntouched, where RowCoef has it
  double log2_own;  // log2 sum 2^(x c - shift)
  double logprob;
};
static_assert(offsetof(PairRow, state) == offsetof(RowCoef, state), "a row's state has one place");

struct ScoreParams {
  const void* logits;
  size_t ld;
  uint32_t vocab;
  uint32_t rows;
  uint32_t mode;
  float c;       // log2(e) / T
  double inv_t;  // 1 / T
  const uint32_t* token;
  const float* weight;  // rows (pairs for the preference loss), or null

  // outputs of a row (or pair)
  float* logprob;
  float* lse;
  float* lse_low;  // what binary32 leaves out of lse
  float* entropy;
  float* loss;
  float* kl;
  pb_inference_error* err;
  void* grad;
  size_t grad_ld;

  // token_logprobs_grad
  const float* in_lse;
  const float* in_lse_low;
  const float* in_entropy;
  const float* grad_logprob;
  const float* grad_entropy;

  // top logits and distillation
  uint32_t k;
  uint32_t* top_id;
  float* top_value;
  const uint32_t* teacher_id;
  const float* teacher_logit;
  const float* teacher_lse;

  // policy loss
  const float* old_logprob;
  const float* advantage;
  const float* ref_logprob;  // and preference: per sequence
  double clip_low, clip_high, kl_coef;

  // preference loss
  const uint32_t* seq_start;
  uint32_t pairs;
  double beta, smoothing;

  // plan and workspace
  uint32_t splits;       // workgroups per row of the statistics pass
  uint32_t span;         // elements per split, a multiple of a tile
  uint32_t grad_splits;  // workgroups per row of the gradient pass
  uint32_t grad_span;
  uint32_t fused;        // threads of a workgroup that takes a whole row, or 0
  uint32_t keep;         // the statistics pass leaves the logits in the caches
  uint32_t tile_shift;   // log2 of the elements of a top-logits tile
  uint32_t* ticket;      // rows: parts of the row that are done, 0 between calls
  RowPart* part;         // rows x splits
  RowCoef* coef;         // rows
  uint32_t* tiles;       // rows x tile count: a top-logits tile's largest value, ordered
  uint32_t* sequence;    // rows: the preference loss' sequence of each, in the tiles' place
};

// Terms of a sum in 32 bits: a thread takes no more logits of a row, and what the
// threads of a row have is joined in 64 bits.
constexpr uint32_t kMaxTerms = 768;
// So the largest part of a row of one workgroup (256 threads) of the statistics
// pass; its marks of the teacher's ids (a bit each) take 24 KB of LDS.
constexpr uint32_t kMaxSpan = 256 * kMaxTerms;
// Top-logits tiles of one row: their words take 16 KB of LDS.
constexpr uint32_t kMaxTiles = 4096;
constexpr uint32_t kMaxSplits = 64;

// Fills splits, span, grad_splits, grad_span and tile_shift.
void plan_scores(uint32_t dtype, ScoreParams* p);
// Workspace of any call on up to `rows` rows of up to `vocab` ids, and where a
// call's parts of it lie.
size_t scores_workspace_bytes(uint32_t rows, size_t vocab);
void place_scores(void* work, ScoreParams* p);

hipError_t launch_token_logprobs(const ScoreParams& p, uint32_t dtype, hipStream_t stream);
hipError_t launch_token_logprobs_grad(const ScoreParams& p, uint32_t dtype, hipStream_t stream);
hipError_t launch_top_logits(const ScoreParams& p, uint32_t dtype, hipStream_t stream);
// Distillation and policy loss.
hipError_t launch_row_loss(const ScoreParams& p, uint32_t dtype, hipStream_t stream);
hipError_t launch_preference(const ScoreParams& p, uint32_t dtype, hipStream_t stream);

}  // namespace pb
