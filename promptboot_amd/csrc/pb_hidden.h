// pb_hidden.h -- launch parameters of the operators on hidden-state rows.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "pbsample.h"

namespace pb {

struct EmbedParams {
  const void* table;
  size_t table_ld;
  uint32_t vocab, cols, rows;
  const uint32_t* token;
  double scale;
  void* out;
  size_t out_ld;
  pb_inference_error* err;
};

// The sort by token: rows that one workgroup sorts, rows of a workgroup of more, bits of a
// pass.  Rows of one part of a sum.
constexpr uint32_t kSortRows = 16384;
constexpr uint32_t kSortTile = 4096;
constexpr uint32_t kSortBits = 9;
constexpr uint32_t kSumRows = 16;

struct EmbedGradParams {
  const void* grad;
  size_t grad_ld;
  uint32_t vocab, cols, rows;
  const uint32_t* token;
  float scale;
  bool accumulate;
  void* table;
  size_t table_ld;
  // workspace: two sets of (id, row) pairs that the passes of the sort go between, the
  // passes' counts [tile][digit], the parts' sums [part][2][cols], and the parts whose last
  // token goes on in the next one, in two lists: how many each has, then those of fewer parts
  // from the front and the others from the back
  uint32_t* id[2];
  uint32_t* row[2];
  uint32_t* count;
  float* part;
  uint32_t* cross;
};

struct NormParams {
  const void* x;
  size_t x_ld;
  uint32_t rows, cols;
  const void* residual;
  size_t residual_ld;
  const void* weight;
  uint32_t weight_dtype;
  bool norm;  // false: rounding to 8 bits alone
  double eps;
  void* sum;
  size_t sum_ld;
  void* out;
  uint32_t out_dtype;
  size_t out_ld;
  int8_t* q;
  size_t q_ld;
  float* scale;
  pb_inference_error* err;
};

struct NormGradParams {
  const void* h;
  size_t h_ld;
  uint32_t rows, cols;
  const void* weight;
  uint32_t weight_dtype;
  double eps;
  const void* grad;
  uint32_t grad_dtype;
  size_t grad_ld;
  const void* grad_sum;
  size_t grad_sum_ld;
  void* grad_h;
  size_t grad_h_ld;
  float* grad_weight;
  bool accumulate;
  uint32_t groups;  // workgroups, each with a row of `part`
  float* part;      // workspace: groups x cols
};

struct Int8Params {
  const int8_t* q;
  size_t q_ld;
  const float* scale;
  uint32_t rows, cols, channels;
  const int8_t* weight;
  size_t weight_ld;
  const float* weight_scale;
  const float* bias;
  void* out;
  size_t out_ld;
};

// Workspace of either gradient on up to `rows` rows of up to `cols` columns, and where a
// call's parts of it lie.
size_t hidden_workspace_bytes(uint32_t rows, size_t cols);
void place_embed_grad(void* work, EmbedGradParams* p);
void place_norm_grad(void* work, NormGradParams* p);
size_t embed_grad_bytes(uint32_t rows, size_t cols);
size_t norm_grad_bytes(uint32_t rows, size_t cols);

hipError_t launch_embed(const EmbedParams& p, uint32_t dtype, uint32_t out_dtype,
                        hipStream_t stream);
hipError_t launch_embed_grad(const EmbedGradParams& p, uint32_t dtype, uint32_t table_dtype,
                             hipStream_t stream);
hipError_t launch_norm(const NormParams& p, uint32_t dtype, hipStream_t stream);
hipError_t launch_norm_grad(const NormGradParams& p, uint32_t dtype, hipStream_t stream);
hipError_t launch_int8(const Int8Params& p, uint32_t out_dtype, hipStream_t stream);

}  // namespace pb
