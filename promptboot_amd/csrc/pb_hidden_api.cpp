// pb_hidden_api.cpp -- C ABI of the operators on hidden-state rows
// (include/pbsample.h): argument checks and the calls' workspace.
// Nothing here allocates but the reservations.
#include <hip/hip_runtime.h>
#include <math.h>

#include <exception>
#include <initializer_list>

#include "pb_hidden.h"
#include "pb_host.h"
#include "pb_internal.h"
#include "pbsample.h"

using pb::clear_error;
using pb::device_error;
using pb::DeviceGuard;
using pb::set_error;

namespace {

uint32_t refuse(pb_inference_error* err, uint32_t status, uint64_t needed, uint64_t available,
                uint32_t kind, uint32_t sub) {
  set_error(err, status, PB_DOMAIN_NONE, needed, available, kind, sub);
  return status;
}

size_t size_of(uint32_t dtype) { return dtype == PB_F32 ? 4 : 2; }

// A buffer of `rows` rows of `cols` elements of `size` bytes; one of no address is not there.
struct Rows {
  const void* at;
  size_t rows, cols, ld, size;
};

bool overlap(const Rows& a, const Rows& b) {
  if (a.at == nullptr || b.at == nullptr || a.rows == 0 || b.rows == 0) return false;
  auto bytes = [](const Rows& r) {
    return pb::ByteRows{r.at, (int64_t)r.rows, (int64_t)(r.cols * r.size),
                        (int64_t)(r.ld * r.size)};
  };
  return pb::share_a_byte(bytes(a), bytes(b));
}

bool same_place(const Rows& a, const Rows& b) {
  return a.at == b.at && a.size == b.size && (a.ld == b.ld || a.rows == 1);
}

bool aligned(const Rows& r) { return ((uintptr_t)r.at & (r.size - 1)) == 0; }

uint32_t check_sizes(size_t rows, size_t cols, pb_inference_error* err) {
  if (cols == 0 || cols > PB_HIDDEN_MAX_COLS)
    return refuse(err, PB_CAPACITY, PB_HIDDEN_MAX_COLS, cols, PB_FIELD_BYTES, 2);
  if (rows > PB_HIDDEN_MAX_ROWS)
    return refuse(err, PB_CAPACITY, PB_HIDDEN_MAX_ROWS, rows, PB_FIELD_BYTES, 8);
  return PB_OK;
}

uint32_t check_channels(size_t n, pb_inference_error* err) {
  if (n == 0 || n > PB_SCORE_MAX_VOCAB)
    return refuse(err, PB_CAPACITY, PB_SCORE_MAX_VOCAB, n, PB_FIELD_LOGITS, 2);
  return PB_OK;
}

uint32_t check_types(std::initializer_list<uint32_t> types, pb_inference_error* err) {
  for (uint32_t t : types)
    if (t > PB_BF16) return refuse(err, PB_STATE, PB_BF16, t, PB_FIELD_NONE, 1);
  return PB_OK;
}

// binary32 holds 1 / sqrt(eps), what a row of zeros is multiplied by.
uint32_t check_eps(double eps, pb_inference_error* err) {
  if (!(eps >= 1e-75 && isfinite(eps))) return refuse(err, PB_ARITHMETIC, 0, 0, PB_FIELD_FINITE, 0);
  return PB_OK;
}

// Distances and addresses of the buffers that are there.  Addresses of a buffer's end stay
// below 2^62 bytes: at most 2^22 rows of 2^38 elements of 4 bytes.
uint32_t check_buffers(std::initializer_list<Rows> all, pb_inference_error* err) {
  for (const Rows& r : all) {
    if (r.at == nullptr) continue;
    if (r.ld < r.cols) return refuse(err, PB_CAPACITY, r.cols, r.ld, PB_FIELD_BYTES, 1);
    if (r.ld >> 38) return refuse(err, PB_CAPACITY, (uint64_t)1 << 38, r.ld, PB_FIELD_BYTES, 4);
    if (!aligned(r)) return refuse(err, PB_ALIGNMENT, r.size, 0, PB_FIELD_ALIGNMENT, 0);
  }
  return PB_OK;
}

// Outputs share nothing with each other and with the inputs, but for the inputs in whose
// place an output may lie: bit i of its mask for input i.
struct Output {
  Rows r;
  uint32_t in_place;
};
uint32_t check_overlap(std::initializer_list<Rows> inputs, std::initializer_list<Output> outputs,
                       pb_inference_error* err) {
  const Output* const end = outputs.end();
  for (const Output* o = outputs.begin(); o != end; ++o) {
    uint32_t i = 0;
    for (const Rows& in : inputs) {
      const bool allowed = (o->in_place >> i++ & 1u) != 0 && same_place(o->r, in);
      if (!allowed && overlap(o->r, in)) return refuse(err, PB_STATE, 0, 0, PB_FIELD_BYTES, 9);
    }
    for (const Output* other = o + 1; other != end; ++other)
      if (overlap(o->r, other->r)) return refuse(err, PB_STATE, 0, 0, PB_FIELD_BYTES, 9);
  }
  return PB_OK;
}

uint32_t missing(pb_inference_error* err) {
  return refuse(err, PB_CAPACITY, 1, 0, PB_FIELD_BYTES, 3);
}
uint32_t no_context(pb_inference_error* err) {
  return refuse(err, PB_STATE, 1, 0, PB_FIELD_NONE, 0);
}

Rows one_row(const void* at, size_t n, size_t size) { return Rows{at, at ? 1u : 0u, n, n, size}; }
// Records start at a word of 8 bytes.
Rows records(const pb_inference_error* at, uint32_t rows) { return Rows{at, rows, 6, 6, 8}; }

uint32_t finish(hipError_t e, pb_inference_error* err) {
  return e == hipSuccess ? PB_OK : device_error(err, e);
}

// A workspace of what `bytes_of` says, or where it grows by doubling of twice the one it
// outgrows, up to what the largest call of either gradient needs.
uint32_t reserve(pb_context* ctx, uint32_t rows, size_t cols,
                 size_t (*bytes_of)(uint32_t rows, size_t cols), bool doubling,
                 pb_inference_error* err) {
  clear_error(err);
  const uint32_t st = check_sizes(rows, cols, err);
  if (st != PB_OK) return st;
  if (ctx == nullptr) return no_context(err);
  const size_t bytes = rows != 0 ? bytes_of(rows, cols) : 0;
  const size_t most =
      doubling ? pb::hidden_workspace_bytes(PB_HIDDEN_MAX_ROWS, PB_HIDDEN_MAX_COLS) : 0;
  try {  // the list of outgrown workspaces grows
    return finish(pb::hidden_reserve(ctx, bytes, most), err);
  } catch (const std::exception&) {
    return device_error(err, hipErrorOutOfMemory);
  }
}

// What pb_norm_rows and pb_quantize_rows have in common, behind their own checks.
uint32_t norm_rows(pb_context* ctx, const pb::NormParams& p, uint32_t dtype, bool required,
                   void* stream, pb_inference_error* err) {
  const size_t size = size_of(dtype);
  const Rows x{p.x, p.rows, p.cols, p.x_ld, size};
  const Rows residual{p.residual, p.rows, p.cols, p.residual_ld, size};
  const Rows weight = one_row(p.weight, p.cols, size_of(p.weight_dtype));
  const Rows sum{p.sum, p.rows, p.cols, p.sum_ld, size};
  const Rows out{p.out, p.rows, p.cols, p.out_ld, size_of(p.out_dtype)};
  const Rows q{p.q, p.rows, p.cols, p.q_ld, 1};
  const Rows scale = one_row(p.scale, p.rows, 4), rec = records(p.err, p.rows);
  uint32_t st = check_buffers({x, residual, weight, sum, out, q, scale, rec}, err);
  if (st != PB_OK) return st;
  if (p.rows == 0) return PB_OK;
  if (!required) return missing(err);
  // (the type of an output in an input's place is the rows')
  const uint32_t out_place = p.out_dtype == dtype ? 3u : 0u;
  st = check_overlap({x, residual, weight},
                     {{sum, 3u}, {out, out_place}, {q, 0}, {scale, 0}, {rec, 0}}, err);
  if (st != PB_OK) return st;
  if (ctx == nullptr) return no_context(err);
  DeviceGuard guard(pb::context_device(ctx));
  return finish(pb::launch_norm(p, dtype, static_cast<hipStream_t>(stream)), err);
}

}  // namespace

extern "C" {

uint32_t pb_context_reserve_hidden(pb_context* ctx, uint32_t rows, size_t cols,
                                   pb_inference_error* err) {
  return reserve(ctx, rows, cols, pb::hidden_workspace_bytes, false, err);
}

uint32_t pb_context_reserve_embed_grad(pb_context* ctx, uint32_t rows, size_t cols,
                                       pb_inference_error* err) {
  return reserve(ctx, rows, cols, pb::embed_grad_bytes, true, err);
}

uint32_t pb_context_reserve_norm_grad(pb_context* ctx, uint32_t rows, size_t cols,
                                      pb_inference_error* err) {
  return reserve(ctx, rows, cols, pb::norm_grad_bytes, true, err);
}

size_t pb_context_hidden_bytes(pb_context* ctx) {
  return ctx ? pb::hidden_access(ctx).bytes : 0;
}

uint32_t pb_embed_rows(pb_context* ctx, const void* d_table, uint32_t dtype, size_t vocab,
                       size_t cols, size_t table_ld, uint32_t rows, const uint32_t* d_token,
                       double scale, void* d_out, uint32_t out_dtype, size_t out_ld,
                       pb_inference_error* d_err, void* stream, pb_inference_error* err) {
  clear_error(err);
  uint32_t st = check_sizes(rows, cols, err);
  if (st != PB_OK || (st = check_channels(vocab, err)) != PB_OK) return st;
  if ((st = check_types({dtype, out_dtype}, err)) != PB_OK) return st;
  if (!isfinite(scale)) return refuse(err, PB_ARITHMETIC, 0, 0, PB_FIELD_FINITE, 0);
  const Rows table{d_table, vocab, cols, table_ld, size_of(dtype)};
  const Rows token = one_row(d_token, rows, 4), rec = records(d_err, rows);
  const Rows out{d_out, rows, cols, out_ld, size_of(out_dtype)};
  if ((st = check_buffers({table, token, out, rec}, err)) != PB_OK) return st;
  if (rows == 0) return PB_OK;
  if (!d_table || !d_token || !d_out) return missing(err);
  if ((st = check_overlap({table, token}, {{out, 0}, {rec, 0}}, err)) != PB_OK) return st;
  if (ctx == nullptr) return no_context(err);
  const pb::EmbedParams p{d_table, table_ld, (uint32_t)vocab, (uint32_t)cols, rows, d_token,
                          scale, d_out, out_ld, d_err};
  DeviceGuard guard(pb::context_device(ctx));
  return finish(pb::launch_embed(p, dtype, out_dtype, static_cast<hipStream_t>(stream)), err);
}

uint32_t pb_embed_rows_grad(pb_context* ctx, const void* d_grad, uint32_t dtype, size_t vocab,
                            size_t cols, size_t grad_ld, uint32_t rows, const uint32_t* d_token,
                            double scale, uint32_t accumulate, void* d_table_grad,
                            uint32_t table_dtype, size_t table_ld, void* stream,
                            pb_inference_error* err) {
  clear_error(err);
  uint32_t st = check_sizes(rows, cols, err);
  if (st != PB_OK || (st = check_channels(vocab, err)) != PB_OK) return st;
  if ((st = check_types({dtype, table_dtype}, err)) != PB_OK) return st;
  if (!isfinite((float)scale)) return refuse(err, PB_ARITHMETIC, 0, 0, PB_FIELD_FINITE, 0);
  const Rows grad{d_grad, rows, cols, grad_ld, size_of(dtype)};
  const Rows token = one_row(d_token, rows, 4);
  const Rows table{d_table_grad, vocab, cols, table_ld, size_of(table_dtype)};
  if ((st = check_buffers({grad, token, table}, err)) != PB_OK) return st;
  // no rows: a gradient that is not added to is zeros all the same
  if (rows == 0 && accumulate) return PB_OK;
  if (!d_table_grad || (rows != 0 && (!d_grad || !d_token))) return missing(err);
  if ((st = check_overlap({grad, token}, {{table, 0}}, err)) != PB_OK) return st;
  if (ctx == nullptr) return no_context(err);
  pb::HiddenAccess work = pb::hidden_access(ctx);
  const size_t need = rows != 0 ? pb::embed_grad_bytes(rows, cols) : 0;
  if (need > work.bytes) return refuse(err, PB_CAPACITY, need, work.bytes, PB_FIELD_BYTES, 6);
  pb::EmbedGradParams p{};
  p.grad = d_grad;
  p.grad_ld = grad_ld;
  p.vocab = (uint32_t)vocab;
  p.cols = (uint32_t)cols;
  p.rows = rows;
  p.token = d_token;
  p.scale = (float)scale;
  p.accumulate = accumulate != 0;
  p.table = d_table_grad;
  p.table_ld = table_ld;
  pb::place_embed_grad(work.work, &p);
  DeviceGuard guard(work.device);
  return finish(pb::launch_embed_grad(p, dtype, table_dtype, static_cast<hipStream_t>(stream)),
                err);
}

uint32_t pb_norm_rows(pb_context* ctx, const void* d_x, uint32_t dtype, size_t cols, size_t x_ld,
                      uint32_t rows, const void* d_residual, size_t residual_ld,
                      const void* d_weight, uint32_t weight_dtype, double eps, void* d_sum,
                      size_t sum_ld, void* d_out, uint32_t out_dtype, size_t out_ld, int8_t* d_q,
                      size_t q_ld, float* d_scale, pb_inference_error* d_err, void* stream,
                      pb_inference_error* err) {
  clear_error(err);
  uint32_t st = check_sizes(rows, cols, err);
  if (st != PB_OK || (st = check_types({dtype, weight_dtype, out_dtype}, err)) != PB_OK) return st;
  if ((st = check_eps(eps, err)) != PB_OK) return st;
  const pb::NormParams p{d_x,  x_ld,   rows,      (uint32_t)cols, d_residual, residual_ld,
                         d_weight, weight_dtype, true, eps,     d_sum,      sum_ld,
                         d_out, out_dtype, out_ld, d_q,          q_ld,       d_scale, d_err};
  const bool required = d_x && (d_out || d_q) && (d_q != nullptr) == (d_scale != nullptr);
  return norm_rows(ctx, p, dtype, required, stream, err);
}

uint32_t pb_quantize_rows(pb_context* ctx, const void* d_x, uint32_t dtype, size_t cols,
                          size_t x_ld, uint32_t rows, int8_t* d_q, size_t q_ld, float* d_scale,
                          pb_inference_error* d_err, void* stream, pb_inference_error* err) {
  clear_error(err);
  uint32_t st = check_sizes(rows, cols, err);
  if (st != PB_OK || (st = check_types({dtype}, err)) != PB_OK) return st;
  const pb::NormParams p{d_x, x_ld, rows, (uint32_t)cols, nullptr, 0, nullptr, PB_F32, false, 0.0,
                         nullptr, 0, nullptr, PB_F32, 0, d_q, q_ld, d_scale, d_err};
  return norm_rows(ctx, p, dtype, d_x && d_q && d_scale, stream, err);
}

uint32_t pb_norm_rows_grad(pb_context* ctx, const void* d_h, uint32_t dtype, size_t cols,
                           size_t h_ld, uint32_t rows, const void* d_weight,
                           uint32_t weight_dtype, double eps, const void* d_grad,
                           uint32_t grad_dtype, size_t grad_ld, const void* d_grad_sum,
                           size_t grad_sum_ld, void* d_grad_h, size_t grad_h_ld,
                           float* d_grad_weight, uint32_t accumulate, void* stream,
                           pb_inference_error* err) {
  clear_error(err);
  uint32_t st = check_sizes(rows, cols, err);
  if (st != PB_OK || (st = check_types({dtype, weight_dtype, grad_dtype}, err)) != PB_OK)
    return st;
  if ((st = check_eps(eps, err)) != PB_OK) return st;
  const size_t size = size_of(dtype);
  const Rows h{d_h, rows, cols, h_ld, size}, grad{d_grad, rows, cols, grad_ld, size_of(grad_dtype)};
  const Rows grad_sum{d_grad_sum, rows, cols, grad_sum_ld, size};
  const Rows weight = one_row(d_weight, cols, size_of(weight_dtype));
  const Rows grad_h{d_grad_h, rows, cols, grad_h_ld, size};
  const Rows grad_weight = one_row(d_grad_weight, cols, 4);
  st = check_buffers({h, grad, grad_sum, weight, grad_h, grad_weight}, err);
  if (st != PB_OK) return st;
  // no rows: a weight's gradient that is not added to is zeros all the same
  if (rows == 0 && (accumulate || !d_grad_weight)) return PB_OK;
  if ((rows != 0 && (!d_h || !d_grad)) || (!d_grad_h && !d_grad_weight)) return missing(err);
  // (the type of an output in an input's place is the rows')
  const uint32_t place = 1u | (grad_dtype == dtype ? 2u : 0u) | 4u;
  st = check_overlap({h, grad, grad_sum, weight}, {{grad_h, place}, {grad_weight, 0}}, err);
  if (st != PB_OK) return st;
  if (ctx == nullptr) return no_context(err);
  pb::HiddenAccess work = pb::hidden_access(ctx);
  const size_t need = d_grad_weight ? pb::norm_grad_bytes(rows, cols) : 0;
  if (need > work.bytes) return refuse(err, PB_CAPACITY, need, work.bytes, PB_FIELD_BYTES, 6);
  pb::NormGradParams p{};
  p.h = d_h;
  p.h_ld = h_ld;
  p.rows = rows;
  p.cols = (uint32_t)cols;
  p.weight = d_weight;
  p.weight_dtype = weight_dtype;
  p.eps = eps;
  p.grad = d_grad;
  p.grad_dtype = grad_dtype;
  p.grad_ld = grad_ld;
  p.grad_sum = d_grad_sum;
  p.grad_sum_ld = grad_sum_ld;
  p.grad_h = d_grad_h;
  p.grad_h_ld = grad_h_ld;
  p.grad_weight = d_grad_weight;
  p.accumulate = accumulate != 0;
  pb::place_norm_grad(work.work, &p);
  DeviceGuard guard(work.device);
  return finish(pb::launch_norm_grad(p, dtype, static_cast<hipStream_t>(stream)), err);
}

uint32_t pb_int8_matmul(pb_context* ctx, const int8_t* d_q, size_t q_ld, const float* d_scale,
                        uint32_t rows, size_t cols, const int8_t* d_weight, size_t weight_ld,
                        const float* d_weight_scale, size_t channels, const float* d_bias,
                        void* d_out, uint32_t out_dtype, size_t out_ld, void* stream,
                        pb_inference_error* err) {
  clear_error(err);
  uint32_t st = check_sizes(rows, cols, err);
  if (st != PB_OK || (st = check_channels(channels, err)) != PB_OK) return st;
  if ((st = check_types({out_dtype}, err)) != PB_OK) return st;
  const Rows q{d_q, rows, cols, q_ld, 1}, weight{d_weight, channels, cols, weight_ld, 1};
  const Rows scale = one_row(d_scale, rows, 4), bias = one_row(d_bias, channels, 4);
  const Rows weight_scale = one_row(d_weight_scale, channels, 4);
  const Rows out{d_out, rows, channels, out_ld, size_of(out_dtype)};
  st = check_buffers({q, weight, scale, weight_scale, bias, out}, err);
  if (st != PB_OK) return st;
  if (rows == 0) return PB_OK;
  if (!d_q || !d_scale || !d_weight || !d_weight_scale || !d_out) return missing(err);
  st = check_overlap({q, weight, scale, weight_scale, bias}, {{out, 0}}, err);
  if (st != PB_OK) return st;
  if (ctx == nullptr) return no_context(err);
  const pb::Int8Params p{d_q, q_ld, d_scale, rows, (uint32_t)cols, (uint32_t)channels, d_weight,
                         weight_ld, d_weight_scale, d_bias, d_out, out_ld};
  DeviceGuard guard(pb::context_device(ctx));
  return finish(pb::launch_int8(p, out_dtype, static_cast<hipStream_t>(stream)), err);
}

}  // extern "C"
