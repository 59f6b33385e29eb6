// pk_block_norm_abi.cpp - C ABI of the norms around a block
// (include/pk_block_norm.h): descriptor checks and the launch.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "pk_abi_internal.h"
#include "pk_block_norm.h"
#include "pk_internal.h"
#include "pk_strided.h"

using namespace pk_abi;

struct pk_block_norm_op {
  pk_abi::CtxRef ctx;
  std::string label;
  uint32_t rows = 0;
  pk::BlockNormArgs args{};
  bool destroyed = false;
};

namespace {

const char* bn_label(const char* label) { return label ? label : "block-norm"; }

// A matrix of the descriptor as bytes (stride 0: packed rows).
Region matrix(const void* p, uint64_t rows, uint32_t channels, uint32_t stride, uint64_t elem) {
  return {p, rows, channels * elem, (stride ? stride : channels) * elem};
}

int check_matrix(const char* label, const char* what, const Region& r, uint64_t bytes, uint64_t elem) {
  if (r.stride < r.row_bytes)
    return fail(PK_RANGE_ERROR, "%s %s stride must be at least the channels", label, what);
  if (!aligned(r.data, elem))
    return fail(PK_INVALID_ARGUMENT, "%s %s must be aligned to its elements", label, what);
  if (bytes < r.extent())
    return fail(PK_RANGE_ERROR, "%s %s needs %llu bytes; arena slice has %llu", label, what,
                (unsigned long long)r.extent(), (unsigned long long)bytes);
  return PK_OK;
}

int check_vector(const char* label, const char* what, const float* p, uint64_t bytes, uint32_t channels) {
  if (bytes != (uint64_t)channels * 4u)
    return fail(PK_INVALID_ARGUMENT, "%s %s must be float32 [%u], %llu bytes", label, what, channels,
                (unsigned long long)channels * 4u);
  if (!aligned(p, 4)) return fail(PK_INVALID_ARGUMENT, "%s %s must be aligned to its elements", label, what);
  return PK_OK;
}

int validate_block_norm(const pk_block_norm_desc* d) {
  if (!d) return fail(PK_INVALID_ARGUMENT, "block norm descriptor is null");
  if (d->struct_size != sizeof(pk_block_norm_desc))
    return fail(PK_INVALID_ARGUMENT, "pk_block_norm_desc.struct_size mismatch");
  const char* label = bn_label(d->label);
  if (d->precision != PK_PRECISION_F16 && d->precision != PK_PRECISION_F32)
    return fail(PK_INVALID_ARGUMENT, "%s has an unsupported precision %d", label, d->precision);
  if (d->kind != PK_NORM_LAYER && d->kind != PK_NORM_RMS)
    return fail(PK_INVALID_ARGUMENT, "%s has an unsupported norm kind %d", label, d->kind);
  if (d->rows == 0 || d->rows > PK_BLOCK_NORM_MAX_ROWS || d->channels == 0 ||
      d->channels > PK_BLOCK_NORM_MAX_CHANNELS)
    return fail(PK_RANGE_ERROR, "Invalid block norm shape for %s", label);
  if (d->has_epsilon && !(d->epsilon >= 0.0f && std::isfinite(d->epsilon)))
    return fail(PK_INVALID_ARGUMENT, "%s epsilon must be a finite number of at least 0", label);
  if (d->has_residual_scale && !std::isfinite(d->residual_scale))
    return fail(PK_INVALID_ARGUMENT, "%s residual scale must be finite", label);
  if (!d->input || !d->output) return fail(PK_INVALID_ARGUMENT, "%s needs an input and an output", label);
  if ((d->beta && !d->gamma) || (d->next_beta && !d->next_gamma))
    return fail(PK_INVALID_ARGUMENT, "%s has a beta without its gamma", label);
  if ((d->next_gamma != nullptr) != (d->next_output != nullptr))
    return fail(PK_INVALID_ARGUMENT, "%s needs next gamma and next output together", label);
  const uint64_t elem = d->precision == PK_PRECISION_F16 ? 2u : 4u;
  const uint64_t gates = !d->gate ? 0u : d->gate_rows ? ((uint64_t)d->rows + d->gate_rows - 1u) / d->gate_rows : 1u;
  const Region in = matrix(d->input, d->rows, d->channels, d->input_stride, elem),
               gate = matrix(d->gate, gates, d->channels, d->gate_stride, elem),
               res = matrix(d->residual, d->rows, d->channels, d->residual_stride, elem),
               out = matrix(d->output, d->rows, d->channels, d->output_stride, elem),
               next = matrix(d->next_output, d->rows, d->channels, d->next_output_stride, elem);
  if (int s = check_matrix(label, "input", in, d->input_bytes, elem)) return s;
  if (d->gate)
    if (int s = check_matrix(label, "gate", gate, d->gate_bytes, elem)) return s;
  if (d->residual)
    if (int s = check_matrix(label, "residual", res, d->residual_bytes, elem)) return s;
  if (int s = check_matrix(label, "output", out, d->output_bytes, elem)) return s;
  if (d->next_output)
    if (int s = check_matrix(label, "next output", next, d->next_output_bytes, elem)) return s;
  const struct {
    const char* name;
    const float* p;
    uint64_t bytes;
  } vectors[4] = {{"gamma", d->gamma, d->gamma_bytes},
                  {"beta", d->beta, d->beta_bytes},
                  {"next gamma", d->next_gamma, d->next_gamma_bytes},
                  {"next beta", d->next_beta, d->next_beta_bytes}};
  for (const auto& v : vectors) {
    if (!v.p) continue;
    if (int s = check_vector(label, v.name, v.p, v.bytes, d->channels)) return s;
  }
  // Each element of a row is read and written by one lane, which reads first:
  // an output may lie on the input's or the residual's own elements, and on
  // nothing else.
  const Region outs[2] = {out, next};
  for (const Region& o : outs) {
    if (!o.data) continue;
    for (const Region& r : {in, res})
      if (overlap(o, r) && !same_rows(o, r))
        return fail(PK_INVALID_ARGUMENT, "%s outputs must be the input or the residual or not overlap them", label);
    if (overlap(o, gate)) return fail(PK_INVALID_ARGUMENT, "%s outputs must not overlap the gate", label);
    for (const auto& v : vectors)
      if (v.p && overlap(o, Region{v.p, 1, v.bytes, v.bytes}))
        return fail(PK_INVALID_ARGUMENT, "%s outputs must not overlap the norms' parameters", label);
  }
  if (overlap(out, next)) return fail(PK_INVALID_ARGUMENT, "%s output and next output must not overlap", label);
  return PK_OK;
}

}  // namespace

extern "C" {

int pk_block_norm_validate(const pk_block_norm_desc* d) { return validate_block_norm(d); }

int pk_block_norm_create(pk_context* ctx, const pk_block_norm_desc* d, pk_block_norm_op** out) try {
  if (int s = check_ctx(ctx)) return s;
  if (!d || !out) return fail(PK_INVALID_ARGUMENT, "block norm descriptor or output is null");
  *out = nullptr;
  if (int s = validate_block_norm(d)) return s;
  std::string label = bn_label(d->label);
  auto* op = new pk_block_norm_op();
  op->ctx = ctx;
  op->label.swap(label);
  op->rows = d->rows;
  const auto stride = [&](uint32_t s) { return (uint64_t)(s ? s : d->channels); };
  pk::BlockNormArgs& a = op->args;
  a.input = d->input;
  a.input_stride = stride(d->input_stride);
  a.gamma = d->gamma;
  a.beta = d->beta;
  a.gate = d->gate;
  a.gate_stride = stride(d->gate_stride);
  a.gate_rows = d->gate_rows;
  a.residual = d->residual;
  a.residual_stride = stride(d->residual_stride);
  a.residual_scale = d->has_residual_scale ? d->residual_scale : 1.0f;
  a.output = d->output;
  a.output_stride = stride(d->output_stride);
  a.next_gamma = d->next_gamma;
  a.next_beta = d->next_beta;
  a.next_output = d->next_output;
  a.next_stride = stride(d->next_output_stride);
  a.rows = d->rows;
  a.channels = d->channels;
  a.rms = d->kind == PK_NORM_RMS;
  a.f16 = d->precision == PK_PRECISION_F16;
  a.epsilon = d->has_epsilon ? d->epsilon : 1e-5f;
  *out = op;
  return ok();
} catch (const std::bad_alloc&) {
  return fail(PK_ALLOCATION_FAILURE, "block norm: out of host memory");
}

int pk_block_norm_enqueue(pk_block_norm_op* op, uint32_t active_rows, void* stream) {
  return pk_block_norm_enqueue_timed(op, active_rows, stream, nullptr, nullptr);
}

int pk_block_norm_enqueue_timed(pk_block_norm_op* op, uint32_t active_rows, void* stream, void* start_event,
                                void* end_event) {
  if (!op) return fail(PK_INVALID_ARGUMENT, "block norm op is null");
  if (op->destroyed) return fail(PK_DESTROYED, "%s was destroyed", op->label.c_str());
  if (active_rows > op->rows)
    return fail(PK_RANGE_ERROR, "%s active rows must be in [1, %u]", op->label.c_str(), op->rows);
  pk::BlockNormArgs args = op->args;
  if (active_rows) args.rows = active_rows;
  DeviceScope device(op->ctx->device);
  PK_HIP(device.status(), "hipSetDevice");
  PK_HIP(pk::launch_block_norm(args, stream_or_default(op->ctx, stream), static_cast<hipEvent_t>(start_event),
                               static_cast<hipEvent_t>(end_event)),
         "block norm launch");
  return ok();
}

int pk_block_norm_destroy(pk_block_norm_op* op) {
  if (op) op->destroyed = true;
  return ok();
}

int pk_block_norm_release(pk_block_norm_op* op) {
  delete op;
  return ok();
}

}  // extern "C"
