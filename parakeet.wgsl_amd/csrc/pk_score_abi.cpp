// pk_score_abi.cpp - C ABI of token scores (include/pk_score.h): descriptor
// checks and the launch.
#include <hip/hip_runtime.h>

#include <string>

#include "pk_abi_internal.h"
#include "pk_internal.h"
#include "pk_score.h"
#include "pk_strided.h"

using namespace pk_abi;

struct pk_score_op {
  pk_abi::CtxRef ctx;
  std::string label;
  uint32_t rows = 0;
  pk::ScoreArgs args{};
  void* workspace = nullptr;
  bool destroyed = false;
};

namespace {

const char* score_label(const char* label) { return label ? label : "token-scores"; }

int validate_score(const pk_score_desc* d) {
  if (!d) return fail(PK_INVALID_ARGUMENT, "token score descriptor is null");
  if (d->struct_size != sizeof(pk_score_desc))
    return fail(PK_INVALID_ARGUMENT, "pk_score_desc.struct_size mismatch");
  const char* label = score_label(d->label);
  if (d->precision != PK_PRECISION_F16 && d->precision != PK_PRECISION_F32)
    return fail(PK_INVALID_ARGUMENT, "%s has an unsupported precision %d", label, d->precision);
  if (d->rows == 0 || d->rows > PK_SCORE_MAX_ROWS || d->columns == 0 || d->columns > PK_SCORE_MAX_COLUMNS)
    return fail(PK_RANGE_ERROR, "Invalid token score shape for %s", label);
  if (d->row_stride && d->row_stride < d->columns)
    return fail(PK_RANGE_ERROR, "%s row stride must be at least the columns", label);
  if (d->alternatives > PK_SCORE_MAX_ALTERNATIVES)
    return fail(PK_RANGE_ERROR, "%s alternatives must be in [0, %u]", label, PK_SCORE_MAX_ALTERNATIVES);
  if (d->has_temperature && !(d->temperature >= 0x1p-20f && d->temperature <= 0x1p20f))
    return fail(PK_RANGE_ERROR, "%s temperature must be in [2^-20, 2^20]", label);
  if (!d->logits) return fail(PK_INVALID_ARGUMENT, "%s needs logits", label);
  if ((d->tokens != nullptr) != (d->log_probs != nullptr))
    return fail(PK_INVALID_ARGUMENT, "%s needs tokens and log probs together", label);
  if ((d->alternatives != 0) != (d->top_tokens != nullptr) || (d->alternatives != 0) != (d->top_log_probs != nullptr))
    return fail(PK_INVALID_ARGUMENT, "%s needs top tokens and top log probs with alternatives, and only then", label);
  if (!d->log_probs && !d->entropies && !d->alternatives)
    return fail(PK_INVALID_ARGUMENT, "%s has no outputs", label);
  const uint64_t elem = d->precision == PK_PRECISION_F16 ? 2u : 4u;
  const uint64_t stride = d->row_stride ? d->row_stride : d->columns;
  const Region logits{d->logits, d->rows, d->columns * elem, stride * elem};
  if (!aligned(d->logits, elem)) return fail(PK_INVALID_ARGUMENT, "%s logits must be aligned to their elements", label);
  if (d->logits_bytes < logits.extent())
    return fail(PK_RANGE_ERROR, "%s logits needs %llu bytes; arena slice has %llu", label,
                (unsigned long long)logits.extent(), (unsigned long long)d->logits_bytes);
  const uint64_t flat = (uint64_t)d->rows * 4u, top = flat * d->alternatives;
  const struct {
    const char* name;
    const void* p;
    uint64_t have, need;
  } slices[5] = {{"tokens", d->tokens, d->tokens_bytes, flat},
                 {"log probs", d->log_probs, d->log_probs_bytes, flat},
                 {"entropies", d->entropies, d->entropies_bytes, flat},
                 {"top tokens", d->top_tokens, d->top_tokens_bytes, top},
                 {"top log probs", d->top_log_probs, d->top_log_probs_bytes, top}};
  for (const auto& s : slices) {
    if (!s.p) continue;
    if (!aligned(s.p, 4)) return fail(PK_INVALID_ARGUMENT, "%s %s must be aligned to its elements", label, s.name);
    if (s.have < s.need)
      return fail(PK_RANGE_ERROR, "%s %s needs %llu bytes; arena slice has %llu", label, s.name,
                  (unsigned long long)s.need, (unsigned long long)s.have);
  }
  for (int i = 1; i < 5; ++i) {  // the outputs, against the logits and every slice before
    if (!slices[i].p) continue;
    const Region out{slices[i].p, 1, slices[i].need, slices[i].need};
    bool shared = overlap(out, Region{d->logits, 1, logits.extent(), logits.extent()});
    for (int j = 0; j < i; ++j) shared = shared || overlap(out, Region{slices[j].p, 1, slices[j].need, slices[j].need});
    if (shared)
      return fail(PK_INVALID_ARGUMENT, "%s outputs must not overlap each other or the inputs", label);
  }
  return PK_OK;
}

}  // namespace

extern "C" {

int pk_score_validate(const pk_score_desc* d) { return validate_score(d); }

int pk_score_create(pk_context* ctx, const pk_score_desc* d, pk_score_op** out) try {
  if (int s = check_ctx(ctx)) return s;
  if (!d || !out) return fail(PK_INVALID_ARGUMENT, "token score descriptor or output is null");
  *out = nullptr;
  if (int s = validate_score(d)) return s;
  std::string label = score_label(d->label);
  pk::ScoreArgs a{};
  a.logits = d->logits;
  a.stride = d->row_stride ? d->row_stride : d->columns;
  a.tokens = d->tokens;
  a.log_probs = d->log_probs;
  a.entropies = d->entropies;
  a.top_tokens = d->top_tokens;
  a.top_log_probs = d->top_log_probs;
  a.rows = d->rows;
  a.columns = d->columns;
  a.alternatives = d->alternatives;
  a.inverse_temperature = d->has_temperature ? 1.0f / d->temperature : 1.0f;
  a.f16 = d->precision == PK_PRECISION_F16;
  void* workspace = nullptr;
  if (const uint64_t records = pk::score_workspace(a)) {
    const uint64_t bytes = pk::score_workspace_bytes(a, records);
    DeviceScope device(ctx->device);
    PK_HIP(device.status(), "hipSetDevice");
    const hipError_t e = hipMalloc(&workspace, bytes);
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return fail(PK_ALLOCATION_FAILURE, "%s: cannot allocate %llu bytes of workspace: %s", label.c_str(),
                  (unsigned long long)bytes, hipGetErrorString(e));
    }
    pk::score_bind_workspace(&a, workspace, records);
  }
  auto* op = new (std::nothrow) pk_score_op();
  if (!op) {
    free_on(ctx->device, workspace);
    return fail(PK_ALLOCATION_FAILURE, "%s: out of host memory", label.c_str());
  }
  op->ctx = ctx;
  op->label.swap(label);
  op->rows = d->rows;
  op->args = a;
  op->workspace = workspace;
  *out = op;
  return ok();
} catch (const std::bad_alloc&) {
  return fail(PK_ALLOCATION_FAILURE, "token scores: out of host memory");
}

int pk_score_enqueue(pk_score_op* op, uint32_t active_rows, void* stream) {
  return pk_score_enqueue_timed(op, active_rows, stream, nullptr, nullptr);
}

int pk_score_enqueue_timed(pk_score_op* op, uint32_t active_rows, void* stream, void* start_event, void* end_event) {
  if (!op) return fail(PK_INVALID_ARGUMENT, "token score op is null");
  if (op->destroyed) return fail(PK_DESTROYED, "%s was destroyed", op->label.c_str());
  if (active_rows > op->rows)
    return fail(PK_RANGE_ERROR, "%s active rows must be in [1, %u]", op->label.c_str(), op->rows);
  pk::ScoreArgs args = op->args;
  if (active_rows) args.rows = active_rows;
  DeviceScope device(op->ctx->device);
  PK_HIP(device.status(), "hipSetDevice");
  PK_HIP(pk::launch_score(args, stream_or_default(op->ctx, stream), static_cast<hipEvent_t>(start_event),
                          static_cast<hipEvent_t>(end_event)),
         "token score launch");
  return ok();
}

int pk_score_destroy(pk_score_op* op) {
  if (!op || op->destroyed) return ok();
  op->destroyed = true;
  free_on(op->ctx->device, op->workspace);
  op->workspace = nullptr;
  return ok();
}

int pk_score_release(pk_score_op* op) {
  if (!op) return ok();
  pk_score_destroy(op);
  delete op;
  return ok();
}

}  // extern "C"
