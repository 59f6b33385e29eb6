// pk_verify_abi.cpp - C ABI of the verification of drafted tokens
// (include/pk_verify.h): descriptor checks and the launch.
#include <hip/hip_runtime.h>

#include <string>

#include "pk_abi_internal.h"
#include "pk_internal.h"
#include "pk_strided.h"
#include "pk_verify.h"

using namespace pk_abi;

struct pk_verify_op {
  pk_abi::CtxRef ctx;
  std::string label;
  uint32_t sequences = 0;
  pk::VerifyArgs args{};
  void* workspace = nullptr;
  bool destroyed = false;
};

namespace {

const char* verify_label(const char* label) { return label ? label : "draft-verification"; }

int validate_verify(const pk_verify_desc* d) {
  if (!d) return fail(PK_INVALID_ARGUMENT, "draft verification descriptor is null");
  if (d->struct_size != sizeof(pk_verify_desc))
    return fail(PK_INVALID_ARGUMENT, "pk_verify_desc.struct_size mismatch");
  const char* label = verify_label(d->label);
  if (d->precision != PK_PRECISION_F16 && d->precision != PK_PRECISION_F32)
    return fail(PK_INVALID_ARGUMENT, "%s has an unsupported precision %d", label, d->precision);
  if (d->mode != PK_VERIFY_SAMPLE && d->mode != PK_VERIFY_GREEDY)
    return fail(PK_INVALID_ARGUMENT, "%s has an unsupported mode %d", label, d->mode);
  if (d->rows == 0 || d->rows > PK_VERIFY_MAX_ROWS || d->sequences == 0 || d->sequences > PK_VERIFY_MAX_SEQUENCES ||
      d->columns == 0 || d->columns > PK_VERIFY_MAX_COLUMNS)
    return fail(PK_RANGE_ERROR, "Invalid draft verification shape [%u sequences, %u, %u] for %s", d->sequences, d->rows,
                d->columns, label);
  const bool greedy = d->mode == PK_VERIFY_GREEDY;
  if (d->has_temperature && !(d->temperature >= 0x1p-20f && d->temperature <= 0x1p20f))
    return fail(PK_RANGE_ERROR, "%s temperature must be in [2^-20, 2^20]", label);
  if (!d->target || !d->row_starts || !d->tokens || !d->accepted || !d->next_tokens)
    return fail(PK_INVALID_ARGUMENT, "%s needs target logits, row starts, tokens and outputs", label);
  if (!greedy && (!d->uniforms || !d->draws))
    return fail(PK_INVALID_ARGUMENT, "%s needs uniforms and draws", label);
  const uint64_t elem = d->precision == PK_PRECISION_F16 ? 2u : 4u;
  const auto logits = [&](const void* p, uint32_t stride) {
    return Region{p, d->rows, d->columns * elem, (stride ? stride : d->columns) * elem};
  };
  const auto words = [](const void* p, uint64_t count) { return Region{p, 1, count * 4u, count * 4u}; };
  const struct {
    const char* name;
    Region region;
    uint64_t have, align;
  } slices[] = {{"target", logits(d->target, d->target_stride), d->target_bytes, elem},
                {"draft", logits(d->draft, d->draft_stride), d->draft_bytes, elem},
                {"row starts", words(d->row_starts, (uint64_t)d->sequences + 1u), d->row_starts_bytes, 4},
                {"tokens", words(d->tokens, d->rows), d->tokens_bytes, 4},
                {"uniforms", words(d->uniforms, d->rows), d->uniforms_bytes, 4},
                {"draws", words(d->draws, d->sequences), d->draws_bytes, 4},
                {"accepted", words(d->accepted, d->sequences), d->accepted_bytes, 4},
                {"next tokens", words(d->next_tokens, d->sequences), d->next_tokens_bytes, 4}};
  for (const auto& s : slices) {
    if (!s.region.data) continue;
    if (s.region.stride < s.region.row_bytes)
      return fail(PK_RANGE_ERROR, "%s %s stride must be at least the columns", label, s.name);
    if (!aligned(s.region.data, s.align))
      return fail(PK_INVALID_ARGUMENT, "%s %s must be aligned to its elements", label, s.name);
    if (s.have < s.region.extent())
      return fail(PK_RANGE_ERROR, "%s %s needs %llu bytes; arena slice has %llu", label, s.name,
                  (unsigned long long)s.region.extent(), (unsigned long long)s.have);
  }
  for (int i = 6; i < 8; ++i)
    for (int j = 0; j < i; ++j)
      if (overlap(slices[i].region, slices[j].region))
        return fail(PK_INVALID_ARGUMENT, "%s outputs must not overlap each other or the inputs", label);
  return PK_OK;
}

}  // namespace

extern "C" {

int pk_verify_validate(const pk_verify_desc* d) { return validate_verify(d); }

int pk_verify_create(pk_context* ctx, const pk_verify_desc* d, pk_verify_op** out) try {
  if (int s = check_ctx(ctx)) return s;
  if (!d || !out) return fail(PK_INVALID_ARGUMENT, "draft verification descriptor or output is null");
  *out = nullptr;
  if (int s = validate_verify(d)) return s;
  std::string label = verify_label(d->label);
  pk::VerifyArgs a{};
  a.target = d->target;
  a.draft = d->draft;
  a.target_stride = d->target_stride ? d->target_stride : d->columns;
  a.draft_stride = d->draft_stride ? d->draft_stride : d->columns;
  a.row_starts = d->row_starts;
  a.tokens = d->tokens;
  a.uniforms = d->uniforms;
  a.draws = d->draws;
  a.accepted = d->accepted;
  a.next_tokens = d->next_tokens;
  a.rows = d->rows;
  a.sequences = d->sequences;
  a.columns = d->columns;
  a.scale = 1.4426950408889634 / (d->has_temperature ? (double)d->temperature : 1.0);
  a.greedy = d->mode == PK_VERIFY_GREEDY;
  a.f16 = d->precision == PK_PRECISION_F16;
  void* workspace = nullptr;
  if (const uint64_t bytes = pk::verify_workspace(a)) {
    DeviceScope device(ctx->device);
    PK_HIP(device.status(), "hipSetDevice");
    const hipError_t e = hipMalloc(&workspace, bytes);
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return fail(PK_ALLOCATION_FAILURE, "%s: cannot allocate %llu bytes of workspace: %s", label.c_str(),
                  (unsigned long long)bytes, hipGetErrorString(e));
    }
    a.workspace = workspace;
  }
  auto* op = new (std::nothrow) pk_verify_op();
  if (!op) {
    free_on(ctx->device, workspace);
    return fail(PK_ALLOCATION_FAILURE, "%s: out of host memory", label.c_str());
  }
  op->ctx = ctx;
  op->label.swap(label);
  op->sequences = d->sequences;
  op->args = a;
  op->workspace = workspace;
  *out = op;
  return ok();
} catch (const std::bad_alloc&) {
  return fail(PK_ALLOCATION_FAILURE, "draft verification: out of host memory");
}

int pk_verify_enqueue(pk_verify_op* op, uint32_t active_sequences, void* stream) {
  return pk_verify_enqueue_timed(op, active_sequences, stream, nullptr, nullptr);
}

int pk_verify_enqueue_timed(pk_verify_op* op, uint32_t active_sequences, void* stream, void* start_event,
                            void* end_event) {
  if (!op) return fail(PK_INVALID_ARGUMENT, "draft verification op is null");
  if (op->destroyed) return fail(PK_DESTROYED, "%s was destroyed", op->label.c_str());
  if (active_sequences > op->sequences)
    return fail(PK_RANGE_ERROR, "%s active sequences must be in [1, %u]", op->label.c_str(), op->sequences);
  pk::VerifyArgs args = op->args;
  if (active_sequences) args.sequences = active_sequences;
  DeviceScope device(op->ctx->device);
  PK_HIP(device.status(), "hipSetDevice");
  PK_HIP(pk::launch_verify(args, stream_or_default(op->ctx, stream), static_cast<hipEvent_t>(start_event),
                           static_cast<hipEvent_t>(end_event)),
         "draft verification launch");
  return ok();
}

int pk_verify_destroy(pk_verify_op* op) {
  if (!op || op->destroyed) return ok();
  op->destroyed = true;
  free_on(op->ctx->device, op->workspace);
  op->workspace = nullptr;
  return ok();
}

int pk_verify_release(pk_verify_op* op) {
  if (!op) return ok();
  pk_verify_destroy(op);
  delete op;
  return ok();
}

}  // extern "C"
