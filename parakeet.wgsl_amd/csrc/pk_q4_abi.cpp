// pk_q4_abi.cpp - C ABI of the product with 4-bit weights and group scales
// (include/pk_q4.h): descriptor checks, the weight's layout and the launch.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "pk_abi_internal.h"
#include "pk_internal.h"
#include "pk_q4.h"
#include "pk_strided.h"

using namespace pk_abi;

struct pk_q4_op {
  pk_abi::CtxRef ctx;
  std::string label;
  uint32_t rows = 0;
  pk::Q4Args args{};
  void* weight = nullptr;
  uint64_t weight_bytes = 0;
  void* workspace = nullptr;
  bool destroyed = false;
};

namespace {

const char* q4_label(const char* label) { return label ? label : "q4-gemm"; }

int validate_q4(const pk_q4_desc* d) {
  if (!d) return fail(PK_INVALID_ARGUMENT, "q4 descriptor is null");
  if (d->struct_size != sizeof(pk_q4_desc)) return fail(PK_INVALID_ARGUMENT, "pk_q4_desc.struct_size mismatch");
  const char* label = q4_label(d->label);
  if (d->precision != PK_PRECISION_F16 && d->precision != PK_PRECISION_F32)
    return fail(PK_INVALID_ARGUMENT, "%s has an unsupported precision %d", label, d->precision);
  // A launch has at most 2^16 - 1 tiles of 16 rows, and less than 2^32
  // threads: the layout one a word, the product 256 a tile of 64 x 128
  // outputs, of which 2^35 outputs take less than 2^24 (65 rows take two).
  const uint64_t blocks = (((uint64_t)d->inner + 127u) / 128u) * (((uint64_t)d->columns + 15u) / 16u);
  if (d->rows == 0 || d->inner == 0 || d->columns == 0 || d->rows > PK_Q4_MAX_ROWS || blocks >= 1u << 24 ||
      (uint64_t)d->rows * d->columns > 1ull << 35)
    return fail(PK_RANGE_ERROR, "Invalid q4 shape [%u, %u, %u] for %s", d->rows, d->inner, d->columns, label);
  // Offsets into a tile of rows are 32 bits.
  if (d->inner > PK_Q4_MAX_STRIDE || d->a_stride > PK_Q4_MAX_STRIDE)
    return fail(PK_RANGE_ERROR, "%s inner and a stride must be at most %u", label, PK_Q4_MAX_STRIDE);
  if (d->group_size && (d->group_size < 32u || (d->group_size & (d->group_size - 1u)) != 0))
    return fail(PK_RANGE_ERROR, "%s group size must be a power of two from 32 on, or 0", label);
  if (d->activation < PK_ACTIVATION_NONE || d->activation > PK_ACTIVATION_RELU)
    return fail(PK_INVALID_ARGUMENT, "%s has an unsupported activation %d", label, d->activation);
  if (d->has_residual_scale && !std::isfinite(d->residual_scale))
    return fail(PK_INVALID_ARGUMENT, "%s residual scale must be finite", label);
  if (d->has_residual_scale && !d->residual)
    return fail(PK_INVALID_ARGUMENT, "%s has a residual scale without a residual", label);
  if (!d->a || !d->packed || !d->scales || !d->output)
    return fail(PK_INVALID_ARGUMENT, "%s needs a, packed, scales and output", label);
  const uint64_t elem = d->precision == PK_PRECISION_F16 ? 2u : 4u;
  const auto matrix = [&](const void* p, uint32_t width, uint32_t stride) {
    return Region{p, d->rows, width * elem, (stride ? stride : width) * elem};
  };
  const struct {
    const char* name;
    Region region;
    uint64_t bytes;
  } matrices[3] = {{"a", matrix(d->a, d->inner, d->a_stride), d->a_bytes},
                   {"output", matrix(d->output, d->columns, d->output_stride), d->output_bytes},
                   {"residual", matrix(d->residual, d->columns, d->residual_stride), d->residual_bytes}};
  for (const auto& m : matrices) {
    if (!m.region.data) continue;
    if (m.region.stride < m.region.row_bytes)
      return fail(PK_RANGE_ERROR, "%s %s stride must be at least its columns", label, m.name);
    if (!aligned(m.region.data, elem))
      return fail(PK_INVALID_ARGUMENT, "%s %s must be aligned to its elements", label, m.name);
    if (m.bytes < m.region.extent())
      return fail(PK_RANGE_ERROR, "%s %s needs %llu bytes; arena slice has %llu", label, m.name,
                  (unsigned long long)m.region.extent(), (unsigned long long)m.bytes);
  }
  const uint64_t packed = ((uint64_t)d->inner * d->columns + 7u) / 8u * 4u;
  if (d->packed_bytes != packed || !aligned(d->packed, 4))
    return fail(PK_INVALID_ARGUMENT, "%s packed must be %llu bytes of whole words", label,
                (unsigned long long)packed);
  const uint32_t group = d->group_size ? d->group_size : d->inner;
  const uint64_t table = (uint64_t)((d->inner + group - 1u) / group) * d->columns * elem;
  if (d->scales_bytes != table || !aligned(d->scales, elem) ||
      (d->offsets && (d->offsets_bytes != table || !aligned(d->offsets, elem))))
    return fail(PK_INVALID_ARGUMENT, "%s scales and offsets must be [%u, %u], %llu bytes", label,
                (d->inner + group - 1u) / group, d->columns, (unsigned long long)table);
  if (d->bias && (d->bias_bytes != (uint64_t)d->columns * 4u || !aligned(d->bias, 4)))
    return fail(PK_INVALID_ARGUMENT, "%s bias must be float32 [%u], %llu bytes", label, d->columns,
                (unsigned long long)d->columns * 4u);
  const Region &a = matrices[0].region, &out = matrices[1].region, &res = matrices[2].region;
  if (overlap(out, a)) return fail(PK_INVALID_ARGUMENT, "%s output must not overlap a", label);
  if (overlap(out, res) && !same_rows(out, res))
    return fail(PK_INVALID_ARGUMENT, "%s output must be the residual or not overlap it", label);
  if (d->bias && overlap(out, Region{d->bias, 1, d->bias_bytes, d->bias_bytes}))
    return fail(PK_INVALID_ARGUMENT, "%s output must not overlap the bias", label);
  return PK_OK;
}

}  // namespace

extern "C" {

int pk_q4_validate(const pk_q4_desc* d) { return validate_q4(d); }

int pk_q4_create(pk_context* ctx, const pk_q4_desc* d, void* stream, pk_q4_op** out) try {
  if (int s = check_ctx(ctx)) return s;
  if (!d || !out) return fail(PK_INVALID_ARGUMENT, "q4 descriptor or output is null");
  *out = nullptr;
  if (int s = validate_q4(d)) return s;
  std::string label = q4_label(d->label);
  DeviceScope device(ctx->device);
  PK_HIP(device.status(), "hipSetDevice");
  const hipStream_t st = stream_or_default(ctx, stream);
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  PK_HIP(hipStreamIsCapturing(st, &capture), "hipStreamIsCapturing");
  if (capture != hipStreamCaptureStatusNone)
    return fail(PK_INVALID_ARGUMENT, "%s cannot be created on a capturing stream", label.c_str());
  pk::Q4Args a{};
  a.a = d->a;
  a.a_stride = d->a_stride ? d->a_stride : d->inner;
  a.out = d->output;
  a.out_stride = d->output_stride ? d->output_stride : d->columns;
  a.bias = d->bias;
  a.residual = d->residual;
  a.residual_stride = d->residual_stride ? d->residual_stride : d->columns;
  a.residual_scale = d->has_residual_scale ? d->residual_scale : 1.0f;
  a.activation = d->activation;
  a.rows = d->rows;
  a.inner = d->inner;
  a.columns = d->columns;
  a.per_block = d->group_size == 32u ? 4u : d->group_size == 64u ? 2u : 1u;
  a.f16 = d->precision == PK_PRECISION_F16;
  const pk::Q4Layout at = pk::q4_layout(a, d->offsets != nullptr);
  void* weight = nullptr;
  const hipError_t got = hipMalloc(&weight, at.bytes);
  if (got != hipSuccess) {
    (void)hipGetLastError();
    return fail(PK_ALLOCATION_FAILURE, "%s: cannot allocate %llu bytes for the weight: %s", label.c_str(),
                (unsigned long long)at.bytes, hipGetErrorString(got));
  }
  uint8_t* base = static_cast<uint8_t*>(weight);
  a.codes = reinterpret_cast<const uint4*>(base);
  a.scales = base + at.scales;
  a.offsets = d->offsets ? base + at.offsets : nullptr;
  void* workspace = nullptr;
  if ((a.part_bytes = pk::q4_workspace(a))) {
    const hipError_t room = hipMalloc(&workspace, a.part_bytes);
    if (room != hipSuccess) {
      (void)hipGetLastError();
      (void)hipFree(weight);
      return fail(PK_ALLOCATION_FAILURE, "%s: cannot allocate %llu bytes of workspace: %s", label.c_str(),
                  (unsigned long long)a.part_bytes, hipGetErrorString(room));
    }
    a.parts = static_cast<float*>(workspace);
  }
  hipError_t e = pk::launch_q4_layout(a, d->packed, d->scales, d->offsets, d->group_size ? d->group_size : d->inner, st);
  const hipError_t done = hipStreamSynchronize(st);
  if (e == hipSuccess) e = done;
  pk_q4_op* op = e == hipSuccess ? new (std::nothrow) pk_q4_op() : nullptr;
  if (!op) {
    (void)hipFree(weight);
    (void)hipFree(workspace);
    if (e == hipSuccess) return fail(PK_ALLOCATION_FAILURE, "%s: out of host memory", label.c_str());
    return fail(PK_DEVICE_ERROR, "%s weight layout failed: %s", label.c_str(), hipGetErrorString(e));
  }
  op->ctx = ctx;
  op->label.swap(label);
  op->rows = d->rows;
  op->args = a;
  op->weight = weight;
  op->weight_bytes = at.bytes;
  op->workspace = workspace;
  *out = op;
  return ok();
} catch (const std::bad_alloc&) {
  return fail(PK_ALLOCATION_FAILURE, "q4: out of host memory");
}

int pk_q4_enqueue(pk_q4_op* op, uint32_t active_rows, void* stream) {
  return pk_q4_enqueue_timed(op, active_rows, stream, nullptr, nullptr);
}

int pk_q4_enqueue_timed(pk_q4_op* op, uint32_t active_rows, void* stream, void* start_event, void* end_event) {
  if (!op) return fail(PK_INVALID_ARGUMENT, "q4 op is null");
  if (op->destroyed) return fail(PK_DESTROYED, "%s was destroyed", op->label.c_str());
  if (active_rows > op->rows)
    return fail(PK_RANGE_ERROR, "%s active rows must be in [1, %u]", op->label.c_str(), op->rows);
  pk::Q4Args args = op->args;
  if (active_rows) args.rows = active_rows;
  DeviceScope device(op->ctx->device);
  PK_HIP(device.status(), "hipSetDevice");
  PK_HIP(pk::launch_q4(args, stream_or_default(op->ctx, stream), static_cast<hipEvent_t>(start_event),
                       static_cast<hipEvent_t>(end_event)),
         "q4 launch");
  return ok();
}

int pk_q4_weight_bytes(const pk_q4_op* op, uint64_t* bytes) {
  if (!op || !bytes) return fail(PK_INVALID_ARGUMENT, "q4 op or output is null");
  *bytes = op->weight_bytes;
  return ok();
}

int pk_q4_destroy(pk_q4_op* op) {
  if (!op || op->destroyed) return ok();
  op->destroyed = true;
  free_on(op->ctx->device, op->weight);
  free_on(op->ctx->device, op->workspace);
  op->weight = op->workspace = nullptr;
  op->weight_bytes = 0;
  return ok();
}

int pk_q4_release(pk_q4_op* op) {
  if (!op) return ok();
  pk_q4_destroy(op);
  delete op;
  return ok();
}

}  // extern "C"
