// pk_cache_abi.cpp - C ABI of the paged cache (include/pk_cache.h): descriptor
// checks and the launches of append and attention.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "pk_abi_internal.h"
#include "pk_cache.h"
#include "pk_internal.h"
#include "pk_strided.h"

using namespace pk_abi;

struct pk_cache_append_op {
  pk_abi::CtxRef ctx;
  std::string label;
  uint32_t sequences = 0;
  pk::CacheAppendArgs args{};
  bool destroyed = false;
};

struct pk_cache_attention_op {
  pk_abi::CtxRef ctx;
  std::string label;
  uint32_t sequences = 0;
  pk::CacheAttentionArgs args{};
  void* workspace = nullptr;
  bool destroyed = false;
};

namespace {

const char* append_label(const char* label) { return label ? label : "cache-append"; }
const char* attention_label(const char* label) { return label ? label : "cache-attention"; }

// A named region that an op reads or writes.
struct Binding {
  const char* name;
  Region region;
  uint64_t have;   // bytes
  uint64_t align;
};

int check_binding(const char* label, const Binding& b) {
  if (b.region.stride < b.region.row_bytes)
    return fail(PK_RANGE_ERROR, "%s %s stride must be at least its columns", label, b.name);
  if (!aligned(b.region.data, b.align))
    return fail(PK_INVALID_ARGUMENT, "%s %s must be aligned to %s", label, b.name,
                b.align == 16 ? "16 bytes" : "its elements");
  if (b.have < b.region.extent())
    return fail(PK_RANGE_ERROR, "%s %s needs %llu bytes; arena slice has %llu", label, b.name,
                (unsigned long long)b.region.extent(), (unsigned long long)b.have);
  return PK_OK;
}

// Rows of [heads][head_dim] elements (stride 0: packed).
Binding matrix(const char* name, const void* p, uint64_t bytes, uint32_t rows, uint32_t heads, uint32_t dim,
               uint32_t stride, uint64_t elem) {
  const uint64_t columns = (uint64_t)heads * dim;
  return {name, {p, rows, columns * elem, (stride ? stride : columns) * elem}, bytes, elem};
}

Binding words(const char* name, const void* p, uint64_t bytes, uint64_t count) {
  return {name, {p, 1, count * 4u, count * 4u}, bytes, 4};
}

// What the descriptors of append and attention have in common: the shape, and
// the bindings of the cache, the tables first.
template <typename Desc>
int check_cache(const Desc* d, const char* label, Binding (&cache)[5]) {
  if (d->precision != PK_PRECISION_F16 && d->precision != PK_PRECISION_F32)
    return fail(PK_INVALID_ARGUMENT, "%s has an unsupported precision %d", label, d->precision);
  if (d->rows == 0 || d->rows > PK_CACHE_MAX_ROWS || d->sequences == 0 || d->sequences > PK_CACHE_MAX_SEQUENCES)
    return fail(PK_RANGE_ERROR, "Invalid cache rows [%u sequences, %u] for %s", d->sequences, d->rows, label);
  if (d->kv_heads == 0 || d->kv_heads > PK_CACHE_MAX_HEADS || d->heads > PK_CACHE_MAX_HEADS || d->head_dim == 0 ||
      d->head_dim > PK_CACHE_MAX_HEAD_DIM || d->head_dim % 8)
    return fail(PK_RANGE_ERROR, "Invalid cache heads [%u over %u, %u] for %s", d->heads, d->kv_heads, d->head_dim,
                label);
  if (d->page_size == 0 || d->page_size > PK_CACHE_MAX_PAGE_SIZE || d->pages == 0 || d->pages_per_sequence == 0 ||
      (uint64_t)d->page_size * d->pages_per_sequence > PK_CACHE_MAX_TOKENS)
    return fail(PK_RANGE_ERROR, "Invalid cache pages [%u of %u, %u of a sequence] for %s", d->pages, d->page_size,
                d->pages_per_sequence, label);
  if (!d->row_starts || !d->lengths || !d->page_table || !d->key_cache || !d->value_cache)
    return fail(PK_INVALID_ARGUMENT, "%s needs row starts, lengths, a page table and caches", label);
  const uint64_t elem = d->precision == PK_PRECISION_F16 ? 2u : 4u;
  const uint64_t page = (uint64_t)d->kv_heads * d->page_size * d->head_dim;
  if (d->page_stride && (d->page_stride < page || d->page_stride % 8 || d->page_stride > PK_CACHE_MAX_BYTES))
    return fail(PK_RANGE_ERROR, "%s page stride must be a multiple of 8 of at least a page", label);
  const uint64_t stride = (d->page_stride ? d->page_stride : page) * elem;
  // The extent, without a product beyond 64 bits.
  if (page * elem > PK_CACHE_MAX_BYTES || (uint64_t)(d->pages - 1) > (PK_CACHE_MAX_BYTES - page * elem) / stride)
    return fail(PK_RANGE_ERROR, "%s caches must be within %llu bytes", label, (unsigned long long)PK_CACHE_MAX_BYTES);
  const Region keys{d->key_cache, d->pages, page * elem, stride}, values{d->value_cache, d->pages, page * elem, stride};
  cache[0] = words("row starts", d->row_starts, d->row_starts_bytes, (uint64_t)d->sequences + 1u);
  cache[1] = words("lengths", d->lengths, d->lengths_bytes, d->sequences);
  cache[2] = words("page table", d->page_table, d->page_table_bytes, (uint64_t)d->sequences * d->pages_per_sequence);
  cache[3] = {"key cache", keys, d->key_cache_bytes, 16};
  cache[4] = {"value cache", values, d->value_cache_bytes, 16};
  for (const Binding& b : cache)
    if (int s = check_binding(label, b)) return s;
  return PK_OK;
}

template <typename Desc>
pk::CacheView cache_view(const Desc* d) {
  pk::CacheView v{};
  v.row_starts = d->row_starts;
  v.lengths = d->lengths;
  v.page_table = d->page_table;
  v.page_stride = d->page_stride ? d->page_stride : (uint64_t)d->kv_heads * d->page_size * d->head_dim;
  v.rows = d->rows;
  v.sequences = d->sequences;
  v.pages_per_sequence = d->pages_per_sequence;
  v.pages = d->pages;
  v.set_page_size(d->page_size);
  v.kv_heads = d->kv_heads;
  v.head_dim = d->head_dim;
  return v;
}

uint64_t stride_of(uint32_t stride, uint32_t heads, uint32_t dim) { return stride ? stride : (uint64_t)heads * dim; }

int validate_append(const pk_cache_append_desc* d) {
  if (!d) return fail(PK_INVALID_ARGUMENT, "cache append descriptor is null");
  if (d->struct_size != sizeof(pk_cache_append_desc))
    return fail(PK_INVALID_ARGUMENT, "pk_cache_append_desc.struct_size mismatch");
  const char* label = append_label(d->label);
  Binding cache[5];
  if (int s = check_cache(d, label, cache)) return s;
  if ((d->heads != 0) != (d->queries != nullptr) || (d->heads != 0) != (d->query_output != nullptr))
    return fail(PK_INVALID_ARGUMENT, "%s needs queries and a query output with heads, and only then", label);
  if (!d->keys || !d->values) return fail(PK_INVALID_ARGUMENT, "%s needs keys and values", label);
  if (d->rotary_dim > d->head_dim || d->rotary_dim % 2)
    return fail(PK_RANGE_ERROR, "%s rotary dim must be even and at most %u", label, d->head_dim);
  if (d->rotary != PK_ROTARY_HALVES && d->rotary != PK_ROTARY_NEIGHBOURS)
    return fail(PK_INVALID_ARGUMENT, "%s has an unsupported rotary kind %d", label, d->rotary);
  if ((d->rotary_dim != 0) != (d->frequencies != nullptr))
    return fail(PK_INVALID_ARGUMENT, "%s needs frequencies with a rotary dim, and only then", label);
  if (d->positions && !d->rotary_dim)
    return fail(PK_INVALID_ARGUMENT, "%s has positions without a rotary dim", label);
  const uint64_t elem = d->precision == PK_PRECISION_F16 ? 2u : 4u;
  const uint32_t dim = d->head_dim;
  const Binding queries = matrix("queries", d->queries, d->queries_bytes, d->rows, d->heads, dim, d->query_stride, elem),
                output = matrix("query output", d->query_output, d->query_output_bytes, d->rows, d->heads, dim,
                                d->query_output_stride, elem);
  const Binding reads[] = {
      queries,
      matrix("keys", d->keys, d->keys_bytes, d->rows, d->kv_heads, dim, d->key_stride, elem),
      matrix("values", d->values, d->values_bytes, d->rows, d->kv_heads, dim, d->value_stride, elem),
      words("frequencies", d->frequencies, d->frequencies_bytes, d->rotary_dim / 2u),
      words("positions", d->positions, d->positions_bytes, d->rows),
      cache[0], cache[1], cache[2]};
  const Binding writes[] = {output, cache[3], cache[4]};
  for (int i = 0; i < 5; ++i)
    if (reads[i].region.data)
      if (int s = check_binding(label, reads[i])) return s;
  if (output.region.data)
    if (int s = check_binding(label, output)) return s;
  for (const Binding& w : writes)
    for (const Binding& r : reads) {
      if (!overlap(w.region, r.region)) continue;
      // A thread reads both elements of a pair before it writes them.
      if (&w == &writes[0] && &r == &reads[0]) {
        if (same_rows(w.region, r.region)) continue;
        return fail(PK_INVALID_ARGUMENT, "%s query output must be the queries or not overlap them", label);
      }
      return fail(PK_INVALID_ARGUMENT, "%s %s must not overlap %s", label, w.name, r.name);
    }
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < i; ++j)
      if (overlap(writes[i].region, writes[j].region))
        return fail(PK_INVALID_ARGUMENT, "%s %s must not overlap %s", label, writes[i].name, writes[j].name);
  return PK_OK;
}

int validate_attention(const pk_cache_attention_desc* d) {
  if (!d) return fail(PK_INVALID_ARGUMENT, "cache attention descriptor is null");
  if (d->struct_size != sizeof(pk_cache_attention_desc))
    return fail(PK_INVALID_ARGUMENT, "pk_cache_attention_desc.struct_size mismatch");
  const char* label = attention_label(d->label);
  Binding cache[5];
  if (int s = check_cache(d, label, cache)) return s;
  if (d->heads == 0 || d->heads % d->kv_heads)
    return fail(PK_RANGE_ERROR, "%s heads must be a multiple of the %u kv heads", label, d->kv_heads);
  // Workgroups of the smallest units, 16 rows of a kv head: as many as a launch holds.
  const uint64_t some = d->sequences < d->rows ? d->sequences : d->rows;
  if ((uint64_t)d->rows * d->heads / 16u + d->kv_heads * some > PK_CACHE_MAX_UNITS)
    return fail(PK_RANGE_ERROR, "%s has more than %u blocks of 16 rows", label, PK_CACHE_MAX_UNITS);
  if (!d->queries || !d->output) return fail(PK_INVALID_ARGUMENT, "%s needs queries and an output", label);
  if (d->causal != 0 && d->causal != 1) return fail(PK_INVALID_ARGUMENT, "%s causal must be 0 or 1", label);
  if (d->window && !d->causal) return fail(PK_INVALID_ARGUMENT, "%s has a window without causal", label);
  if (d->has_scale && !(std::fabs(d->scale) <= 0x1p60f))
    return fail(PK_RANGE_ERROR, "%s scale must be at most 2^60 in magnitude", label);
  if (!(d->score_cap == 0.0f || (d->score_cap >= 0x1p-20f && d->score_cap <= 0x1p20f)))
    return fail(PK_RANGE_ERROR, "%s score cap must be 0 or in [2^-20, 2^20]", label);
  const uint64_t elem = d->precision == PK_PRECISION_F16 ? 2u : 4u;
  const Binding queries = matrix("queries", d->queries, d->queries_bytes, d->rows, d->heads, d->head_dim,
                                 d->query_stride, elem),
                output = matrix("output", d->output, d->output_bytes, d->rows, d->heads, d->head_dim,
                                d->output_stride, elem);
  if (int s = check_binding(label, queries)) return s;
  if (int s = check_binding(label, output)) return s;
  for (const Binding& r : {queries, cache[0], cache[1], cache[2], cache[3], cache[4]})
    if (overlap(output.region, r.region))
      return fail(PK_INVALID_ARGUMENT, "%s output must not overlap %s", label, r.name);
  return PK_OK;
}

// The op's arguments for a launch over the first `active` sequences.
template <typename Op, typename Args>
int active_args(const Op* op, const char* what, uint32_t active, Args* args) {
  if (!op) return fail(PK_INVALID_ARGUMENT, "%s op is null", what);
  if (op->destroyed) return fail(PK_DESTROYED, "%s was destroyed", op->label.c_str());
  if (active > op->sequences)
    return fail(PK_RANGE_ERROR, "%s active sequences must be in [1, %u]", op->label.c_str(), op->sequences);
  *args = op->args;
  if (active) args->cache.sequences = active;
  return PK_OK;
}

}  // namespace

extern "C" {

int pk_cache_append_validate(const pk_cache_append_desc* d) { return validate_append(d); }

int pk_cache_append_create(pk_context* ctx, const pk_cache_append_desc* d, pk_cache_append_op** out) try {
  if (int s = check_ctx(ctx)) return s;
  if (!d || !out) return fail(PK_INVALID_ARGUMENT, "cache append descriptor or output is null");
  *out = nullptr;
  if (int s = validate_append(d)) return s;
  std::string label = append_label(d->label);
  auto* op = new (std::nothrow) pk_cache_append_op();
  if (!op) return fail(PK_ALLOCATION_FAILURE, "%s: out of host memory", label.c_str());
  pk::CacheAppendArgs a{};
  a.cache = cache_view(d);
  a.queries = d->queries;
  a.keys = d->keys;
  a.values = d->values;
  a.query_output = d->query_output;
  a.key_cache = d->key_cache;
  a.value_cache = d->value_cache;
  a.frequencies = d->frequencies;
  a.positions = d->positions;
  a.query_stride = stride_of(d->query_stride, d->heads, d->head_dim);
  a.query_output_stride = stride_of(d->query_output_stride, d->heads, d->head_dim);
  a.key_stride = stride_of(d->key_stride, d->kv_heads, d->head_dim);
  a.value_stride = stride_of(d->value_stride, d->kv_heads, d->head_dim);
  a.heads = d->heads;
  a.rotary_dim = d->rotary_dim;
  a.neighbours = d->rotary == PK_ROTARY_NEIGHBOURS;
  a.f16 = d->precision == PK_PRECISION_F16;
  op->ctx = ctx;
  op->label.swap(label);
  op->sequences = d->sequences;
  op->args = a;
  *out = op;
  return ok();
} catch (const std::bad_alloc&) {
  return fail(PK_ALLOCATION_FAILURE, "cache append: out of host memory");
}

int pk_cache_append_enqueue(pk_cache_append_op* op, uint32_t active_sequences, void* stream) {
  return pk_cache_append_enqueue_timed(op, active_sequences, stream, nullptr, nullptr);
}

int pk_cache_append_enqueue_timed(pk_cache_append_op* op, uint32_t active_sequences, void* stream, void* start_event,
                                  void* end_event) {
  pk::CacheAppendArgs args;
  if (int s = active_args(op, "cache append", active_sequences, &args)) return s;
  DeviceScope device(op->ctx->device);
  PK_HIP(device.status(), "hipSetDevice");
  PK_HIP(pk::launch_cache_append(args, stream_or_default(op->ctx, stream), static_cast<hipEvent_t>(start_event),
                                 static_cast<hipEvent_t>(end_event)),
         "cache append launch");
  return ok();
}

int pk_cache_append_destroy(pk_cache_append_op* op) {
  if (op) op->destroyed = true;
  return ok();
}

int pk_cache_append_release(pk_cache_append_op* op) {
  if (!op) return ok();
  pk_cache_append_destroy(op);
  delete op;
  return ok();
}

int pk_cache_attention_validate(const pk_cache_attention_desc* d) { return validate_attention(d); }

int pk_cache_attention_create(pk_context* ctx, const pk_cache_attention_desc* d, pk_cache_attention_op** out) try {
  if (int s = check_ctx(ctx)) return s;
  if (!d || !out) return fail(PK_INVALID_ARGUMENT, "cache attention descriptor or output is null");
  *out = nullptr;
  if (int s = validate_attention(d)) return s;
  std::string label = attention_label(d->label);
  pk::CacheAttentionArgs a{};
  a.cache = cache_view(d);
  a.queries = d->queries;
  a.output = d->output;
  a.key_cache = d->key_cache;
  a.value_cache = d->value_cache;
  a.query_stride = stride_of(d->query_stride, d->heads, d->head_dim);
  a.output_stride = stride_of(d->output_stride, d->heads, d->head_dim);
  a.heads = d->heads;
  a.group.set(d->heads / d->kv_heads);
  a.window = d->window;
  a.scale = d->has_scale ? d->scale : (float)(1.0 / std::sqrt((double)d->head_dim));
  a.cap = d->score_cap;
  a.causal = d->causal != 0;
  a.f16 = d->precision == PK_PRECISION_F16;
  const uint64_t elem = a.f16 ? 2u : 4u;
  a.wide_rows = aligned(a.queries, 16) && aligned(a.output, 16) && a.query_stride * elem % 16u == 0 &&
                a.output_stride * elem % 16u == 0;
  void* workspace = nullptr;
  if (const uint64_t bytes = pk::cache_attention_workspace(a)) {
    DeviceScope device(ctx->device);
    PK_HIP(device.status(), "hipSetDevice");
    const hipError_t e = hipMalloc(&workspace, bytes);
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return fail(PK_ALLOCATION_FAILURE, "%s: cannot allocate %llu bytes of workspace: %s", label.c_str(),
                  (unsigned long long)bytes, hipGetErrorString(e));
    }
    a.workspace = workspace;
    a.workspace_bytes = bytes;
  }
  auto* op = new (std::nothrow) pk_cache_attention_op();
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
  return fail(PK_ALLOCATION_FAILURE, "cache attention: out of host memory");
}

int pk_cache_attention_enqueue(pk_cache_attention_op* op, uint32_t active_sequences, void* stream) {
  return pk_cache_attention_enqueue_timed(op, active_sequences, stream, nullptr, nullptr);
}

int pk_cache_attention_enqueue_timed(pk_cache_attention_op* op, uint32_t active_sequences, void* stream,
                                     void* start_event, void* end_event) {
  pk::CacheAttentionArgs args;
  if (int s = active_args(op, "cache attention", active_sequences, &args)) return s;
  DeviceScope device(op->ctx->device);
  PK_HIP(device.status(), "hipSetDevice");
  PK_HIP(pk::launch_cache_attention(args, stream_or_default(op->ctx, stream), static_cast<hipEvent_t>(start_event),
                                    static_cast<hipEvent_t>(end_event)),
         "cache attention launch");
  return ok();
}

int pk_cache_attention_destroy(pk_cache_attention_op* op) {
  if (!op || op->destroyed) return ok();
  op->destroyed = true;
  free_on(op->ctx->device, op->workspace);
  op->workspace = nullptr;
  return ok();
}

int pk_cache_attention_release(pk_cache_attention_op* op) {
  if (!op) return ok();
  pk_cache_attention_destroy(op);
  delete op;
  return ok();
}

}  // extern "C"
