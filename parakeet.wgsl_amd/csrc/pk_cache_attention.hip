// pk_cache_attention.hip - attention of new tokens over a paged cache for
// gfx950 (include/pk_cache.h has the formulas and what the arrays may hold).
#include "pk_internal.h"

namespace pk {
namespace {

constexpr float kInf = __builtin_inff();
constexpr float kLog2E = 1.4426950408889634f;
constexpr int kThreads = 256;
constexpr int kMaxDim = 256;

// Tokens [low, high) that the row at `position` of a sequence of `length` sees.
struct Seen {
  uint32_t low, high;
};
__device__ __forceinline__ Seen seen_by(const CacheAttentionArgs& args, uint32_t length, int64_t position) {
  const uint32_t held = min(length, args.cache.capacity());
  if (!args.causal) return {0u, held};
  if (position < 0) return {0u, 0u};
  const uint32_t p = (uint32_t)position, high = min(p + 1u, held);
  const uint32_t low = args.window && p >= args.window ? p - args.window + 1u : 0u;
  return {min(low, high), high};
}

__device__ __forceinline__ float block_reduce(float x, bool largest, float* scratch) {
#pragma unroll
  for (int off = 32; off; off >>= 1) {
    const float y = __shfl_xor(x, off, 64);
    x = largest ? fmaxf(x, y) : x + y;
  }
  __syncthreads();  // the readers of the reduction before
  if ((threadIdx.x & 63u) == 0) scratch[threadIdx.x >> 6] = x;
  __syncthreads();
  x = scratch[0];
  for (int w = 1; w < kThreads / 64; ++w) x = largest ? fmaxf(x, scratch[w]) : x + scratch[w];
  return x;
}

// One row of one head: a thread scores a token, then sums an element.
template <typename T>
__global__ __launch_bounds__(kThreads) void cache_attention_row_kernel(CacheAttentionArgs args) {
  __shared__ float query[kMaxDim], weight[kThreads], scratch[kThreads / 64];
  __shared__ uint64_t places[kThreads];
  __shared__ uint32_t owner;
  const CacheView& cache = args.cache;
  const uint32_t at = threadIdx.x, row = blockIdx.x, head = blockIdx.y, dim = cache.head_dim;
  if (at == 0) owner = ~0u;
  __syncthreads();
  for (uint32_t s = at; s < cache.sequences; s += kThreads)
    if (row >= min(cache.row_starts[s], cache.rows) && row < min(cache.row_starts[s + 1], cache.rows)) owner = s;
  __syncthreads();
  const uint32_t s = owner;
  if (s >= cache.sequences) return;
  const uint32_t length = cache.lengths[s];
  const int64_t position = (int64_t)length - (min(cache.row_starts[s + 1], cache.rows) - row);
  const Seen seen = seen_by(args, length, position);
  const uint64_t kv = (uint64_t)(head / (args.heads / cache.kv_heads)) * cache.page_size * dim;
  const T* q = static_cast<const T*>(args.queries) + row * args.query_stride + (uint64_t)head * dim;
  if (at < dim) query[at] = (float)q[at];
  float m = -kInf, l = 0.0f, out = 0.0f;
  for (uint32_t t0 = seen.low; t0 < seen.high; t0 += kThreads) {
    __syncthreads();
    const uint32_t t = t0 + at;
    const uint64_t place = t < seen.high ? cache.place(s, t) : CacheView::no_place;
    float z = -kInf;
    if (place != CacheView::no_place) {
      const T* k = static_cast<const T*>(args.key_cache) + place + kv;
      float dot = 0.0f;
      for (uint32_t d = 0; d < dim; ++d) dot = __builtin_fmaf(query[d], (float)k[d], dot);
      z = dot * args.scale;
      if (args.cap > 0.0f) z = args.cap * tanhf(z / args.cap);
    }
    places[at] = place;
    const float top = fmaxf(m, block_reduce(z, true, scratch));
    const float base = top == -kInf ? 0.0f : top;
    const float p = __builtin_amdgcn_exp2f((z - base) * kLog2E), old = __builtin_amdgcn_exp2f((m - base) * kLog2E);
    m = top;
    weight[at] = p;
    l = l * old + block_reduce(place != CacheView::no_place ? p : 0.0f, false, scratch);
    __syncthreads();
    if (at < dim) {
      out *= old;
      const uint32_t count = min((uint32_t)kThreads, seen.high - t0);
      for (uint32_t i = 0; i < count; ++i)
        if (places[i] != CacheView::no_place)
          out = __builtin_fmaf(weight[i], (float)(static_cast<const T*>(args.value_cache) + places[i] + kv)[at], out);
    }
  }
  if (at < dim)
    (static_cast<T*>(args.output) + row * args.output_stride + (uint64_t)head * dim)[at] =
        (T)(m == -kInf && l == 0.0f ? 0.0f : out / l);
}

}  // namespace

hipError_t launch_cache_attention(const CacheAttentionArgs& args, hipStream_t stream, hipEvent_t start,
                                  hipEvent_t stop) {
  const auto kernel = args.f16 ? cache_attention_row_kernel<_Float16> : cache_attention_row_kernel<float>;
  const dim3 grid(args.cache.rows, args.heads), block(kThreads);
  if (start || stop)
    hipExtLaunchKernelGGL(kernel, grid, block, 0, stream, start, stop, 0, args);
  else
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, args);
  return hipGetLastError();
}

}  // namespace pk
