// pk_cache_append.hip - the append to a paged cache for gfx950
// (include/pk_cache.h has the formulas and what the arrays may hold).
//
// Bound by memory, each element read and written once, and by the launch where
// rows are few. A workgroup holds whole rows. Its threads first turn the
// angles of their rows into sines and cosines in LDS, once for all heads; the
// position times the frequency is a product of 32 by 24 bits, exact in f64 but
// for 3 bits that a second fma gives, and nothing is rounded to f32 before the
// sines and cosines are. Then a thread takes VEC pairs of a head at
// a time: 16 bytes of each half, or 32 together.
#include "pk_internal.h"

namespace pk {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRows = 8;        // rows of a workgroup
constexpr uint32_t kMaxPairs = 128;

// cos and sin of position * frequency radians, each within a step of f32: the
// angle less whole quarter turns, then the Taylor series up to pi / 4.
__device__ __forceinline__ float2 unit_of(uint32_t position, float frequency) {
#pragma clang fp contract(off)  // `low` is what the rounding of `turns` left, which has to take place
  constexpr double kTurn = 0.15915494309189535, kTurnLow = -9.839338337591835e-18;  // 1 / (2 pi)
  const double p = position, f = frequency, a = p * f, a_low = __builtin_fma(p, f, -a);
  const double turns = a * kTurn;
  const double low = __builtin_fma(a, kTurn, -turns) + (a * kTurnLow + a_low * kTurn);
  const double part = (turns - __builtin_rint(turns)) + low;
  const double quarters = __builtin_rint(4.0 * part);
  const double x = (part - 0.25 * quarters) * 6.283185307179586, x2 = x * x;
  double s = -1.0 / 39916800, c = 1.0 / 479001600;
  constexpr double kSin[5] = {1.0, -1.0 / 6, 1.0 / 120, -1.0 / 5040, 1.0 / 362880};
  constexpr double kCos[6] = {1.0, -1.0 / 2, 1.0 / 24, -1.0 / 720, 1.0 / 40320, -1.0 / 3628800};
#pragma unroll
  for (int i = 4; i >= 0; --i) s = __builtin_fma(s, x2, kSin[i]);
#pragma unroll
  for (int i = 5; i >= 0; --i) c = __builtin_fma(c, x2, kCos[i]);
  const int turned = (int)quarters & 3;
  const float sine = (float)(s * x), cosine = (float)c;
  const float u = (turned & 1) ? sine : cosine, v = (turned & 1) ? cosine : sine;
  return make_float2(turned == 1 || turned == 2 ? -u : u, turned >= 2 ? -v : v);
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Run {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Run<T, VEC> load_run(const T* p) {
  return *reinterpret_cast<const Run<T, VEC>*>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_run(T* p, const Run<T, VEC>& r) {
  *reinterpret_cast<Run<T, VEC>*>(p) = r;
}

template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void cache_append_kernel(CacheAppendArgs args, uint32_t group_rows) {
  __shared__ float2 units[kMaxRows * kMaxPairs];
  __shared__ uint32_t sequence_of[kMaxRows];
  const CacheView& cache = args.cache;
  const uint32_t at = threadIdx.x, first = blockIdx.x * group_rows;
  if (at < kMaxRows) sequence_of[at] = ~0u;
  __syncthreads();
  for (uint32_t s = at; s < cache.sequences; s += kThreads) {
    const uint32_t from = min(cache.row_starts[s], cache.rows), to = min(cache.row_starts[s + 1], cache.rows);
    for (uint32_t r = 0; r < group_rows; ++r)
      if (first + r >= from && first + r < to) sequence_of[r] = s;
  }
  __syncthreads();

  const uint32_t pairs = args.rotary_dim / 2, dim = cache.head_dim;
  // The position of row `first + r` in its sequence; false: none, or before the first.
  const auto position_of = [&](uint32_t r, uint32_t* sequence, uint32_t* position) {
    const uint32_t s = sequence_of[r];
    *sequence = s;
    if (s >= cache.sequences) return false;
    const uint32_t behind = min(cache.row_starts[s + 1], cache.rows) - (first + r), length = cache.lengths[s];
    *position = length - behind;
    return length >= behind;
  };
  for (uint32_t i = at; i < group_rows * pairs; i += kThreads) {
    const uint32_t r = i / pairs, j = i - r * pairs;
    uint32_t s, position = 0;
    if (!position_of(r, &s, &position)) continue;
    units[i] = unit_of(args.positions ? args.positions[first + r] : position, args.frequencies[j]);
  }
  __syncthreads();

  // A head is `turned` items of VEC pairs that are rotated and `copied` of 2 VEC elements that are not.
  const uint32_t turned = pairs / VEC, each = dim / (2 * VEC);
  const uint32_t heads = args.heads + 2 * cache.kv_heads, row_items = heads * each;
  for (uint32_t i = at; i < group_rows * row_items; i += kThreads) {
    const uint32_t r = i / row_items, rest = i - r * row_items, h = rest / each, item = rest - h * each;
    uint32_t s, position;
    if (!position_of(r, &s, &position)) continue;
    const uint64_t row = first + r;
    const T* from;
    T* to;
    const bool value = h >= args.heads + cache.kv_heads;
    if (h < args.heads) {
      from = static_cast<const T*>(args.queries) + row * args.query_stride + (uint64_t)h * dim;
      to = static_cast<T*>(args.query_output) + row * args.query_output_stride + (uint64_t)h * dim;
    } else {
      const uint32_t kv = h - args.heads - (value ? cache.kv_heads : 0u);
      const uint64_t place = position < cache.capacity() ? cache.place(s, position) : CacheView::no_place;
      if (place == CacheView::no_place) continue;
      from = (value ? static_cast<const T*>(args.values) + row * args.value_stride
                    : static_cast<const T*>(args.keys) + row * args.key_stride) + (uint64_t)kv * dim;
      to = static_cast<T*>(value ? args.value_cache : args.key_cache) + place + (uint64_t)kv * cache.page_size * dim;
    }
    const bool turn = !value && item < turned;
    // The elements of the item: two runs, side by side but for rotated halves.
    const uint32_t x_at = turn && !args.neighbours ? item * VEC : value || turn ? item * 2 * VEC
                                                                : args.rotary_dim + (item - turned) * 2 * VEC;
    const uint32_t y_at = turn && !args.neighbours ? x_at + pairs : x_at + VEC;
    const Run<T, VEC> x = load_run<T, VEC>(from + x_at), y = load_run<T, VEC>(from + y_at);
    if (!turn) {
      store_run<T, VEC>(to + x_at, x);
      store_run<T, VEC>(to + y_at, y);
      continue;
    }
    const float2* unit = units + r * pairs + item * VEC;
    Run<T, VEC> a, b;
    if (!args.neighbours) {
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        const float p = (float)x.v[c], q = (float)y.v[c];
        a.v[c] = (T)(p * unit[c].x - q * unit[c].y);
        b.v[c] = (T)(q * unit[c].x + p * unit[c].y);
      }
    } else {
      T both[2 * VEC], out[2 * VEC];
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        both[c] = x.v[c];
        both[VEC + c] = y.v[c];
      }
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        const float p = (float)both[2 * c], q = (float)both[2 * c + 1];
        out[2 * c] = (T)(p * unit[c].x - q * unit[c].y);
        out[2 * c + 1] = (T)(q * unit[c].x + p * unit[c].y);
      }
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        a.v[c] = out[c];
        b.v[c] = out[VEC + c];
      }
    }
    store_run<T, VEC>(to + x_at, a);
    store_run<T, VEC>(to + y_at, b);
  }
}

typedef void (*Kernel)(CacheAppendArgs, uint32_t);

// Whether runs of `vec` elements are aligned in every binding and whole in
// every part of a head.
bool fits(const CacheAppendArgs& a, uint32_t vec) {
  const uint64_t e = a.f16 ? 2u : 4u, bytes = vec * e;
  const auto rows = [&](const void* p, uint64_t stride) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * e % bytes == 0;
  };
  const uint32_t half = a.rotary_dim / 2;
  return half % vec == 0 && a.cache.head_dim % (2 * vec) == 0 && (a.cache.head_dim - a.rotary_dim) % (2 * vec) == 0 &&
         rows(a.keys, a.key_stride) && rows(a.values, a.value_stride) &&
         (!a.queries || (rows(a.queries, a.query_stride) && rows(a.query_output, a.query_output_stride)));
}

}  // namespace

hipError_t launch_cache_append(const CacheAppendArgs& args, hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
  uint32_t vec = 1;
  Kernel kernel = args.f16 ? cache_append_kernel<_Float16, 1> : cache_append_kernel<float, 1>;
  if (args.f16 && fits(args, 8)) {
    vec = 8;
    kernel = cache_append_kernel<_Float16, 8>;
  } else if (fits(args, 4)) {
    vec = 4;
    kernel = args.f16 ? cache_append_kernel<_Float16, 4> : cache_append_kernel<float, 4>;
  }
  // Rows of a workgroup: as many as give each thread an item.
  const uint32_t items = (args.heads + 2u * args.cache.kv_heads) * (args.cache.head_dim / (2u * vec));
  uint32_t rows = (kThreads + items - 1u) / items;
  rows = rows > (uint32_t)kMaxRows ? (uint32_t)kMaxRows : rows;
  const dim3 grid((args.cache.rows + rows - 1u) / rows), block(kThreads);
  if (start || stop)
    hipExtLaunchKernelGGL(kernel, grid, block, 0, stream, start, stop, 0, args, rows);
  else
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, args, rows);
  return hipGetLastError();
}

}  // namespace pk
