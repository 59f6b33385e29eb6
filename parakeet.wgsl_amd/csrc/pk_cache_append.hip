// pk_cache_append.hip - the append to a paged cache for gfx950
// (include/pk_cache.h has the formulas and what the arrays may hold).
//
// Bound by memory, each element read and written once, and by the launch where
// rows are few: 8192 rows of 32 + 2 * 8 heads of 128 f16 channels 44.5 us, 4.5 TB/s where a
// large copy reaches 5.1; 1616 of 8 + 2 * 8 6.5 us; one row 3.5 to 4.
//
// A workgroup holds whole rows. Where a row's token goes takes three loads in turn (row
// starts, length, page table), so the first elements are loaded before it, the rest of the chain is gone
// through once for a workgroup, and of many rows a workgroup takes several: 1 row each
// was 46 us in the first case, two workgroups for each row 52. Sines and cosines are made in LDS, once for all
// heads; the position times the frequency is a product of 32 by 24 bits, exact in
// f64 but for 3 bits that a second fma gives, and nothing is rounded to f32 before the
// sines and cosines are. A thread takes VEC pairs of a head at a time: 16 bytes of each half, or 32
// together; narrower where strides or head sizes ask for it.
#include "pk_internal.h"

namespace pk {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRows = 8;        // rows of a workgroup
constexpr int kHeld = 2;           // items of a thread at a time, where it has several
constexpr uint32_t kMany = 2048;   // workgroups that many rows are left to
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

// An item of a row: VEC pairs of a head that are rotated, or 2 VEC elements that are not.
struct Item {
  uint32_t row, head, x, y;  // of the workgroup's rows; of all heads; elements of the head where its runs start
  bool live, turn;
};

// Of a row: whether it has a position, the one of its rotation, and its token's place in the caches.
struct Where {
  bool live;
  uint32_t position;
  uint64_t place;
};

template <typename T, int VEC, int HELD>
__global__ __launch_bounds__(kThreads) void cache_append_kernel(CacheAppendArgs args, uint32_t group_rows) {
  __shared__ float2 units[kMaxRows * kMaxPairs];
  __shared__ uint32_t sequence_of[kMaxRows], behind_of[kMaxRows];
  __shared__ Where where[kMaxRows];
  const CacheView& cache = args.cache;
  const uint32_t at = threadIdx.x, first = blockIdx.x * group_rows;
  const uint32_t pairs = args.rotary_dim / 2, dim = cache.head_dim;
  // A head has `turned` items that are rotated and then those that are copied.
  const uint32_t turned = pairs / VEC, each = dim / (2 * VEC);
  const uint32_t row_items = (args.heads + 2 * cache.kv_heads) * each;
  const uint32_t items = min(group_rows, cache.rows - first) * row_items;
  const auto item_of = [&](uint32_t i) {
    Item t;
    t.live = i < items;
    t.row = i / row_items;
    const uint32_t rest = i - t.row * row_items;
    t.head = rest / each;
    const uint32_t index = rest - t.head * each;
    const bool value = t.head >= args.heads + cache.kv_heads;
    t.turn = !value && index < turned;
    const bool halves = t.turn && !args.neighbours;
    t.x = halves ? index * VEC : value || t.turn ? index * 2 * VEC : args.rotary_dim + (index - turned) * 2 * VEC;
    t.y = halves ? t.x + pairs : t.x + VEC;
    return t;
  };
  const auto source = [&](const Item& t) {
    const uint64_t row = first + t.row;
    const uint32_t kv = t.head - args.heads;
    return t.head < args.heads ? static_cast<const T*>(args.queries) + row * args.query_stride + (uint64_t)t.head * dim
           : kv < cache.kv_heads
               ? static_cast<const T*>(args.keys) + row * args.key_stride + (uint64_t)kv * dim
               : static_cast<const T*>(args.values) + row * args.value_stride + (uint64_t)(kv - cache.kv_heads) * dim;
  };
  // HELD items at a time; the first ones' elements are loaded before it is known where they go.
  Item held[HELD];
  Run<T, VEC> x[HELD], y[HELD];
  const auto load = [&](uint32_t from_item) {
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      held[h] = item_of(from_item + h * kThreads);
      if (held[h].live) {
        const T* from = source(held[h]);
        x[h] = load_run<T, VEC>(from + held[h].x);
        y[h] = load_run<T, VEC>(from + held[h].y);
      }
    }
  };
  load(at);

  if (at < kMaxRows) sequence_of[at] = ~0u;
  __syncthreads();
  for (uint32_t s = at; s < cache.sequences; s += kThreads) {
    const uint32_t from = min(cache.row_starts[s], cache.rows), to = min(cache.row_starts[s + 1], cache.rows);
    for (uint32_t r = 0; r < group_rows; ++r)
      if (first + r >= from && first + r < to) {
        sequence_of[r] = s;
        behind_of[r] = to - (first + r);
      }
  }
  __syncthreads();
  // Of each row whether it has a position, which, and where its token lies.
  if (at < group_rows) {
    const uint32_t s = sequence_of[at];
    Where w = {false, 0, CacheView::no_place};
    if (s < cache.sequences) {
      const uint32_t behind = behind_of[at], length = cache.lengths[s];
      w.live = length >= behind;
      w.position = length - behind;
      if (w.live && w.position < cache.capacity()) w.place = cache.place(s, w.position);
      if (args.positions) w.position = args.positions[first + at];
    }
    where[at] = w;
  }
  __syncthreads();
  for (uint32_t i = at; i < group_rows * pairs; i += kThreads) {
    const uint32_t r = i / pairs;
    if (where[r].live) units[i] = unit_of(where[r].position, args.frequencies[i - r * pairs]);
  }
  if (pairs) __syncthreads();

  const auto store = [&](const Item& item, const Run<T, VEC>& x, const Run<T, VEC>& y) {
    const Where w = where[item.row];
    if (!w.live) return;
    T* to;
    if (item.head < args.heads) {
      to = static_cast<T*>(args.query_output) + (uint64_t)(first + item.row) * args.query_output_stride +
           (uint64_t)item.head * dim;
    } else {
      if (w.place == CacheView::no_place) return;
      const bool value = item.head >= args.heads + cache.kv_heads;
      const uint32_t kv = item.head - args.heads - (value ? cache.kv_heads : 0u);
      to = static_cast<T*>(value ? args.value_cache : args.key_cache) + w.place + (uint64_t)kv * cache.page_size * dim;
    }
    if (!item.turn) {
      store_run<T, VEC>(to + item.x, x);
      store_run<T, VEC>(to + item.y, y);
      return;
    }
    const float2* unit = units + item.row * pairs + (args.neighbours ? item.x / 2 : item.x);
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
    store_run<T, VEC>(to + item.x, a);
    store_run<T, VEC>(to + item.y, b);
  };
  for (uint32_t from_item = at;; load(from_item)) {
#pragma unroll
    for (int h = 0; h < HELD; ++h)
      if (held[h].live) store(held[h], x[h], y[h]);
    from_item += HELD * kThreads;
    if (from_item - at >= items) break;
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
  const uint32_t vec = args.f16 && fits(args, 8) ? 8u : fits(args, 4) ? 4u : 1u;
  // Rows of a workgroup: as many as give each thread an item, or, of many rows, as many as
  // leave kMany workgroups, whose threads then go through several items.
  const uint32_t items = (args.heads + 2u * args.cache.kv_heads) * (args.cache.head_dim / (2u * vec));
  const uint32_t few = kThreads / items, many = args.cache.rows / kMany;
  uint32_t rows = many > few ? many : few;
  rows = rows > (uint32_t)kMaxRows ? (uint32_t)kMaxRows : rows ? rows : 1u;
  const bool one = rows * items <= (uint32_t)kThreads;
  const Kernel kernel = vec == 8u   ? (one ? cache_append_kernel<_Float16, 8, 1> : cache_append_kernel<_Float16, 8, kHeld>)
                        : args.f16  ? (vec == 4u ? cache_append_kernel<_Float16, 4, 1> : cache_append_kernel<_Float16, 1, 1>)
                        : vec == 4u ? (one ? cache_append_kernel<float, 4, 1> : cache_append_kernel<float, 4, kHeld>)
                                    : cache_append_kernel<float, 1, 1>;
  const dim3 grid((args.cache.rows + rows - 1u) / rows), block(kThreads);
  if (start || stop)
    hipExtLaunchKernelGGL(kernel, grid, block, 0, stream, start, stop, 0, args, rows);
  else
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, args, rows);
  return hipGetLastError();
}

}  // namespace pk
