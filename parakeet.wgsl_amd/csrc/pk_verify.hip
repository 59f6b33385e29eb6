// pk_verify.hip - verification of drafted tokens for gfx950
// (include/pk_verify.h has the formulas and what rows of infinities, NaN and
// strange numbers give).
//
// Decisions are whole numbers, so probabilities and sums are f64: a sum of
// 131072 f32 exponentials moves with its order by more than the gap between two
// neighbouring tokens of a flat distribution.
#include "pk_internal.h"

namespace pk {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kNoToken = 0xffffffffu;
constexpr float kInf = __builtin_inff();

// 2^x, x <= 0: the whole part goes to the exponent, and the Taylor series of
// 2^f, |f| <= 1/2, is cut where its terms fall below 2^-53.
__device__ __forceinline__ double exp2_of(double x) {
  x = x < -1100.0 ? -1100.0 : x;  // 0 from there on; a NaN passes
  const double n = __builtin_rint(x), f = (x - n) * 0.6931471805599453;
  double r = 1.0 / 6227020800.0;
  constexpr double kInverse[13] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320,
                                   1.0 / 362880, 1.0 / 3628800, 1.0 / 39916800, 1.0 / 479001600};
#pragma unroll
  for (int i = 12; i >= 0; --i) r = __builtin_fma(r, f, kInverse[i]);
  return __builtin_ldexp(r, (int)n);
}

// Sums (or maxima) over the workgroup, in every thread, in a fixed order.
template <typename V, typename Op>
__device__ __forceinline__ V reduce(V x, V* scratch, Op op) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) x = op(x, __shfl_xor(x, off, 64));
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) scratch[threadIdx.x >> 6] = x;
  __syncthreads();
  x = scratch[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) x = op(x, scratch[w]);
  return x;
}

// A row of logits: its maximum, the sum of 2^((z - m) scale), and whether
// it has no probabilities.
struct RowSum {
  double m, sum;
  bool bad;
};

template <typename T>
__device__ RowSum sum_row(const T* z, uint32_t columns, double scale, double* scratch) {
  float m = -kInf;
  int strange = 0;
  for (uint32_t i = threadIdx.x; i < columns; i += kThreads) {
    const float v = (float)z[i];
    strange |= !(v < kInf);
    m = fmaxf(m, v);
  }
  float* f = reinterpret_cast<float*>(scratch);
  m = reduce(m, f, [](float a, float b) { return fmaxf(a, b); });
  strange = reduce(strange, reinterpret_cast<int*>(scratch), [](int a, int b) { return a | b; });
  RowSum row = {m, 0.0, strange || m == -kInf};
  if (row.bad) return row;
  double sum = 0.0;
  for (uint32_t i = threadIdx.x; i < columns; i += kThreads) sum += exp2_of(((double)(float)z[i] - row.m) * scale);
  row.sum = reduce(sum, scratch, [](double a, double b) { return a + b; });
  return row;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyArgs args) {
  __shared__ double scratch[kThreads / 64];
  const uint32_t s = blockIdx.x, at = threadIdx.x, columns = args.columns;
  const uint32_t start = min(args.row_starts[s], args.rows), end = min(args.row_starts[s + 1], args.rows);
  uint32_t accepted = 0, token = kNoToken;
  for (uint32_t row = start; row < end; ++row) {
    const T* z = static_cast<const T*>(args.target) + row * args.target_stride;
    const uint32_t draft = row + 1 < end ? args.tokens[row + 1] : kNoToken;
    const bool last = draft >= columns;
    if (args.greedy) {
      // The largest, the lowest index of equal ones; 0 where there is none.
      uint64_t best = 0;
      for (uint32_t i = at; i < columns; i += kThreads) {
        const float v = (float)z[i] + 0.0f;
        const uint32_t bits = __float_as_uint(v), order = (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
        const uint64_t key = v > -kInf ? ((uint64_t)order << 32) | (uint32_t)~i : 0;
        best = key > best ? key : best;
      }
      unsigned long long all = best;
      all = reduce(all, reinterpret_cast<unsigned long long*>(scratch),
                   [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
      token = all ? ~(uint32_t)all : kNoToken;
      if (last || token != draft) break;
      ++accepted;
      continue;
    }
    const T* y = args.draft ? static_cast<const T*>(args.draft) + row * args.draft_stride : nullptr;
    const RowSum p = sum_row(z, columns, args.scale, scratch);
    RowSum q = {0.0, 1.0, false};
    if (!last && y) q = sum_row(y, columns, args.scale, scratch);
    if (p.bad || q.bad) {
      token = kNoToken;
      break;
    }
    const auto target_of = [&](uint32_t i) { return exp2_of(((double)(float)z[i] - p.m) * args.scale) / p.sum; };
    const auto draft_of = [&](uint32_t i) {
      return y ? exp2_of(((double)(float)y[i] - q.m) * args.scale) / q.sum : i == draft ? 1.0 : 0.0;
    };
    if (!last && (double)args.uniforms[row] * draft_of(draft) < target_of(draft)) {
      ++accepted;
      continue;
    }
    bool residual = !last;
    const auto weight = [&](uint32_t i) {
      if (i >= columns) return 0.0;
      const double w = target_of(i) - (residual ? draft_of(i) : 0.0);
      return w > 0.0 ? w : 0.0;
    };
    const auto add = [](double a, double b) { return a + b; };
    double whole = 0.0;
    for (;;) {
      whole = 0.0;
      for (uint32_t i = 0; i < columns; i += kThreads) whole += reduce(weight(i + at), scratch, add);
      if (whole > 0.0 || !residual) break;
      residual = false;
    }
    const float draw = args.draws[s];
    const double want = draw > 0.0f ? (draw < 1.0f ? (double)draw * whole : whole) : draw <= 0.0f ? 0.0 : whole;
    double before = 0.0;
    uint32_t behind = 0;  // the last token with a weight
    token = kNoToken;
    for (uint32_t i = 0; i < columns && token == kNoToken; i += kThreads) {
      const double mine = weight(i + at);
      double running = mine;  // of the wavefront up to this lane, then of the workgroup
      for (int off = 1; off < 64; off <<= 1) {
        const double other = __shfl_up(running, off, 64);
        if ((int)(at & 63u) >= off) running += other;
      }
      __syncthreads();
      if ((at & 63u) == 63u) scratch[at >> 6] = running;
      __syncthreads();
      double base = before, total = 0.0;
      for (uint32_t w = 0; w < kThreads / 64; ++w) {
        if (w < (at >> 6)) base += scratch[w];
        total += scratch[w];
      }
      uint32_t hit = mine > 0.0 && base + running > want ? i + at : kNoToken;
      __syncthreads();
      hit = reduce(hit, reinterpret_cast<uint32_t*>(scratch), [](uint32_t a, uint32_t b) { return a < b ? a : b; });
      const uint32_t live = reduce(mine > 0.0 ? i + at : 0u, reinterpret_cast<uint32_t*>(scratch),
                                   [](uint32_t a, uint32_t b) { return a > b ? a : b; });
      token = hit;
      behind = live > behind ? live : behind;
      before += total;
    }
    if (token == kNoToken) token = behind;
    break;
  }
  if (at == 0) {
    args.accepted[s] = accepted;
    args.next_tokens[s] = token;
  }
}

}  // namespace

hipError_t launch_verify(const VerifyArgs& args, hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
  const auto kernel = args.f16 ? verify_kernel<_Float16> : verify_kernel<float>;
  const dim3 grid(args.sequences), block(kThreads);
  if (start || stop)
    hipExtLaunchKernelGGL(kernel, grid, block, 0, stream, start, stop, 0, args);
  else
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, args);
  return hipGetLastError();
}

}  // namespace pk
