// pk_score.hip - token scores for gfx950 (include/pk_score.h has the
// formulas and what rows of infinities and NaN give).
//
// One workgroup per row: the maximum, then the sums relative to it, then one
// scan per alternative for the best key below the last.
#include "pk_internal.h"
#include "pk_wave.h"

namespace pk {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2E = 1.4426950408889634f;

// A logit's place in the order of alternatives: larger logits first, equal
// ones by index. 0 for what is never an alternative: minus infinity and NaN.
__device__ __forceinline__ uint64_t score_key(float x, uint32_t index) {
  if (!(x > -__builtin_inff())) return 0;
  const uint32_t bits = __float_as_uint(x + 0.0f);  // one zero
  const uint32_t order = (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
  return ((uint64_t)order << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t order = (uint32_t)(key >> 32);
  return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void score_kernel(ScoreArgs args) {
  __shared__ float red[4][kThreads / 64];
  __shared__ uint64_t best[kThreads / 64];
  const uint32_t row = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
  const T* x = static_cast<const T*>(args.logits) + row * args.stride;
  const float scale = args.inverse_temperature;
  const float inf = __builtin_inff();

  float m = -inf;
  for (uint32_t i = tid; i < args.columns; i += kThreads) m = fmaxf(m, (float)x[i]);
  m = wave::max(m);
  if ((tid & 63u) == 0) red[0][wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) m = fmaxf(m, red[0][w]);
  const float centre = m == -inf ? 0.0f : m;

  float r = 0.0f, t = 0.0f, equal = 0.0f;  // sums over the logits below the maximum, and how many are the maximum
  for (uint32_t i = tid; i < args.columns; i += kThreads) {
    const float v = (float)x[i], d = (v - centre) * scale;
    const float e = __builtin_amdgcn_exp2f(d * kLog2E);
    if (v == m) {
      equal += m == -inf ? 0.0f : d == 0.0f ? 1.0f : e;
    } else {
      r += e;
      t = __builtin_fmaf(e, fmaxf(d, -200.0f), t);
    }
  }
  r = wave::sum(r);
  t = wave::sum(t);
  equal = wave::sum(equal);
  if ((tid & 63u) == 0) {
    red[1][wave] = r;
    red[2][wave] = t;
    red[3][wave] = equal;
  }
  __syncthreads();
  r = t = equal = 0.0f;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    r += red[1][w];
    t += red[2][w];
    equal += red[3][w];
  }
  const bool empty = m == -inf && r == 0.0f;
  r += equal - 1.0f;
  const float spread = log1pf(r);  // NaN where a logit is NaN or plus infinity
  auto log_prob = [&](float v) { return empty ? -inf : (v - m) * scale - spread; };
  if (tid == 0) {
    if (args.entropies) args.entropies[row] = empty ? 0.0f : spread - t / (1.0f + r);
    if (args.tokens) {
      const uint32_t token = args.tokens[row];
      float p = 0.0f;
      if (token < args.columns) p = log_prob((float)x[token]);
      else if (token != 0xffffffffu) p = __builtin_nanf("");
      args.log_probs[row] = p;
    }
  }
  uint64_t last = ~0ull;
  for (uint32_t k = 0; k < args.alternatives; ++k) {
    uint64_t key = 0;
    for (uint32_t i = tid; i < args.columns; i += kThreads) {
      const uint64_t mine = score_key((float)x[i], i);
      if (mine < last && mine > key) key = mine;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)key, off, 64);
      key = other > key ? other : key;
    }
    __syncthreads();  // the readers of the round before
    if ((tid & 63u) == 0) best[wave] = key;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) key = best[w] > key ? best[w] : key;
    last = key;
    if (tid == 0) {
      const uint64_t at = (uint64_t)row * args.alternatives + k;
      args.top_tokens[at] = key ? ~(uint32_t)key : 0xffffffffu;
      args.top_log_probs[at] = key ? log_prob(key_logit(key)) : -inf;
    }
  }
}

}  // namespace

hipError_t launch_score(const ScoreArgs& args, hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
  void (*kernel)(ScoreArgs) = args.f16 ? score_kernel<_Float16> : score_kernel<float>;
  if (start || stop)
    hipExtLaunchKernelGGL(kernel, dim3(args.rows), dim3(kThreads), 0, stream, start, stop, 0, args);
  else
    hipLaunchKernelGGL(kernel, dim3(args.rows), dim3(kThreads), 0, stream, args);
  return hipGetLastError();
}

}  // namespace pk
