// pk_block_norm.hip - the norms around a block for gfx950: the norm of the
// block's output, its gate and residual, and the norm of the sum, in one pass
// (include/pk_block_norm.h has the formulas).
//
// Bound by memory: each matrix is read or written once (2 to 5 elements of
// traffic for some 20 operations). A row lies in the registers of GROUP
// threads (a wavefront up to 2048 channels, then 256 or 1024 threads), HELD
// vectors a thread, as f32 from the first load to the last store, so the
// second norm costs no memory trip. Variances are of the differences from
// the mean, a second sum over registers, since E[x^2] - E[x]^2 loses every
// digit of a row whose mean is far from zero.
#include "pk_internal.h"
#include "pk_wave.h"

namespace pk {
namespace {

constexpr int kThreads = 256;  // of a workgroup, unless one row takes more

template <typename T, int VEC>
struct VectorOf {
  typedef T type __attribute__((ext_vector_type(VEC)));
};
template <typename T>
struct VectorOf<T, 1> {
  typedef T type;
};

template <typename T, int VEC, int GROUP, int HELD>
__global__ __launch_bounds__(GROUP > kThreads ? GROUP : kThreads) void block_norm_kernel(BlockNormArgs args) {
  typedef typename VectorOf<T, VEC>::type V;
  constexpr int kRows = GROUP < kThreads ? kThreads / GROUP : 1;  // rows of a workgroup
  constexpr int kWaves = GROUP / 64;
  __shared__ float partial[4][kWaves];  // a slot for each of the sums: no sum waits for the readers of another
  const uint32_t row = blockIdx.x * kRows + threadIdx.x / GROUP;
  const uint32_t at = threadIdx.x % GROUP;
  if (row >= args.rows) return;  // whole wavefronts, and whole workgroups where they meet
  const uint32_t vectors = args.channels / VEC;
  const float inverse = 1.0f / (float)args.channels;

  auto load = [&](const void* p, uint64_t from, V (&dst)[HELD]) {
    const V* v = reinterpret_cast<const V*>(static_cast<const T*>(p) + from);
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (at + i * GROUP < vectors) dst[i] = v[at + i * GROUP];
  };
  auto element = [](const V& v, int c) -> float {
    if constexpr (VEC == 1) return (float)v;
    else return (float)v[c];
  };
  // The sum of f(x) over the row, the same in every thread of the group.
  auto total = [&](int slot, auto f, const float (&x)[HELD][VEC]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (at + i * GROUP < vectors)
#pragma unroll
        for (int c = 0; c < VEC; ++c) s += f(x[i][c]);
    s = wave::sum(s);
    if constexpr (kWaves > 1) {
      if ((threadIdx.x & 63) == 0) partial[slot][threadIdx.x >> 6] = s;
      __syncthreads();
      s = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) s += partial[slot][w];
    }
    return s;
  };
  auto normalize = [&](int slot, const float* gamma, const float* beta, float (&x)[HELD][VEC]) {
    float mean = 0.0f;
    if (!args.rms) mean = total(slot, [](float v) { return v; }, x) * inverse;
    const float power = total(slot + 1, [mean](float v) { return (v - mean) * (v - mean); }, x) * inverse;
    const float scale = 1.0f / __builtin_sqrtf(power + args.epsilon);
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const uint32_t v = at + i * GROUP;
      if (v >= vectors) continue;
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        const float b = beta ? beta[v * VEC + c] : 0.0f;
        x[i][c] = __builtin_fmaf((x[i][c] - mean) * scale, gamma[v * VEC + c], b);
      }
    }
  };
  auto store = [&](void* p, uint64_t from, const float (&x)[HELD][VEC]) {
    V* out = reinterpret_cast<V*>(static_cast<T*>(p) + from);
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      if (at + i * GROUP >= vectors) continue;
      V v;
#pragma unroll
      for (int c = 0; c < VEC; ++c)
        if constexpr (VEC == 1) v = (T)x[i][c];
        else v[c] = (T)x[i][c];
      out[at + i * GROUP] = v;
    }
  };

  V in[HELD], gate[HELD], residual[HELD];
  load(args.input, row * args.input_stride, in);
  if (args.gate) load(args.gate, (args.gate_rows ? row / args.gate_rows : 0u) * args.gate_stride, gate);
  if (args.residual) load(args.residual, row * args.residual_stride, residual);
  float x[HELD][VEC];
#pragma unroll
  for (int i = 0; i < HELD; ++i)
#pragma unroll
    for (int c = 0; c < VEC; ++c) x[i][c] = element(in[i], c);
  if (args.gamma) normalize(0, args.gamma, args.beta, x);
#pragma unroll
  for (int i = 0; i < HELD; ++i)
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
      if (args.gate) x[i][c] *= element(gate[i], c);
      x[i][c] = __builtin_fmaf(args.residual_scale, x[i][c], args.residual ? element(residual[i], c) : 0.0f);
    }
  store(args.output, row * args.output_stride, x);
  if (args.next_output) {
    normalize(2, args.next_gamma, args.next_beta, x);
    store(args.next_output, row * args.next_stride, x);
  }
}

typedef void (*Kernel)(BlockNormArgs);

// Threads of a row's group by channels, and the vectors each holds.
template <typename T, int VEC>
Kernel pick(uint32_t channels, uint32_t* group) {
  *group = channels <= 2048u ? 64u : channels <= 8192u ? 256u : 1024u;
  if (channels <= 512u) return block_norm_kernel<T, VEC, 64, 8 / VEC>;
  if (channels <= 1024u) return block_norm_kernel<T, VEC, 64, 16 / VEC>;
  if (channels <= 2048u) return block_norm_kernel<T, VEC, 64, 32 / VEC>;
  if (channels <= 4096u) return block_norm_kernel<T, VEC, 256, 16 / VEC>;
  if (channels <= 8192u) return block_norm_kernel<T, VEC, 256, 32 / VEC>;
  return block_norm_kernel<T, VEC, 1024, 16 / VEC>;
}

}  // namespace

hipError_t launch_block_norm(const BlockNormArgs& args, hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
  const uint32_t elem = args.f16 ? 2u : 4u;
  // 16-byte vectors where every row of every matrix starts on 16 bytes.
  uint64_t bits = (uint64_t)args.channels * elem;
  const auto rows_at = [&](const void* p, uint64_t stride) {
    if (p) bits |= reinterpret_cast<uintptr_t>(p) | stride * elem;
  };
  rows_at(args.input, args.input_stride);
  rows_at(args.gate, args.gate_stride);
  rows_at(args.residual, args.residual_stride);
  rows_at(args.output, args.output_stride);
  rows_at(args.next_output, args.next_stride);
  const bool wide = bits % 16u == 0u;
  uint32_t group = 0;
  const Kernel kernel = args.f16 ? (wide ? pick<_Float16, 8>(args.channels, &group) : pick<_Float16, 1>(args.channels, &group))
                                 : (wide ? pick<float, 4>(args.channels, &group) : pick<float, 1>(args.channels, &group));
  const uint32_t threads = group > (uint32_t)kThreads ? group : (uint32_t)kThreads, each = threads / group;
  const dim3 grid((args.rows + each - 1u) / each), block(threads);
  if (start || stop)
    hipExtLaunchKernelGGL(kernel, grid, block, 0, stream, start, stop, 0, args);
  else
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, args);
  return hipGetLastError();
}

}  // namespace pk
