// pk_block_norm.hip - the norms around a block for gfx950: the norm of the
// block's output, its gate and residual, and the norm of the sum, in one pass
// (include/pk_block_norm.h has the formulas).
//
// Bound by memory: each matrix is read or written once (2 to 5 elements of
// traffic for some 20 operations): 8192 rows of 4096 f16 channels with gate,
// residual and both norms 61.7 us, 5.4 TB/s where a copy reaches 4.9; 3008 of
// 1024 7.4 us (5.0 at that rate). A row lies in the registers of GROUP
// threads, at most 16 channels a thread (one wavefront up to 1024 channels,
// 1024 threads for 16384), as f32 from the first load to the last store, so
// the second norm costs no memory trip, and every load of the row and of both
// norms' parameters is issued before the first sum waits for any. Variances
// are of the differences from the mean, a second sum over registers, since
// E[x^2] - E[x]^2 loses every digit of a row whose mean is far from zero.
// Vectors of 16 bytes load and store at any address of an element (gfx9's
// global memory takes unaligned ones); channels beyond the last whole vector
// are one extra element of the first threads.
#include "pk_internal.h"
#include "pk_wave.h"

namespace pk {
namespace {

constexpr int kThreads = 256;  // of a workgroup whose rows take a wavefront each

template <typename T, int GROUP, int HELD, bool TAIL>
__global__ __launch_bounds__(GROUP == 64 ? kThreads : GROUP) void block_norm_kernel(BlockNormArgs args) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int kWaves = GROUP / 64;
  constexpr bool kLate = GROUP == 1024;  // see normalize
  typedef T V __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));
  __shared__ float partial[4][kWaves];  // a slot for each of the sums: no sum waits for the readers of another
  const uint32_t row = GROUP == 64
                           ? blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6))
                           : blockIdx.x;
  const uint32_t at = threadIdx.x % GROUP;
  if (row >= args.rows) return;  // whole wavefronts
  const uint32_t vectors = args.channels / VEC, tail = TAIL ? args.channels % VEC : 0u;
  const float inverse = 1.0f / (float)args.channels;

  // What a thread holds of a row: HELD vectors, and an element of the tail.
  // Loads are unconditional, of the row's last vector where a thread has no
  // i-th one; sums and stores leave those out.
  struct Raw {
    V v[HELD];
    T edge;
  };
  struct Row {
    float v[HELD][VEC];
    float edge;
  };
  const auto has = [&](int i) { return at + i * GROUP < vectors; };
  const auto place = [&](int i) { return min(at + i * GROUP, vectors - 1u); };
  const bool has_edge = at < tail;
  const uint32_t edge = args.channels - 1u - (has_edge ? at : 0u);
  const auto load = [&](const void* p, uint64_t from) {
    const T* source = static_cast<const T*>(p) + from;
    Raw raw;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      if (TAIL && !vectors) raw.v[i] = (V)(T)0.0f;
      else raw.v[i] = reinterpret_cast<const V*>(source)[place(i)];
    }
    raw.edge = TAIL ? source[edge] : (T)0.0f;
    return raw;
  };
  const auto load_vector = [&](const float* p) {
    Row x;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
#pragma unroll
      for (int f = 0; f < VEC / 4; ++f) {
        F4 q;
        if (TAIL && !vectors) q = (F4)0.0f;
        else q = reinterpret_cast<const F4*>(p)[place(i) * (VEC / 4) + f];
#pragma unroll
        for (int c = 0; c < 4; ++c) x.v[i][4 * f + c] = q[c];
      }
    x.edge = TAIL ? p[edge] : 0.0f;
    return x;
  };
  // The sum of f(x) over the row, the same in every thread of the group.
  const auto total = [&](int slot, auto f, const Row& x) {
    float s = TAIL && has_edge ? f(x.edge) : 0.0f;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      float part = 0.0f;
#pragma unroll
      for (int c = 0; c < VEC; ++c) part += f(x.v[i][c]);
      s += has(i) ? part : 0.0f;
    }
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
  // The parameters are loaded ahead, with the row (loading them behind the
  // sums took 5% to 15% longer at 1 to 8192 rows of 768 to 8192 channels),
  // but for 1024 threads, whose 128 registers do not hold them: 1 to 256 rows
  // of 12000 f32 channels 8.2 to 13.9 us ahead, 6.5 to 12.0 behind.
  const auto normalize = [&](int slot, Row& gamma, Row& beta, const float* gammas, const float* betas, Row& x) {
    float mean = 0.0f;
    if (!args.rms) mean = total(slot, [](float v) { return v; }, x) * inverse;
    const float power = total(slot + 1, [mean](float v) { return (v - mean) * (v - mean); }, x) * inverse;
    const float scale = 1.0f / __builtin_sqrtf(power + args.epsilon);
    if constexpr (kLate) {
      gamma = load_vector(gammas);
      if (betas) beta = load_vector(betas);
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i)
#pragma unroll
      for (int c = 0; c < VEC; ++c)
        x.v[i][c] = __builtin_fmaf((x.v[i][c] - mean) * scale, gamma.v[i][c], beta.v[i][c]);
    x.edge = __builtin_fmaf((x.edge - mean) * scale, gamma.edge, beta.edge);
  };
  const auto store = [&](void* p, uint64_t from, const Row& x) {
    T* target = static_cast<T*>(p) + from;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      if (!has(i)) continue;
      V v;
#pragma unroll
      for (int c = 0; c < VEC; ++c) v[c] = (T)x.v[i][c];
      reinterpret_cast<V*>(target)[at + i * GROUP] = v;
    }
    if (TAIL && has_edge) target[edge] = (T)x.edge;
  };

  const Raw in = load(args.input, row * args.input_stride);
  Raw residual, gate;
  if (args.residual) residual = load(args.residual, row * args.residual_stride);
  if (args.gate) gate = load(args.gate, (args.gate_rows ? row / args.gate_rows : 0u) * args.gate_stride);
  Row gamma, beta = {}, next_gamma, next_beta = {};
  if constexpr (!kLate) {
    if (args.gamma) gamma = load_vector(args.gamma);
    if (args.beta) beta = load_vector(args.beta);
    if (args.next_output) next_gamma = load_vector(args.next_gamma);
    if (args.next_beta) next_beta = load_vector(args.next_beta);
  }
  Row x;
#pragma unroll
  for (int i = 0; i < HELD; ++i)
#pragma unroll
    for (int c = 0; c < VEC; ++c) x.v[i][c] = (float)in.v[i][c];
  x.edge = (float)in.edge;
  if (args.gamma) normalize(0, gamma, beta, args.gamma, args.beta, x);
  if (args.gate) {
#pragma unroll
    for (int i = 0; i < HELD; ++i)
#pragma unroll
      for (int c = 0; c < VEC; ++c) x.v[i][c] *= (float)gate.v[i][c];
    x.edge *= (float)gate.edge;
  }
  const float scale = args.residual_scale;
  if (args.residual) {
#pragma unroll
    for (int i = 0; i < HELD; ++i)
#pragma unroll
      for (int c = 0; c < VEC; ++c) x.v[i][c] = __builtin_fmaf(scale, x.v[i][c], (float)residual.v[i][c]);
    x.edge = __builtin_fmaf(scale, x.edge, (float)residual.edge);
  } else {
#pragma unroll
    for (int i = 0; i < HELD; ++i)
#pragma unroll
      for (int c = 0; c < VEC; ++c) x.v[i][c] *= scale;
    x.edge *= scale;
  }
  store(args.output, row * args.output_stride, x);
  if (args.next_output) {
    normalize(2, next_gamma, next_beta, args.next_gamma, args.next_beta, x);
    store(args.next_output, row * args.next_stride, x);
  }
}

typedef void (*Kernel)(BlockNormArgs);

// The kernel for rows of `channels`, and the threads of a row.
template <typename T, bool TAIL>
Kernel pick(uint32_t channels, uint32_t* group) {
  constexpr int VEC = 16 / sizeof(T);
  *group = channels <= 1024u ? 64u : channels <= 2048u ? 128u : channels <= 4096u ? 256u : channels <= 8192u ? 512u
                                                                                                             : 1024u;
  if (channels <= 512u) return block_norm_kernel<T, 64, 8 / VEC, TAIL>;
  if (channels <= 1024u) return block_norm_kernel<T, 64, 16 / VEC, TAIL>;
  if (channels <= 2048u) return block_norm_kernel<T, 128, 16 / VEC, TAIL>;
  if (channels <= 4096u) return block_norm_kernel<T, 256, 16 / VEC, TAIL>;
  if (channels <= 8192u) return block_norm_kernel<T, 512, 16 / VEC, TAIL>;
  return block_norm_kernel<T, 1024, 16 / VEC, TAIL>;
}
template <typename T>
Kernel pick(uint32_t channels, uint32_t* group) {
  return channels % (16 / sizeof(T)) ? pick<T, true>(channels, group) : pick<T, false>(channels, group);
}

}  // namespace

hipError_t launch_block_norm(const BlockNormArgs& args, hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
  uint32_t group = 0;
  const Kernel kernel = args.f16 ? pick<_Float16>(args.channels, &group) : pick<float>(args.channels, &group);
  const uint32_t threads = group == 64u ? (uint32_t)kThreads : group, each = threads / group;
  const dim3 grid((args.rows + each - 1u) / each), block(threads);
  if (start || stop)
    hipExtLaunchKernelGGL(kernel, grid, block, 0, stream, start, stop, 0, args);
  else
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, args);
  return hipGetLastError();
}

}  // namespace pk
