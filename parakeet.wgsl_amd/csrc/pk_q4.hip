// pk_q4.hip - the product with 4-bit weights and group scales for gfx950
// (include/pk_q4.h has the formula).
//
// The weight lies in blocks of 16 columns x 128 k, the columns of a block
// row by row along K: lane l of a wavefront owns column l & 15 at
// k = 32 i + 8 (l >> 4) + j, word i of its four holding j = 0..7. That is the
// B operand of v_mfma_f32_16x16x32_f16 as it stands, so a block is one
// 16-byte load a lane and four matrix instructions. Within a word the codes
// 2t and 2t + 1 are nibble t of the low and of the high half: one mask takes
// a pair out as two f16 (1024 + code or 1024 + 16 code, whose ulp is a code),
// and one packed operation makes them code - 8.
// Scales follow in the same order, per_block (1, 2 or 4) a column and block.
#include "pk_internal.h"

namespace pk {
namespace {

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;  // wavefronts that share the K blocks of a tile

// Bit of code j (0..7) in its word.
__host__ __device__ constexpr uint32_t nibble_at(uint32_t j) { return 4u * (j >> 1) + 16u * (j & 1u); }

__global__ void layout_codes(const uint32_t* packed, uint32_t* codes, uint32_t inner, uint32_t columns,
                             uint32_t kblocks, uint64_t words) {
  const uint64_t id = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (id >= words) return;
  const uint32_t i = id & 3u, lane = (id >> 2) & 63u;
  const uint64_t block = id >> 8;
  const uint32_t n = (uint32_t)(block / kblocks) * 16u + (lane & 15u);
  const uint32_t k0 = (uint32_t)(block % kblocks) * 128u + 32u * i + 8u * (lane >> 4);
  uint32_t word = 0;
#pragma unroll
  for (uint32_t j = 0; j < 8u; ++j) {
    uint32_t code = 8u;  // the weight 0 behind the edges
    if (n < columns && k0 + j < inner) {
      const uint64_t at = (uint64_t)(k0 + j) * columns + n;
      code = (packed[at >> 3] >> (4u * (uint32_t)(at & 7u))) & 15u;
    }
    word |= code << nibble_at(j);
  }
  codes[id] = word;
}

template <typename T>
__global__ void layout_scales(const T* source, T* target, uint32_t inner, uint32_t columns, uint32_t group,
                              uint32_t kblocks, uint32_t per_block, uint64_t count) {
  const uint64_t id = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (id >= count) return;
  const uint32_t part = (uint32_t)(id % per_block);
  const uint64_t rest = id / per_block;
  const uint64_t block = rest >> 4;
  const uint32_t n = (uint32_t)(block / kblocks) * 16u + (uint32_t)(rest & 15u);
  const uint32_t k = (uint32_t)(block % kblocks) * 128u + part * (128u / per_block);
  target[id] = n < columns && k < inner ? source[(uint64_t)(k / group) * columns + n] : (T)0.0f;
}

// Codes of a word as f16 of code - 8: a[2t], a[2t + 1] from nibble t.
__device__ __forceinline__ half8 decode(uint32_t word) {
  const half2 low = {(_Float16)-1032.0f, (_Float16)-1032.0f}, high = {(_Float16)-72.0f, (_Float16)-72.0f};
  const half2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
  half8 f;
#pragma unroll
  for (int t = 0; t < 4; t += 2) {
    const uint32_t w = word >> (4 * t);
    const half2 p = __builtin_bit_cast(half2, (w & 0x000f000fu) | 0x64006400u) + low;
    const half2 q = __builtin_elementwise_fma(__builtin_bit_cast(half2, (w & 0x00f000f0u) | 0x64006400u), sixteenth, high);
    f[2 * t] = p[0];
    f[2 * t + 1] = p[1];
    f[2 * t + 2] = q[0];
    f[2 * t + 3] = q[1];
  }
  return f;
}

// Eight elements of a row of `a` from k on, zero from K on.
template <typename T>
__device__ __forceinline__ void load_row(const T* row, uint32_t k, uint32_t inner, bool wide, T (&dst)[8]) {
  if (wide && k + 8u <= inner) {
    typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int p = 0; p < 8 / N; ++p) {
      const V v = *reinterpret_cast<const V*>(row + k + N * p);
#pragma unroll
      for (int c = 0; c < N; ++c) dst[N * p + c] = v[c];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) dst[j] = k + j < inner ? row[k + j] : (T)0.0f;
  }
}

// One workgroup: 16 rows x 16 columns, its wavefronts every kWaves-th block.
template <typename T, int PER>
__global__ __launch_bounds__(64 * kWaves) void q4_kernel(Q4Args args, bool wide) {
  __shared__ float partial[kWaves][16][17];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t column = lane & 15u, quad = lane >> 4;
  const uint32_t nb = blockIdx.x, m0 = blockIdx.y * 16u;
  const uint32_t kblocks = (args.inner + 127u) / 128u;
  const T* row = static_cast<const T*>(args.a) + (uint64_t)min(m0 + column, args.rows - 1u) * args.a_stride;
  floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t kb = wave; kb < kblocks; kb += kWaves) {
    const uint64_t block = (uint64_t)nb * kblocks + kb;
    const uint4 words = args.codes[block * 64u + lane];
    const uint32_t w[4] = {words.x, words.y, words.z, words.w};
    floatx4 part = {0.0f, 0.0f, 0.0f, 0.0f}, sums = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T a[8];
      load_row(row, kb * 128u + 32u * i + 8u * quad, args.inner, wide, a);
      const half8 b = decode(w[i]);
      if constexpr (sizeof(T) == 2) {
        half8 av, one;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          av[j] = a[j];
          one[j] = (_Float16)1.0f;
        }
        part = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, b, part, 0, 0, 0);
        if (args.offsets) sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, one, sums, 0, 0, 0);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          part = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], (float)b[j], part, 0, 0, 0);
          if (args.offsets) sums = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], 1.0f, sums, 0, 0, 0);
        }
      }
      if ((i + 1) % (4 / PER) == 0) {  // the end of a group, or of the block
        const uint64_t at = (block * 16u + column) * PER + i / (4 / PER);
        const float scale = (float)static_cast<const T*>(args.scales)[at];
        const float offset = args.offsets ? (float)static_cast<const T*>(args.offsets)[at] : 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[r] = __builtin_fmaf(part[r], scale, acc[r]);
          if (args.offsets) acc[r] = __builtin_fmaf(sums[r], offset, acc[r]);
          part[r] = sums[r] = 0.0f;
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) partial[wave][4 * quad + r][column] = acc[r];
  __syncthreads();
  const uint32_t m = m0 + threadIdx.x / 16u, n = nb * 16u + threadIdx.x % 16u;
  if (m >= args.rows || n >= args.columns) return;
  float v = 0.0f;
#pragma unroll
  for (int p = 0; p < kWaves; ++p) v += partial[p][threadIdx.x / 16u][threadIdx.x % 16u];
  if (args.bias) v += args.bias[n];
  if (args.activation == kActSilu) v = v / (1.0f + __expf(-v));
  else if (args.activation == kActRelu) v = v > 0.0f ? v : (v != v ? v : 0.0f);
  if (args.residual)
    v = __builtin_fmaf(args.residual_scale, v,
                       (float)static_cast<const T*>(args.residual)[(uint64_t)m * args.residual_stride + n]);
  static_cast<T*>(args.out)[(uint64_t)m * args.out_stride + n] = (T)v;
}

}  // namespace

Q4Layout q4_layout(const Q4Args& args, bool offsets) {
  const uint64_t blocks = (uint64_t)((args.inner + 127u) / 128u) * ((args.columns + 15u) / 16u);
  const uint64_t table = (blocks * 16u * args.per_block * (args.f16 ? 2u : 4u) + 255u) / 256u * 256u;
  Q4Layout at;
  at.scales = blocks * 1024u;
  at.offsets = at.scales + table;
  at.bytes = at.offsets + (offsets ? table : 0u);
  return at;
}

hipError_t launch_q4_layout(const Q4Args& args, const uint32_t* packed, const void* scales, const void* offsets,
                            uint32_t group, hipStream_t stream) {
  const uint32_t kblocks = (args.inner + 127u) / 128u;
  const uint64_t blocks = (uint64_t)kblocks * ((args.columns + 15u) / 16u);
  const uint64_t words = blocks * 256u, count = blocks * 16u * args.per_block;
  const auto grid = [](uint64_t n) { return dim3((uint32_t)((n + 255u) / 256u)); };
  hipLaunchKernelGGL(layout_codes, grid(words), dim3(256), 0, stream, packed,
                     reinterpret_cast<uint32_t*>(const_cast<uint4*>(args.codes)), args.inner, args.columns, kblocks,
                     words);
  if (const hipError_t e = hipGetLastError()) return e;
  const void* sources[2] = {scales, offsets};
  void* targets[2] = {const_cast<void*>(args.scales), const_cast<void*>(args.offsets)};
  for (int i = 0; i < 2; ++i) {
    if (!sources[i]) continue;
    if (args.f16)
      hipLaunchKernelGGL(layout_scales<_Float16>, grid(count), dim3(256), 0, stream,
                         static_cast<const _Float16*>(sources[i]), static_cast<_Float16*>(targets[i]), args.inner,
                         args.columns, group, kblocks, args.per_block, count);
    else
      hipLaunchKernelGGL(layout_scales<float>, grid(count), dim3(256), 0, stream,
                         static_cast<const float*>(sources[i]), static_cast<float*>(targets[i]), args.inner,
                         args.columns, group, kblocks, args.per_block, count);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

hipError_t launch_q4(const Q4Args& args, hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
  typedef void (*Kernel)(Q4Args, bool);
  static const Kernel kernels[2][3] = {
      {q4_kernel<float, 1>, q4_kernel<float, 2>, q4_kernel<float, 4>},
      {q4_kernel<_Float16, 1>, q4_kernel<_Float16, 2>, q4_kernel<_Float16, 4>}};
  const Kernel kernel = kernels[args.f16][args.per_block >> 1];
  const uint64_t elem = args.f16 ? 2u : 4u;
  const bool wide = (reinterpret_cast<uintptr_t>(args.a) | args.a_stride * elem) % 16u == 0;
  const dim3 grid((args.columns + 15u) / 16u, (args.rows + 15u) / 16u);
  if (start || stop)
    hipExtLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, stream, start, stop, 0, args, wide);
  else
    hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, stream, args, wide);
  return hipGetLastError();
}

}  // namespace pk
