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
//
// One row is bound by the weight's bytes: 1 x 4096 x 8192 5.7 us (3.5 at the
// rate of a copy, 4.9 TB/s). From some 32 rows on it is the instructions: a
// SIMD issues a matrix instruction (8.05 ns) or an fma (1.25 ns) but hardly
// both at once, one and 8 fma take 17.1 ns, so that decoding and scaling
// count in full: per 32 k and 16 columns 9 and, once a group, 16 operations
// for 4 matrix instructions. 64 x 8192 x 8192 with offsets 24.2 us, of which
// 10.2 are these instructions and the rest waits for rows and codes; 1504 x
// 1024 x 4096 20.1 us, 0.63 PFLOP/s, and x 4096 x 4096 60 us, 0.84.
#include "pk_internal.h"
#include "pk_wave.h"

namespace pk {
namespace {

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

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

// The constants of decode in registers: as literals each pair would take two
// instructions (and, or) where one has three operands.
struct Decoder {
  uint32_t low = 0x000f000fu, high = 0x00f000f0u, base = 0x64006400u;
  __device__ __forceinline__ Decoder() {
    asm("" : "+s"(low));
    asm("" : "+s"(high));
    asm("" : "+v"(base));
  }
  // Codes of a word as f16 of code - 8: f[2t], f[2t + 1] from nibble t.
  __device__ __forceinline__ half8 operator()(uint32_t word) const {
    const half2 minus_1032 = (half2)(_Float16)-1032.0f, minus_72 = (half2)(_Float16)-72.0f;
    half8 f;
#pragma unroll
    for (int t = 0; t < 4; t += 2) {
      const uint32_t w = word >> (4 * t);
      const half2 p = __builtin_bit_cast(half2, (w & low) | base) + minus_1032;
      const half2 q = __builtin_elementwise_fma(__builtin_bit_cast(half2, (w & high) | base),
                                                (half2)(_Float16)0.0625f, minus_72);
      f[2 * t] = p[0];
      f[2 * t + 1] = p[1];
      f[2 * t + 2] = q[0];
      f[2 * t + 3] = q[1];
    }
    return f;
  }
};

// 16 bytes of a row of `a`.
template <typename T>
struct Chunk {
  static constexpr int N = 16 / sizeof(T);
  typedef T V __attribute__((ext_vector_type(N)));
  V v;
  typedef T U __attribute__((ext_vector_type(N), aligned(sizeof(T))));  // at any address of an element
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const U*>(p); }
  // p[0] is element k of a row; what lies from K on is zero. Without a branch
  // for each chunk, which would have it wait for the one before: the row's
  // last 16 bytes, shifted by what lies behind K (64 x 1000 x 1000 7.4 us, with a
  // branch for each 9.3).
  __device__ __forceinline__ void load(const T* p, uint32_t k, uint32_t inner) {
    if (inner < (uint32_t)N) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = k + j < inner ? p[j] : (T)0.0f;
      return;
    }
    const uint32_t behind = k + N > inner ? k + N - inner : 0u;
    load(p - behind);
    typedef uint64_t words __attribute__((ext_vector_type(2)));
    const words w = __builtin_bit_cast(words, v);
    const uint32_t bits = behind * (8u * sizeof(T)), part = bits & 63u;
    const uint64_t low = bits < 64u ? w[0] : w[1], high = bits < 64u ? w[1] : 0u;
    const words shifted = {low >> part | (high << 1) << (63u - part), high >> part};
    v = __builtin_bit_cast(V, bits < 128u ? shifted : (words)0);
  }
};

// Eight elements of a row in k order: a lane's operand of 32 k.
template <typename T>
struct Fragment {
  Chunk<T> c[8 / Chunk<T>::N];
};

// acc += a . b over 32 k.
__device__ __forceinline__ void multiply(const Fragment<_Float16>& a, const half8& b, floatx4& acc) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.c[0].v, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void multiply(const Fragment<float>& a, const half8& b, floatx4& acc) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.c[j / 4].v[j % 4], (float)b[j], acc, 0, 0, 0);
}

// acc[mt][nt] += a[mt] . b; one f32 instruction waits for the one whose sum it
// adds to, so those of a k go before the next k.
template <int MT, int NT>
__device__ __forceinline__ void multiply(const Fragment<_Float16> (&a)[MT], const half8& b, floatx4 (&acc)[MT][NT],
                                         int nt) {
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) multiply(a[mt], b, acc[mt][nt]);
}
template <int MT, int NT>
__device__ __forceinline__ void multiply(const Fragment<float> (&a)[MT], const half8& b, floatx4 (&acc)[MT][NT],
                                         int nt) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      acc[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[mt].c[j / 4].v[j % 4], (float)b[j], acc[mt][nt], 0, 0, 0);
}

// The sums of 16 rows over the k of a group, in each lane those of its four
// rows of output: a product with ones. f32: a lane adds what it holds and one
// instruction a group adds the lanes, where a product would take eight for
// each 32 k (1504 x 1024 x 4096, groups of 32: 130 us, 161 with those).
template <typename T>
struct RowSums;
template <>
struct RowSums<_Float16> {
  floatx4 s;
  __device__ __forceinline__ void clear() { s = (floatx4)0.0f; }
  __device__ __forceinline__ void add(const Fragment<_Float16>& a) { multiply(a, (half8)(_Float16)1.0f, s); }
  __device__ __forceinline__ floatx4 total() const { return s; }
};
template <>
struct RowSums<float> {
  float s;
  __device__ __forceinline__ void clear() { s = 0.0f; }
  __device__ __forceinline__ void add(const Fragment<float>& a) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s += a.c[j / 4].v[j % 4];
  }
  __device__ __forceinline__ floatx4 total() const {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(s, 1.0f, (floatx4)0.0f, 0, 0, 0);
  }
};

// The activation of one output.
__device__ __forceinline__ float activate(int activation, float v) {
  if (activation == kActSilu) return v * __builtin_amdgcn_rcpf(1.0f + __expf(-v));
  if (activation == kActRelu) return v > 0.0f ? v : (v != v ? v : 0.0f);
  return v;
}

// What an output adds: its bias and residual.
struct Extra {
  float bias = 0.0f, residual = 0.0f;
};
template <typename T>
__device__ __forceinline__ Extra load_extra(const Q4Args& args, uint32_t m, uint32_t n) {
  Extra e;
  if (args.bias) e.bias = args.bias[n];
  if (args.residual) e.residual = (float)static_cast<const T*>(args.residual)[(uint64_t)m * args.residual_stride + n];
  return e;
}
// bias, activation and residual of one output, stored.
template <typename T>
__device__ __forceinline__ void finish(const Q4Args& args, uint32_t m, uint32_t n, float v, const Extra& e) {
  v = activate(args.activation, args.bias ? v + e.bias : v);
  if (args.residual) v = __builtin_fmaf(args.residual_scale, v, e.residual);
  static_cast<T*>(args.out)[(uint64_t)m * args.out_stride + n] = (T)v;
}

// The same for 8 columns from n on, those behind the edge left out.
template <typename T>
__device__ __forceinline__ void finish_row(const Q4Args& args, uint32_t m, uint32_t n, float (&v)[8]) {
  constexpr int N = Chunk<T>::N;
  typedef float F __attribute__((ext_vector_type(4), aligned(4)));
  if (n + 8u > args.columns) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n + j < args.columns) finish<T>(args, m, n + j, v[j], load_extra<T>(args, m, n + j));
    return;
  }
  if (args.bias) {
    const F lo = *reinterpret_cast<const F*>(args.bias + n), hi = *reinterpret_cast<const F*>(args.bias + n + 4u);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += j < 4 ? lo[j] : hi[j - 4];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = activate(args.activation, v[j]);
#pragma unroll
  for (int p = 0; p < 8; p += N) {
    Chunk<T> x;
    if (args.residual) {
      x.load(static_cast<const T*>(args.residual) + (uint64_t)m * args.residual_stride + n + p);
#pragma unroll
      for (int j = 0; j < N; ++j) v[p + j] = __builtin_fmaf(args.residual_scale, v[p + j], (float)x.v[j]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) x.v[j] = (T)v[p + j];
    *reinterpret_cast<typename Chunk<T>::U*>(static_cast<T*>(args.out) + (uint64_t)m * args.out_stride + n + p) = x.v;
  }
}

// LDS bytes of the rows of `a` in a panel kernel.
constexpr uint32_t kPanelBytes = 80u * 1024u;
// Elements from row to row of the panel: whole blocks of K and 16 bytes, so
// that the rows of a fragment lie in different banks.
template <typename T>
__host__ __device__ constexpr uint32_t panel_stride(uint32_t inner) {
  return (inner + 127u) / 128u * 128u + 16u / sizeof(T);
}

// Copies all rows of `a` into LDS, zeros behind K, four chunks a thread at a
// time.
template <typename T>
__device__ __forceinline__ void copy_panel(const Q4Args& args, void* lds) {
  constexpr uint32_t kChunks = 128u / Chunk<T>::N;
  const uint32_t chunks = (args.inner + 127u) / 128u * kChunks;
  // Thread and step as rows and chunks; one row needs no division.
  uint32_t r = 0u, c = threadIdx.x, step_rows = 0u, step = blockDim.x;
  if (args.rows > 1u) {
    r = threadIdx.x / chunks;
    c = threadIdx.x % chunks;
    step_rows = blockDim.x / chunks;
    step = blockDim.x % chunks;
  }
  while (r < args.rows) {
    Chunk<T> x[4];
    uint32_t to[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const bool has = r < args.rows && c < chunks;
      to[t] = has ? r * panel_stride<T>(args.inner) + c * Chunk<T>::N : ~0u;
      if (has) {  // the shift only where K ends: 16 x 1024 x 4096 4.1 us, 5.2 with it in every chunk
        const T* from = static_cast<const T*>(args.a) + r * args.a_stride + c * Chunk<T>::N;
        if ((c + 1u) * Chunk<T>::N <= args.inner) x[t].load(from);
        else x[t].load(from, c * Chunk<T>::N, args.inner);
      }
      r += step_rows;
      c += step;
      if (c >= chunks) {
        c -= min(c, chunks);
        ++r;
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (to[t] != ~0u) *reinterpret_cast<Chunk<T>*>(static_cast<T*>(lds) + to[t]) = x[t];
  }
}

// Wavefronts of a workgroup: as many as have registers for what they hold.
template <typename T, int MT, int NT, bool PANEL>
__host__ __device__ constexpr int most_waves() {
  return MT * NT >= 4 || (sizeof(T) == 4 && !PANEL) ? 8 : 16;
}

// Few rows. One workgroup: up to 16 MT rows x 16 NT columns; its wavefronts
// take every W-th block of K and their sums meet in LDS, so no memory is
// shared between workgroups. Codes and scales are loaded two blocks ahead.
// Fragments are read from LDS, since loaded as they are the lanes of one
// instruction touch 16 rows four times over: PANEL copies the rows whole
// before the first block, otherwise each wavefront copies its own block of
// 128 k, loaded a block ahead, through an area of its own.
template <typename T, int PER, int MT, int NT, bool OFFSETS, bool PANEL>
__global__ __launch_bounds__((64 * most_waves<T, MT, NT, PANEL>())) void q4_rows_kernel(Q4Args args) {
  constexpr int kMost = most_waves<T, MT, NT, PANEL>();
  constexpr int kStep = 4 / PER;           // matrix instructions of a group
  constexpr int kChunks = 128 / Chunk<T>::N;        // of a row and block
  constexpr int kStage = 16 * MT * kChunks;         // of a wavefront's area
  constexpr int kCopies = kStage / 64;              // chunks a lane copies
  constexpr uint32_t kRowsBytes = PANEL ? kPanelBytes : kMost * kStage * 16u;
  constexpr uint32_t kSumsBytes = kMost * 16 * MT * (16 * NT + 1) * 4u;
  __shared__ uint4 lds[(kRowsBytes > kSumsBytes ? kRowsBytes : kSumsBytes) / 16u];
  const uint32_t lane = threadIdx.x & 63u, waves = blockDim.x >> 6;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));  // addresses stay scalar
  const uint32_t column = lane & 15u, quad = lane >> 4;
  const uint32_t m0 = blockIdx.y * (16u * MT);
  const uint32_t kblocks = (args.inner + 127u) / 128u, nblocks = (args.columns + 15u) / 16u;
  typedef T S __attribute__((ext_vector_type(PER == 1 ? 2 : PER)));  // a column's scales of a block

  uint64_t base[NT];  // first block of each column block (the last one again behind the edge)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) base[nt] = (uint64_t)min(blockIdx.x * NT + nt, nblocks - 1u) * kblocks;
  struct Weight {
    uint4 codes[NT];
    S scales[NT], offsets[NT];
  };
  const auto load_weight = [&](uint32_t kb, Weight& w) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint64_t block = base[nt] + kb;
      w.codes[nt] = (args.codes + block * 64u)[lane];
      const T* scales = static_cast<const T*>(args.scales) + block * (16u * PER);
      const T* offsets = static_cast<const T*>(args.offsets) + block * (16u * PER);
      if constexpr (PER == 1) {
        w.scales[nt][0] = scales[column];
        if (OFFSETS) w.offsets[nt][0] = offsets[column];
      } else {
        w.scales[nt] = reinterpret_cast<const S*>(scales)[column];
        if (OFFSETS) w.offsets[nt] = reinterpret_cast<const S*>(offsets)[column];
      }
    }
  };

  // A wavefront's block of rows: chunk c of row r lies at c ^ (r & 15), which
  // spreads the 16 rows of a fragment over the banks.
  Chunk<T>* stage = reinterpret_cast<Chunk<T>*>(lds) + (PANEL ? 0 : wave * kStage);
  Chunk<T> copy[PANEL ? 1 : kCopies];
  const T* tile = static_cast<const T*>(args.a) + (uint64_t)m0 * args.a_stride;
  uint32_t from[PANEL ? 1 : kCopies];  // of a chunk in the tile's rows, in elements from the block's first
  if constexpr (!PANEL)
#pragma unroll
    for (int t = 0; t < kCopies; ++t) {
      const uint32_t id = t * 64u + lane, r = id / kChunks, c = (id % kChunks) ^ (r & 15u);
      from[t] = (min(m0 + r, args.rows - 1u) - m0) * (uint32_t)args.a_stride + c * Chunk<T>::N;
    }
  const auto load_rows = [&](uint32_t kb) {
    const T* block = tile + kb * 128u;
    if (kb * 128u + 128u <= args.inner) {
#pragma unroll
      for (int t = 0; t < kCopies; ++t) copy[t].load(block + from[t]);
    } else {
#pragma unroll
      for (int t = 0; t < kCopies; ++t) {
        const uint32_t id = t * 64u + lane, c = (id % kChunks) ^ ((id / kChunks) & 15u);
        copy[t].load(block + from[t], kb * 128u + c * Chunk<T>::N, args.inner);
      }
    }
  };
  // Fragment of the 16 rows mt, step i of block kb.
  const auto fragment = [&](uint32_t kb, int i, int mt) {
    Fragment<T> f;
    constexpr int kParts = 8 / Chunk<T>::N;
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      if constexpr (PANEL) {
        const uint32_t r = min(column, args.rows - 1u);
        f.c[p] = *reinterpret_cast<const Chunk<T>*>(reinterpret_cast<const T*>(lds) + r * panel_stride<T>(args.inner) +
                                                    kb * 128u + 32u * i + 8u * quad + p * Chunk<T>::N);
      } else {
        const uint32_t r = 16u * mt + column, c = (4u * i + quad) * kParts + p;
        f.c[p] = stage[r * kChunks + (c ^ (r & 15u))];
      }
    }
    return f;
  };

  // Workgroups of an XCD (every eighth) start at different blocks of K, so
  // that they do not all ask its L2 for the same lines: 3% to 8% at 16 to 64
  // rows of 4096 and 8192.
  const uint32_t shift = PANEL ? 0u : (blockIdx.x >> 3) % kblocks;
  const auto turned = [&](uint32_t kb) { return kb + shift < kblocks ? kb + shift : kb + shift - kblocks; };
  Weight ahead[2];
  if constexpr (PANEL) {
    copy_panel<T>(args, lds);  // m0 is 0: a panel has at most 16 rows
  } else {
    if (wave < kblocks) load_rows(turned(wave));
  }
  if (wave < kblocks) load_weight(turned(wave), ahead[0]);
  if (wave + waves < kblocks) load_weight(turned(wave + waves), ahead[1]);
  if constexpr (PANEL) __syncthreads();

  floatx4 acc[MT][NT], part[MT][NT];
  RowSums<T> sums[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = (floatx4)0.0f;
  const Decoder decode;

  for (uint32_t kb = wave; kb < kblocks; kb += waves) {
    const Weight w = ahead[0];
    ahead[0] = ahead[1];
    if (kb + 2u * waves < kblocks) load_weight(turned(kb + 2u * waves), ahead[1]);
    if constexpr (!PANEL) {
#pragma unroll
      for (int t = 0; t < kCopies; ++t) stage[t * 64u + lane] = copy[t];
      wave::sync();  // a lane reads what others copied
      if (kb + waves < kblocks) load_rows(turned(kb + waves));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      Fragment<T> a[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) a[mt] = fragment(kb, i, mt);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const half8 b = decode(reinterpret_cast<const uint32_t(&)[4]>(w.codes[nt])[i]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          if (i % kStep == 0) part[mt][nt] = (floatx4)0.0f;  // the first of a group adds to the constant
          multiply(a[mt], b, part[mt][nt]);
        }
      }
      if constexpr (OFFSETS)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          if (i % kStep == 0) sums[mt].clear();
          sums[mt].add(a[mt]);
        }
      if ((i + 1) % kStep == 0) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          floatx4 sum;
          if constexpr (OFFSETS) sum = sums[mt].total();
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              acc[mt][nt][r] = __builtin_fmaf(part[mt][nt][r], (float)w.scales[nt][i / kStep], acc[mt][nt][r]);
              if (OFFSETS)
                acc[mt][nt][r] = __builtin_fmaf(sum[r], (float)w.offsets[nt][i / kStep], acc[mt][nt][r]);
            }
        }
      }
    }
    if constexpr (!PANEL) wave::sync();  // every lane has read, and the next block is copied
  }
  float* partial = reinterpret_cast<float*>(lds);  // [waves][16 MT][16 NT + 1]
  constexpr int kWidth = 16 * NT + 1;
  __syncthreads();  // every wavefront has read its rows
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        partial[(wave * 16u * MT + 16 * mt + 4 * quad + r) * kWidth + 16 * nt + column] = acc[mt][nt][r];
  __syncthreads();
  const uint32_t outputs = min(args.rows - m0, 16u * MT) * (16u * NT);
  // kBatch outputs a thread at a time, whose residuals are under way together.
  constexpr uint32_t kBatch = MT == 1 ? 1u : 4u;
  for (uint32_t from = threadIdx.x; from < outputs; from += kBatch * blockDim.x) {
    Extra extra[kBatch];
    bool has[kBatch];
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b) {
      const uint32_t id = from + b * blockDim.x, n = blockIdx.x * (16u * NT) + id % (16u * NT);
      has[b] = id < outputs && n < args.columns;
      if (has[b]) extra[b] = load_extra<T>(args, m0 + id / (16u * NT), n);
    }
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b) {
      if (!has[b]) continue;
      const uint32_t id = from + b * blockDim.x, m = id / (16u * NT), n = id % (16u * NT);
      float v = 0.0f;
#pragma unroll 4
      for (uint32_t w = 0; w < waves; ++w) v += partial[(w * 16u * MT + m) * kWidth + n];
      finish<T>(args, m0 + m, blockIdx.x * (16u * NT) + n, v, extra[b]);
    }
  }
}

// One to four f32 rows on the VALU: a matrix instruction of f32 operands takes
// 32 cycles for 4 k whatever the rows, an fma that reads its weight as f16
// (v_fma_mix_f32) 4 for each row. The rows lie in LDS whole, a lane
// multiplies the codes of its column and quarter of 32 k, and the quarters
// and wavefronts meet at the end.
template <int PER, int ROWS, bool OFFSETS>
__global__ __launch_bounds__(1024) void q4_vector_kernel(Q4Args args) {
  constexpr int kStep = 4 / PER;
  __shared__ uint4 lds[kPanelBytes / 16u];
  const uint32_t lane = threadIdx.x & 63u, waves = blockDim.x >> 6;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t column = lane & 15u, quad = lane >> 4;
  const uint32_t kblocks = (args.inner + 127u) / 128u;
  const uint64_t base = (uint64_t)blockIdx.x * kblocks;
  const uint32_t stride = panel_stride<float>(args.inner);
  typedef float S __attribute__((ext_vector_type(PER == 1 ? 2 : PER)));
  struct Weight {
    uint4 codes;
    S scales, offsets;
  };
  const auto load_weight = [&](uint32_t kb, Weight& w) {
    w.codes = (args.codes + (base + kb) * 64u)[lane];
    const float* scales = static_cast<const float*>(args.scales) + (base + kb) * (16u * PER);
    const float* offsets = static_cast<const float*>(args.offsets) + (base + kb) * (16u * PER);
    if constexpr (PER == 1) {
      w.scales[0] = scales[column];
      if (OFFSETS) w.offsets[0] = offsets[column];
    } else {
      w.scales = reinterpret_cast<const S*>(scales)[column];
      if (OFFSETS) w.offsets = reinterpret_cast<const S*>(offsets)[column];
    }
  };
  copy_panel<float>(args, lds);
  Weight ahead[2];
  if (wave < kblocks) load_weight(wave, ahead[0]);
  if (wave + waves < kblocks) load_weight(wave + waves, ahead[1]);
  __syncthreads();

  const Decoder decode;
  const float* rows = reinterpret_cast<const float*>(lds) + 8u * quad;
  float acc[ROWS] = {}, part[ROWS], sums[ROWS];
  for (uint32_t kb = wave; kb < kblocks; kb += waves) {
    const Weight w = ahead[0];
    ahead[0] = ahead[1];
    if (kb + 2u * waves < kblocks) load_weight(kb + 2u * waves, ahead[1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const half8 b = decode(reinterpret_cast<const uint32_t(&)[4]>(w.codes)[i]);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const Chunk<float>* from = reinterpret_cast<const Chunk<float>*>(
            rows + min((uint32_t)r, args.rows - 1u) * stride + kb * 128u + 32u * i);
        const Chunk<float> a[2] = {from[0], from[1]};
        if (i % kStep == 0) part[r] = sums[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          part[r] = __builtin_fmaf(a[j / 4].v[j % 4], (float)b[j], part[r]);
          if (OFFSETS) sums[r] += a[j / 4].v[j % 4];
        }
        if ((i + 1) % kStep == 0) {
          acc[r] = __builtin_fmaf(part[r], w.scales[i / kStep], acc[r]);
          if (OFFSETS) acc[r] = __builtin_fmaf(sums[r], w.offsets[i / kStep], acc[r]);
        }
      }
    }
  }
  float* partial = reinterpret_cast<float*>(lds);  // [waves][ROWS][16]
  __syncthreads();                                 // every wavefront has read its rows
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    acc[r] += __shfl_xor(acc[r], 16, 64);
    acc[r] += __shfl_xor(acc[r], 32, 64);
    if (quad == 0) partial[(wave * ROWS + r) * 16u + column] = acc[r];
  }
  __syncthreads();
  for (uint32_t id = threadIdx.x; id < args.rows * 16u; id += blockDim.x) {
    const uint32_t m = id / 16u, n = blockIdx.x * 16u + id % 16u;
    if (n >= args.columns) continue;
    float v = 0.0f;
#pragma unroll 4
    for (uint32_t w = 0; w < waves; ++w) v += partial[(w * ROWS + m) * 16u + id % 16u];
    finish<float>(args, m, n, v, load_extra<float>(args, m, n));
  }
}

// Many rows. One workgroup: 64 rows x 128 columns, a wavefront 32 of the
// columns. The rows go through LDS, a block of 128 k at a time in two
// buffers; codes go from memory to registers, where each wavefront makes its
// own operands of them: 9 VALU operations per 4 matrix instructions, beside
// the 16 that a group's scales take for each 16 columns. Of few tiles
// blockIdx.y is a part of K, whose sums go to a workspace as they lie in the
// lanes, and a second launch adds the parts in their order.
constexpr int kTileRows = 64, kTileColumns = 128;
constexpr uint32_t kTileVectors = kTileRows * kTileColumns / 4;  // of a lane's four rows
constexpr uint32_t kMostSplitTiles = 256;  // one for each compute unit: more are not split along K
template <typename T, int PER, bool OFFSETS>
__global__ __launch_bounds__(256, OFFSETS || sizeof(T) == 4 ? 2 : 3) void q4_tile_kernel(Q4Args args) {
  constexpr int kStep = 4 / PER;
  constexpr int kChunks = 128 / Chunk<T>::N, kCopies = kTileRows * kChunks / 256;
  constexpr int kWidth = 32 + 4;  // f32 columns of a wavefront's part on its way out
  typedef T S __attribute__((ext_vector_type(PER == 1 ? 2 : PER)));
  __shared__ uint4 lds[2][kTileRows * kChunks];
  static_assert(sizeof(lds) >= 4 * 32 * kWidth * sizeof(float), "the outputs pass through the rows' buffers");
  const uint32_t lane = threadIdx.x & 63u, column = lane & 15u, quad = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t kblocks = (args.inner + 127u) / 128u, nblocks = (args.columns + 15u) / 16u;
  // Workgroups of one XCD (every eighth) take neighbouring tiles of one
  // column of tiles: its weights stay in their L2.
  const uint32_t row_tiles = (args.rows + kTileRows - 1u) / kTileRows;
  const uint32_t id = xcd_local_order(blockIdx.x, gridDim.x);
  const uint32_t m0 = id % row_tiles * kTileRows, n0 = id / row_tiles * kTileColumns;
  const uint32_t wn = wave * 32u;

  uint64_t base[2];
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) base[nt] = (uint64_t)min((n0 + wn) / 16u + nt, nblocks - 1u) * kblocks;
  struct Weight {
    uint4 codes[2];
    S scales[2], offsets[2];
  };
  const auto load_weight = [&](uint32_t kb, Weight& w) {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const uint64_t block = base[nt] + kb;
      w.codes[nt] = (args.codes + block * 64u)[lane];
      const T* scales = static_cast<const T*>(args.scales) + block * (16u * PER);
      const T* offsets = static_cast<const T*>(args.offsets) + block * (16u * PER);
      if constexpr (PER == 1) {
        w.scales[nt][0] = scales[column];
        if (OFFSETS) w.offsets[nt][0] = offsets[column];
      } else {
        w.scales[nt] = reinterpret_cast<const S*>(scales)[column];
        if (OFFSETS) w.offsets[nt] = reinterpret_cast<const S*>(offsets)[column];
      }
    }
  };
  const T* tile = static_cast<const T*>(args.a) + (uint64_t)m0 * args.a_stride;
  uint32_t from[kCopies];
#pragma unroll
  for (int t = 0; t < kCopies; ++t) {
    const uint32_t at = t * 256u + threadIdx.x, r = at / kChunks, c = (at % kChunks) ^ (r & 15u);
    from[t] = (min(m0 + r, args.rows - 1u) - m0) * (uint32_t)args.a_stride + c * Chunk<T>::N;
  }
  Chunk<T> copy[kCopies];
  const auto load_rows = [&](uint32_t kb) {
    const T* block = tile + kb * 128u;
#pragma unroll
    for (int t = 0; t < kCopies; ++t) copy[t].load(block + from[t]);
  };
  const auto load_last_rows = [&](uint32_t kb) {  // K ends within this block
    const T* block = tile + kb * 128u;
#pragma unroll
    for (int t = 0; t < kCopies; ++t) {
      const uint32_t at = t * 256u + threadIdx.x, c = (at % kChunks) ^ ((at / kChunks) & 15u);
      copy[t].load(block + from[t], kb * 128u + c * Chunk<T>::N, args.inner);
    }
  };
  const auto store_rows = [&](int buffer) {
#pragma unroll
    for (int t = 0; t < kCopies; ++t) reinterpret_cast<Chunk<T>*>(lds[buffer])[t * 256u + threadIdx.x] = copy[t];
  };

  const Decoder decode;
  floatx4 acc[4][2];
#pragma unroll
  for (int mt = 0; mt < 4; ++mt)
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) acc[mt][nt] = (floatx4)0.0f;

  const auto multiply_block = [&](uint32_t kb, const Weight& w) {
    const Chunk<T>* rows = reinterpret_cast<const Chunk<T>*>(lds[kb & 1u]);
    floatx4 part[4][2];
    RowSums<T> sums[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      Fragment<T> a[4];
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const uint32_t r = 16u * mt + column;
        constexpr int kParts = 8 / Chunk<T>::N;
#pragma unroll
        for (int p = 0; p < kParts; ++p) a[mt].c[p] = rows[r * kChunks + (((4u * i + quad) * kParts + p) ^ column)];
      }
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const half8 b = decode(reinterpret_cast<const uint32_t(&)[4]>(w.codes[nt])[i]);
        if (i % kStep == 0)
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) part[mt][nt] = (floatx4)0.0f;
        multiply(a, b, part, nt);
      }
      if constexpr (OFFSETS)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          if (i % kStep == 0) sums[mt].clear();
          sums[mt].add(a[mt]);
        }
      if ((i + 1) % kStep == 0) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          floatx4 sum;
          if constexpr (OFFSETS) sum = sums[mt].total();
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              acc[mt][nt][r] = __builtin_fmaf(part[mt][nt][r], (float)w.scales[nt][i / kStep], acc[mt][nt][r]);
              if (OFFSETS)
                acc[mt][nt][r] = __builtin_fmaf(sum[r], (float)w.offsets[nt][i / kStep], acc[mt][nt][r]);
            }
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // one step's operands at a time in registers
    }
  };
  // This part's whole blocks, the next one's loads under way while one is
  // multiplied, then the block that K ends in.
  const uint32_t first = blockIdx.y * args.span, last = min(first + args.span, kblocks);
  const uint32_t whole = min(args.inner / 128u, last);
  Weight w, next;
  load_weight(first, w);
  if (whole > first) load_rows(first);
  else load_last_rows(first);
  store_rows(first & 1u);
  __syncthreads();
  for (uint32_t kb = first; kb + 1u < whole; ++kb) {
    load_rows(kb + 1u);
    load_weight(kb + 1u, next);
    multiply_block(kb, w);
    store_rows((kb + 1u) & 1u);
    w = next;
    __syncthreads();
  }
  if (whole > first && last > whole) {
    load_last_rows(whole);
    load_weight(whole, next);
    multiply_block(whole - 1u, w);
    store_rows(whole & 1u);
    w = next;
    __syncthreads();
  }
  multiply_block(last - 1u, w);
  if (gridDim.y > 1u) {
    floatx4* sums = reinterpret_cast<floatx4*>(args.parts) + ((uint64_t)blockIdx.y * gridDim.x + id) * kTileVectors;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) sums[(wave * 8u + 2 * mt + nt) * 64u + lane] = acc[mt][nt];
    return;
  }
  __syncthreads();

  // Out through LDS, 32 rows at a time, so that a lane stores 8 columns.
  float* part_out = reinterpret_cast<float*>(lds) + wave * (32 * kWidth);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          part_out[(16 * mt + 4 * quad + r) * kWidth + 16 * nt + column] = acc[2 * half + mt][nt][r];
    wave::sync();
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      const uint32_t r = 16u * pass + (lane >> 2), c = 8u * (lane & 3u);
      const uint32_t m = m0 + 32u * half + r, n = n0 + wn + c;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = part_out[r * kWidth + c + j];
      if (m < args.rows) finish_row<T>(args, m, n, v);
    }
    wave::sync();
  }
}

// Adds the parts of tiles split along K, four rows of a column a thread.
template <typename T>
__global__ __launch_bounds__(256) void q4_join_kernel(Q4Args args, uint32_t tiles, uint32_t parts) {
  const uint32_t at = blockIdx.x * 256u + threadIdx.x, tile = at / kTileVectors, v = at % kTileVectors;
  const uint32_t row_tiles = (args.rows + kTileRows - 1u) / kTileRows;
  const uint32_t lane = v & 63u, nt = (v >> 6) & 1u, mt = (v >> 7) & 3u, wave = v >> 9;
  const uint32_t m = tile % row_tiles * kTileRows + 16u * mt + 4u * (lane >> 4);
  const uint32_t n = tile / row_tiles * kTileColumns + 32u * wave + 16u * nt + (lane & 15u);
  if (m >= args.rows || n >= args.columns) return;
  const floatx4* sums = reinterpret_cast<const floatx4*>(args.parts) + at;
  floatx4 sum = (floatx4)0.0f;
#pragma unroll 8
  for (uint32_t p = 0; p < parts; ++p) sum += sums[(uint64_t)p * tiles * kTileVectors];
  Extra extra[4];
#pragma unroll
  for (uint32_t r = 0; r < 4u; ++r)
    if (m + r < args.rows) extra[r] = load_extra<T>(args, m + r, n);
#pragma unroll
  for (uint32_t r = 0; r < 4u; ++r)
    if (m + r < args.rows) finish<T>(args, m + r, n, sum[r], extra[r]);
}

typedef void (*Kernel)(Q4Args);
// The instantiation of a kernel template for a weight.
#define PK_Q4_PICK(args, KERNEL)                                                                            \
  ((args).offsets ? ((args).per_block == 1u ? KERNEL(1, true) : (args).per_block == 2u ? KERNEL(2, true)    \
                                                                                        : KERNEL(4, true))  \
                  : ((args).per_block == 1u ? KERNEL(1, false) : (args).per_block == 2u ? KERNEL(2, false)  \
                                                                                         : KERNEL(4, false)))
template <typename T, int MT, int NT, bool PANEL>
Kernel pick_rows(const Q4Args& args) {
#define PK_Q4_ROWS(PER, OFFSETS) q4_rows_kernel<T, PER, MT, NT, OFFSETS, PANEL>
  return PK_Q4_PICK(args, PK_Q4_ROWS);
#undef PK_Q4_ROWS
}
template <int ROWS>
Kernel pick_vector(const Q4Args& args) {
#define PK_Q4_VECTOR(PER, OFFSETS) q4_vector_kernel<PER, ROWS, OFFSETS>
  return PK_Q4_PICK(args, PK_Q4_VECTOR);
#undef PK_Q4_VECTOR
}
Kernel pick_tile(const Q4Args& args) {
#define PK_Q4_TILE(PER, OFFSETS) q4_tile_kernel<_Float16, PER, OFFSETS>
#define PK_Q4_TILE_F32(PER, OFFSETS) q4_tile_kernel<float, PER, OFFSETS>
  return args.f16 ? PK_Q4_PICK(args, PK_Q4_TILE) : PK_Q4_PICK(args, PK_Q4_TILE_F32);
#undef PK_Q4_TILE
#undef PK_Q4_TILE_F32
}

// A launch: kernel, grid and threads.
struct Q4Plan {
  Kernel kernel;
  dim3 grid;  // y of a tile kernel: parts of K, `span` blocks each
  uint32_t threads;
  uint32_t span;  // 0: no tile kernel
  uint64_t part_bytes() const { return span && grid.y > 1u ? (uint64_t)grid.x * grid.y * kTileVectors * 16u : 0u; }
};

// f16 kernels of few rows: rows and columns of a workgroup in 16, wavefronts
// at most, and the us that a compute unit takes for a block of K and for the
// rest of a workgroup, fitted to products of 32 to 300 rows, K 512 to 8192, N
// 256 to 8192, groups of 128 without offsets. Smaller groups and offsets make
// all kernels slower alike: over 63 products of 17 to 1504 rows each, the
// choice takes 1.012 to 1.019 times the fastest kernel's time in the mean for
// groups of 32, 64 and 128, with offsets and without, and 1.18 at most.
struct RowsShape {
  uint32_t mt, nt, waves;
  float block, rest;
};
// Two columns share the reads of 32 and 64 rows.
constexpr RowsShape kRowsShapes[] = {
    {1, 1, 16, 0.07f, 0.3f}, {1, 2, 16, 0.115f, 0.35f}, {2, 2, 8, 0.165f, 0.8f}, {4, 2, 8, 0.26f, 2.0f}};
// The kernels of kRowsShapes.
Kernel pick_rows_f16(const Q4Args& args, uint32_t shape) {
  switch (shape) {
    case 0: return pick_rows<_Float16, 1, 1, false>(args);
    case 1: return pick_rows<_Float16, 1, 2, false>(args);
    case 2: return pick_rows<_Float16, 2, 2, false>(args);
    default: return pick_rows<_Float16, 4, 2, false>(args);
  }
}
// us of a launch of f16 tiles, `blocks` of K each, fitted to the same products:
// a compute unit holds three (with offsets two), of which one leaves it idle
// half the time.
float tile_time(uint64_t tiles, uint32_t blocks) {
  const float each = (float)((tiles + 255u) / 256u);
  return 1.5f * each + (each > 1.0f ? 0.55f * each : 0.72f) * (float)blocks;
}

Q4Plan plan(const Q4Args& args) {
  const auto tiles = [](uint32_t n, uint32_t size) { return (n + size - 1u) / size; };
  const uint32_t kblocks = tiles(args.inner, 128u), nblocks = tiles(args.columns, 16u);
  // Four wavefronts at least, for the outputs if not for K: 64 x 60 x 614 with
  // a residual 7.2 us, with one for its one block 11.1.
  const auto threads = [&](uint32_t most) { return 64u * (kblocks < 4u ? 4u : kblocks < most ? kblocks : most); };
  // Wavefronts of the kernels with the rows in LDS: two blocks of K each,
  // from 4 (1 x 640 x 1032 3.2 us, 3.6 with one block each) to `most`.
  const auto panel_threads = [&](uint32_t most) {
    const uint32_t two = kblocks / 2u < 4u ? 4u : kblocks / 2u;
    return threads(two < most ? two : most);
  };
  const uint64_t row_bytes =
      args.f16 ? panel_stride<_Float16>(args.inner) * 2ull : panel_stride<float>(args.inner) * 4ull;
  const bool panel = args.rows <= 16u && args.rows * row_bytes <= kPanelBytes;
  // Tiles whole, or too few to fill the compute units in as many parts along K
  // as make two for each, but 16, which a thread of the join adds in turn.
  const uint64_t tiled = (uint64_t)tiles(args.rows, kTileRows) * tiles(args.columns, kTileColumns);
  const uint32_t most_parts =
      tiled <= 32u ? 16u : tiled <= kMostSplitTiles ? 2u * kMostSplitTiles / (uint32_t)tiled : 1u;
  const uint32_t span = tiles(kblocks, most_parts), parts = tiles(kblocks, span);
  const auto tile_plan = [&](uint32_t blocks) {
    return Q4Plan{pick_tile(args), dim3((uint32_t)tiled, tiles(kblocks, blocks)), 256u, blocks};
  };
  if (!args.f16) {
    // A block of a tile takes eight times as long as in f16: parts, whose
    // second launch takes some 4 us, win from 1024 blocks of K and tile on: 128
    // x 4096 x 4096 44.2 us and rows 55.9, 256 x 1024 x 4096 28.2 and 36.8, 64 x
    // 4096 x 4096 27.8 and 28.8; but 48 x 4096 x 4096 27.2 and 23.3, 64 x 1024 x
    // 4096 13.5 and 10.4, and 1504 x 1024 x 1024 (192 tiles, 8 blocks along K)
    // 44.3, whole 41.9. Whole tiles: 216 (1504 x 640 x 1032) 30.0 and rows 48.6.
    if (args.rows > 48u && parts > 1u && kblocks >= (tiled < 160u ? 8u : 32u) && tiled * kblocks >= 1024u)
      return tile_plan(span);
    if (args.rows > 64u && tiled >= 160u) return tile_plan(kblocks);
    // 1 x 4096 x 4096: 4.2 us on the VALU, 8.1 on the matrix units; 4 rows 7.8 and 9.5.
    if (panel && args.rows <= 4u)
      return {args.rows == 1u ? pick_vector<1>(args) : args.rows == 2u ? pick_vector<2>(args) : pick_vector<4>(args),
              dim3(nblocks), panel_threads(16u), 0u};
    if (panel) return {pick_rows<float, 1, 1, true>(args), dim3(nblocks), panel_threads(16u), 0u};
    return {pick_rows<float, 1, 1, false>(args), dim3(nblocks, tiles(args.rows, 16u)), threads(8u), 0u};
  }
  // 8 wavefronts (1 x 8192 x 8192 8.3 us, 16 8.8; 8 x 2048 x 8192 4.5 and 5.2).
  if (panel) return {pick_rows<_Float16, 1, 1, true>(args), dim3(nblocks), panel_threads(8u), 0u};
  // The kernel that the times above make the fastest: 64 x 4096 x 2048 6.4 us
  // with 16 rows a workgroup, 7.0 with 32, 9.7 with 64, parts of tiles 12.5; 64 x
  // 4096 x 4096 10.9, 8.6, 10.8 and 13.3; 64 x 4096 x 8192 21.4, 16.1, 12.9 and 15.3;
  // 300 x 8192 x 1024 22.9, 22.3, 29.3 and 17.0; 300 x 2048 x 8192 54.4, 45.2, 35.5
  // and tiles whole 22.3. Parts: 5.5 us for the sums' way through memory and
  // the second launch.
  uint32_t best = 0;
  float time = 0.0f;
  dim3 grid;
  for (uint32_t i = 0; i < sizeof(kRowsShapes) / sizeof(kRowsShapes[0]); ++i) {
    const RowsShape& s = kRowsShapes[i];
    if (s.mt > 1u && args.rows <= 8u * s.mt) break;  // half of its rows at most
    const uint32_t x = tiles(nblocks, s.nt), y = tiles(args.rows, 16u * s.mt);
    const float t = (float)(((uint64_t)x * y + 255u) / 256u) * (s.rest + s.block * (float)kblocks);
    if (i && t >= time) continue;
    best = i;
    time = t;
    grid = dim3(x, y);
  }
  const float whole = tile_time(tiled, kblocks), split = 5.5f + tile_time(tiled * parts, span);
  if (parts > 1u && split < time && split < whole) return tile_plan(span);
  if (whole < time) return tile_plan(kblocks);
  return {pick_rows_f16(args, best), grid, threads(kRowsShapes[best].waves), 0u};
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

uint64_t q4_workspace(const Q4Args& args) {
  Q4Args some = args;
  uint64_t bytes = 0;
  const auto count = [&](uint32_t rows) {
    some.rows = rows;
    const uint64_t wanted = plan(some).part_bytes();
    if (wanted > bytes) bytes = wanted;
  };
  // A plan depends on the rows in 16, and takes a tile at least for 64.
  for (uint32_t rows = 16u; rows < args.rows && rows <= kMostSplitTiles * kTileRows; rows += 16u) count(rows);
  count(args.rows);
  return bytes;
}

hipError_t launch_q4(const Q4Args& given, hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
  Q4Args args = given;
  const Q4Plan p = plan(args);
  args.span = p.span;
  const uint64_t bytes = p.part_bytes();
  if (bytes > args.part_bytes) return hipErrorInvalidValue;
  if (start || (stop && !bytes))
    hipExtLaunchKernelGGL(p.kernel, p.grid, dim3(p.threads), 0, stream, start, bytes ? nullptr : stop, 0, args);
  else
    hipLaunchKernelGGL(p.kernel, p.grid, dim3(p.threads), 0, stream, args);
  if (const hipError_t e = hipGetLastError()) return e;
  if (!bytes) return hipSuccess;
  const dim3 grid(p.grid.x * (kTileVectors / 256u));
  const auto join = args.f16 ? q4_join_kernel<_Float16> : q4_join_kernel<float>;
  if (stop)
    hipExtLaunchKernelGGL(join, grid, dim3(256), 0, stream, nullptr, stop, 0, args, p.grid.x, p.grid.y);
  else
    hipLaunchKernelGGL(join, grid, dim3(256), 0, stream, args, p.grid.x, p.grid.y);
  return hipGetLastError();
}

}  // namespace pk
