// pk_score.hip - token scores for gfx950 (include/pk_score.h has the formulas
// and what rows of infinities and NaN give).
//
// Bound by memory where rows are many and f32: 2048 of 32000 logits 50.3 us,
// 5.2 TB/s where a copy reaches 4.9. f16 is bound by the VALU, some 10
// operations a logit (two converts, fma, exponential, sums): 3008 of 1025 5.4
// us, 3.0 of them the launch. A logit is loaded once and stays in registers,
// as 16-byte vectors, through the maximum, the sums relative to it and the search for
// alternatives. A group of 64, 256 or 1024 threads holds a row, or a part of
// one: rows longer than a group holds, and long rows when there are few, are
// split, and a second launch joins the parts' maxima, sums and alternatives.
//
// Alternatives: 64 subsets of the group know their largest logits. At least K
// logits reach the K-th largest of these maxima, and where large logits lie
// anywhere in the row few others do, so a threshold just below it (found by
// halving the interval, counting with ballots) leaves a short list. Each
// entry of the list then counts the entries that go before it: its place. A
// row that leaves too many (a plateau of equal logits, large ones side by
// side, a mask of the lowest number that leaves fewer than K subsets with
// another) is searched again, K times for the best below the last: 2048 rows
// of 32000 f32 logits masked so but for 4 of each 510 us, masked by minus
// infinity 44; 3008 of 1025 f16 15.7 and 5.5.
#include "pk_internal.h"
#include "pk_wave.h"

namespace pk {
namespace {

constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_inff();
constexpr int kList = 256;      // entries of a group's list
constexpr int kJoining = 256;   // threads of the groups that split a row

// A logit's place in the order of alternatives: larger logits first, equal
// ones by index. 0 is below every key.
__device__ __forceinline__ uint64_t score_key(float x, uint32_t index) {
  const uint32_t bits = __float_as_uint(x + 0.0f);  // one zero
  const uint32_t order = (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
  return ((uint64_t)order << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t order = (uint32_t)(key >> 32);
  return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}

// The largest key of the wavefront, in every lane: the largest upper half,
// then the largest lower half among those.
__device__ __forceinline__ uint64_t wave_max_key(uint64_t key) {
  const auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  const uint32_t high = wave::reduce_bits((uint32_t)(key >> 32), 0u, larger);
  const uint32_t low = wave::reduce_bits((uint32_t)(key >> 32) == high ? (uint32_t)key : 0u, 0u, larger);
  return ((uint64_t)high << 32) | low;
}

// Orders LDS traffic between the threads of a group.
template <int GROUP>
__device__ __forceinline__ void group_sync() {
  if constexpr (GROUP > 64) __syncthreads();
  else wave::sync();
}

// A threshold that at least `count` of the 64 lanes' values reach, close to
// the largest one such; minus infinity if fewer are above that.
__device__ __forceinline__ float wave_threshold(float value, uint32_t count) {
  const auto reached = [&](float at) { return (uint32_t)__popcll(__ballot(value >= at)); };
  float high = wave::max(value);
  if ((uint32_t)__popcll(__ballot(value > -kInf)) < count) return -kInf;
  float low = -wave::max(value > -kInf ? -value : -kInf);
  for (int step = 0; step < 12; ++step) {
    const float mid = 0.5f * low + 0.5f * high;
    const uint32_t n = reached(mid);
    if (n >= count) low = mid;
    else high = mid;
    if (n >= count && n <= count + 2u) break;
  }
  return low;
}

// What the compiler knew of the held logits it knows no longer: their f32
// values do not stay in registers from one phase to the next.
template <typename V, int N>
__device__ __forceinline__ void forget(V (&held)[N]) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    words w = __builtin_bit_cast(words, held[i]);
    asm volatile("" : "+v"(w));
    held[i] = __builtin_bit_cast(V, w);
  }
}

// Calls store(place, key) for the K first of the `found` different keys of
// `list`, and store(place, 0) for the places behind them.
template <int GROUP, typename Store>
__device__ __forceinline__ void place_keys(const uint64_t* list, uint32_t found, uint32_t at, uint32_t K, Store store) {
  if (found <= 64u) {  // in the lanes of one wavefront
    if (GROUP > 64 && at >= 64u) return;
    const uint64_t key = at < found ? list[at] : 0;
    uint32_t place = 0;
    for (uint32_t j = 0; j < found; ++j) {
      const uint32_t low = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)key, (int)j);
      const uint32_t high = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(key >> 32), (int)j);
      place += (((uint64_t)high << 32) | low) > key;
    }
    if (at >= found) place = at;
    if (place < K) store(place, key);
    return;
  }
  for (uint32_t i = at; i < found; i += GROUP) {
    const uint64_t key = list[i];
    uint32_t place = 0;
    for (uint32_t j = 0; j < found; ++j) place += list[j] > key;
    if (place < K) store(place, key);
  }
}

template <int GROUP>
struct Shared {
  float subset[64];
  float sums[3][GROUP / 64 > 1 ? GROUP / 64 : 1];
  uint64_t list[kList];
  uint64_t best[GROUP / 64 > 1 ? GROUP / 64 : 1];
  uint32_t count;
};

// log(1 + r), r >= 0: the logarithm of u = 1 + r rounded, times r / (u - 1),
// which takes out what the rounding of u did (W. Kahan's form). Logarithm and
// reciprocal are the hardware's, within 1 ulp.
__device__ __forceinline__ float log_one_plus(float r) {
  const float u = 1.0f + r;
  return u == 1.0f ? r : __builtin_amdgcn_logf(u) * kLn2 * (r * __builtin_amdgcn_rcpf(u - 1.0f));
}

// The row's results from its whole sums.
struct RowScores {
  float m, scale, spread;
  bool empty;
  __device__ RowScores(const ScoreArgs& args, const ScorePart& p)
      : m(p.m), scale(args.inverse_temperature), spread(log_one_plus(p.r)), empty(p.m == -kInf && p.r == 0.0f) {}
  // The entropy and the log probability of `token`, whose logit is given.
  __device__ void store_row(const ScoreArgs& args, uint32_t row, const ScorePart& p, uint32_t token,
                            float logit) const {
    if (args.entropies) args.entropies[row] = empty ? 0.0f : spread - p.t * kLn2 * __builtin_amdgcn_rcpf(1.0f + p.r);
    if (args.tokens)
      args.log_probs[row] = token < args.columns ? log_prob(logit) : token == 0xffffffffu ? 0.0f : __builtin_nanf("");
  }
  // Halves of x and m: their difference is a number where that of x and m is
  // beyond f32, and twice the scale brings a temperature above 1 back.
  __device__ float log_prob(float x) const {
    return empty ? -kInf : (0.5f * x - 0.5f * m) * (2.0f * scale) - spread;
  }
  // Alternative k of the row; key 0: none.
  __device__ void store(const ScoreArgs& args, uint32_t row, uint32_t k, uint64_t key) const {
    const uint64_t at = (uint64_t)row * args.alternatives + k;
    args.top_tokens[at] = key ? ~(uint32_t)key : 0xffffffffu;
    args.top_log_probs[at] = key ? log_prob(key_logit(key)) : -kInf;
  }
};

// Calls store(k, key) for the K largest of key_of(0..count), 0 where there
// are no more, by one scan for each.
template <int GROUP, typename KeyOf, typename Store>
__device__ __forceinline__ void best_keys(Shared<GROUP>& s, uint32_t at, uint32_t K, uint32_t count, KeyOf key_of,
                                          Store store) {
  uint64_t last = ~0ull;
  for (uint32_t k = 0; k < K; ++k) {
    uint64_t key = 0;
#pragma unroll 1
    for (uint32_t i = at; i < count; i += GROUP) {
      const uint64_t other = key_of(i);
      if (other < last && other > key) key = other;
    }
    key = wave_max_key(key);
    if constexpr (GROUP > 64) {
      __syncthreads();  // the readers of the round before
      if ((at & 63u) == 0) s.best[at >> 6] = key;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < GROUP / 64; ++w) key = s.best[w] > key ? s.best[w] : key;
    }
    last = key;
    if (at == 0) store(k, key);
  }
}

// One group: part blockIdx.y of a row, elements [part * span, part * span +
// span), HELD vectors a thread. What lies before the first and behind the
// last 16-byte boundary goes to single threads, one element each.
template <typename T, int GROUP, int HELD>
__global__ __launch_bounds__(GROUP < 256 ? 256 : GROUP, GROUP > 256 ? 8 : 1) void score_kernel(ScoreArgs args) {
  constexpr int kRows = GROUP < 256 ? 256 / GROUP : 1;
  constexpr int VEC = 16 / sizeof(T);
  constexpr int kWaves = GROUP / 64;
  constexpr bool kHalf = sizeof(T) == 2;
  typedef T V __attribute__((ext_vector_type(VEC)));
  __shared__ Shared<GROUP> shared[kRows];
  Shared<GROUP>& s = shared[threadIdx.x / GROUP];
  const uint32_t row = blockIdx.x * kRows + threadIdx.x / GROUP, at = threadIdx.x % GROUP;
  const uint32_t lane = threadIdx.x & 63u, wave = at >> 6;
  if (row >= args.rows) return;  // a whole group
  const uint32_t first = blockIdx.y * args.span, size = min(args.columns - first, args.span);
  const T* x = static_cast<const T*>(args.logits) + row * args.stride + first;
  const uint32_t head = min(size, (uint32_t)(-reinterpret_cast<uintptr_t>(x) % 16u / sizeof(T)));
  const uint32_t vectors = (size - head) / VEC, tail = size - head - vectors * VEC;
  const uint32_t K = args.alternatives;

  // The given token and its logit, before and behind the row's loads.
  const bool leads = at == 0;
  uint32_t token = 0xffffffffu;
  if (leads && args.tokens) token = args.tokens[row];
  V held[HELD];
  const V* body = reinterpret_cast<const V*>(x + head);
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const uint32_t v = at + i * GROUP;
    if (v < vectors) held[i] = body[v];
    else
#pragma unroll
      for (int c = 0; c < VEC; ++c) held[i][c] = (T)-kInf;
  }
  const uint32_t edge = at < head ? at : head + vectors * VEC + (at - head);  // this thread's single element
  const float single = at < head + tail ? (float)x[edge] : -kInf;
  const float target = leads && token < args.columns
                           ? (float)(static_cast<const T*>(args.logits) + row * args.stride)[token]
                           : 0.0f;
  if (kWaves > 1 && at == 0) s.count = 0;

  // Maxima: of each vector, the thread, its subset (GROUP / 64 lanes) and the group.
  // The operands of a maximum are quiet first: of a signalling NaN and a
  // number it is a NaN, and the next one loses the number.
  float top[HELD], mine = __builtin_canonicalizef(single);
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const V w = held[i];
    if constexpr (kHalf) {
      const auto pairs = __builtin_elementwise_max(__builtin_shufflevector(w, w, 0, 1, 2, 3),
                                                   __builtin_shufflevector(w, w, 4, 5, 6, 7));
      const auto pair = __builtin_elementwise_max(__builtin_shufflevector(pairs, pairs, 0, 1),
                                                  __builtin_shufflevector(pairs, pairs, 2, 3));
      top[i] = fmaxf((float)pair[0], (float)pair[1]);
    } else {
      top[i] = fmaxf(fmaxf(__builtin_canonicalizef(w[0]), __builtin_canonicalizef(w[1])),
                     fmaxf(__builtin_canonicalizef(w[2]), __builtin_canonicalizef(w[3])));
    }
    mine = fmaxf(mine, top[i]);
  }
  float subset = mine;
  if constexpr (GROUP > 64) {
#pragma unroll
    for (int off = 1; off < kWaves; off <<= 1) subset = fmaxf(subset, __shfl_xor(subset, off, 64));
    if (at % kWaves == 0) s.subset[at / kWaves] = subset;
    __syncthreads();
    subset = s.subset[lane];
  }
  const float m = wave::max(subset);
  // No alternative is minus infinity: the lowest number is below all others.
  const float threshold = K ? fmaxf(wave_threshold(subset, K), -3.402823466e38f) : 0.0f;
  uint32_t found = 0;

  // Sums. f16: the exponent (x - m) s is x s - c in one operation, c = m s
  // rounded, the same c for every x, and what the rounding leaves at x = m
  // is taken out of the sums. f32: x - m first, exact where it matters.
  const float scale = args.inverse_temperature * kLog2E, centre = m == -kInf ? 0.0f : m;
  const float shift = -(centre * scale);
  const auto exponent = [&](float v) {
    if constexpr (kHalf) return __builtin_fmaf(v, scale, shift);
    return (v - centre) * scale;
  };
  const float zero = m == -kInf ? 0.0f : exponent(m);
  float r = 0.0f, t = 0.0f;
  uint32_t equal = 0;  // of the wavefront, counted on the scalar unit
  const auto add = [&](float v, bool watch) {
    const float d = exponent(v);
    float e = __builtin_amdgcn_exp2f(d);
    if (watch) {
      const bool is_top = d == zero;
      e = is_top ? 0.0f : e;
      equal += (uint32_t)__popcll(__ballot(is_top));
    }
    r += e;
    t = __builtin_fmaf(e, fmaxf(d, -200.0f), t);  // 0 times minus infinity is 0 here
  };
  const auto add_all = [&](bool watch) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
#pragma unroll
      for (int c = 0; c < VEC; ++c) add((float)held[i][c], watch);
      __builtin_amdgcn_sched_barrier(0);  // one vector's values at a time in registers
    }
    add(single, watch);
  };
  if constexpr (kWaves == 1 || HELD == 8) {  // the second pass would take registers that 8 vectors need
    add_all(true);
  } else {
    // Only a wavefront that holds a maximum looks for it, in a second pass.
    add_all(false);
    forget(held);
    if (__any(mine == m)) {
      r = t = 0.0f;
      add_all(true);
    }
  }
  r = wave::sum(r);
  t = wave::sum(t);
  float maxima = (float)equal;
  if constexpr (kWaves > 1) {
    if (lane == 0) {
      s.sums[0][wave] = r;
      s.sums[1][wave] = t;
      s.sums[2][wave] = maxima;
    }
  }

  // The list of what reaches the threshold.
  if constexpr (kHalf) forget(held);
  if (K && __any(mine >= threshold)) {
    const auto offer = [&](float v, uint32_t index) {
      const uint64_t hits = __ballot(v >= threshold);
      if (!hits) return;
      uint32_t place = 0;
      if constexpr (kWaves > 1) {
        if (lane == 0) place = atomicAdd(&s.count, (uint32_t)__popcll(hits));
        place = (uint32_t)__builtin_amdgcn_readfirstlane((int)place);
      } else {
        place = found;
        found += (uint32_t)__popcll(hits);
      }
      place += __builtin_amdgcn_mbcnt_hi((uint32_t)(hits >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hits, 0u));
      if (v >= threshold && place < (uint32_t)kList) s.list[place] = score_key(v, index);
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      if (__any(top[i] >= threshold))
#pragma unroll
        for (int c = 0; c < VEC; ++c) offer((float)held[i][c], first + head + (at + i * GROUP) * VEC + c);
      __builtin_amdgcn_sched_barrier(0);
    }
    offer(single, first + edge);
  }
  group_sync<GROUP>();
  if constexpr (kWaves > 1) {
    r = t = maxima = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      r += s.sums[0][w];
      t += s.sums[1][w];
      maxima += s.sums[2][w];
    }
  }
  ScorePart part;
  part.m = m;
  part.unused = 0.0f;
  if (m == -kInf) {
    part.r = r;
    part.t = 0.0f;
  } else {
    // zero is at most half a step of c, a step of an f16 logit 2^13 times that:
    // where zero is far from 0 every other term is 0, and 2^-zero infinite.
    const float correction = kHalf ? __builtin_amdgcn_exp2f(fmaxf(-100.0f, fminf(100.0f, -zero))) : 1.0f;
    part.t = correction * __builtin_fmaf(-zero, r, t);
    part.r = __builtin_fmaf(correction, r, maxima - 1.0f);
  }

  if constexpr (kWaves > 1) found = s.count;
  const auto alternatives = [&](auto store) {
    if (found <= (uint32_t)kList) {
      place_keys<GROUP>(s.list, found, at, K, store);
    } else {
      // From the cache: the rare way holds no registers of the usual one.
      best_keys<GROUP>(s, at, K, size, [&](uint32_t i) {
        const float v = (float)x[i];
        return v > -kInf ? score_key(v, first + i) : 0;
      }, store);
    }
  };
  if (gridDim.y == 1) {
    const RowScores scores(args, part);
    if (leads) scores.store_row(args, row, part, token, target);
    if (K) alternatives([&](uint32_t k, uint64_t key) { scores.store(args, row, k, key); });
  } else {
    const uint64_t record = (uint64_t)row * gridDim.y + blockIdx.y;
    if (leads) args.parts[record] = part;
    if (K) alternatives([&](uint32_t k, uint64_t key) { args.part_keys[record * K + k] = key; });
  }
}

// Joins the parts of a row, one workgroup each. A second launch: for 8 rows
// of 131072 f16 logits in 32 parts each both take 9.7 us; one launch whose last
// workgroup joins waits for its stores, its arrival and its loads at the agent's
// coherence point in turn, 1.2 us more.
__global__ __launch_bounds__(kJoining) void score_join_kernel(ScoreArgs args, uint32_t parts) {
  __shared__ Shared<kJoining> s;
  const uint32_t row = blockIdx.x, at = threadIdx.x;
  uint32_t token = 0xffffffffu;
  if (at == 0 && args.tokens) token = args.tokens[row];
  constexpr int kWaves = kJoining / 64;
  const uint32_t lane = at & 63u, wave = at >> 6, K = args.alternatives, keys_count = parts * K;
  const ScorePart* p = args.parts + (uint64_t)row * parts;
  const uint64_t* keys = args.part_keys + (uint64_t)row * keys_count;
  // This thread's first part and key, together: most rows have no more.
  ScorePart mine = {-kInf, 0.0f, 0.0f, 0.0f};
  uint64_t key = 0, threshold = 1;
  if (at < parts) mine = p[at];
  if (at < keys_count) key = keys[at];
  float target = 0.0f;
  if (at == 0 && token < args.columns) {
    const uint64_t from = row * args.stride + token;
    target = args.f16 ? (float)static_cast<const _Float16*>(args.logits)[from]
                      : static_cast<const float*>(args.logits)[from];
  }
  // No key below a part's K-th is one of the row's K best: that part has K.
  float m = mine.m;
  if (K)
    for (uint32_t i = at; i < parts; i += kJoining) {
      const uint64_t lowest = keys[i * K + K - 1u];
      threshold = lowest > threshold ? lowest : threshold;
    }
  for (uint32_t i = at + kJoining; i < parts; i += kJoining) m = fmaxf(m, p[i].m);
  m = wave::max(m);
  threshold = wave_max_key(threshold);
  if (lane == 0) {
    s.subset[wave] = m;
    s.best[wave] = threshold;
  }
  if (at == 0) s.count = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    m = fmaxf(m, s.subset[w]);
    threshold = s.best[w] > threshold ? s.best[w] : threshold;
  }
  // Each part's sums relative to the row's maximum; a part with that maximum
  // leaves its own one out, which all but one of them add again.
  const float scale = args.inverse_temperature * kLog2E;
  float r = 0.0f, t = 0.0f, equal = 0.0f;
  for (uint32_t i = at; i < parts; i += kJoining) {
    const ScorePart part = i == at ? mine : p[i];
    if (part.m == m || part.m == -kInf) {
      r += part.r;
      t += part.t;
      equal += part.m == -kInf ? 0.0f : 1.0f;
    } else {
      const float d = (part.m - m) * scale, f = __builtin_amdgcn_exp2f(d), all = 1.0f + part.r;
      r = __builtin_fmaf(f, all, r);
      t = __builtin_fmaf(f, __builtin_fmaf(fmaxf(d, -200.0f), all, part.t), t);
    }
  }
  r = wave::sum(r);
  t = wave::sum(t);
  equal = wave::sum(equal);
  if (lane == 0) {
    s.sums[0][wave] = r;
    s.sums[1][wave] = t;
    s.sums[2][wave] = equal;
  }
  for (uint32_t i = at; i < keys_count; i += kJoining) {
    if (i != at) key = keys[i];
    if (key >= threshold) {
      const uint32_t place = atomicAdd(&s.count, 1u);
      if (place < (uint32_t)kList) s.list[place] = key;
    }
  }
  __syncthreads();
  ScorePart whole = {m, 0.0f, 0.0f, 0.0f};
  equal = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    whole.r += s.sums[0][w];
    whole.t += s.sums[1][w];
    equal += s.sums[2][w];
  }
  if (m > -kInf) whole.r += equal - 1.0f;
  const RowScores scores(args, whole);
  if (at == 0) scores.store_row(args, row, whole, token, target);
  if (!K) return;
  const auto store = [&](uint32_t k, uint64_t key) { scores.store(args, row, k, key); };
  const uint32_t found = s.count;
  if (found <= (uint32_t)kList) place_keys<kJoining>(s.list, found, at, K, store);
  else best_keys<kJoining>(s, at, K, keys_count, [&](uint32_t i) { return keys[i]; }, store);
}

typedef void (*Kernel)(ScoreArgs);
struct Variant {
  uint32_t group, held;  // threads, vectors a thread
  Kernel kernel;
};
template <typename T>
constexpr Variant kVariants[] = {
    {64, 1, score_kernel<T, 64, 1>},     {64, 2, score_kernel<T, 64, 2>},   {64, 4, score_kernel<T, 64, 4>},
    {256, 2, score_kernel<T, 256, 2>},   {256, 4, score_kernel<T, 256, 4>}, {256, 8, score_kernel<T, 256, 8>},
    {1024, 4, score_kernel<T, 1024, 4>}, {1024, 8, score_kernel<T, 1024, 8>},
};
// In place of a {64, 4} and a {256, 8} where every group has a compute unit
// to itself: 32 rows of 2048 f16 logits 4.2 us instead of 5.2, of 16384 6.0
// instead of 7.1; from 512 rows on they are slower.
template <typename T>
constexpr Variant kFewRows[] = {{256, 1, score_kernel<T, 256, 1>}, {1024, 2, score_kernel<T, 1024, 2>}};

// The parts of a row, and the kernel that holds one.
struct ScorePlan {
  uint32_t parts, span;
  const Variant* variant;
};
ScorePlan plan(const ScoreArgs& args) {
  const uint32_t vec = args.f16 ? 8u : 4u;
  const Variant* table = args.f16 ? kVariants<_Float16> : kVariants<float>;
  const uint32_t most = 1024u * 8u * vec;  // the longest part of one group
  uint32_t parts = (args.columns + most - 1u) / most;
  // Few long rows: parts of at least 4096 logits instead, as many as make
  // kScoreFill groups. The second launch takes some 4 us, which a group gains
  // back on 65536 logits and 2048 for each row (f16, 8 alternatives): 32 rows of
  // 65536 10.4 us (whole 11.3), 8 of 131072 9.7 (14.6) and 64 13.0 (16.2), but 1
  // row of 32000 8.9 (6.1). 64 of 65536 stay whole, 11.3, and would take 10.3.
  if ((uint64_t)args.rows * parts < kScoreFill && args.columns >= 65536u && args.columns / args.rows >= 2048u) {
    const uint32_t wanted = (kScoreFill + args.rows - 1u) / args.rows, smallest = (args.columns + 4095u) / 4096u;
    const uint32_t more = wanted < smallest ? wanted : smallest;
    if (more > parts) parts = more;
  }
  ScorePlan p;
  p.span = (uint32_t)(((uint64_t)args.columns + parts - 1u) / parts + vec - 1u) / vec * vec;
  p.parts = (args.columns + p.span - 1u) / p.span;
  p.variant = table;
  const uint32_t vectors = (p.span < args.columns ? p.span : args.columns) / vec;
  while (p.variant->group * p.variant->held < vectors) ++p.variant;
  if ((uint64_t)args.rows * p.parts <= kScoreFill) {
    const Variant* few = args.f16 ? kFewRows<_Float16> : kFewRows<float>;
    if (p.variant == table + 2) p.variant = few;
    if (p.variant == table + 5) p.variant = few + 1;
  }
  return p;
}

}  // namespace

uint64_t score_workspace(const ScoreArgs& args) {
  // From kScoreFill rows on the parts of a row stay as they are; below, any
  // number of rows may have the most.
  ScoreArgs some = args;
  uint64_t records = 0;
  const auto count = [&](uint32_t rows) {
    some.rows = rows;
    const uint64_t parts = plan(some).parts;
    if (parts > 1 && parts * rows > records) records = parts * rows;
  };
  for (uint32_t rows = 1; rows <= args.rows && rows <= kScoreFill; ++rows) count(rows);
  count(args.rows);
  return records;
}

uint64_t score_workspace_bytes(const ScoreArgs& args, uint64_t records) {
  return records * (sizeof(ScorePart) + 8u * args.alternatives);
}

void score_bind_workspace(ScoreArgs* args, void* workspace, uint64_t records) {
  args->parts = static_cast<ScorePart*>(workspace);
  args->part_keys = reinterpret_cast<uint64_t*>(args->parts + records);
  args->records = records;
}

hipError_t launch_score(const ScoreArgs& given, hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
  ScoreArgs args = given;
  const ScorePlan p = plan(args);
  args.span = p.span;
  const bool split = p.parts > 1;
  if (split && (uint64_t)args.rows * p.parts > args.records) return hipErrorInvalidValue;
  const uint32_t each = p.variant->group < 256u ? 256u / p.variant->group : 1u;
  const dim3 grid((args.rows + each - 1u) / each, p.parts), block(p.variant->group < 256u ? 256u : p.variant->group);
  if (start || (stop && !split))
    hipExtLaunchKernelGGL(p.variant->kernel, grid, block, 0, stream, start, split ? nullptr : stop, 0, args);
  else
    hipLaunchKernelGGL(p.variant->kernel, grid, block, 0, stream, args);
  if (const hipError_t e = hipGetLastError()) return e;
  if (!split) return hipSuccess;
  if (stop)
    hipExtLaunchKernelGGL(score_join_kernel, dim3(args.rows), dim3(kJoining), 0, stream, nullptr, stop, 0, args,
                          p.parts);
  else
    hipLaunchKernelGGL(score_join_kernel, dim3(args.rows), dim3(kJoining), 0, stream, args, p.parts);
  return hipGetLastError();
}

}  // namespace pk
