// pk_verify.hip - verification of drafted tokens for gfx950
// (include/pk_verify.h has the formulas and what rows of infinities, NaN and
// strange numbers give).
//
// Decisions are whole numbers, so probabilities and sums are f64: a sum of
// 131072 f32 exponentials moves with its order by more than the gap between two
// neighbouring tokens of a flat distribution. An exponential through the table is
// 10 operations of f64 and 7 others, and they bound the sums: 64 logits take a SIMD 115
// cycles, where memory would feed twice as many.
//
// Short rows: one launch, a workgroup for each sequence. Its wavefronts take the
// rows' sums, target and draft, side by side, the decisions are read from
// them in turn, and all threads look for the next token. Long rows: a launch
// for the sums of parts of all rows; one for each sequence and part that decides, every
// workgroup for itself, and sums the part's weights; and one for each
// sequence that finds the part and in it the token. f16: a chunk of 5 rows of 1025 columns
// 10.5 us; 32 chunks of 3 to 8 rows of 131072 with as many of the draft model's 50.5 to 52.7, of which the
// sums of 36 million logits are 28, the weights 11 and the token 5, these two chains of dependent loads; f32
// 51; greedy 15.8 and 18.5, by two launches that bytes bound.
#include "pk_internal.h"
#include "pk_wave.h"

namespace pk {
namespace {

constexpr uint32_t kNoToken = 0xffffffffu;
constexpr float kInf = __builtin_inff();
constexpr int kThreads = 256;       // of a workgroup that holds a part of a row
// Pieces of 16 bytes in a thread that sums a part of a row, and one that sums the
// weights of a smaller part: those launches have fewer rows. 4 pieces for the sums take 53.5 us and not
// 52.4 (32 x 8 x 131072), 8 for the weights 61.4.
constexpr int kSumsHeld = 8, kHeld = 4;
constexpr int kSequence = 1024;     // threads of a workgroup that holds a sequence
constexpr uint32_t kShort = 4096;   // columns of a row that is short
template <typename T>
constexpr uint32_t kSumsSpan = kThreads * kSumsHeld * 16 / sizeof(T);  // columns of a part for the sums
template <typename T>
constexpr uint32_t kSpan = kThreads * kHeld * 16 / sizeof(T);          // and for the weights

typedef uint32_t Words __attribute__((ext_vector_type(2)));  // of a double, the low one first

// 2^x, x <= 0 but for roundings, within 2^-45 of it: x less its nearest whole number goes
// through a polynomial that meets 2^f at the 10 Chebyshev points of [-1/2, 1/2]; the whole number is
// in the low bits of x + 1.5 * 2^52 and is added to the exponent. 0 below 2^-1000.
__device__ __forceinline__ double exp2_of(double x) {
#pragma clang fp contract(off)
  constexpr double kWhole = 6755399441055744.0;
  const double shifted = x + kWhole, f = x - (shifted - kWhole);
  constexpr double c[10] = {1.0000000000000135, 0.6931471805599462, 0.2402265069564034, 0.05550410866465166,
                            0.00961812919393429, 0.0013333558200796013, 0.0001540343375126647, 1.5252672924257465e-05,
                            1.3259645241948732e-06, 1.020590550210069e-07};
  double r = c[9];
#pragma unroll
  for (int i = 8; i >= 0; --i) r = __builtin_fma(r, f, c[i]);
  const Words w = __builtin_bit_cast(Words, r), k = __builtin_bit_cast(Words, shifted);
  const Words all = {w.x, w.y + (k.x << 20)};
  return x > -1000.0 ? __builtin_bit_cast(double, all) : 0.0;
}

// The many exponentials of a row, 2^((z - m) scale) within 2^-45: the whole number k of 512ths of
// the exponent goes to the table of 2^(j / 512) in LDS, j = k mod 512, and to the exponent of what
// it finds there, the rest, at most a 1024th, through the Taylor series up to its third power. The
// table has j taken from its exponents already, so that k as it is can be added.
constexpr int kTable = 512;
// What is below stands for 0: a masked token has 2^-1000.
constexpr double kLeast = 0x1p-990;
template <int THREADS>
__device__ __forceinline__ void make_table(double* table) {
  for (int j = threadIdx.x; j < kTable; j += THREADS) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, 2.0 * exp2_of((double)(j - kTable) / kTable));
    table[j] = __builtin_bit_cast(double, bits - ((uint64_t)j << 43));
  }
  __syncthreads();
}
template <typename T>
struct Powers {
  const double* table;
  double m, scale, c;
  double right;  // of the true power over at()
  // f16: the exponent is one operation, z * scale - c, c the product of m and scale
  // rounded, the same for every z; what that rounding left, below 2^-16, is put right for the
  // whole row. f32: z - m first, since where logits are as large as f32's largest, c has no digits left.
  __device__ Powers(const double* table, double m, double scale_of_one)
      : table(table), m(m), scale(scale_of_one * kTable), c(m * scale) {
    right = sizeof(T) == 2 ? exp2_of(-__builtin_fma(m, scale, -c) / kTable) : 1.0;
  }
  __device__ __forceinline__ double at(float z) const {
#pragma clang fp contract(off)
    const double exponent = sizeof(T) == 2 ? __builtin_fma((double)z, scale, -c) : ((double)z - m) * scale;
    const double x = __builtin_fmax(exponent, -1000.0 * kTable);
    constexpr double kWhole = 6755399441055744.0, kLn2 = 0.6931471805599453 / kTable;
    const double shifted = x + kWhole, f = x - (shifted - kWhole);
    const uint32_t k = __builtin_bit_cast(Words, shifted).x;
    const Words found = __builtin_bit_cast(Words, table[k % kTable]), moved = {found.x, found.y + (k << 11)};
    const double power = __builtin_bit_cast(double, moved);
    const double rest = f * __builtin_fma(__builtin_fma(kLn2 * kLn2 * kLn2 / 6, f, kLn2 * kLn2 / 2), f, kLn2);
    return __builtin_fma(power, rest, power);
  }
};

// Up to N elements from `row` on, `count` of them there: 16 bytes at a time where they lie so.
template <int N, typename T>
__device__ __forceinline__ void load_run(const T* row, uint32_t count, float (&to)[N]) {
  constexpr int VEC = 16 / sizeof(T);
  typedef T V __attribute__((ext_vector_type(VEC)));
  if (count >= (uint32_t)N && reinterpret_cast<uintptr_t>(row) % 16u == 0) {
    V v[N / VEC];
#pragma unroll
    for (int i = 0; i < N / VEC; ++i) v[i] = reinterpret_cast<const V*>(row)[i];
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = (float)v[i / VEC][i % VEC];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = (uint32_t)i < count ? (float)row[i] : -kInf;
  }
}

// Over the lanes of a wavefront, or over WIDTH neighbouring ones, in every lane and in a fixed order.
template <int WIDTH, typename V, typename Op>
__device__ __forceinline__ V reduce_lanes(V x, Op op) {
#pragma unroll
  for (int off = 1; off < WIDTH; off <<= 1) x = op(x, __shfl_xor(x, off, 64));
  return x;
}
template <int THREADS, typename V, typename Op>
__device__ __forceinline__ V reduce_group(V x, double* scratch, Op op) {
  static_assert(sizeof(V) <= sizeof(double), "a word of scratch each");
  if constexpr (sizeof(V) == 8 && Op::kSum) x = wave::sum(x);
  else x = reduce_lanes<64>(x, op);
  V* all = reinterpret_cast<V*>(scratch);
  __syncthreads();  // the readers of the one before
  if ((threadIdx.x & 63u) == 0) all[threadIdx.x >> 6] = x;
  __syncthreads();
  x = all[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) x = op(x, all[w]);
  return x;
}
struct Add {
  static constexpr bool kSum = true;
  __device__ double operator()(double a, double b) const { return a + b; }
};
struct Larger {
  static constexpr bool kSum = false;
  template <typename V>
  __device__ V operator()(V a, V b) const { return a > b ? a : b; }
};

// Of a row of logits, or a part: the maximum m and the sum of 2^((z - m) scale);
// greedy: the key of the best. A sum below 0: a NaN or plus infinity is among them.
struct RowSum {
  union {
    double m;
    uint64_t best;
  };
  double sum;
};
__device__ __forceinline__ bool has_none(const RowSum& r) { return !(r.sum > 0.0); }

// Larger logits first, equal ones by index; 0 for what is none (NaN, minus infinity).
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
  const uint32_t bits = __float_as_uint(v + 0.0f), order = (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
  return v > -kInf ? ((uint64_t)order << 32) | (uint32_t)~index : 0;
}

// Joins sums of parts whose maxima are `m` and sums `sum` to the whole's maximum.
__device__ __forceinline__ double scaled(double m, double sum, double top, double scale) {
  return sum > 0.0 ? sum * exp2_of((m - top) * scale) : 0.0;
}

// The rows of a sequence, and the draft that a row judges.
struct Rows {
  uint32_t start, end;
  __device__ Rows(const VerifyArgs& args, uint32_t s)
      : start(min(args.row_starts[s], args.rows)), end(min(args.row_starts[s + 1], args.rows)) {}
  __device__ uint32_t draft(const VerifyArgs& args, uint32_t row) const {
    return row + 1 < end ? args.tokens[row + 1] : kNoToken;
  }
};

// What a sequence came to: accepted drafts, and the row that its next token is drawn from.
struct End {
  uint32_t accepted, row;
  uint32_t draft;      // refused there; kNoToken: the row is the last
  uint32_t token;      // decided already (kNoToken), or to be drawn (0)
  RowSum p, q;
};

// What decides about a row but for its sums, which are on their way meanwhile.
struct Judged {
  uint32_t draft;
  float uniform, target, drafted;  // and the draft's logits
  template <typename T>
  __device__ void load(const VerifyArgs& args, const Rows& rows, uint32_t row, T) {
    uniform = target = drafted = 0.0f;
    draft = row < rows.end ? rows.draft(args, row) : kNoToken;
    if (draft >= args.columns || args.greedy) return;
    uniform = args.uniforms[row];
    target = (float)(static_cast<const T*>(args.target) + row * args.target_stride)[draft];
    if (args.draft) drafted = (float)(static_cast<const T*>(args.draft) + row * args.draft_stride)[draft];
  }
  __device__ bool stands(const VerifyArgs& args, const RowSum& p, const RowSum& q) const {
    const double power = exp2_of(((double)target - p.m) * args.scale) / p.sum, pd = power > kLeast ? power : 0.0;
    const double qd = args.draft ? exp2_of(((double)drafted - q.m) * args.scale) / q.sum : 1.0;
    return (double)uniform * qd < pd;
  }
};

// The weights that the next token is drawn by.
template <typename T>
struct Weights {
  static constexpr int kRun = kSpan<T> / kSequence;  // columns of a thread, of those that hold a sequence
  const T *z, *y;  // y null: no draft logits, or the last row
  uint32_t refused;
  Powers<T> p, q;
  double inverse, draft_inverse;
  bool residual;
  __device__ Weights(const VerifyArgs& args, const double* table, const End& end, bool residual)
      : z(static_cast<const T*>(args.target) + end.row * args.target_stride),
        y(args.draft && residual ? static_cast<const T*>(args.draft) + end.row * args.draft_stride : nullptr),
        refused(end.draft), p(table, end.p.m, args.scale), q(table, y ? end.q.m : 0.0, args.scale),
        inverse(p.right / end.p.sum), draft_inverse(y ? q.right / end.q.sum : 0.0), residual(residual) {}
  __device__ __forceinline__ double of(float target, float draft, uint32_t i) const {
#pragma clang fp contract(off)  // equal probabilities leave 0
    double w = p.at(target) * inverse;
    if (y) w -= q.at(draft) * draft_inverse;
    else if (residual && i == refused) w -= 1.0;
    return w > kLeast ? w : 0.0;
  }
  // Of N columns from `first` on, `count` of them there; the others' are 0.
  template <int N>
  __device__ __forceinline__ void run(uint32_t first, uint32_t count, double (&w)[N]) const {
    float target[N], draft[N];
    load_run<N>(z + first, count, target);
    if (y) load_run<N>(y + first, count, draft);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = (uint32_t)i < count ? of(target[i], y ? draft[i] : 0.0f, first + i) : 0.0;
  }
};

// A draw of [0, 1) of the whole weight; below it none. Above it, or NaN, more than all: not the whole
// itself, which a running sum, taken in another order, may pass by a rounding before the last token.
__device__ __forceinline__ double wanted(float draw, double whole) {
  return draw <= 0.0f ? 0.0 : draw < 1.0f ? (double)draw * whole : (double)kInf;
}

// Of a workgroup of kSequence threads: the sum of x over the threads before this one, and over all.
struct Running {
  double before, whole;
};
__device__ __forceinline__ Running running_sum(double x, double* scratch) {
  const uint32_t at = threadIdx.x, lane = at & 63u;
  const double running = wave::running_sum(x);
  __syncthreads();
  if (lane == 63u) scratch[at >> 6] = running;
  __syncthreads();
  Running r = {0.0, 0.0};
#pragma unroll
  for (uint32_t w = 0; w < kSequence / 64; ++w) {
    if (w == (at >> 6)) r.before = r.whole + (running - x);
    r.whole += scratch[w];
  }
  return r;
}

// The first column whose running sum of weights exceeds `want`, `before` being the sum in front of
// this thread's run of N from `first` on; the last with a weight if none does, kNoToken if none has
// one. Threads have their runs in order, so the first lane of the first wavefront with one has it.
template <int N>
__device__ __forceinline__ uint32_t find_token(const double (&w)[N], uint32_t first, double before, double want,
                                               double* scratch) {
  uint32_t hit = kNoToken, behind = kNoToken;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    before += w[i];
    if (w[i] > 0.0) {
      behind = first + i;
      if (before > want && hit == kNoToken) hit = first + i;
    }
  }
  const uint64_t hits = __ballot(hit != kNoToken), weights = __ballot(behind != kNoToken);
  hit = hits ? wave::of_lane(hit, (uint32_t)__builtin_ctzll(hits)) : kNoToken;
  behind = weights ? wave::of_lane(behind, 63u - (uint32_t)__builtin_clzll(weights)) : kNoToken;
  uint2* found = reinterpret_cast<uint2*>(scratch);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) found[threadIdx.x >> 6] = make_uint2(hit, behind);
  __syncthreads();
  hit = behind = kNoToken;
#pragma unroll
  for (int i = 0; i < kSequence / 64; ++i) {
    hit = hit == kNoToken ? found[i].x : hit;
    behind = found[i].y == kNoToken ? behind : found[i].y;
  }
  return hit != kNoToken ? hit : behind;
}

// The rows [first, first + count) of a sequence in turn, from their sums (`each` apart: of the target, and of the
// draft behind it): where it ends, if it does. Threads decide a row each first.
__device__ __forceinline__ bool decide(const VerifyArgs& args, const Rows& rows, const Judged& judged, uint32_t first,
                                       uint32_t count, const RowSum* sums, uint32_t each, uint32_t* states, End* end) {
  enum { kStands = 0, kDraws = 1, kNone = 2 };
  if (threadIdx.x < count) {
    const uint32_t draft = judged.draft;
    const RowSum p = sums[threadIdx.x * each], q = sums[threadIdx.x * each + each - 1u];
    const bool last = draft >= args.columns;
    uint32_t state;
    if (args.greedy) {
      state = !has_none(p) && !last && ~(uint32_t)p.best == draft ? kStands : kDraws;
    } else if (has_none(p) || (!last && args.draft && has_none(q))) {
      state = kNone;
    } else {
      state = !last && judged.stands(args, p, q) ? kStands : kDraws;
    }
    states[threadIdx.x] = state;
  }
  __syncthreads();
  for (uint32_t i = 0; i < count; ++i) {
    const uint32_t state = states[i];
    if (state == kStands) continue;
    const uint32_t draft = rows.draft(args, first + i);
    end->p = sums[i * each];
    end->q = sums[i * each + each - 1u];
    end->row = first + i;
    end->accepted = end->row - rows.start;
    end->draft = draft >= args.columns ? kNoToken : draft;
    end->token = args.greedy ? (has_none(end->p) ? kNoToken : ~(uint32_t)end->p.best) : state == kNone ? kNoToken : 0u;
    return true;
  }
  return false;
}

// ------------------------------------------------------------- short rows

// A wavefront's sum of a whole row, pieces of kRun columns a lane. Rows of up to kAll columns stay
// in registers, longer ones are read a second time from the cache.
template <typename T>
__device__ __forceinline__ RowSum sum_row(const T* z, const double* table, uint32_t columns, double scale, bool greedy) {
  constexpr int kRun = 16 / sizeof(T), kPieces = 4;
  constexpr uint32_t kAll = 64 * kRun * kPieces;
  const uint32_t lane = threadIdx.x & 63u;
  float v[kPieces][kRun];
  const auto load = [&](uint32_t base) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const uint32_t from = base + (i * 64u + lane) * kRun;
      load_run<kRun>(z + from, columns > from ? columns - from : 0u, v[i]);
    }
  };
  // Calls use(value, column) for the columns that there are.
  const auto each = [&](bool loaded, auto use) {
    for (uint32_t base = 0; base < columns; base += kAll) {
      if (!loaded) load(base);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const uint32_t from = base + (i * 64u + lane) * kRun;
        if (from < columns)
#pragma unroll
          for (int c = 0; c < kRun; ++c) use(v[i][c], from + c);
      }
    }
  };
  RowSum row;
  if (greedy) {
    unsigned long long best = 0;
    each(false, [&](float x, uint32_t i) { best = Larger()(best, (unsigned long long)key_of(x, i)); });
    row.best = reduce_lanes<64>(best, Larger());
    row.sum = row.best ? 1.0 : 0.0;
    return row;
  }
  float m = -kInf;
  bool strange = false;
  each(false, [&](float x, uint32_t) {
    strange |= !(x < kInf);
    m = fmaxf(m, x);
  });
  m = wave::max(m);
  row.m = m;
  row.sum = -1.0;
  if (__any(strange)) return row;
  double sum = 0.0;
  if (m > -kInf) {
    const Powers<T> powers(table, row.m, scale);
    each(columns <= kAll, [&](float x, uint32_t) { sum += powers.at(x); });
    sum *= powers.right;
  }
  row.sum = wave::sum(sum);
  return row;
}

template <typename T>
__global__ __launch_bounds__(kSequence) void verify_sequence_kernel(VerifyArgs args) {
  constexpr uint32_t kWaves = kSequence / 64;
  constexpr int kRun = 16 / sizeof(T);
  static_assert(kRun * kSequence >= (int)kShort, "a thread's columns");
  __shared__ double scratch[kWaves];
  __shared__ RowSum sums[kWaves];
  __shared__ uint32_t states[kWaves];
  __shared__ double table[kTable];
  const uint32_t s = blockIdx.x, wave = threadIdx.x >> 6;
  if (!args.greedy) make_table<kSequence>(table);
  const Rows rows(args, s);
  const bool two = args.draft && !args.greedy;
  const uint32_t each = two ? 2u : 1u;
  End end = {0, rows.start, kNoToken, kNoToken, {}, {}};
  for (uint32_t first = rows.start; first < rows.end; first += kWaves / each) {
    const uint32_t row = first + wave / each;
    Judged judged;
    judged.load(args, rows, threadIdx.x < kWaves / each ? first + threadIdx.x : rows.end, T());
    RowSum sum = {{0.0}, 0.0};
    if (row < rows.end) {
      // The row of a sequence's last token has no draft.
      const bool of_draft = two && (wave & 1u);
      const T* z = of_draft ? static_cast<const T*>(args.draft) + row * args.draft_stride
                            : static_cast<const T*>(args.target) + row * args.target_stride;
      if (!of_draft || rows.draft(args, row) < args.columns) sum = sum_row(z, table, args.columns, args.scale, args.greedy);
    }
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) sums[wave] = sum;
    __syncthreads();
    if (decide(args, rows, judged, first, min(kWaves / each, rows.end - first), sums, each, states, &end)) break;
  }
  if (!args.greedy && end.token != kNoToken) {
    const uint32_t first = threadIdx.x * kRun, count = args.columns > first ? args.columns - first : 0u;
    double w[kRun];
    Running running;
    for (bool residual = end.draft != kNoToken;; residual = false) {
      Weights<T>(args, table, end, residual).run(first, count, w);
      double mine = 0.0;
#pragma unroll
      for (int i = 0; i < kRun; ++i) mine += w[i];
      running = running_sum(mine, scratch);
      if (running.whole > 0.0 || !residual) break;  // or p is nowhere above q
    }
    end.token = find_token(w, first, running.before, wanted(args.draws[s], running.whole), scratch);
  }
  if (threadIdx.x == 0) {
    args.accepted[s] = end.accepted;
    args.next_tokens[s] = end.token;
  }
}

// -------------------------------------------------------------- long rows

// Memory of the op: for each row of target and draft the sums of its parts;
// for each sequence where it ended, and the weights of the parts of that row.
struct Workspace {
  RowSum* sums;     // [rows][2][sums parts]
  End* ends;        // [sequences]
  double* weights;  // [sequences][parts]: of max(p - q, 0), or of p
};
template <typename T>
__host__ __device__ uint32_t parts_of(uint32_t columns) {
  return (columns + kSpan<T> - 1u) / kSpan<T>;
}
template <typename T>
__host__ __device__ uint32_t sums_parts_of(uint32_t columns) {
  return (columns + kSumsSpan<T> - 1u) / kSumsSpan<T>;
}
template <typename T>
__host__ __device__ Workspace bind(const VerifyArgs& args, uint64_t sequences) {
  Workspace w;
  w.sums = static_cast<RowSum*>(args.workspace);
  w.ends = reinterpret_cast<End*>(w.sums + 2ull * args.rows * sums_parts_of<T>(args.columns));
  w.weights = reinterpret_cast<double*>(w.ends + sequences);
  return w;
}

// The columns of a part as a thread holds them: pieces of 16 bytes from the first
// boundary on, and a single one of those before and behind.
template <typename T>
struct Part {
  static constexpr int VEC = 16 / sizeof(T);
  typedef T V __attribute__((ext_vector_type(VEC)));
  uint32_t first, head, vectors, tail;
  __device__ Part(const T* row, uint32_t columns, uint32_t part) : first(part * kSumsSpan<T>) {
    const uint32_t size = min(kSumsSpan<T>, columns - first);
    head = min(size, (uint32_t)(-reinterpret_cast<uintptr_t>(row + first) % 16u / sizeof(T)));
    vectors = (size - head) / VEC;
    tail = size - head - vectors * VEC;
  }
};

// Whether a row belongs to a sequence, and, of the draft's, is not a last one. Lanes look for the
// last sequence that starts at or before it.
__device__ __forceinline__ bool is_needed(const VerifyArgs& args, uint32_t row, bool of_draft) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t low = 0, count = args.sequences;
  while (count > 1u) {
    const uint32_t step = (count + 63u) / 64u, at = lane * step;
    const bool before = at < count && args.row_starts[low + at] <= row;
    const uint32_t last = 63u - (uint32_t)__builtin_clzll(__ballot(before) | 1ull);
    low += last * step;
    count = min(step, count - last * step);
  }
  const Rows rows(args, low);
  return row >= rows.start && row < rows.end && (!of_draft || rows.draft(args, row) < args.columns);
}

// The sums of a part of a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs args, uint32_t parts) {
  typedef typename Part<T>::V V;
  constexpr int VEC = Part<T>::VEC;
  __shared__ double scratch[kThreads / 64];
  __shared__ double table[kTable];
  const uint32_t at = threadIdx.x, row = blockIdx.x, which = blockIdx.y / parts, part_index = blockIdx.y - which * parts;
  const T* z = which ? static_cast<const T*>(args.draft) + row * args.draft_stride
                     : static_cast<const T*>(args.target) + row * args.target_stride;
  const Part<T> part(z, args.columns, part_index);
  const V* body = reinterpret_cast<const V*>(z + part.first + part.head);
  V held[kSumsHeld];
#pragma unroll
  for (int i = 0; i < kSumsHeld; ++i) {
    const uint32_t v = at + i * kThreads;
    if (v < part.vectors) held[i] = body[v];
    else
#pragma unroll
      for (int c = 0; c < VEC; ++c) held[i][c] = (T)-kInf;
  }
  const uint32_t edge = part.first + (at < part.head ? at : part.head + part.vectors * VEC + (at - part.head));
  const float single = at < part.head + part.tail ? (float)z[edge] : -kInf;
  const bool needed = is_needed(args, row, which);
  if (!args.greedy) make_table<kThreads>(table);
  if (!needed) return;
  RowSum sum;
  if (args.greedy) {
    unsigned long long best = at < part.head + part.tail ? key_of(single, edge) : 0;
#pragma unroll
    for (int i = 0; i < kSumsHeld; ++i)
#pragma unroll
      for (int c = 0; c < VEC; ++c)
        best = Larger()(best, (unsigned long long)key_of((float)held[i][c],
                                                         part.first + part.head + (at + i * kThreads) * VEC + c));
    sum.best = reduce_group<kThreads>(best, scratch, Larger());
    sum.sum = sum.best ? 1.0 : 0.0;
  } else {
    float m = single;
    bool strange = !(single < kInf);
#pragma unroll
    for (int i = 0; i < kSumsHeld; ++i)
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        strange |= !((float)held[i][c] < kInf);
        m = fmaxf(m, (float)held[i][c]);
      }
    // Plus infinity stands for what is no number.
    float* tops = reinterpret_cast<float*>(scratch);
    m = __any(strange) ? kInf : wave::max(m);
    if ((at & 63u) == 0) tops[at >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) m = fmaxf(m, tops[w]);
    sum.m = m;
    double mine = 0.0;
    if (m > -kInf && m < kInf) {
      const Powers<T> powers(table, sum.m, args.scale);
      mine = powers.at(single);
#pragma unroll
      for (int i = 0; i < kSumsHeld; ++i)
        if (at + i * kThreads < part.vectors)
#pragma unroll
          for (int c = 0; c < VEC; ++c) mine += powers.at((float)held[i][c]);
      mine *= powers.right;
    }
    sum.sum = reduce_group<kThreads>(mine, scratch, Add());
    if (m == kInf) sum.sum = -1.0;
  }
  if (at == 0) bind<T>(args, 0).sums[((uint64_t)row * 2 + which) * parts + part_index] = sum;
}

// Where a sequence ends: groups of 16 lanes join the parts of a row each, 8 rows at a time,
// and the decisions are read from them in turn.
template <typename T>
__device__ __forceinline__ End find_end(const VerifyArgs& args, const Workspace& work, uint32_t s, uint32_t parts,
                                        RowSum* sums, uint32_t* states) {
  constexpr uint32_t kTogether = kThreads / 32;
  const Rows rows(args, s);
  const uint32_t group = threadIdx.x / 16, lane = threadIdx.x % 16;
  End end = {0, rows.start, kNoToken, kNoToken, {}, {}};
  for (uint32_t first = rows.start; first < rows.end; first += kTogether) {
    const uint32_t row = first + group / 2, which = group & 1u;
    const bool needed = row < rows.end && (!which || (args.draft && !args.greedy && rows.draft(args, row) < args.columns));
    Judged judged;
    judged.load(args, rows, threadIdx.x < kTogether ? first + threadIdx.x : rows.end, T());
    RowSum sum = {{0.0}, 0.0};
    const RowSum* from = work.sums + ((uint64_t)row * 2 + which) * parts;
    if (args.greedy) {
      unsigned long long best = 0;
      if (needed)
        for (uint32_t i = lane; i < parts; i += 16u) best = Larger()(best, (unsigned long long)from[i].best);
      sum.best = reduce_lanes<16>(best, Larger());
      sum.sum = sum.best ? 1.0 : 0.0;
    } else {
      double m = -(double)kInf, all = 0.0;
      bool strange = false;
      if (needed)
        for (uint32_t i = lane; i < parts; i += 16u) {
          m = Larger()(m, from[i].m);
          strange |= from[i].sum < 0.0;
        }
      m = reduce_lanes<16>(m, Larger());
      if (needed)
        for (uint32_t i = lane; i < parts; i += 16u) all += scaled(from[i].m, from[i].sum, m, args.scale);
      sum.m = m;
      sum.sum = reduce_lanes<16>(all, Add());
      strange = reduce_lanes<16>((int)strange, Larger());
      if (strange) sum.sum = -1.0;
    }
    __syncthreads();
    if (lane == 0) sums[group] = sum;
    __syncthreads();
    if (decide(args, rows, judged, first, min(kTogether, rows.end - first), sums, 2u, states, &end)) break;
  }
  return end;
}

// Decides a sequence, and sums the weights of a part of the row where it ends.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_weights_kernel(VerifyArgs args, uint32_t parts, uint32_t sequences) {
  __shared__ double scratch[kThreads / 64];
  __shared__ RowSum sums[kThreads / 16];
  __shared__ uint32_t states[kThreads / 32];
  __shared__ double table[kTable];
  if (!args.greedy) make_table<kThreads>(table);
  const uint32_t s = blockIdx.x, part_index = blockIdx.y, at = threadIdx.x;
  const Workspace work = bind<T>(args, sequences);
  const End end = find_end<T>(args, work, s, sums_parts_of<T>(args.columns), sums, states);
  if (part_index == 0 && at == 0) {
    args.accepted[s] = end.accepted;
    if (args.greedy || end.token == kNoToken) args.next_tokens[s] = end.token;
    work.ends[s] = end;
  }
  if (args.greedy || end.token == kNoToken) return;
  const Weights<T> weights(args, table, end, end.draft != kNoToken);
  constexpr int kRun = 16 / sizeof(T);
  double mine = 0.0;
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const uint32_t first = part_index * kSpan<T> + (j * kThreads + at) * kRun;
    double w[kRun];
    weights.run(first, args.columns > first ? args.columns - first : 0u, w);
#pragma unroll
    for (int i = 0; i < kRun; ++i) mine += w[i];
  }
  mine = reduce_group<kThreads>(mine, scratch, Add());
  if (at == 0) work.weights[(uint64_t)s * parts + part_index] = mine;
}

// Finds the part of the row whose weights the draw ends in, and in it the token.
template <typename T>
__global__ __launch_bounds__(kSequence) void verify_token_kernel(VerifyArgs args, uint32_t parts, uint32_t sequences) {
  __shared__ double scratch[kSequence / 64];
  __shared__ double found_before;
  __shared__ uint32_t found_part;
  __shared__ double table[kTable];
  make_table<kSequence>(table);
  const uint32_t s = blockIdx.x, at = threadIdx.x;
  const Workspace work = bind<T>(args, sequences);
  const End end = work.ends[s];
  if (end.token == kNoToken) return;
  bool residual = end.draft != kNoToken;
  constexpr int kRun = Weights<T>::kRun;
  double* part_weights = work.weights + (uint64_t)s * parts;
  const auto sum_parts = [&] {
    double mine = 0.0;
    for (uint32_t i = at; i < parts; i += kSequence) mine += part_weights[i];
    return reduce_group<kSequence>(mine, scratch, Add());
  };
  // This thread's weights of a part, and where they start.
  double w[kRun];
  uint32_t first = 0;
  const auto weigh = [&](uint32_t part) {
    first = part * kSpan<T> + at * kRun;
    Weights<T>(args, table, end, residual).run(first, args.columns > first ? args.columns - first : 0u, w);
    double mine = 0.0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) mine += w[i];
    return mine;
  };
  double whole = sum_parts();
  if (!(whole > 0.0) && residual) {  // p is nowhere above q, which is rare: the parts' weights of p
    residual = false;
    for (uint32_t i = 0; i < parts; ++i) {
      const double mine = reduce_group<kSequence>(weigh(i), scratch, Add());
      if (at == 0) part_weights[i] = mine;
    }
    __syncthreads();
    whole = sum_parts();
  }
  const double want = wanted(args.draws[s], whole);
  if (at < 64u) {  // the first wavefront, 64 parts at a time
    double before = 0.0, last_before = 0.0;
    uint32_t part = kNoToken, last = kNoToken;
    for (uint32_t base = 0; base < parts && part == kNoToken; base += 64u) {
      const double w = base + at < parts ? part_weights[base + at] : 0.0;
      const double running = wave::running_sum(w);
      const uint64_t hit = __ballot(w > 0.0 && before + running > want), live = __ballot(w > 0.0);
      const int lane = hit ? __builtin_ctzll(hit) : live ? 63 - __builtin_clzll(live) : 0;
      const double to = before + wave::of_lane(running - w, (uint32_t)lane);
      if (hit) part = base + lane;
      if (live) {
        last = base + lane;
        last_before = to;
      }
      before += wave::of_lane(running, 63u);
    }
    if (at == 0) {
      found_part = part != kNoToken ? part : last;
      found_before = last_before;
    }
  }
  __syncthreads();
  if (found_part == kNoToken) {  // no weight at all
    if (at == 0) args.next_tokens[s] = kNoToken;
    return;
  }
  const double mine = weigh(found_part);
  const uint32_t token = find_token(w, first, found_before + running_sum(mine, scratch).before, want, scratch);
  if (at == 0) args.next_tokens[s] = token;
}

// One workgroup for a sequence, or its rows in parts over many: the exponentials of 16 rows at a time, 8
// with drafts, against two launches more. 12 rows of 1025 f16 columns, refused early or accepted to
// the end: 14.6 and 20 us by one, 20.2 either way by many; 5 rows of 4096 16.8 and 19.8, 12 of 4096 19.1 to
// 27.7 and 20.4, 30 of 4096 up to 56 and 25; 5 of 8192 26.8 and 23.1. f32: 5 of 4096 16 and 18.
bool together(const VerifyArgs& args) { return args.columns <= kShort && args.rows <= 16ull * args.sequences; }

template <typename Kernel, typename... Args>
hipError_t launch(Kernel kernel, dim3 grid, dim3 block, hipStream_t stream, hipEvent_t start, hipEvent_t stop,
                  Args... args) {
  if (start || stop)
    hipExtLaunchKernelGGL(kernel, grid, block, 0, stream, start, stop, 0, args...);
  else
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, args...);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_typed(const VerifyArgs& args, hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
  if (together(args))
    return launch(verify_sequence_kernel<T>, dim3(args.sequences), dim3(kSequence), stream, start, stop, args);
  if (!args.workspace) return hipErrorInvalidValue;
  const uint32_t parts = parts_of<T>(args.columns), sequences = args.sequences;
  const bool two = args.draft && !args.greedy;
  const uint32_t sums_parts = sums_parts_of<T>(args.columns);
  if (const hipError_t e = launch(verify_sums_kernel<T>, dim3(args.rows, sums_parts * (two ? 2u : 1u)), dim3(kThreads),
                                  stream, start, nullptr, args, sums_parts))
    return e;
  const hipError_t e = launch(verify_weights_kernel<T>, dim3(sequences, args.greedy ? 1u : parts), dim3(kThreads), stream,
                              nullptr, args.greedy ? stop : nullptr, args, parts, sequences);
  if (e || args.greedy) return e;
  return launch(verify_token_kernel<T>, dim3(sequences), dim3(kSequence), stream, nullptr, stop, args, parts, sequences);
}

template <typename T>
uint64_t workspace_typed(const VerifyArgs& args) {
  // Fewer active sequences may no longer be together.
  VerifyArgs one = args;
  one.sequences = 1;
  if (together(one)) return 0;
  const uint64_t parts = parts_of<T>(args.columns);
  return 2ull * args.rows * sums_parts_of<T>(args.columns) * sizeof(RowSum) +
         args.sequences * (sizeof(End) + parts * sizeof(double));
}

}  // namespace

uint64_t verify_workspace(const VerifyArgs& args) {
  return args.f16 ? workspace_typed<_Float16>(args) : workspace_typed<float>(args);
}

hipError_t launch_verify(const VerifyArgs& args, hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
  return args.f16 ? launch_typed<_Float16>(args, stream, start, stop) : launch_typed<float>(args, stream, start, stop);
}

}  // namespace pk
