// pk_cache_attention.hip - attention of new tokens over a paged cache for
// gfx950 (include/pk_cache.h has the formulas and what the arrays may hold).
//
// A unit is one kv head of one sequence and up to R of the rows that read it: the
// G = heads / kv_heads query heads of the sequence's new tokens, token by
// token. Lengths are known on the device alone, so the launch brings more
// workgroups than there are units, and each finds its item from the arrays:
// the tokens of all units over the workgroups left give the longest part, and
// units longer than that are split into equal parts, so that one long sequence
// among short ones fills the device too. Parts meet in memory of the op and a second
// launch joins them in their order.
//
// Single tokens and drafts are bound by memory where sequences are long, else by the chain of
// loads to a unit's first keys and the launches; chunks by the matrix instructions and the exponentials
// beside them. Each kernel has its figures.
//
// Scores are computed transposed, S^T = K Q^T: a lane then holds scores of
// one row, its running maximum and sum stay in that lane, and the exponentials
// are at once the operand of O^T = V^T P^T.
#include "pk_internal.h"
#include "pk_wave.h"

namespace pk {
namespace {

constexpr float kInf = __builtin_inff();
constexpr float kLog2E = 1.4426950408889634f;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kMaxDim = 256;
// Exponentials are taken of a score less a base, in log2 units, which follows the maximum of the scores: it
// is moved to kLift below it when a score passes the base by kMargin and that, so that most
// tiles move nothing. f16: the largest weight is 2^7 to 2^15 (the type ends at 2^16), and one of 2^-32
// of it is not yet 0; with the base at the maximum itself, weights 17 nats below it are off by 44 %, and 17.5
// nats below it 0. f32 has the range anyway.
constexpr float kMargin = 8.0f;
template <typename T>
constexpr float kLift = sizeof(T) == 2 ? 7.0f : 0.0f;
// The exponent of the kernels is fma(product, factor, -base): exact, where the maximum was rounded. From scores
// of 2^24 on that rounding is a factor of 2 and more, in the end beyond the type: a base that far becomes
// kLost, for which every exponential is 0 and which no score passes, and its item goes to the
// plain loop, which takes the rounded score of all.
constexpr float kFar = 16777216.0f, kLost = 3.0e38f;
__device__ __forceinline__ float base_at(float base) { return fabsf(base) < kFar || base == -kInf ? base : kLost; }

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));

// Tokens [low, high).
struct Seen {
  uint32_t low, high;
};
// What a row at `position` of a sequence of `length` tokens sees.
__device__ __forceinline__ Seen seen_by(const CacheAttentionArgs& args, uint32_t length, int64_t position) {
  const uint32_t held = min(length, args.cache.capacity());
  if (!args.causal) return {0u, held};
  if (position < 0) return {0u, 0u};
  const uint32_t p = (uint32_t)position, high = min(p + 1u, held);
  const uint32_t low = args.window && p >= args.window ? p - args.window + 1u : 0u;
  return {min(low, high), high};
}
// What any of `count` rows from `first` on sees.
__device__ __forceinline__ Seen seen_by(const CacheAttentionArgs& args, uint32_t length, int64_t first,
                                        uint32_t count) {
  const Seen last = seen_by(args, length, first + count - 1);
  const Seen start = seen_by(args, length, first < 0 ? 0 : first);
  return {min(start.low, last.high), last.high};
}

// A unit, as the launch that joins finds it.
struct Unit {
  uint32_t slot, parts;        // the record of its first item, and how many
  uint32_t row, rows;          // first row of the sequence, rows of all heads in the unit
  uint32_t head, first;        // kv head, first of the sequence's rows of all heads
};
// What the host chose for a launch: most_units + more workgroups.
struct Plan {
  uint32_t most_units;
  uint32_t more;      // 0: no unit is split
  uint32_t shortest;  // tokens of a part, at least
  uint32_t listed;    // sequences of the list that a launch of its own makes; 0: none
};
// A sequence in the order of the items: its number, first row, rows, blocks of rows, tokens that any of its rows
// sees, length; and, up to and with it, the items, the units, and the records of split units.
struct Listed {
  uint32_t sequence, start, count, tiles, span, length;
  uint32_t parts, items_to, units_to, slots_to;
};
// Memory of the op: the number of units, the list, the units, then a record of each
// item of a split unit: maxima and sums of its rows, then their outputs before the division.
// A unit of more than `longest` tokens has less than 2 span / longest parts, and all
// spans add up to at most `more` times longest: 2 * more records.
struct Workspace {
  uint32_t* units_count;
  Listed* list;
  Unit* units;
  float2* sums;    // [records][R]
  float* outputs;  // [records][R][dim]
};
constexpr uint64_t kHeader = 256;
__host__ __device__ constexpr uint64_t list_bytes(const Plan& p) {
  return (p.listed * sizeof(Listed) + 255u) / 256u * 256u;
}
__host__ __device__ constexpr uint64_t units_bytes(const Plan& p) {
  return (p.most_units * sizeof(Unit) + 255u) / 256u * 256u;
}
uint64_t workspace_bytes(const Plan& p, uint32_t R, uint32_t dim) {
  return kHeader + list_bytes(p) + units_bytes(p) + 2ull * p.more * R * (sizeof(float2) + 4u * dim);
}
__device__ inline Workspace bind(void* memory, const Plan& plan, uint32_t R) {
  uint8_t* p = static_cast<uint8_t*>(memory);
  Workspace w;
  w.units_count = reinterpret_cast<uint32_t*>(p);
  w.list = reinterpret_cast<Listed*>(p + kHeader);
  w.units = reinterpret_cast<Unit*>(p + kHeader + list_bytes(plan));
  w.sums = reinterpret_cast<float2*>(p + kHeader + list_bytes(plan) + units_bytes(plan));
  w.outputs = reinterpret_cast<float*>(w.sums + 2ull * plan.more * R);
  return w;
}

// What a workgroup does: a part of a unit.
struct Item {
  uint32_t sequence, head;   // kv head
  uint32_t row;              // first row of the sequence
  uint32_t first, rows;      // rows of all heads: the first of the sequence's, how many
  uint32_t length;
  int64_t position;          // of the sequence's first row
  uint32_t new_tokens;
  uint32_t parts, part;
  uint32_t unit;             // number of the unit
  uint32_t slot;             // of the unit's first part, if it has several
  bool live;
};

// The item of a workgroup. Workgroups go to the 8 XCDs in turn; 8 neighbouring items, blocks of rows
// of one kv head, go to one, whose L2 has their keys and values then: 4 chunks of 1024 rows 268 us
// and not 272, 16 of up to 188 in f32 44 and not 46.
__device__ __forceinline__ uint32_t item_index() {
  const uint32_t i = blockIdx.x, base = i & ~63u, j = i & 63u;
  return base + 64u <= gridDim.x ? base + (j & 7u) * 8u + (j >> 3) : i;
}

// Sequence s; one behind the last has nothing.
template <int R>
__device__ __forceinline__ Listed look_at(const CacheAttentionArgs& args, uint32_t s) {
  const CacheView& cache = args.cache;
  Listed x = {s, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  if (s < cache.sequences) {
    x.start = min(cache.row_starts[s], cache.rows);
    const uint32_t end = min(cache.row_starts[s + 1], cache.rows), length = cache.lengths[s];
    x.length = length;
    x.count = end > x.start ? end - x.start : 0u;
    x.tiles = (x.count * args.group.by + R - 1u) / R;
    const Seen seen = seen_by(args, length, (int64_t)length - x.count, x.count);
    x.span = x.count ? max(1u, seen.high - seen.low) : 0u;
  }
  return x;
}
// Parts of at most so many tokens, from all units and all their tokens: sum(ceil(span /
// longest)) over the units is at most tokens / longest + units. The quotient is rounded up by
// more than its and the sum's roundings. More units than there can be come from row starts
// that decrease: those are not split, and none is joined.
__device__ __forceinline__ uint32_t longest_part(const Plan& plan, uint32_t units, float tokens) {
  if (!plan.more || units > plan.most_units) return 0x7fffffffu;
  return max(plan.shortest, (uint32_t)min(tokens / (float)plan.more * 1.0001f + 1.0f, 2e9f));
}
__device__ __forceinline__ uint32_t parts_of(uint32_t span, uint32_t longest) {
  return span ? (span + longest - 1u) / longest : 0u;
}

// Item `index` of a sequence whose sums count it: the sums of those before it are these less its own.
template <int R>
__device__ __forceinline__ Item item_in(const CacheAttentionArgs& args, const Listed& x, uint32_t index) {
  const uint32_t units = x.tiles * args.cache.kv_heads, items = units * x.parts, group = args.group.by;
  const uint32_t local = index - (x.items_to - items), unit = local / x.parts;
  Item item;
  item.live = local < items;  // else from sums past 32 bits: of row starts that decrease
  item.sequence = x.sequence;
  item.parts = x.parts;
  item.part = local - unit * x.parts;
  item.head = unit / x.tiles;
  item.first = (unit - item.head * x.tiles) * R;
  item.row = x.start;
  item.new_tokens = x.count;
  item.rows = min((uint32_t)R, x.count * group - item.first);
  item.length = x.length;
  item.position = (int64_t)x.length - x.count;
  item.unit = x.units_to - units + unit;
  item.slot = x.slots_to - (x.parts > 1u ? items : 0u) + unit * x.parts;
  return item;
}

// Finds item `index`; every wavefront for itself, lanes over up to 64 sequences, or over the list.
constexpr uint32_t kUnlisted = 64;
template <int R>
__device__ __forceinline__ Item find_item(const CacheAttentionArgs& args, const Plan& plan, const Workspace& work,
                                          uint32_t index) {
  const CacheView& cache = args.cache;
  const uint32_t lane = threadIdx.x & 63u;
  Item none;
  none.live = false;
  if (plan.listed) {
    // The 64 sequences that the item is in, by the last of each 64, then the one.
    uint32_t at = min((lane + 1u) * 64u, plan.listed) - 1u;
    uint64_t hit = __ballot(index < work.list[at].items_to);
    if (!hit) return none;
    const uint32_t base = (uint32_t)__builtin_ctzll(hit) * 64u;
    at = min(base + lane, plan.listed - 1u);
    hit = __ballot(index < work.list[at].items_to);
    at = base + (uint32_t)__builtin_ctzll(hit);
    return item_in<R>(args, work.list[at], index);
  }
  if (cache.sequences == 1u) {  // no sums over lanes: one token over 300 to 2000 0.4 us less
    Listed only = look_at<R>(args, 0);
    const uint32_t units = only.tiles * cache.kv_heads;
    only.parts = parts_of(only.span, longest_part(plan, units, (float)units * (float)only.span));
    only.units_to = units;
    only.items_to = units * only.parts;
    only.slots_to = only.parts > 1u ? only.items_to : 0u;
    if (plan.more && blockIdx.x == 0 && threadIdx.x == 0) *work.units_count = units > plan.most_units ? 0u : units;
    return index < only.items_to ? item_in<R>(args, only, index) : none;
  }
  Listed mine = look_at<R>(args, lane);
  const uint32_t units = wave::reduce_bits(mine.tiles * cache.kv_heads, 0u, [](uint32_t a, uint32_t b) { return a + b; });
  const float tokens = wave::sum((float)(mine.tiles * cache.kv_heads) * (float)mine.span);
  if (plan.more && blockIdx.x == 0 && threadIdx.x == 0) *work.units_count = units > plan.most_units ? 0u : units;
  // The longest of the sequences first, so that the last workgroups are short ones.
  if (cache.sequences > 1u) {
    uint32_t rank = 0;
    for (uint32_t j = 0; j < cache.sequences; ++j) {
      const uint32_t other = wave::of_lane(mine.span, j);
      rank += other > mine.span || (other == mine.span && j < lane);
    }
    if (lane >= cache.sequences) rank = lane;
    const auto sorted = [&](uint32_t x) { return (uint32_t)__builtin_amdgcn_ds_permute((int)(rank * 4u), (int)x); };
    mine = {sorted(lane), sorted(mine.start), sorted(mine.count), sorted(mine.tiles), sorted(mine.span),
            sorted(mine.length), 0, 0, 0, 0};
  }
  mine.parts = parts_of(mine.span, longest_part(plan, units, tokens));
  const uint32_t have = mine.tiles * cache.kv_heads, items = have * mine.parts;
  mine.items_to = wave::running_sum(items);
  mine.units_to = wave::running_sum(have);
  mine.slots_to = wave::running_sum(mine.parts > 1u ? items : 0u);
  const uint64_t hit = __ballot(index < mine.items_to);
  if (!hit) return none;
  const uint32_t at = (uint32_t)__builtin_ctzll(hit);
  const auto its = [&](uint32_t x) { return wave::of_lane(x, at); };
  const Listed found = {its(mine.sequence), its(mine.start), its(mine.count), its(mine.tiles), its(mine.span),
                        its(mine.length), its(mine.parts), its(mine.items_to), its(mine.units_to), its(mine.slots_to)};
  return item_in<R>(args, found, index);
}

// The list of more than kUnlisted sequences, by one workgroup, instead of a pass of every item over all of
// them: 32 query heads over 8, one token each of up to 500 in f16, take 14.2 us without and 17
// with it at 32 sequences, 20.1 and 21 at 64, 36.8 and 29.4 at 96, 122 and 69 at 256. In
// descending order of the spans, as far as 8 classes to an octave go; which of a class
// comes first may change, and with it who works on what, but no sum.
constexpr int kListThreads = 1024;
constexpr uint32_t kEach = 4;  // sequences of a thread: 4096
template <int R>
__global__ __launch_bounds__(kListThreads) void cache_attention_list_kernel(CacheAttentionArgs args, Plan plan) {
  __shared__ uint32_t order[kListThreads * kEach], classes[256], totals[4][kListThreads / 64];
  __shared__ float all_tokens[kListThreads / 64];
  const Workspace work = bind(args.workspace, plan, R);
  const uint32_t at = threadIdx.x, lane = at & 63u, wave_at = at >> 6, kv = args.cache.kv_heads, n = plan.listed;
  const auto class_of = [](uint32_t span) {
    if (span < 8u) return 255u - span;
    const uint32_t octave = 31u - (uint32_t)__builtin_clz(span);
    return 255u - (octave * 8u + (span >> (octave - 3u) & 7u) - 16u);
  };
  if (at < 256u) classes[at] = 0;
  __syncthreads();
  uint32_t units = 0, place[kEach], kind[kEach];
  float tokens = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    const uint32_t s = at + i * kListThreads;
    if (s >= n) continue;
    const Listed x = look_at<R>(args, s);
    units += x.tiles * kv;
    tokens += (float)(x.tiles * kv) * (float)x.span;
    kind[i] = class_of(x.span);
    place[i] = atomicAdd(&classes[kind[i]], 1u);
  }
  units = wave::reduce_bits(min(units, plan.most_units + 1u), 0u, [](uint32_t a, uint32_t b) { return a + b; });
  units = min(units, plan.most_units + 1u);  // decreasing row starts: no sum past 32 bits
  tokens = wave::sum(tokens);
  if (lane == 0) {
    totals[3][wave_at] = units;
    all_tokens[wave_at] = tokens;
  }
  __syncthreads();
  if (at < 64u) {  // classes before each class
    uint32_t here[4], sum = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      here[c] = sum;
      sum += classes[at * 4u + c];
    }
    const uint32_t before = wave::running_sum(sum) - sum;
#pragma unroll
    for (int c = 0; c < 4; ++c) classes[at * 4u + c] = before + here[c];
  }
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i)
    if (at + i * kListThreads < n) order[classes[kind[i]] + place[i]] = at + i * kListThreads;
  units = 0;
  tokens = 0.0f;
#pragma unroll
  for (int w = 0; w < kListThreads / 64; ++w) {
    units += totals[3][w];
    tokens += all_tokens[w];
  }
  __syncthreads();
  const uint32_t longest = longest_part(plan, units, tokens);
  // A thread's neighbours in this order, and the sums over those before them.
  Listed mine[kEach];
  uint32_t items = 0, have = 0, slots = 0;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    const uint32_t p = at * kEach + i;
    if (p < n) {
      mine[i] = look_at<R>(args, order[p]);
      mine[i].parts = parts_of(mine[i].span, longest);
      const uint32_t own = mine[i].tiles * kv;
      items += own * mine[i].parts;
      have += own;
      slots += mine[i].parts > 1u ? own * mine[i].parts : 0u;
    }
    if (p < n) {
      mine[i].items_to = items;
      mine[i].units_to = have;
      mine[i].slots_to = slots;
    }
  }
  const uint32_t items_to = wave::running_sum(items), units_to = wave::running_sum(have),
                 slots_to = wave::running_sum(slots);
  if (lane == 63u) {
    totals[0][wave_at] = items_to;
    totals[1][wave_at] = units_to;
    totals[2][wave_at] = slots_to;
  }
  __syncthreads();
  uint32_t before[3] = {items_to - items, units_to - have, slots_to - slots};
  for (uint32_t w = 0; w < wave_at; ++w)
#pragma unroll
    for (int c = 0; c < 3; ++c) before[c] += totals[c][w];
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    const uint32_t p = at * kEach + i;
    if (p >= n) continue;
    mine[i].items_to += before[0];
    mine[i].units_to += before[1];
    mine[i].slots_to += before[2];
    work.list[p] = mine[i];
  }
  if (at == 0) *work.units_count = units > plan.most_units ? 0u : units;
}

// tanh: by the exponential, within 2^-23 of 1; NEAR: near 0, where that has lost digits, by its
// series, relative to it.
template <bool NEAR>
__device__ __forceinline__ float tanh_of(float x) {
  const float e = __builtin_amdgcn_exp2f(2.0f * kLog2E * x);
  const float far = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
  if constexpr (!NEAR) return far;
  const float x2 = x * x;
  const float near = __builtin_fmaf(
      x * x2, __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, 0.021869489f, -0.053968254f), 0.13333333f),
                             -0.33333333f), x);
  return fabsf(x) < 0.25f ? near : far;
}

// From the product of a query and a key to the score in log2 units: a capped
// product is the score over `factor`, any other the score itself, with factor > 0:
// queries take the sign of the scale (and 0) with them, exactly. NEAR: any cap. Without, as f16 kernels are
// but for those of large caps, caps up to kNearCap, of which 2^-23 is a tenth of what the rounding of the
// weights to f16 comes to (16 drafts 22.6 us and not 24); of larger ones it is most of the error, and in the end the score.
// Both ways in one kernel cost its registers: 4 chunks of 1024 444 us and not 274, without a cap.
constexpr float kNearCap = 256.0f;
template <bool NEAR>
struct Score {
  float factor, sign, before, after;
  bool capped;
  __device__ explicit Score(const CacheAttentionArgs& args)
      : factor(args.cap > 0.0f || args.scale == 0.0f ? 1.0f : fabsf(args.scale) * kLog2E),
        sign(args.scale > 0.0f ? 1.0f : args.scale < 0.0f ? -1.0f : 0.0f), before(fabsf(args.scale) / args.cap),
        after(args.cap * kLog2E), capped(args.cap > 0.0f) {}
  __device__ __forceinline__ float cap(float dot) const { return after * tanh_of<NEAR>(dot * before); }
};

// Where the tokens of one kv head of a sequence lie, in pieces of 16 bytes
// from the start of a cache: 64 GiB of cache are 2^32 of them.
template <typename T>
struct Places {
  const uint32_t* table;
  uint32_t row, page, head;  // pieces of a token, from page to page, and to the head
  uint32_t count, size, magic, shift;
  __device__ Places(const CacheView& c, uint32_t sequence, uint32_t kv)
      : table(c.page_table + (uint64_t)sequence * c.pages_per_sequence),
        row((uint32_t)(c.head_dim * sizeof(T) / 16u)), page((uint32_t)(c.page_stride * sizeof(T) / 16u)),
        head(kv * c.page_size * (uint32_t)(c.head_dim * sizeof(T) / 16u)), count(c.pages), size(c.page_size),
        magic(c.page.magic), shift(c.page.shift) {}
  static constexpr uint32_t none = 0xffffffffu;
  __device__ __forceinline__ uint32_t at(uint32_t token) const {
    return (uint32_t)(((uint64_t)token * magic) >> shift);
  }
  // The table's entry of a token below `end`.
  __device__ __forceinline__ uint32_t entry(uint32_t token, uint32_t end) const {
    return token < end ? table[at(token)] : none;
  }
  __device__ __forceinline__ uint32_t place(uint32_t token, uint32_t entry) const {
    return entry * page + head + (token - at(token) * size) * row;
  }
};

// The part [from, to) of the tokens that an item works on.
__device__ __forceinline__ Seen part_of(const CacheAttentionArgs& args, const Item& item) {
  const uint32_t token = args.group.under(item.first), last = args.group.under(item.first + item.rows - 1u);
  const Seen all = seen_by(args, item.length, item.position + token, last - token + 1u);
  if (item.parts == 1u) return all;
  const uint32_t each = ((all.high - all.low) / item.parts + 32u) & ~31u;
  const uint64_t low = all.low + (uint64_t)item.part * each;
  return {(uint32_t)min(low, (uint64_t)all.high), (uint32_t)min(low + each, (uint64_t)all.high)};
}

// Writes element d of row r of an item: the output, or what the join needs.
template <typename T, int R>
struct Result {
  const CacheAttentionArgs& args;
  const Item& item;
  const Workspace& work;
  __device__ T* output(uint32_t r) const {
    const uint32_t group = args.group.by, i = item.first + r, token = args.group.under(i);
    return static_cast<T*>(args.output) + (item.row + token) * args.output_stride +
           (uint64_t)(item.head * group + (i - token * group)) * args.cache.head_dim;
  }
  __device__ float* partial(uint32_t r) const {
    return work.outputs + ((uint64_t)(item.slot + item.part) * R + r) * args.cache.head_dim;
  }
  __device__ void sums(uint32_t r, float m, float l) const {
    work.sums[(uint64_t)(item.slot + item.part) * R + r] = make_float2(m, l);
  }
};
// 1 / l, and 0 where no score counted.
__device__ __forceinline__ float inverse(float m, float l) { return m == -kInf && l == 0.0f ? 0.0f : 1.0f / l; }

// Outputs before they are rounded. Weights that were rounded up, and a sum that was not, put a mean of f16's
// largest values beyond the type; a number stays one, and an infinity an infinity.
template <typename T, typename V>
__device__ __forceinline__ V kept_finite(V x, int count) {
  constexpr float kMost = 65504.0f;
  if constexpr (sizeof(T) == 2) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < count; ++i) most = fmaxf(most, fabsf(x[i]));
    if (most > kMost)
#pragma unroll
      for (int i = 0; i < count; ++i) x[i] = fabsf(x[i]) < kInf ? __builtin_amdgcn_fmed3f(x[i], -kMost, kMost) : x[i];
  }
  return x;
}

// Of 64 tokens from t0 on, those below `end`.
__device__ __forceinline__ uint64_t tokens_below(uint32_t t0, uint32_t end) {
  const uint32_t n = end > t0 ? end - t0 : 0u;
  return n >= 64u ? ~0ull : (1ull << n) - 1ull;
}

__device__ __forceinline__ float block_reduce(float x, bool largest, float* scratch) {
#pragma unroll
  for (int off = 32; off; off >>= 1) {
    const float y = __shfl_xor(x, off, 64);
    x = largest ? fmaxf(x, y) : x + y;
  }
  __syncthreads();  // the readers of the reduction before
  if ((threadIdx.x & 63u) == 0) scratch[threadIdx.x >> 6] = x;
  __syncthreads();
  x = scratch[0];
  for (int w = 1; w < kWaves; ++w) x = largest ? fmaxf(x, scratch[w]) : x + scratch[w];
  return x;
}

// An item without matrix instructions: a thread scores a token, then sums an element.
// A product of matrices multiplies every value of a tile by every row's exponential, so that an
// infinity or a NaN that only a later row sees would reach the earlier ones as
// 0 * inf: items whose output is not finite come here, and those of far scores.
template <typename T, int R, bool NEAR>
__device__ __forceinline__ void careful_item(const CacheAttentionArgs& args, const Item& item, const Workspace& work,
                                             float* lds) {
  float *query = lds, *weight = lds + kMaxDim, *scratch = weight + kThreads;
  uint32_t* places = reinterpret_cast<uint32_t*>(scratch + kWaves);
  const CacheView& cache = args.cache;
  const uint32_t at = threadIdx.x, dim = cache.head_dim, group = args.group.by;
  const Seen part = part_of(args, item);
  const Places<T> map(cache, item.sequence, item.head);
  const Score<NEAR> score(args);
  const Result<T, R> result{args, item, work};
  constexpr uint32_t kPiece = 16 / sizeof(T);
  for (uint32_t r = 0; r < item.rows; ++r) {
    const uint32_t i = item.first + r, token = args.group.under(i);
    const Seen own = seen_by(args, item.length, item.position + token);
    const uint32_t low = max(own.low, part.low), high = min(own.high, part.high);
    const T* q = static_cast<const T*>(args.queries) + (item.row + token) * args.query_stride +
                 (uint64_t)(item.head * group + (i - token * group)) * dim;
    __syncthreads();
    if (at < dim) query[at] = (float)q[at] * score.sign;
    float m = -kInf, l = 0.0f, out = 0.0f;
    for (uint32_t t0 = low; t0 < high; t0 += kThreads) {
      __syncthreads();
      const uint32_t t = t0 + at, entry = map.entry(t, high);
      const uint32_t place = entry < map.count ? map.place(t, entry) : Places<T>::none;
      float z = -kInf;
      if (place != Places<T>::none) {
        const T* k = static_cast<const T*>(args.key_cache) + (uint64_t)place * kPiece;
        float dot = 0.0f;
        for (uint32_t d = 0; d < dim; ++d) dot = __builtin_fmaf(query[d], (float)k[d], dot);
        z = (score.capped ? score.cap(dot) : dot) * score.factor;
      }
      places[at] = place;
      const float top = fmaxf(m, block_reduce(z, true, scratch));
      const float base = top == -kInf ? 0.0f : top;
      const float p = __builtin_amdgcn_exp2f(z - base), old = __builtin_amdgcn_exp2f(m - base);
      m = top;
      weight[at] = p;
      l = l * old + block_reduce(p, false, scratch);
      __syncthreads();
      if (at < dim) {
        out *= old;
        const uint32_t count = min((uint32_t)kThreads, high - t0);
        for (uint32_t j = 0; j < count; ++j)
          if (places[j] != Places<T>::none) {
            const T* v = static_cast<const T*>(args.value_cache) + (uint64_t)places[j] * kPiece;
            out = __builtin_fmaf(weight[j], (float)v[at], out);
          }
      }
    }
    if (item.parts == 1u) {
      const floatx4 x = {out * inverse(m, l)};
      if (at < dim) result.output(r)[at] = (T)kept_finite<T>(x, 1)[0];
    } else {
      if (at < dim) result.partial(r)[at] = out;
      if (at == 0) result.sums(r, m, l);
    }
  }
}

// The kernels of few rows: the wavefronts of a workgroup hold the same RB blocks of
// 16 rows and take the steps of tokens in turn, each with maxima, sums and
// outputs of its own, which meet in LDS at the end.
//
// f16: steps of 32 tokens. Keys come from the cache straight into the operand
// of v_mfma_f32_16x16x32_f16 (a lane has 16 bytes of one token, the order of
// the channels being free as long as queries have the same); values go
// through LDS, whose transposed reads give four tokens of a channel, in the
// order in which the scores lie. f32: steps of 16 tokens, v_mfma_f32_16x16x4_f32,
// whose operands take keys and values as they lie.
//
// The loads of a step's keys are issued when the step before has used its own, those of
// its values likewise, and the entries of the page table a step ahead of the keys, before
// the values: loads return in their order, and nothing waits for more than it needs; of the first
// step the queries come between keys and values (f32 chunks below 40 us, behind them 41). Keys and values
// two steps ahead leave one wavefront a SIMD and twice the code: 201 us for 64 sequences below and
// not 182, 10.2 for one token where one was 9.5. Eight wavefronts a workgroup: 197, and 9.7.
//
// f16, 32 heads over 8 of 128 channels: 4 sequences with 131072 tokens 367 us, 5.8 TB/s of keys and
// values, 64 with 200 to 16384 182, 5.3. One token of 8 heads over 376 9.0 us, by the clock from the
// first instruction on: 0.7 for the item, 0.5 for the pages, 2.1 for keys, values and queries, 3.1 for
// three steps, 1.4 for the end; the launch is the rest. 16 drafts of 4 to 8 tokens over up to 6000 (16
// heads over 2 of 64 channels, a window, capped scores) 20.6 us: 1.8, 0.9, 1.8, 8 for four steps,
// 2.7, then the join. f32, 16 chunks of up to 188 rows with windows of 376: 40 us; a SIMD has one wavefront or
// two, and over all of them the matrix instructions are busy 30 % of the time. f32 tokens: 64 sequences 351 us,
// 6.1 TB/s, one over 376 14.7; 16 drafts 38.
template <typename T>
struct Step;
template <>
struct Step<_Float16> {
  static constexpr int kTokens = 32;
};
template <>
struct Step<float> {
  static constexpr int kTokens = 16;
};

template <typename T, int DP, int RB>
struct FewShape {
  static constexpr int kTokens = Step<T>::kTokens;
  static constexpr int kValueBytes = sizeof(T) == 2 ? kTokens * DP * 2 : 0;  // of a wavefront
  static constexpr int kSlice = 64, kSliceRow = kSlice + 4;                  // channels that are joined at a time
  static constexpr int kJoinBytes = kWaves * RB * 16 * kSliceRow * 4;
  static constexpr int kCarefulBytes = (int)(kMaxDim + kThreads + kWaves + kThreads) * 4;
  static constexpr int kSums = 2 * kWaves * RB * 16 * 4;
  // One block of f16 queries stays in registers; others are read from LDS for each step, rows
  // 16 bytes longer than they are, so that 16 of them lie on different banks.
  static constexpr bool kQueriesInLds = sizeof(T) == 4 || RB > 1;
  static constexpr int kQueryRow = DP * (int)sizeof(T) + 16;
  static constexpr int kQueryBytes = kQueriesInLds ? RB * 16 * kQueryRow : 0;
  static constexpr int largest(int a, int b) { return a > b ? a : b; }
  static constexpr int kLds =
      kSums + 16 + largest(largest(kWaves * kValueBytes + kQueryBytes, kJoinBytes), kCarefulBytes);
};

template <typename T, int DP, int RB, bool WHOLE, bool NEAR>
__global__ __launch_bounds__(kThreads, RB > 1 && DP <= 128 && DP * RB <= 256 ? 2 : 1) void cache_attention_few_kernel(
    CacheAttentionArgs args, Plan plan) {
  typedef FewShape<T, DP, RB> Shape;
  constexpr int R = 16 * RB, STEP = Shape::kTokens, TB = STEP / 16;  // token blocks of a step
  constexpr bool kHalf = sizeof(T) == 2;
  constexpr int PIECE = 16 / sizeof(T);
  constexpr int KS = DP / (4 * PIECE);         // pieces of a key in a lane
  constexpr int VR = DP / PIECE;               // pieces of a value row
  constexpr int VS = STEP * VR / 64;           // pieces of a step's values in a lane
  constexpr int OB = DP / 16;                  // blocks of 16 channels
  typedef T V __attribute__((ext_vector_type(PIECE)));
  __shared__ __attribute__((aligned(16))) uint8_t lds[Shape::kLds];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, col = lane & 15u, quarter = lane >> 4;
  const CacheView& cache = args.cache;

  const Workspace work = bind(args.workspace, plan, R);
  const Item item = find_item<R>(args, plan, work, item_index());
  if (!item.live) return;
  if (plan.more && item.part == 0 && item.unit < plan.most_units && threadIdx.x == 0)
    work.units[item.unit] = {item.slot, item.parts, item.row, item.rows, item.head, item.first};
  const Seen part = part_of(args, item);
  const uint32_t group = args.group.by, dim = cache.head_dim;
  const Places<T> map(cache, item.sequence, item.head);
  const Score<NEAR> score(args);
  const uint32_t pieces = dim / PIECE;

  // Queries, and what their rows see.
  constexpr bool kInLds = Shape::kQueriesInLds;
  uint8_t* query_rows = lds + Shape::kSums + 16 + kWaves * Shape::kValueBytes;
  const auto query_piece = [&](uint32_t r, uint32_t c) {
    const uint32_t i = item.first + r, token = args.group.under(i);
    const T* q = static_cast<const T*>(args.queries) + (item.row + token) * args.query_stride +
                 (uint64_t)(item.head * group + (i - token * group)) * dim + c * PIECE;
    V x = V{};
    if (r < item.rows && (WHOLE || c < pieces)) {
      if (args.wide_rows) {
        x = *reinterpret_cast<const V*>(q);
      } else {
#pragma unroll
        for (int e = 0; e < PIECE; ++e) x[e] = q[e];
      }
    }
    return x;
  };
  constexpr int QUERIES = kInLds ? R * VR / kThreads : KS;  // pieces of a thread; on their way to LDS
  static_assert(!kInLds || R * VR % kThreads == 0, "whole rounds of pieces");
  V held[QUERIES];
  const auto query = [&](int b, int k) {
    if constexpr (kInLds)
      return *reinterpret_cast<const V*>(query_rows + (16u * b + col) * Shape::kQueryRow + (4u * k + quarter) * 16u);
    else
      return held[k];
  };
  uint32_t low[RB], high[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const uint32_t r = 16u * b + col;
    const Seen own = seen_by(args, item.length, item.position + args.group.under(item.first + r));
    low[b] = r < item.rows ? own.low : 0u;
    high[b] = r < item.rows ? own.high : 0u;
  }
  // Tokens that all rows of the unit see.
  uint32_t common_low = 0, common_high = 0xffffffffu;
  {
    const uint32_t t0 = args.group.under(item.first), t1 = args.group.under(item.first + item.rows - 1u);
    common_high = seen_by(args, item.length, item.position + t0).high;
    common_low = seen_by(args, item.length, item.position + t1).low;
  }

  float m[RB], l[RB];
  floatx4 out[RB][OB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    m[b] = -kInf;
    l[b] = 0.0f;
#pragma unroll
    for (int o = 0; o < OB; ++o) out[b][o] = floatx4{};
  }

  const uint8_t *keys = static_cast<const uint8_t*>(args.key_cache), *values = static_cast<const uint8_t*>(args.value_cache);
  _Float16* tile = reinterpret_cast<_Float16*>(lds + Shape::kSums + 16 + wave * Shape::kValueBytes);
  V key[TB][KS], value[VS];
  const auto shuffled = [&](uint32_t x, uint32_t from) {
    return (uint32_t)__builtin_amdgcn_ds_bpermute((int)(from * 4u), (int)x);
  };
  const auto load_keys = [&](uint32_t places) {
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      const uint64_t from = (uint64_t)shuffled(places, 16u * t + col) * 16u;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint32_t c = 4u * k + quarter;
        if (WHOLE || c < pieces) key[t][k] = *reinterpret_cast<const V*>(keys + from + c * 16u);
        else key[t][k] = V{};
      }
    }
  };
  // f16: 16 bytes of a row of the step, in their order; f32: channels 64 s + 4
  // col + c of the tokens 4 quarter + r.
  const auto value_token = [&](int i) { return kHalf ? (uint32_t)i * (64u / VR) + lane / VR : 4u * quarter + (i & 3); };
  const auto value_piece = [&](int i) { return kHalf ? lane % VR : (uint32_t)(i >> 2) * 16u + col; };
  const auto load_values = [&](uint32_t places, uint32_t live) {
    if (WHOLE && live == (uint32_t)((1ull << STEP) - 1ull)) {
#pragma unroll
      for (int i = 0; i < VS; ++i)
        value[i] = *reinterpret_cast<const V*>(values + ((uint64_t)shuffled(places, value_token(i)) + value_piece(i)) * 16u);
    } else {
#pragma unroll
      for (int i = 0; i < VS; ++i) {
        const uint32_t token = value_token(i), c = value_piece(i), place = shuffled(places, token);
        value[i] = V{};
        if ((live >> token & 1u) && (WHOLE || c < pieces))
          value[i] = *reinterpret_cast<const V*>(values + ((uint64_t)place + c) * 16u);
      }
    }
  };

  constexpr uint32_t kStride = kWaves * STEP;
  const uint32_t mine = lane % STEP;
  uint32_t t0 = part.low + wave * STEP;
  uint32_t entry = map.entry(t0 + mine, part.high);
  const auto places_of = [&](uint32_t from, uint32_t* live) {
    const bool held = entry < map.count;
    *live = (uint32_t)__ballot(held) & (uint32_t)((1ull << STEP) - 1ull);
    return held ? map.place(from + mine, entry) : 0u;
  };
  uint32_t live = 0, places = 0;
  if (t0 < part.high) {
    places = places_of(t0, &live);
    load_keys(places);
    entry = map.entry(t0 + kStride + mine, part.high);
  }
#pragma unroll
  for (int i = 0; i < QUERIES; ++i) {
    const uint32_t at = threadIdx.x + i * kThreads;
    held[i] = kInLds ? query_piece(at / VR, at % VR) : query_piece(col, 4u * i + quarter);
  }
  if (t0 < part.high) load_values(places, live);
#pragma unroll
  for (int i = 0; i < QUERIES; ++i) held[i] *= (T)score.sign;
  if constexpr (kInLds) {
#pragma unroll
    for (int i = 0; i < QUERIES; ++i) {
      const uint32_t at = threadIdx.x + i * kThreads;
      *reinterpret_cast<V*>(query_rows + at / VR * Shape::kQueryRow + at % VR * 16u) = held[i];
    }
    __syncthreads();
  }
  for (; t0 < part.high; t0 += kStride) {
    floatx4 s[RB][TB];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int t = 0; t < TB; ++t) s[b][t] = floatx4{};
    // f32 chunks leave out pieces that are all behind the head: of 96 and 80 channels 390 and 364 us, not 433 and
    // 422. Single rows do not, which wait for memory and not for this: 179 and not 149.
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      if (!kHalf && !WHOLE && RB > 1 && 4u * k >= pieces) continue;
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const V q = query(b, k);
#pragma unroll
        for (int t = 0; t < TB; ++t) {
          if constexpr (kHalf) {
            s[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key[t][k], q, s[b][t], 0, 0, 0);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[b][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(key[t][k][e], q[e], s[b][t], 0, 0, 0);
          }
        }
      }
    }
    const uint32_t live_now = live;
    const bool more = t0 + kStride < part.high;
    if (more) {
      places = places_of(t0 + kStride, &live);
      load_keys(places);
      entry = map.entry(t0 + 2u * kStride + mine, part.high);
    }
    // Scores, and the hidden ones among them.
    const bool whole = live_now == (uint32_t)((1ull << STEP) - 1ull) && t0 >= common_low && t0 + STEP <= common_high;
    V weights[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      if (score.capped) {
#pragma unroll
        for (int t = 0; t < TB; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[b][t][j] = score.cap(s[b][t][j]);
      }
      if (!whole) {
        const uint32_t seen =
            (live_now & (uint32_t)(tokens_below(t0, high[b]) & ~tokens_below(t0, low[b]))) >> (4u * quarter);
#pragma unroll
        for (int t = 0; t < TB; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[b][t][j] = (seen & (1u << (16 * t + j))) ? s[b][t][j] : -kInf;
      }
      float top = -kInf;
#pragma unroll
      for (int t = 0; t < TB; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, s[b][t][j]);
      top *= score.factor;
      if (__any(top > m[b] + (kMargin + kLift<T>))) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        top = base_at(fmaxf(top - kLift<T>, m[b]));
        const float old = m[b] == top ? 1.0f : __builtin_amdgcn_exp2f(m[b] - top);
        m[b] = top;
        l[b] *= old;
#pragma unroll
        for (int o = 0; o < OB; ++o) out[b][o] *= old;
      }
      const float base = m[b] == -kInf ? 0.0f : m[b];
#pragma unroll
      for (int t = 0; t < TB; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][t][j], score.factor, -base));
          l[b] += p;
          if constexpr (kHalf) weights[b][4 * t + j] = (_Float16)p;
          else weights[b][j] = p;
        }
    }
    if constexpr (kHalf) {
      // 32 bytes of a row, a granule, are found at the row's granule xor a number of the
      // row, so that the 8 rows of a read lie on different banks.
      const auto turned = [](uint32_t row) { return DP >= 128 ? row & 7u : row >> 1 & 3u; };
      wave::sync();
#pragma unroll
      for (int i = 0; i < VS; ++i) {
        const uint32_t row = value_token(i), c = value_piece(i);
        *reinterpret_cast<V*>(tile + row * DP + ((c >> 1) ^ turned(row)) * 16u + (c & 1u) * 8u) = value[i];
      }
      if (more) load_values(places, live);
      wave::sync();
#pragma unroll
      for (int o = 0; o < OB; ++o) {
        V v;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t row = 16u * t + 4u * quarter + (col >> 2);
          const _Float16* from = tile + row * DP + ((uint32_t)o ^ turned(row)) * 16u + (col & 3u) * 4u;
          const half4 four = __builtin_bit_cast(
              half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)from));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * t + e] = four[e];
        }
#pragma unroll
        for (int b = 0; b < RB; ++b) out[b][o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, weights[b], out[b][o], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VS; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int b = 0; b < RB; ++b)
            out[b][(i >> 2) * 4 + c] =
                __builtin_amdgcn_mfma_f32_16x16x4f32(value[i][c], weights[b][i & 3], out[b][(i >> 2) * 4 + c], 0, 0, 0);
      if (more) load_values(places, live);
    }
  }

  // The wavefronts' maxima and sums, and whether an output that another row's
  // tokens could have spoiled is not a number.
  float* sums = reinterpret_cast<float*>(lds);
  uint32_t* strange = reinterpret_cast<uint32_t*>(lds + Shape::kSums);
  if (threadIdx.x == 0) *strange = 0;
  bool odd = false;
  if (args.causal && item.new_tokens > 1u)  // rows that do not all see the same
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int o = 0; o < OB; ++o)
#pragma unroll
        for (int j = 0; j < 4; ++j) odd |= !(fabsf(out[b][o][j]) < kInf);
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    odd |= m[b] == kLost;
    l[b] += __shfl_xor(l[b], 16, 64);
    l[b] += __shfl_xor(l[b], 32, 64);
    if (quarter == 0) {
      sums[wave * R + 16 * b + col] = m[b];
      sums[kWaves * R + wave * R + 16 * b + col] = l[b];
    }
  }
  __syncthreads();
  if (__any(odd) && lane == 0) *strange = 1;
  float scale[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    float top = -kInf;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sums[w * R + 16 * b + col]);
    scale[b] = m[b] == top ? 1.0f : __builtin_amdgcn_exp2f(m[b] - top);
  }
  __syncthreads();
  if (*strange) {
    careful_item<T, R, NEAR>(args, item, work, reinterpret_cast<float*>(lds + Shape::kSums + 16));
    return;
  }
  float* slices = reinterpret_cast<float*>(lds + Shape::kSums + 16);
  const Result<T, R> result{args, item, work};
#pragma unroll
  for (int at = 0; at < DP; at += Shape::kSlice) {
    if (at) __syncthreads();
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      float* to = slices + (wave * R + 16 * b + col) * Shape::kSliceRow;
#pragma unroll
      for (int o = 0; o < 4; ++o) {
        const floatx4 x = out[b][at / 16 + o] * scale[b];
        if constexpr (kHalf) {
          *reinterpret_cast<floatx4*>(to + 16 * o + 4 * quarter) = x;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) to[16 * quarter + 4 * j + o] = x[j];
        }
      }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < item.rows * (Shape::kSlice / 4); i += kThreads) {
      const uint32_t r = i / (Shape::kSlice / 4), d = i % (Shape::kSlice / 4) * 4u;
      if (at + d >= dim) continue;
      floatx4 x = *reinterpret_cast<const floatx4*>(slices + r * Shape::kSliceRow + d);
      float top = sums[r];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) {
        x += *reinterpret_cast<const floatx4*>(slices + (w * R + r) * Shape::kSliceRow + d);
        top = fmaxf(top, sums[w * R + r]);
      }
      float all = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float own = sums[w * R + r];
        all = __builtin_fmaf(sums[kWaves * R + w * R + r], own == top ? 1.0f : __builtin_amdgcn_exp2f(own - top), all);
      }
      if (item.parts > 1u) {
        *reinterpret_cast<floatx4*>(result.partial(r) + at + d) = x;
        if (at + d == 0) result.sums(r, top, all);
        continue;
      }
      x = kept_finite<T>(x * inverse(top, all), 4);
      T* to = result.output(r) + at + d;
      if (args.wide_rows) {
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 four;
#pragma unroll
        for (int e = 0; e < 4; ++e) four[e] = (T)x[e];
        *reinterpret_cast<T4*>(to) = four;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = (T)x[e];
      }
    }
  }
}

// The kernel of many rows, f16: a workgroup of 4 wavefronts with 32 rows each,
// which share tiles of 64 tokens in LDS, two of them: while one is used, the next one
// is loaded straight to the other, 16 tokens by each wavefront; where some of these 16 are hidden or
// have no page they go through registers, zeros in their places. Keys are read as operands of
// v_mfma_f32_32x32x16_f16, 16 bytes of a token, values transposed, four tokens of a channel, in the order
// in which the scores lie: scores 8u .. 8u + 7 of a lane are tokens 16u + 4 half + 0..3 and 8 more.
// Both are laid out so that the lanes that read together read different banks: pieces
// of 16 bytes of a key, and of 32 bytes of a value, are exchanged by a number of the row.
//
// 4 chunks of 700 to 1024 rows over up to 8192 tokens, 32 heads over 8 of 128 channels: 252 to 267 us, 780
// TF where a large product reaches 1032; blocks of 64 rows by the kernel above took 1024. Matrix
// instructions are busy 36 % of the time and the VALU, by its instructions, some 48 %: two wavefronts
// share a SIMD, and these hardly overlap. Pages of 8, 24 or 100 tokens take 270 to 274 us (through
// registers 378). Of DP channels of a tile USED take part in the products, all or three quarters: heads of 96
// and 80 channels 236 and 224 us, of 192 among 256 380; with all 259, 250 and 447.
template <int DP>
struct ManyShape {
  static constexpr int kTokens = 64, kRows = 128;
  static constexpr int kTile = kTokens * DP;  // elements of a tile of keys or of values
  static constexpr int kLds = 4 * kTile * 2 + 16;
  static_assert(4 * kTile * 2 >= (int)(kMaxDim + kThreads + kWaves + kThreads) * 4, "the careful way's LDS");
};

template <int DP, int USED, bool WHOLE, bool NEAR>
__global__ __launch_bounds__(kThreads, DP > 128 ? 1 : 2) void cache_attention_many_kernel(CacheAttentionArgs args,
                                                                                          Plan plan) {
  typedef _Float16 T;
  typedef ManyShape<DP> Shape;
  constexpr int R = Shape::kRows, STEP = Shape::kTokens;
  constexpr int KS = USED / 16, DB = USED / 32, VR = DP / 8;
  constexpr int LOADS = STEP * VR / kThreads;  // pieces of keys, and of values, of a thread
  __shared__ __attribute__((aligned(16))) uint8_t lds[Shape::kLds];
  const uint32_t lane = threadIdx.x & 63u, col = lane & 31u, half = lane >> 5;
  const CacheView& cache = args.cache;

  const Workspace work = bind(args.workspace, plan, R);
  const Item item = find_item<R>(args, plan, work, item_index());
  if (!item.live) return;
  if (plan.more && item.part == 0 && item.unit < plan.most_units && threadIdx.x == 0)
    work.units[item.unit] = {item.slot, item.parts, item.row, item.rows, item.head, item.first};
  const Seen part = part_of(args, item);
  const uint32_t group = args.group.by, dim = cache.head_dim;
  const Places<T> map(cache, item.sequence, item.head);
  const Score<NEAR> score(args);
  const uint32_t pieces = dim / 8u;

  // This lane's query, what its row sees, what all rows of the wavefront see, and any.
  half8 query[KS];
  uint32_t low = 0, high = 0;
  const uint32_t wave = wave::of_lane(threadIdx.x >> 6, 0u), r = 32u * wave + col;
#pragma unroll
  for (int k = 0; k < KS; ++k) query[k] = half8{};
  if (r < item.rows) {
    const uint32_t i = item.first + r, token = args.group.under(i);
    const Seen own = seen_by(args, item.length, item.position + token);
    low = own.low;
    high = own.high;
    const T* q = static_cast<const T*>(args.queries) + (item.row + token) * args.query_stride +
                 (uint64_t)(item.head * group + (i - token * group)) * dim;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const uint32_t c = 2u * k + half;
      if (WHOLE || c < pieces) {
        if (args.wide_rows) {
          query[k] = *reinterpret_cast<const half8*>(q + c * 8u);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) query[k][e] = q[c * 8u + e];
        }
        query[k] *= (T)score.sign;
      }
    }
  }
  Seen any = {0, 0}, all = {0, 0};
  if (32u * wave < item.rows) {
    const uint32_t first = args.group.under(item.first + 32u * wave),
                   last = args.group.under(item.first + min(item.rows, 32u * wave + 32u) - 1u);
    const Seen a = seen_by(args, item.length, item.position + first), b = seen_by(args, item.length, item.position + last);
    all = {b.low, a.high};
    any = {a.low, b.high};
  }

  float m = -kInf, l = 0.0f;
  floatx16 out[DB];
#pragma unroll
  for (int o = 0; o < DB; ++o) out[o] = floatx16{};

  T* tiles = reinterpret_cast<T*>(lds);  // keys, values, keys, values
  const auto key_turn = [](uint32_t row) { return DP == 64 ? row >> 1 & 7u : row & 15u; };
  const auto value_turn = [](uint32_t row) { return (DP == 64 ? (row & 2u) : (row & 3u) << 1) | (row >> 2 & 1u); };

  const uint8_t *keys = static_cast<const uint8_t*>(args.key_cache), *values = static_cast<const uint8_t*>(args.value_cache);
  // Each wavefront stages 16 tokens of a tile, its lanes pieces of 64 / VR of them at a time, each
  // lane the piece that belongs where lanes in their order put 16 bytes each.
  const auto staged_row = [&](int i) { return (uint32_t)i * (64u / VR) + lane / VR; };
  const uint32_t slot = lane % VR;
  // A key's and a value's piece for this lane, of row `row` of the 16: rows turn alike in each 16.
  const auto key_piece = [&](uint32_t row) { return slot ^ key_turn(row); };
  const auto value_piece = [&](uint32_t row) { return (((slot >> 1) ^ value_turn(row)) << 1) | (slot & 1u); };
  // Tiles start at multiples of 16. Where pages hold a multiple of 16 tokens, the wavefront's 16 lie side by
  // side, and what differs from lane to lane is the same for all tiles (4 chunks of 1024: 252 and not 268 us). Not
  // beyond 128 channels, where its registers are not left: two chunks of 1024 131 us and not 241.
  const bool runs = DP <= 128 && cache.page_size % 16u == 0;
  const uint32_t begin = part.low & ~15u;
  uint32_t key_offset[LOADS], value_offset[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const uint32_t row = staged_row(i);
    key_offset[i] = (row * map.row + key_piece(row)) * 16u;
    value_offset[i] = (row * map.row + value_piece(row)) * 16u;
    if constexpr (!WHOLE)  // pieces behind a head are never loaded
#pragma unroll
      for (int stage = 0; stage < 2; ++stage) {
        T* k_to = tiles + stage * 2 * Shape::kTile + 16u * wave * DP + i * 512 + lane * 8u;
        if (key_piece(row) >= pieces) *reinterpret_cast<half8*>(k_to) = half8{};
        if (value_piece(row) >= pieces) *reinterpret_cast<half8*>(k_to + Shape::kTile) = half8{};
      }
  }
  const auto to_lds = [&](const uint8_t* from, T* to, bool there) {
    if (WHOLE || there)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                       (__attribute__((address_space(3))) void*)to, 16, 0, 0);
  };
  // The entries of the next tile's tokens, or, of runs, of its four 16s in lanes 0 to 3.
  const auto next_entry = [&](uint32_t t0) { return map.entry(runs ? t0 + 16u * (lane & 3u) : t0 + lane, part.high); };
  uint32_t entry = next_entry(begin);
  uint64_t live_next = 0;
  const auto load = [&](uint32_t t0, uint32_t stage) {
    T* k_to = tiles + stage * 2u * Shape::kTile + 16u * wave * DP;
    T* v_to = k_to + Shape::kTile;
    const uint32_t ours = t0 + 16u * wave;
    uint32_t places = 0;
    bool whole;
    if (runs) {
      const uint32_t held = (uint32_t)__ballot(entry < map.count) & 15u;
      const uint32_t spread = (held | held << 15) & 0x10001u, more = (held >> 2 | held << 13) & 0x10001u;
      live_next = (((uint64_t)(more * 0xffffu) << 32) | (spread * 0xffffu)) & tokens_below(t0, part.high) &
                  ~tokens_below(t0, part.low);
      whole = (held >> wave & 1u) && ours >= part.low && ours + 16u <= part.high;
      if (whole) {
        const uint64_t from = (uint64_t)map.place(ours, wave::of_lane(entry, wave)) * 16u;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          to_lds(keys + from + key_offset[i], k_to + i * 512, key_piece(staged_row(i)) < pieces);
          to_lds(values + from + value_offset[i], v_to + i * 512, value_piece(staged_row(i)) < pieces);
        }
      } else {
        places = held >> wave & 1u ? map.place(ours, wave::of_lane(entry, wave)) : 0u;
      }
    } else {
      const bool held = entry < map.count && t0 + lane >= part.low;
      live_next = __ballot(held);
      whole = (live_next >> (16u * wave) & 0xffffu) == 0xffffu;
      places = held ? map.place(t0 + lane, entry) : 0u;
      if (whole) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const uint32_t row = staged_row(i);
          const uint64_t place = (uint32_t)__builtin_amdgcn_ds_bpermute((int)((16u * wave + row) * 4u), (int)places);
          to_lds(keys + (place + key_piece(row)) * 16u, k_to + i * 512, key_piece(row) < pieces);
          to_lds(values + (place + value_piece(row)) * 16u, v_to + i * 512, value_piece(row) < pieces);
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint32_t row = staged_row(i), at = 16u * wave + row;
        const uint32_t place = runs ? places + row * map.row
                                    : (uint32_t)__builtin_amdgcn_ds_bpermute((int)(at * 4u), (int)places);
        half8 key = half8{}, value = half8{};
        if (live_next >> at & 1u) {
          if (WHOLE || key_piece(row) < pieces)
            key = *reinterpret_cast<const half8*>(keys + ((uint64_t)place + key_piece(row)) * 16u);
          if (WHOLE || value_piece(row) < pieces)
            value = *reinterpret_cast<const half8*>(values + ((uint64_t)place + value_piece(row)) * 16u);
        }
        *reinterpret_cast<half8*>(k_to + i * 512 + lane * 8u) = key;
        *reinterpret_cast<half8*>(v_to + i * 512 + lane * 8u) = value;
      }
    }
    entry = next_entry(t0 + STEP);
  };
  uint64_t live = 0;
  if (begin < part.high) {
    load(begin, 0);
    live = live_next;
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // what this wavefront loads to LDS is there
  __syncthreads();
  uint32_t stage = 0;
  for (uint32_t t0 = begin; t0 < part.high; t0 += STEP) {
    const bool more = t0 + STEP < part.high;
    if (more) load(t0 + STEP, stage ^ 1u);
    if (t0 < any.high && t0 + STEP > any.low) {
      const T* k_from = tiles + stage * 2u * Shape::kTile;
      const T* v_from = k_from + Shape::kTile;
      floatx16 s[2];
      s[0] = s[1] = floatx16{};
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t piece = (2u * k + half) ^ key_turn(col);
          const half8 x = *reinterpret_cast<const half8*>(k_from + (32u * t + col) * DP + piece * 8u);
          s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, query[k], s[t], 0, 0, 0);
        }
      const bool whole = live == ~0ull && t0 >= all.low && t0 + STEP <= all.high;
      if (score.capped) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[t][j] = score.cap(s[t][j]);
      }
      if (!whole) {
        const uint64_t seen = (live & tokens_below(t0, high) & ~tokens_below(t0, low)) >> (4u * half);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            s[t][j] = ((uint32_t)(seen >> (32 * t)) & (1u << (8 * (j >> 2) + (j & 3)))) ? s[t][j] : -kInf;
      }
      float top = -kInf;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, s[t][j]);
      top *= score.factor;
      if (__any(top > m + (kMargin + kLift<T>))) {
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        top = base_at(fmaxf(top - kLift<T>, m));
        const float old = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= old;
#pragma unroll
        for (int o = 0; o < DB; ++o) out[o] *= old;
      }
      const float base = m == -kInf ? 0.0f : m;
      half8 weights[2][2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][j], score.factor, -base));
          l += p;
          weights[t][j >> 3][j & 7] = (T)p;
        }
      const uint32_t row = 4u * half + (lane >> 2 & 3u), turn = value_turn(row);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int o = 0; o < DB; ++o) {
            half8 v;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const T* from = v_from + (32u * t + 16u * u + 8u * j + row) * DP +
                              ((2u * o + (lane >> 4 & 1u)) ^ turn) * 16u + (lane & 3u) * 4u;
              const half4 four = __builtin_bit_cast(
                  half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)from));
#pragma unroll
              for (int e = 0; e < 4; ++e) v[4 * j + e] = four[e];
            }
            out[o] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, weights[t][u], out[o], 0, 0, 0);
          }
    }
    stage ^= 1u;
    live = live_next;
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
  }

  uint32_t* strange = reinterpret_cast<uint32_t*>(lds + Shape::kLds - 16);
  if (threadIdx.x == 0) *strange = 0;
  bool odd = m == kLost;
  l += __shfl_xor(l, 32, 64);
  if (args.causal && item.new_tokens > 1u)
#pragma unroll
    for (int o = 0; o < DB; ++o)
#pragma unroll
      for (int j = 0; j < 16; ++j) odd |= !(fabsf(out[o][j]) < kInf);
  __syncthreads();
  if (__any(odd) && lane == 0) *strange = 1;
  __syncthreads();
  if (*strange) {
    careful_item<T, R, NEAR>(args, item, work, reinterpret_cast<float*>(lds));
    return;
  }
  if (r >= item.rows) return;
  const Result<T, R> result{args, item, work};
  const float scale = item.parts > 1u ? 1.0f : inverse(m, l);
  T* to = result.output(r);
  float* part_to = result.partial(r);
#pragma unroll
  for (int o = 0; o < DB; ++o) {
    out[o] *= scale;
    if (item.parts == 1u) out[o] = kept_finite<T>(out[o], 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t d = 32u * o + 8u * j + 4u * half;
      if (!WHOLE && d >= dim) continue;
      const floatx4 x = {out[o][4 * j], out[o][4 * j + 1], out[o][4 * j + 2], out[o][4 * j + 3]};
      if (item.parts > 1u) {
        *reinterpret_cast<floatx4*>(part_to + d) = x;
      } else {
        half4 four;
#pragma unroll
        for (int e = 0; e < 4; ++e) four[e] = (T)x[e];
        if (args.wide_rows) {
          *reinterpret_cast<half4*>(to + d) = four;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) to[d + e] = four[e];
        }
      }
    }
  }
  if (item.parts > 1u && half == 0) result.sums(r, m, l);
}

// Joins the parts of a unit: a wavefront takes a row, its lanes 4 channels each, 8 parts' loads at a
// time. 4 to 6 us, the launch among them, whether there are parts or not. 4 rows a workgroup, 0.8 us less
// for 16 drafts than 16 rows; units of 128 rows keep 16, as few of them are split (4 chunks of 1024 5.8 and 7.7).
__host__ __device__ constexpr int join_rows(int R) { return R > 64 ? 16 : 4; }
template <typename T, int R>
__global__ __launch_bounds__(64 * join_rows(R)) void cache_attention_join_kernel(CacheAttentionArgs args, Plan plan) {
  const Workspace work = bind(args.workspace, plan, R);
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const Unit unit = work.units[blockIdx.x];
  if (blockIdx.x >= *work.units_count || unit.parts <= 1u) return;
  const uint32_t group = args.group.by, dim = args.cache.head_dim;
  const uint32_t d = 4u * lane < dim ? 4u * lane : 0u;  // all lanes take part in the exchange
  const uint32_t r = blockIdx.y * join_rows(R) + wave;
  if (r >= unit.rows) return;
  const float2* sums = work.sums + (uint64_t)unit.slot * R + r;
  float top = -kInf;
  for (uint32_t p = lane; p < unit.parts; p += 64u) top = fmaxf(top, sums[(uint64_t)p * R].x);
  top = wave::max(top);
  float all = 0.0f;
  floatx4 x = floatx4{};
  for (uint32_t p0 = 0; p0 < unit.parts; p0 += 64u) {
    const uint32_t p = p0 + lane;
    float factor = 0.0f;
    if (p < unit.parts) {
      const float2 own = sums[(uint64_t)p * R];
      factor = own.x == top ? 1.0f : __builtin_amdgcn_exp2f(own.x - top);
      all += own.y * factor;
    }
    const uint32_t count = min(64u, unit.parts - p0);
    const float* from = work.outputs + ((uint64_t)(unit.slot + p0) * R + r) * dim + d;
    const auto add = [&](const floatx4& part, uint32_t lane_of) {
      x += part * __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(factor), (int)lane_of));
    };
    uint32_t i = 0;
    for (; i + 8u <= count; i += 8u) {  // eight loads at a time
      floatx4 some[8];
#pragma unroll
      for (uint32_t j = 0; j < 8u; ++j) some[j] = *reinterpret_cast<const floatx4*>(from + (uint64_t)(i + j) * R * dim);
#pragma unroll
      for (uint32_t j = 0; j < 8u; ++j) add(some[j], i + j);
    }
    if (i < count) {  // those behind the last are loaded and not added: 0 times an infinity is none
      floatx4 some[7];
#pragma unroll
      for (uint32_t j = 0; j < 7u; ++j)
        some[j] = *reinterpret_cast<const floatx4*>(from + (uint64_t)min(i + j, count - 1u) * R * dim);
#pragma unroll
      for (uint32_t j = 0; j < 7u; ++j)
        if (i + j < count) add(some[j], i + j);
    }
  }
  all = wave::sum(all);
  x = kept_finite<T>(x * inverse(top, all), 4);
  const uint32_t i = unit.first + r, token = args.group.under(i);
  T* to = static_cast<T*>(args.output) + (unit.row + token) * args.output_stride +
          (uint64_t)(unit.head * group + (i - token * group)) * dim + d;
  if (4u * lane < dim)
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = (T)x[e];
}

typedef void (*Kernel)(CacheAttentionArgs, Plan);
struct Variant {
  Kernel kernel, list, join;
  uint32_t rows;  // of a unit
};

// Of large caps in f16 one kernel for heads of any width.
template <typename T, int DP, int RB>
Variant few(bool whole, bool near) {
  constexpr bool kNear = sizeof(T) == 4;
  return {near && !kNear ? cache_attention_few_kernel<T, DP, RB, false, true>
          : whole        ? cache_attention_few_kernel<T, DP, RB, true, kNear>
                         : cache_attention_few_kernel<T, DP, RB, false, kNear>,
          cache_attention_list_kernel<16 * RB>, cache_attention_join_kernel<T, 16 * RB>, 16 * RB};
}

template <int DP>
Variant many(uint32_t dim, bool near) {
  constexpr int kNarrow = DP > 64 ? DP / 4 * 3 : DP;
  return {near                       ? cache_attention_many_kernel<DP, DP, false, true>
          : dim == (uint32_t)DP      ? cache_attention_many_kernel<DP, DP, true, false>
          : dim <= (uint32_t)kNarrow ? cache_attention_many_kernel<DP, kNarrow, false, false>
                                     : cache_attention_many_kernel<DP, DP, false, false>,
          cache_attention_list_kernel<ManyShape<DP>::kRows>, cache_attention_join_kernel<_Float16, ManyShape<DP>::kRows>,
          ManyShape<DP>::kRows};
}

// Rows of a unit: 16, 32 or 64 where the rows of an average sequence need no more, else
// 128 (f16). f16 units have 64 rows for heads of up to 64 channels: beyond, their outputs and keys
// fill the registers. f32 units end at 64, 32 and 16 rows for heads of up to 64, 128 and 256
// channels. 16 sequences with 32 to 64 rows of 64 channels, 1500 to 6000 tokens: 64 rows 22.2 us,
// 128 30.1. 8 sequences with 48 to 64 rows of 128 channels, up to 8192 tokens: 47 us by 64 rows, 29
// by 128, 41 by 32; 24 to 32 rows 25.8 by 32 rows, 25.6 by 128, and 64 such sequences of up to
// 1000 24.6 and 28.7. Of 256 channels, 8 with 64 rows, up to 4000 tokens: 55.7 by 32, 38.7 by 128; with
// 32 rows 32 and 36.5. f32, 256 channels, 4 chunks of 512: 937 us by 16 rows, 1402 by 32, which spill.
uint32_t unit_rows(const CacheAttentionArgs& args) {
  const uint64_t group = args.group.by;
  const uint64_t rows = (args.cache.rows * group + args.cache.sequences - 1u) / args.cache.sequences;
  const uint32_t dim = args.cache.head_dim, most = args.f16 ? 128u : dim <= 64u ? 64u : dim <= 128u ? 32u : 16u;
  const uint32_t wanted = rows <= 16u ? 16u : rows <= 32u ? 32u : rows > 64u ? 128u : dim <= 64u ? 64u : 128u;
  return wanted < most ? wanted : most;
}

template <typename T, int DP>
Variant choose(uint32_t rows, uint32_t dim, bool near) {
  constexpr bool kHalf = sizeof(T) == 2;
  if constexpr (kHalf || DP <= 128)
    if (rows == 32u) return few<T, DP, 2>(dim == (uint32_t)DP, near);
  if constexpr (DP <= 64)
    if (rows == 64u) return few<T, DP, 4>(dim == (uint32_t)DP, near);
  if constexpr (kHalf)
    if (rows == 128u) return many<DP>(dim, near);
  return few<T, DP, 1>(dim == (uint32_t)DP, near);
}
template <typename T>
Variant choose(const CacheAttentionArgs& args) {
  const uint32_t dim = args.cache.head_dim, rows = unit_rows(args);
  const bool near = args.cap > kNearCap;
  if (dim <= 64u) return choose<T, 64>(rows, dim, near);
  if (dim <= 128u) return choose<T, 128>(rows, dim, near);
  return choose<T, 256>(rows, dim, near);
}

// Tokens of a part at least, and workgroups beside one for each unit, of which parts are made: a
// part costs its start, and its record's way to the join. Parts of 256, 512 and 1024: one token of 32 over 8
// heads of 128 channels in f16 over 2000 tokens takes 12, 14.9 and 20.6 us, 8 such over 500 to 2000
// 16.7, 15.5 and 20.5; 16 drafts over up to 6000 22.8, 22.4 and 27.5. Twice as many workgroups: one token over 131072 132
// us and not 113, 64 over up to 16384 187 and not 183 (half as many 198); of 32 rows, 4 drafts over 32768
// 71 and not 61 (60); of 64 rows 82 and not 67 (117). Of 128 rows half as many: two chunks of 512
// over 16000 206 us and not 181 (twice as many 199), eight of 100 to 300 over up to 8192 52 and not 59.
constexpr uint32_t kShortest = 512;

Plan plan_of(const CacheAttentionArgs& args, uint32_t R) {
  const uint64_t group = args.group.by;
  const uint32_t some = args.cache.sequences < args.cache.rows ? args.cache.sequences : args.cache.rows;
  Plan plan;
  // Full tiles of rows, and one that is not full for each sequence.
  plan.most_units = (uint32_t)(args.cache.kv_heads * (args.cache.rows * group / R + some));
  // Tokens that the rows of a unit see: of a window those before its first row's, and the unit's own.
  const uint64_t own = (R - 1u) / group + 2u, seen = args.causal && args.window ? args.window + own : ~0ull;
  plan.more = args.cache.capacity() > kShortest && seen > kShortest ? (R == 16u ? 1024u : R == 64u ? 256u : 512u) : 0u;
  plan.shortest = kShortest;
  plan.listed = args.cache.sequences > kUnlisted ? args.cache.sequences : 0u;
  return plan;
}

}  // namespace

uint64_t cache_attention_workspace(const CacheAttentionArgs& args) {
  // Any number of active sequences: the rows of a unit follow from it.
  CacheAttentionArgs one = args;
  one.cache.sequences = 1;
  uint64_t most = 0;
  for (uint32_t rows = unit_rows(args); rows <= unit_rows(one); rows *= 2) {
    const Plan plan = plan_of(args, rows);
    const uint64_t bytes = workspace_bytes(plan, rows, args.cache.head_dim);
    if ((plan.more || plan.listed) && bytes > most) most = bytes;
  }
  return most;
}

hipError_t launch_cache_attention(const CacheAttentionArgs& args, hipStream_t stream, hipEvent_t start,
                                  hipEvent_t stop) {
  const Variant variant = args.f16 ? choose<_Float16>(args) : choose<float>(args);
  const Plan plan = plan_of(args, variant.rows);
  if ((plan.more || plan.listed) && workspace_bytes(plan, variant.rows, args.cache.head_dim) > args.workspace_bytes)
    return hipErrorInvalidValue;
  const dim3 grid(plan.most_units + plan.more), block(kThreads);
  if (plan.listed) {
    if (start)
      hipExtLaunchKernelGGL(variant.list, dim3(1), dim3(kListThreads), 0, stream, start, nullptr, 0, args, plan);
    else
      hipLaunchKernelGGL(variant.list, dim3(1), dim3(kListThreads), 0, stream, args, plan);
    if (const hipError_t e = hipGetLastError()) return e;
    start = nullptr;
  }
  if (start || (stop && !plan.more))
    hipExtLaunchKernelGGL(variant.kernel, grid, block, 0, stream, start, plan.more ? nullptr : stop, 0, args, plan);
  else
    hipLaunchKernelGGL(variant.kernel, grid, block, 0, stream, args, plan);
  if (const hipError_t e = hipGetLastError()) return e;
  if (!plan.more) return hipSuccess;
  // Each unit that is split has one of the workgroups beside the units' at least; of sorted sequences its units come first.
  const uint32_t split = plan.listed || plan.most_units < plan.more ? plan.most_units : plan.more;
  const dim3 units(split, variant.rows / join_rows(variant.rows)), joining(64 * join_rows(variant.rows));
  if (stop)
    hipExtLaunchKernelGGL(variant.join, units, joining, 0, stream, nullptr, stop, 0, args, plan);
  else
    hipLaunchKernelGGL(variant.join, units, joining, 0, stream, args, plan);
  return hipGetLastError();
}

}  // namespace pk
