// One new token a stream against a window's cache held in 4 bits: the step of
// attention.cu over rows of codes, x ~ (c - 7.5) step + middle with c in 0..15.
//
//   score_t = scale q . k_t = scale (step_t (q . c_t) + (middle_t - 7.5 step_t) sum q)
//   out = sum p_t v_t = sum (p_t step_t) (c_t - 7.5) + sum p_t middle_t
//
// so that codes go to the products as they are, as float16 numbers, which
// is exact, and the ranges stay outside: a key's in two numbers a score, a value's in
// its weight p_t step_t and in one float sum a head, which no rounding meets. q and the
// weights are scaled by powers of two into float16's range, whatever the tokens' type:
// of a head's q nothing is lost within 2^-25 of its largest channel, and the weights
// are rounded once, to 11 bits: the products take no wider operands, codes in 16 bits are
// exact, and a second product of what the rounding takes would be the dearest part made twice
// (3 long memories in float16: error against 64 bits 3.1e-4, with float weights 2.1e-4).
//
// The cache is read once; taking a word of eight codes apart costs 5 or 6 instructions
// though, which with the rest weigh about as much as the reading. So the work is cut evenly:
// the turns of 32 slots of all streams and key-value heads (up to 16 query heads; more:
// several times) in one line, of which every warp has the same share, wherever that
// begins and ends. A warp keeps a ring in shared memory filled some turns ahead, waits for
// no other, and leaves the sums of its part of each stream's head in a workspace, which
// a second kernel joins in order.
//
// 96 streams of 4100 slots, 16 heads (4) of 128 channels, 214 MB: 58 us (3.7 TB/s); 3 streams
// of 65,536 slots, 24 heads (8) of 96 channels, 164 MB: 44 us. The first's reading alone
// takes 40 to 48 us, all but the reading 44, starting and ending about 7 of either: the
// two do not overlap entirely. Joining takes 6 to 8 us. Between 12 and 20 warps a
// multiprocessor, deeper rings, turns loaded by whole blocks or clusters: none was faster;
// the kernels for more than 64 channels spill 50 to 170 bytes a thread at 16 warps, and were no
// faster with fewer warps that spill nothing. Rows that are not whole 16-byte words come by
// 4-byte copies: of 120 channels 146 us, of 72 103, where 128 and 96 take 59 and 54. One stream
// of 1028 slots: 7 and 5 us, launches and latency.
//
//   scores [slots x heads] = K q^T: a lane's words of two key rows are its parts of
//     the products, with q's channels permuted alike;
//   out [dim x heads] += V^T P^T: a lane's words of two value rows, interleaved, are
//     its parts of four products; P turns around in registers (movmatrix).
//
// So slots and channels fill the products' 16 rows, and 8 heads their columns.
#include <algorithm>

#include "tensorcore.cuh"

namespace gs {
namespace {

// Set when a bounded wait ran out (window_attention_4bit_status).
__device__ uint32_t g_timeout;

constexpr int kMaxDim = 128;
constexpr int kWarps = 4, kThreads = 32 * kWarps;
// What registers and shared memory allow.
constexpr int blocks_per_sm(int dim, int sets) { return sets == 1 ? 4 : dim == 64 ? 3 : 2; }
constexpr int kSlots = 32;  // of a warp's turn
constexpr float kLog2e = 1.44269504f;
// As in attention.cu: growth (log2) of the scores' maximum that passes without
// rescaling, and the weights' place above it in float16.
constexpr float kSlack = 8.0f, kLift = 7.0f;

template <int kDim>
struct Stage {
  static constexpr int kCount = kDim == 128 ? 3 : 5;  // of a warp's ring
  static constexpr int kRow = kDim / 2;  // bytes; shorter rows leave the rest as it is
  alignas(16) unsigned char codes[2][kSlots * kRow];  // keys', values'
};

// What a slot's ranges come to: score = (dot with c - 7.5) * key_step + (sum of q) *
// key_middle.
// Each twice, for instructions on two floats (a lane's two heads).
struct Slot {
  float2 key_step, key_middle, value_step, value_middle;
};

template <int kDim>
struct Shared {
  Stage<kDim> stage[kWarps][Stage<kDim>::kCount];
  alignas(16) Slot slot[kWarps][kSlots];
  uint64_t full[kWarps][Stage<kDim>::kCount];
};

// What a warp leaves of its part of an item, for each of `heads` query heads: outputs
// times the sum, then the heads' maxima and sums. A part with a unit of values from 2^20 on is
// large: its outputs are 2^-64 as large, and its sums negative to show it.
template <int kDim>
struct Parts {
  float* data;
  int32_t heads;
  __host__ __device__ int64_t floats() const { return int64_t{heads} * (kDim + 2) + (heads & 1) * 2; }
  __device__ float* out(int64_t part, int h) const { return data + part * floats() + h * kDim; }
  __device__ float* top(int64_t part, int h) const {
    return data + part * floats() + heads * kDim + h;
  }
  __device__ float* sum(int64_t part, int h) const { return top(part, h) + heads; }
};
constexpr uint32_t kLargeUnit = (127 + 20) << 23;  // 2^20's bits
constexpr float kLargeScale = 0x1p64f;
constexpr float kFar = 0x1p100f, kFarScale = 0x1p64f;  // of queries' channels

// The warps that have an item's first and last turn.
struct Reach {
  int32_t first, last;
};

// A stream's slots that count (0: idle), and its turns.
struct Stream {
  int64_t position;
  int count, turns;
};
__device__ __forceinline__ Stream stream_at(const gs_window_attention_step_4bit_args& a, int64_t b) {
  const int64_t position = a.positions[b];
  const int count = position < 0 ? 0 : static_cast<int>(min(position, int64_t{a.slots} - 1)) + 1;
  return {position, count, (count + kSlots - 1) / kSlots};
}

// The line of turns: stream after stream, each `heads` (key-value heads times pieces of
// query heads) times its turns. (More than kCounted streams are not counted first, which
// would take a microsecond a thousand: each is in the line with the turns of a full cache,
// and a warp passes over those that it lacks.) Warp w of `warps` has turns [w total / warps,
// (w + 1) total / warps) of it, one at least.
struct Line {
  int64_t total, warps;
  int64_t stream, before;  // the stream that has the warp's first turn, the turns before it
};
constexpr int kCounted = 1024;
__device__ __forceinline__ int turns_in_line(const gs_window_attention_step_4bit_args& a,
                                             const Stream& s) {
  return a.batch > kCounted ? (a.slots + kSlots - 1) / kSlots : s.turns;
}
// By a whole warp.
__device__ Line find_turn(const gs_window_attention_step_4bit_args& a, int heads, int64_t w,
                          int64_t warps) {
  const int lane = threadIdx.x & 31;
  if (a.batch > kCounted) {
    const int64_t each = int64_t{turns_in_line(a, {})} * heads;
    const int64_t total = a.batch * each, at = w * total / min(warps, total);
    return {total, min(warps, total), at / each, at / each * each};
  }
  int64_t total = 0;
  for (int64_t b = lane; b < a.batch; b += 32) total += int64_t{stream_at(a, b).turns} * heads;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  warps = min(warps, total);
  Line line = {total, warps, 0, 0};
  if (w >= warps) return line;
  const int64_t at = w * total / warps;
  for (int64_t b0 = 0; b0 < a.batch; b0 += 32) {
    const int64_t mine = b0 + lane < a.batch ? int64_t{stream_at(a, b0 + lane).turns} * heads : 0;
    int64_t through = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, through, o);
      if (lane >= o) through += x;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, line.before + through > at);
    if (past) {
      const int first = __ffs(past) - 1;
      line.stream = b0 + first;
      line.before += __shfl_sync(0xffffffffu, through - mine, first);
      return line;
    }
    line.before += __shfl_sync(0xffffffffu, through, 31);
  }
  line.stream = a.batch;
  return line;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// The code of x. In double: (x - middle) and the quotient are then far more exact than
// any two codes' border is close (step has 8 or 11 bits), so that ties are ties.
__device__ __forceinline__ uint32_t code_of(float x, float step, float middle) {
  if (!(step > 0.0f && step < INFINITY)) return 8;
  const double place = rint((static_cast<double>(x) - middle) / static_cast<double>(step) + 7.5);
  return static_cast<uint32_t>(fmin(fmax(place, 0.0), 15.0));
}

// The new token's rows as they are held: lanes 0 to 15 have a word of eight channels of
// the key's row each, lanes 16 to 31 of the value's.
struct Fresh {
  uint32_t codes, range;
};
template <class T>
__device__ __forceinline__ Fresh round_row(const T* row, int dim) {
  const int word = threadIdx.x & 15;
  float x[8], high = -INFINITY, low = INFINITY;
  if (8 * word < dim) {
    load_pack<8>(row + 8 * word, x);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      high = max_nan(high, x[k]);
      low = min_nan(low, x[k]);
    }
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, o));
    low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  // Where the spread leaves float's range, by halves.
  const float spread = high - low;
  const T step = from_float<T>(isinf(spread) ? (0.5f * high - 0.5f * low) / 15.0f * 2.0f
                                             : spread / 15.0f);
  const T middle = from_float<T>(0.5f * high + 0.5f * low);
  Fresh f = {0, 0};
  if (8 * word < dim)
#pragma unroll
    for (int k = 0; k < 8; ++k)
      f.codes |= code_of(x[k], to_float(step), to_float(middle)) << 4 * k;
  f.range = static_cast<uint32_t>(reinterpret_cast<const uint16_t&>(step)) |
            static_cast<uint32_t>(reinterpret_cast<const uint16_t&>(middle)) << 16;
  return f;
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t word) {
  const T* v = reinterpret_cast<const T*>(&word);
  return make_float2(to_float(v[0]), to_float(v[1]));
}

// Codes 0 to 3 of both halves of a word as four pairs of float16 numbers, with nothing to
// convert: the bits 0 to 3 of a half are the subnormal number c 2^-24, bits 4 to 7 are 16 c
// 2^-24, which the products take exactly. So pairs 1 and 3 are 16 times as large.
constexpr float kCodeUnit = 16777216.0f;  // 2^24
__device__ __forceinline__ void spread(uint32_t word, uint32_t (&pair)[4]) {
  const uint32_t next = word >> 8;
  pair[0] = word & 0x000f000fu;
  pair[1] = word & 0x00f000f0u;
  pair[2] = next & 0x000f000fu;
  pair[3] = next & 0x00f000f0u;
}

// The same of two slots' words, for values: pairs 0 and 2 are the low codes, and pairs 1 and
// 3 whole bytes, low + 16 high: one instruction less, and their sums are told apart at the end.
__device__ __forceinline__ void spread_bytes(uint32_t word, uint32_t (&pair)[4]) {
  pair[0] = word & 0x000f000fu;
  pair[1] = word & 0x00ff00ffu;
  pair[3] = __byte_perm(word, 0, 0x4341);
  pair[2] = pair[3] & 0x000f000fu;
}

// c += a b, 16 x 16 by 16 x 8.
__device__ __forceinline__ void multiply(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c = a b.
__device__ __forceinline__ void multiply_new(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// An 8 x 8 matrix of pairs, a row in four lanes, turned around.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int kWords>
__device__ __forceinline__ void read_words(const unsigned char* p, uint32_t (&w)[kWords]) {
  static_assert(kWords <= 4);
  if constexpr (kWords == 1 || kWords == 3) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  } else if constexpr (kWords == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x;
    w[1] = x.y;
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x;
    w[1] = x.y;
    w[2] = x.z;
    w[3] = x.w;
  }
}

// kKeyWords: a lane's words of a key's row, which four share. kSets: of 8 heads. kMasked: with validity of the slots. kAligned: rows of codes are
// whole 16-byte words.
template <class T, int kDim, int kKeyWords, int kSets, bool kMasked, bool kAligned>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(kDim, kSets))
    step_kernel(gs_window_attention_step_4bit_args a, Parts<kDim> parts, Reach* reach) {
  using S = Shared<kDim>;
  constexpr int kRow = Stage<kDim>::kRow, kStages = Stage<kDim>::kCount;
  constexpr int kValueWords = kDim / 64;  // a lane's words of a value's row, which eight share
  constexpr int kHeads = 8 * kSets;
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  S& s = *reinterpret_cast<S*>(shared_bytes);
  chain_wait();
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // one for the whole warp
  const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const int group = a.heads / a.kv_heads, pieces = (group + kHeads - 1) / kHeads;
  const int row_bytes = a.dim / 2;
  const int pitch = kAligned ? row_bytes : kRow;  // of a staged row
  if constexpr (kAligned) {
    if (lane == 0) {
      for (uint64_t& bar : s.full[warp]) tc::barrier_init(tc::shared_address(&bar), 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      tc::fence_async_shared();
    }
    __syncwarp();
  }
  const int64_t me = int64_t{blockIdx.x} * kWarps + warp;
  const Line line = find_turn(a, a.kv_heads * pieces, me, int64_t{gridDim.x} * kWarps);
  if (me >= line.warps) return;
  int64_t at = me * line.total / line.warps, b = line.stream;
  int64_t before = line.before;  // turns before the stream's
  const int64_t end = (me + 1) * line.total / line.warps;
  bool good = true;
  // The ring goes on from part to part: the next turn's stage, and its barrier's phase.
  uint32_t stage = 0, phase = 0;
  while (at < end) {
  const Stream stream = stream_at(a, b);
  const int places = turns_in_line(a, stream);
  if (at - before >= int64_t{places} * a.kv_heads * pieces) {
    before += int64_t{places} * a.kv_heads * pieces;
    ++b;
    continue;
  }
  const int64_t head_piece = (at - before) / places;
  const int first_turn = static_cast<int>((at - before) % places);
  const int here = static_cast<int>(min(int64_t{places - first_turn}, end - at));
  const int turns = min(here, stream.turns - first_turn);
  at += here;
  if (turns <= 0) continue;
  const int piece = static_cast<int>(head_piece % pieces);
  const int kv_head = static_cast<int>(head_piece / pieces);
  const int head0 = kv_head * group + piece * kHeads;
  const int heads = min(kHeads, group - piece * kHeads);
  const int64_t position = stream.position;
  const int count = stream.count;
  const int slot = static_cast<int>(
      position < a.first ? position : a.first + (position - a.first) % (a.slots - a.first));
  const int64_t row0 = (b * a.kv_heads + kv_head) * a.slots;
  uint8_t* const codes[2] = {a.k_codes + row0 * row_bytes, a.v_codes + row0 * row_bytes};
  uint32_t* const range[2] = {static_cast<uint32_t*>(a.k_range) + row0,
                              static_cast<uint32_t*>(a.v_range) + row0};
  uint8_t* const slots_valid = kMasked ? a.cache_valid + b * a.slots : nullptr;
  const bool token_valid = !kMasked || !a.valid || a.valid[b];

  const int base0 = first_turn * kSlots;
  const int end_slot = min(count, base0 + turns * kSlots);  // the part's
  int next_base = base0;  // of the next turn to load
  const uint8_t* next_codes[2] = {codes[0] + int64_t{base0} * row_bytes,
                                  codes[1] + int64_t{base0} * row_bytes};
  const auto load = [&](uint32_t to) {  // it, to stage `to`
    if constexpr (kAligned) {  // the turn's rows are one run of memory
      if (next_base < end_slot && good && lane == 0) {
        const uint32_t bytes = min(kSlots, end_slot - next_base) * row_bytes;
        const uint32_t bar = tc::shared_address(&s.full[warp][to]);
        tc::barrier_expect(bar, 2 * bytes);
#pragma unroll
        for (int side = 0; side < 2; ++side)
          asm volatile(
              "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, "
              "[%3];" ::"r"(tc::shared_address(s.stage[warp][to].codes[side])),
              "l"(next_codes[side]), "r"(bytes), "r"(bar)
              : "memory");
      }
    } else {
      if (next_base < end_slot) {
        Stage<kDim>& st = s.stage[warp][to];
        const int row = min(lane, end_slot - 1 - next_base);
#pragma unroll
        for (int side = 0; side < 2; ++side)
          for (int w = 0; w < row_bytes; w += 4)
            cp_async4(st.codes[side] + lane * kRow + w, next_codes[side] + row * row_bytes + w);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    next_base += kSlots;
    next_codes[0] += kSlots * row_bytes;
    next_codes[1] += kSlots * row_bytes;
  };
  // The ranges of the lane's slot of a turn, keys' and values', zeros behind the last one.
  const uint32_t* const lane_range[2] = {range[0] + lane, range[1] + lane};
  const auto ranges_of = [&](int base) {
    if (base + lane >= end_slot) return make_uint2(0, 0);
    return make_uint2(__ldcg(lane_range[0] + base), __ldcg(lane_range[1] + base));
  };
  const auto seen_in = [&](int base) {  // whether the lane's slot of a turn may be seen
    const int at = base + lane;
    if (at >= end_slot) return false;
    return !kMasked || (at == slot ? token_valid : slots_valid[at] != 0);
  };
#pragma unroll
  for (uint32_t t = 0; t < kStages - 1; ++t)
    load(stage + t < kStages ? stage + t : stage + t - kStages);
  bool seen_next = seen_in(base0);
  uint2 range_next = ranges_of(base0), range_after = ranges_of(base0 + kSlots);  // two turns ahead

  // The warp whose turn has the new token's slot rounds its rows.
  const bool owner = slot >= base0 && slot < end_slot;
  Fresh fresh = {0, 0};
  if (owner) {
    const bool value = lane >= 16;
    fresh = round_row(value ? static_cast<const T*>(a.v) + b * a.v_stride + kv_head * a.v_head_stride
                            : static_cast<const T*>(a.k) + b * a.k_stride + kv_head * a.k_head_stride,
                      a.dim);
    if (piece == 0) {
      if (8 * (lane & 15) < a.dim)
        *reinterpret_cast<uint32_t*>(codes[value] + int64_t{slot} * row_bytes + 4 * (lane & 15)) =
            fresh.codes;
      if ((lane & 15) == 0) range[value][slot] = fresh.range;
      if (kMasked && kv_head == 0 && lane == 0) slots_valid[slot] = token_valid;
    }
  }

  // Head g's q (and head g + 8's), channels in the order of the keys' products: a word's
  // are pairs (0, 4), (1, 5) of one product and (2, 6), (3, 7) of the next. A head's largest
  // channel goes to 2^10, or 2^6 where codes are 16 times as large.
  uint32_t q[kSets][kKeyWords][4];
  // Of the lane's columns, heads 2j and 2j + 1: what takes their dots to those with c - 7.5,
  // and the sums of q; both in base 2.
  float2 dot_scale[kSets], dot_offset[kSets], q_sum[kSets];
  // Where a head's q has channels from 2^100 on, these are 2^-64 as large and the keys' ranges
  // 2^64: then no part of a score leaves float's range that the score does not. (The group's
  // other heads share the ranges: they lose keys of 2^64 and more, which leave that head
  // no finite scores.)
  constexpr bool kWideRange = std::is_same_v<T, __nv_bfloat16>;  // float16 ends at 2^16
  bool far[kSets], any_far = false;
#pragma unroll
  for (int r = 0; r < kSets; ++r) {
    float x[kKeyWords][8], total = 0.0f, largest = 0.0f;
#pragma unroll
    for (int w = 0; w < kKeyWords; ++w) {
      const int channel = 8 * (kKeyWords * j + w);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[w][k] = 0.0f;
      if (g + 8 * r < heads && channel < a.dim)
        load_pack<8>(static_cast<const T*>(a.q) + b * a.q_stride +
                         (head0 + g + 8 * r) * a.q_head_stride + channel,
                     x[w]);
#pragma unroll
      for (int k = 0; k < 8; ++k) largest = max_nan(largest, fabsf(x[w][k]));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1)
      largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    far[r] = kWideRange && __any_sync(0xffffffffu, largest >= kFar);
    any_far = any_far || far[r];
    const float shrink = far[r] ? 1.0f / kFarScale : 1.0f;
#pragma unroll
    for (int w = 0; w < kKeyWords; ++w)
#pragma unroll
      for (int k = 0; k < 8; ++k) total += x[w][k] * shrink;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const uint32_t exponent = max(__float_as_uint(largest) & 0x7f800000u, 11u << 23);
    const float up = __uint_as_float((264u << 23) - exponent);
    const float down = __uint_as_float((254u << 23) - __float_as_uint(up));
#pragma unroll
    for (int w = 0; w < kKeyWords; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        q[r][w][e] = tc::pack2<__half>(x[w][e] * (e & 1 ? 0.0625f * up : up),
                                       x[w][e + 4] * (e & 1 ? 0.0625f * up : up));
    const float scale = a.scale * kLog2e;
    const auto heads_of = [&](float x) {
      return make_float2(__shfl_sync(0xffffffffu, x, 8 * j), __shfl_sync(0xffffffffu, x, 8 * j + 4));
    };
    dot_scale[r] = heads_of(kCodeUnit * (down * shrink) * scale);
    dot_offset[r] = heads_of(-7.5f * total * scale);
    q_sum[r] = heads_of(total * scale);
  }
#pragma unroll
  for (int r = 0; r < kSets; ++r)
    if (any_far && !far[r]) {
      dot_scale[r] = tc::mul2(dot_scale[r], both(1.0f / kFarScale));
      dot_offset[r] = tc::mul2(dot_offset[r], both(1.0f / kFarScale));
      q_sum[r] = tc::mul2(q_sum[r], both(1.0f / kFarScale));
    }
  float2 out[kSets][kValueWords][4][2] = {};  // of both heads: channels e, and e + 4
  float top[kSets][2];
  float2 sum[kSets] = {}, middle_sum[kSets] = {}, weight_sum[kSets] = {};
#pragma unroll
  for (int r = 0; r < kSets; ++r) top[r][0] = top[r][1] = -INFINITY;
  // Value steps and middles are taken relative to a power of two above the largest step so
  // far, so that sums of weights times values stay finite wherever the values are; and above
  // 2^-60 of the largest middle, for rows without a spread. (A step 2^-21 of another's
  // that is seen as little as it weighs loses digits of its weight in float16: all of
  // them together are less than 2^-29 of that other's spread a slot.)
  uint32_t unit = 0;  // its bits
  float per_unit = 1.0f;

  // Slots in the order of the products' rows: row n of 8 is slot n / 2 + 4 (n % 2), so that
  // a lane's four slots of V, j, 4 + j, 8 + j and 12 + j, and its neighbours', lie next to one
  // another.
  const int key_row = (g >> 1) + 4 * (g & 1);
  for (int base = base0; base < end_slot && good; base += kSlots) {
    load(stage == 0 ? kStages - 1 : stage - 1);  // the turn before's
    Stage<kDim>& st = s.stage[warp][stage];
    const bool seen = seen_next;
    uint2 ranges = range_next;
    seen_next = seen_in(base + kSlots);
    range_next = range_after;
    range_after = ranges_of(base + 2 * kSlots);
    if constexpr (kAligned) {
      good = tc::barrier_wait_warp(tc::shared_address(&s.full[warp][stage]), phase);
      if (!good) break;
    } else {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
    }
    if (owner && static_cast<uint32_t>(slot - base) < kSlots) {
      const int side = lane >> 4, word = lane & 15;
      if (8 * word < a.dim)
        *reinterpret_cast<uint32_t*>(st.codes[side] + (slot - base) * pitch + 4 * word) = fresh.codes;
      const uint32_t key = __shfl_sync(0xffffffffu, fresh.range, 0);
      const uint32_t value = __shfl_sync(0xffffffffu, fresh.range, 16);
      if (lane == slot - base) ranges = make_uint2(key, value);
      tc::fence_async_shared();  // before the stage's next load
      __syncwarp();
    }
    // A slot a lane: its ranges, zeros where it is not seen.
    const uint32_t visible = __ballot_sync(0xffffffffu, seen);
    {
      float2 key = unpack2<T>(seen ? ranges.x : 0);
      if (any_far) key = tc::mul2(key, both(kFarScale));
      const float2 value = unpack2<T>(seen ? ranges.y : 0);
      const uint32_t largest = __reduce_max_sync(
          0xffffffffu, __float_as_uint(fmaxf(fabsf(value.x), 0x1p-60f * fabsf(value.y))));
      if (largest >= unit) {  // the same for the whole warp
        const uint32_t next = min(largest & 0x7f800000u, 0x7e000000u) + 0x00800000u;
        const float shrink = unit ? __uint_as_float(unit) / __uint_as_float(next) : 0.0f;
#pragma unroll
        for (int r = 0; r < kSets; ++r) {
          weight_sum[r] = tc::mul2(weight_sum[r], both(shrink));
          middle_sum[r] = tc::mul2(middle_sum[r], both(shrink));
        }
#pragma unroll
        for (int r = 0; r < kSets; ++r)
#pragma unroll
          for (int h = 0; h < kValueWords; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int c = 0; c < 2; ++c) out[r][h][i][c] = tc::mul2(out[r][h][i][c], both(shrink));
        unit = next;
        per_unit = __uint_as_float(0x7f000000u - next);
      }
      s.slot[warp][lane] = {both(key.x), both(key.y), both(value.x * per_unit),
                            both(value.y * per_unit)};
    }
    __syncwarp();
    Slot of[4];  // the lane's slots as rows of the scores: key_row, + 8, + 16, + 24
#pragma unroll
    for (int i = 0; i < 4; ++i) of[i] = s.slot[warp][key_row + 8 * i];
    float x[kSets][2][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {  // 16 slots
      uint32_t low[kKeyWords], high[kKeyWords];
      read_words<kKeyWords>(st.codes[0] + (16 * half + key_row) * pitch + 4 * kKeyWords * j, low);
      read_words<kKeyWords>(st.codes[0] + (16 * half + 8 + key_row) * pitch + 4 * kKeyWords * j, high);
#pragma unroll
      for (int w = 0; w < kKeyWords; ++w) {
        uint32_t p0[4], p8[4];
        spread(low[w], p0);
        spread(high[w], p8);
#pragma unroll
        for (int r = 0; r < kSets; ++r) {
          if (w == 0) multiply_new(x[r][half], p0[0], p8[0], p0[1], p8[1], q[r][w][0], q[r][w][1]);
          else multiply(x[r][half], p0[0], p8[0], p0[1], p8[1], q[r][w][0], q[r][w][1]);
          multiply(x[r][half], p0[2], p8[2], p0[3], p8[3], q[r][w][2], q[r][w][3]);
        }
      }
    }
    uint32_t weight[kSets][4];  // of the slots of[i], both heads, then turned around
#pragma unroll
    for (int r = 0; r < kSets; ++r) {
      float2 score[4];  // of the lane's two heads
      float next[2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* const c = x[r][i >> 1] + 2 * (i & 1);
        score[i] = tc::fma2(tc::fma2(make_float2(c[0], c[1]), dot_scale[r], dot_offset[r]),
                            of[i].key_step, tc::mul2(q_sum[r], of[i].key_middle));
      }
      if (visible != 0xffffffffu)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(visible >> (key_row + 8 * i) & 1)) score[i].x = score[i].y = -INFINITY;
      next[0] = fmaxf(tc::max3(score[0].x, score[1].x, score[2].x), score[3].x);
      next[1] = fmaxf(tc::max3(score[0].y, score[1].y, score[2].y), score[3].y);
      if (__any_sync(0xffffffffu, next[0] > top[r][0] + kSlack || next[1] > top[r][1] + kSlack)) {
        float shrink[2] = {1.0f, 1.0f};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1)
            next[e] = fmaxf(next[e], __shfl_xor_sync(0xffffffffu, next[e], o));
          if (next[e] > top[r][e] + kSlack) {
            shrink[e] = tc::exp2_approx(top[r][e] - next[e]);
            top[r][e] = next[e];
          }
        }
        const float2 shrinks = make_float2(shrink[0], shrink[1]);
        sum[r] = tc::mul2(sum[r], shrinks);
        middle_sum[r] = tc::mul2(middle_sum[r], shrinks);
        weight_sum[r] = tc::mul2(weight_sum[r], shrinks);
#pragma unroll
        for (int h = 0; h < kValueWords; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c) out[r][h][i][c] = tc::mul2(out[r][h][i][c], shrinks);
      }
      const float2 shift = make_float2(top[r][0] == -INFINITY ? 0.0f : kLift - top[r][0],
                                       top[r][1] == -INFINITY ? 0.0f : kLift - top[r][1]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 y = tc::add2(score[i], shift);
        const float2 p = make_float2(tc::exp2_approx(y.x), tc::exp2_approx(y.y));
        sum[r] = tc::add2(sum[r], p);
        middle_sum[r] = tc::fma2(p, of[i].value_middle, middle_sum[r]);
        const float2 w = tc::mul2(p, of[i].value_step);
        weight[r][i] = transposed(tc::pack2<__half>(w.x, w.y));
      }
    }
    // The turn's sums of weights times codes, all of them positive, are added to the others'
    // in float arithmetic: the products' own sums, which are cut and not rounded, would
    // all err to one side, by more than the few digits that are left once 7.5 times the
    // weights is taken off (`weight_sum`, the weights as they were rounded).
    float turn[kSets][kValueWords][4][4], turn_weight[kSets][4];
#pragma unroll
    for (int r = 0; r < kSets; ++r) {
      constexpr uint32_t kOnes = 0x3c003c00u;
      multiply_new(turn_weight[r], kOnes, kOnes, kOnes, kOnes, weight[r][0], weight[r][1]);
      multiply(turn_weight[r], kOnes, kOnes, kOnes, kOnes, weight[r][2], weight[r][3]);
      weight_sum[r] = tc::add2(weight_sum[r], make_float2(turn_weight[r][0], turn_weight[r][1]));
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t word[4][kValueWords];  // of the slots j, 4 + j, 8 + j, 12 + j
#pragma unroll
      for (int i = 0; i < 4; ++i)
        read_words<kValueWords>(
            st.codes[1] + (16 * half + 4 * i + j) * pitch + 4 * kValueWords * g, word[i]);
#pragma unroll
      for (int h = 0; h < kValueWords; ++h) {
        uint32_t a0[4], a1[4], a2[4], a3[4];  // channels 0 to 3 and 4 to 7, two slots each
        spread_bytes(__byte_perm(word[0][h], word[1][h], 0x5410), a0);
        spread_bytes(__byte_perm(word[0][h], word[1][h], 0x7632), a1);
        spread_bytes(__byte_perm(word[2][h], word[3][h], 0x5410), a2);
        spread_bytes(__byte_perm(word[2][h], word[3][h], 0x7632), a3);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int r = 0; r < kSets; ++r)
            if (half == 0)
              multiply_new(turn[r][h][e], a0[e], a1[e], a2[e], a3[e], weight[r][0], weight[r][1]);
            else
              multiply(turn[r][h][e], a0[e], a1[e], a2[e], a3[e], weight[r][2], weight[r][3]);
      }
    }
#pragma unroll
    for (int r = 0; r < kSets; ++r)
#pragma unroll
      for (int h = 0; h < kValueWords; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            out[r][h][e][c] = tc::add2(out[r][h][e][c], make_float2(turn[r][h][e][2 * c],
                                                                   turn[r][h][e][2 * c + 1]));
    __syncwarp();  // all lanes are done with the stage that the next turn fills
    if (++stage == kStages) stage = 0, phase ^= 1;
  }
  if (!good) {  // let what is in flight land, and show that the result is not valid
    for (uint64_t& bar : s.full[warp]) tc::barrier_settle(tc::shared_address(&bar));
    for (float2& x : sum) x = make_float2(NAN, NAN);
    if (lane == 0) atomicExch(&g_timeout, 1u);
  }

  // What the warp leaves: row g of product (h, e) is channel 8 (kValueWords g + h) + e, row g
  // + 8 channel e + 4. Parts are numbered by warp and item together: both only grow.
  const int64_t item = (b * a.kv_heads + kv_head) * pieces + piece;
  if (lane == 0 && first_turn == 0) reach[item].first = static_cast<int32_t>(me);
  if (lane == 0 && first_turn + turns == stream.turns) reach[item].last = static_cast<int32_t>(me);
  const bool large = unit >= kLargeUnit;
  const float unit_size = __uint_as_float(unit) * (large ? 1.0f / kLargeScale : 1.0f);
#pragma unroll
  for (int r = 0; r < kSets; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int head = 8 * r + 2 * j + e;
      float total = e ? sum[r].y : sum[r].x, middle = e ? middle_sum[r].y : middle_sum[r].x;
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        middle += __shfl_xor_sync(0xffffffffu, middle, o);
      }
      if (head >= heads) continue;
      if (g == 0) {
        *parts.top(me + item, head) = top[r][e];
        *parts.sum(me + item, head) = large ? -total : total;
      }
      // Weights times codes are in units of 2^-24, and the weights in `unit`. Odd channels' come
      // 16 times as large and on top of their neighbours'.
      const float size = unit_size * kCodeUnit;
      const float off = unit_size * fmaf(-7.5f, e ? weight_sum[r].y : weight_sum[r].x, middle);
      const auto low = [&](float2 x) { return fmaf(e ? x.y : x.x, size, off); };
      const auto high = [&](float2 x, float2 both) {
        return fmaf(e ? both.y - x.y : both.x - x.x, 0.0625f * size, off);
      };
#pragma unroll
      for (int h = 0; h < kValueWords; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<float4*>(parts.out(me + item, head) + 8 * (kValueWords * g + h) + 4 * i) =
              make_float4(low(out[r][h][0][i]), high(out[r][h][0][i], out[r][h][1][i]),
                          low(out[r][h][2][i]), high(out[r][h][2][i], out[r][h][3][i]));
    }
  __syncwarp();  // the next part's slots
  }
  if constexpr (!kAligned) asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// An item's parts joined in order, a block an item and head: the threads of a channel take
// every so many parts. What is left of the time is latency, so what a thread needs first
// is requested before it is known what it is multiplied by.
constexpr int kMostParts = 128, kAhead = 8;  // at a time: threads of the smallest block
template <class T, int kDim, int kSets>
__global__ void __launch_bounds__(1024)
    join_kernel(gs_window_attention_step_4bit_args a, Parts<kDim> parts, const Reach* reach) {
  constexpr int kHeads = 8 * kSets;
  __shared__ float joined[1024], scales[kMostParts], sums[kMostParts], tops[32];
  chain_wait();
  const int group = a.heads / a.kv_heads, pieces = (group + kHeads - 1) / kHeads;
  const int64_t item = blockIdx.x, b = item / pieces / a.kv_heads;
  const int kv_head = static_cast<int>(item / pieces % a.kv_heads);
  const int piece = static_cast<int>(item % pieces), h = blockIdx.y;
  if (h >= min(kHeads, group - piece * kHeads)) return;
  const Reach r = reach[item];  // of an idle stream's items: whatever was there
  T* const out = static_cast<T*>(a.out) +
                 (b * a.heads + kv_head * group + piece * kHeads + h) * a.dim;
  if (a.positions[b] < 0) {
    if (threadIdx.x < a.dim) out[threadIdx.x] = from_float<T>(0.0f);
    return;
  }
  const int count = r.last - r.first + 1, threads = blockDim.x, thread = threadIdx.x;
  const int d = thread % kDim, groups = threads / kDim, mine = thread / kDim;
  const int64_t from = item + r.first;
  float ahead[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    ahead[k] = mine + k * groups < count ? parts.out(from + mine + k * groups, h)[d] : 0.0f;
  float top = -INFINITY, sum = 0.0f;
  if (thread < count) top = *parts.top(from + thread, h), sum = *parts.sum(from + thread, h);
  float whole = top;
  bool large = signbit(sum);
  for (int i = thread + threads; i < count; i += threads) {
    whole = fmaxf(whole, *parts.top(from + i, h));
    large = large || signbit(*parts.sum(from + i, h));
  }
  whole = warp_max(whole);
  if ((thread & 31) == 0) tops[thread >> 5] = whole;
  const bool any_large = __syncthreads_or(large);
  for (int w = 0; w < threads / 32; ++w) whole = fmaxf(whole, tops[w]);
  const float shift = whole == -INFINITY ? 0.0f : whole;
  float o = 0.0f, total = 0.0f;
  for (int i0 = 0; i0 < count; i0 += kMostParts) {
    __syncthreads();
    const int some = min(kMostParts, count - i0);
    if (thread < some) {
      if (i0 > 0) top = *parts.top(from + i0 + thread, h), sum = *parts.sum(from + i0 + thread, h);
      const float scale = tc::exp2_approx(top - shift);
      scales[thread] = any_large && !signbit(sum) ? scale / kLargeScale : scale;
      sums[thread] = fabsf(sum) * scale;
    }
    __syncthreads();
    int i = mine;
    if (i0 == 0) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k, i += groups)
        if (i < some) o = fmaf(ahead[k], scales[i], o);
    }
#pragma unroll 8
    for (; i < some; i += groups) o = fmaf(parts.out(from + i0 + i, h)[d], scales[i], o);
    if (thread < a.dim)
      for (int k = 0; k < some; ++k) total += sums[k];
  }
  joined[thread] = o;
  __syncthreads();
  if (thread < a.dim) {
    for (int i = 1; i < groups; ++i) o += joined[i * kDim + d];
    out[d] = from_float<T>(total == 0.0f ? 0.0f : any_large ? o / total * kLargeScale : o / total);
  }
}

// Blocks of the first kernel: all that are resident at once, as far as every warp has a turn.
int64_t blocks_of(const gs_window_attention_step_4bit_args& a, int64_t items, int sets) {
  const int64_t turns = items * ceil_div(a.slots, kSlots);
  return std::min<int64_t>(blocks_per_sm(a.dim <= 64 ? 64 : 128, sets) * kSmCount,
                           (turns + kWarps - 1) / kWarps);
}

int64_t items_of(const gs_window_attention_step_4bit_args& a, int sets) {
  return a.batch * a.kv_heads * ceil_div(a.heads / a.kv_heads, 8 * sets);
}

uint64_t reach_bytes(int64_t items) { return (sizeof(Reach) * static_cast<uint64_t>(items) + 15) / 16 * 16; }

int part_heads(const gs_window_attention_step_4bit_args& a, int sets) {
  return std::min(a.heads / a.kv_heads, 8 * sets);
}

template <class T, int kDim, int kKeyWords, int kSets, bool kMasked, bool kAligned>
int32_t step(const gs_window_attention_step_4bit_args& a, cudaStream_t stream) {
  const int64_t items = items_of(a, kSets), blocks = blocks_of(a, items, kSets);
  if (items > INT32_MAX) return GS_ERR_CAPACITY;
  Reach* const reach = static_cast<Reach*>(a.workspace);
  const Parts<kDim> parts = {
      reinterpret_cast<float*>(static_cast<unsigned char*>(a.workspace) + reach_bytes(items)),
      part_heads(a, kSets)};
  constexpr size_t kShared = sizeof(Shared<kDim>);
  GS_TRY((allow_shared<step_kernel<T, kDim, kKeyWords, kSets, kMasked, kAligned>>(kShared)));
  launch_chained_shared(step_kernel<T, kDim, kKeyWords, kSets, kMasked, kAligned>,
                        dim3(static_cast<unsigned>(blocks)), dim3(kThreads), kShared, stream, a,
                        parts, reach);
  GS_TRY(check_launch());
  // Threads by the parts of an item: few parts, many items; many parts, few items.
  const int64_t each = blocks * kWarps / items;
  const int threads = each >= 16 ? 1024 : each >= 8 ? 256 : 128;
  launch_chained(join_kernel<T, kDim, kSets>,
                 dim3(static_cast<unsigned>(items), parts.heads),
                 threads, stream, a, parts, static_cast<const Reach*>(reach));
  return check_launch();
}

int sets_of(const gs_window_attention_step_4bit_args& a) { return a.heads / a.kv_heads <= 8 ? 1 : 2; }

int32_t check_args(const gs_window_attention_step_4bit_args& a) {
  if (a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.heads > 65535 || a.dim < 8 ||
      a.dim % 8)
    return GS_ERR_INVALID_ARGUMENT;
  if (a.dim > kMaxDim || (a.dtype != GS_BFLOAT16 && a.dtype != GS_FLOAT16))
    return GS_ERR_UNSUPPORTED;
  if (a.batch < 0 || a.first < 0 || a.slots <= a.first ||
      a.batch > GS_MAX_SEQUENCE_TOKENS / a.slots || !(a.scale > 0.0f && a.scale < INFINITY))
    return GS_ERR_INVALID_ARGUMENT;
  return GS_OK;
}

bool strided16(const void* p, int64_t stride, int64_t head_stride) {
  return is_aligned(p, 16) && stride % 8 == 0 && head_stride % 8 == 0;
}

}  // namespace

uint64_t window_attention_step_4bit_workspace_size(const gs_window_attention_step_4bit_args& a) {
  if (check_args(a) != GS_OK || a.batch == 0) return 0;
  const int sets = sets_of(a);
  const int64_t items = items_of(a, sets);
  const int heads = part_heads(a, sets);
  const uint64_t part = 4 * (a.dim <= 64 ? Parts<64>{nullptr, heads}.floats()
                                         : Parts<128>{nullptr, heads}.floats());
  return reach_bytes(items) +
         part * static_cast<uint64_t>(blocks_of(a, items, sets) * kWarps + items);
}

int32_t window_attention_4bit_status(cudaStream_t stream) { return take_timeout(g_timeout, stream); }

int32_t launch_window_attention_step_4bit(const gs_window_attention_step_4bit_args& a,
                                          cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (a.batch == 0) return GS_OK;
  if (!a.q || !a.k || !a.v || !a.k_codes || !a.v_codes || !a.k_range || !a.v_range ||
      !a.positions || !a.out || !a.workspace || (a.valid && !a.cache_valid))
    return GS_ERR_INVALID_ARGUMENT;
  if (!strided16(a.q, a.q_stride, a.q_head_stride) ||
      !strided16(a.k, a.k_stride, a.k_head_stride) ||
      !strided16(a.v, a.v_stride, a.v_head_stride) || !is_aligned(a.k_codes, 16) ||
      !is_aligned(a.v_codes, 16) || !is_aligned(a.k_range, 16) || !is_aligned(a.v_range, 16) ||
      !is_aligned(a.out, 16) || !is_aligned(a.positions, 8) || !is_aligned(a.workspace, 16))
    return GS_ERR_MISALIGNED;
  if (a.workspace_size < window_attention_step_4bit_workspace_size(a)) return GS_ERR_CAPACITY;
  const auto typed = [&](auto t) {
    using T = decltype(t);
    const auto shaped = [&](auto masked, auto aligned) {
      constexpr bool kMasked = decltype(masked)::value, kAligned = decltype(aligned)::value;
      // Keys of up to 96 channels in three words a lane: 44 us against 47 with four (3
      // streams of 65,536 slots, 24 heads of 96).
      const auto with_sets = [&](auto sets) {
        constexpr int kSets = decltype(sets)::value;
        return a.dim <= 64   ? step<T, 64, 2, kSets, kMasked, kAligned>(a, stream)
               : a.dim <= 96 ? step<T, 128, 3, kSets, kMasked, kAligned>(a, stream)
                             : step<T, 128, 4, kSets, kMasked, kAligned>(a, stream);
      };
      return sets_of(a) == 1 ? with_sets(std::integral_constant<int, 1>{})
                             : with_sets(std::integral_constant<int, 2>{});
    };
    const bool aligned = a.dim % 32 == 0;
    if (a.cache_valid)
      return aligned ? shaped(std::true_type{}, std::true_type{})
                     : shaped(std::true_type{}, std::false_type{});
    return aligned ? shaped(std::false_type{}, std::true_type{})
                   : shaped(std::false_type{}, std::false_type{});
  };
  return a.dtype == GS_BFLOAT16 ? typed(__nv_bfloat16{}) : typed(__half{});
}

}  // namespace gs
