// One new token a stream against a window's cache held in 4 bits: the step of
// attention.cu over rows of codes, x ~ (c - 7.5) step + middle with c in 0..15.
//
//   score_t = scale q . k_t = scale (step_t (q . c_t) + (middle_t - 7.5 step_t) sum q)
//   out = sum p_t v_t = sum (p_t step_t) (c_t - 7.5) + sum p_t middle_t
//
// so that codes go to the products as they are, small whole numbers in float16, which
// are exact, and the ranges stay outside: a key's in two numbers a score, a value's in
// its weight p_t step_t and in one float sum a head, which no rounding meets. q and the
// weights are scaled by powers of two into float16's range, whatever the tokens' type:
// of a head's q nothing is lost within 2^-25 of its largest channel, and the weights
// are rounded once, to 11 bits.
//
// The cache is read once; taking a word of eight codes apart costs 9 to 10 instructions
// though, which together weigh about as much as the reading. A cluster of blocks shares
// the slots of a stream and key-value head, up to 16 query heads (more: more clusters). A
// warp takes 32 slots at a time from a ring in shared memory of its own, filled some
// turns ahead by cp.async, so that warps never wait for one another:
//
//   scores [slots x heads] = K q^T: a lane's words of two key rows are its parts of
//     the products, with q's channels permuted alike;
//   out [dim x heads] += V^T P^T: a lane's words of two value rows, interleaved, are
//     its parts of four products; P turns around in registers (movmatrix).
//
// So slots and channels fill the products' 16 rows, and 8 heads their columns. Sums are
// joined at the end in order, in the block and across the cluster: one launch, no
// workspace, no atomics.
#include "step.cuh"

namespace gs {
namespace {

constexpr int kMaxDim = 128;
constexpr int kWarps = 4, kThreads = 32 * kWarps;
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
  uint32_t range[2][kSlots];  // step in the low half, middle in the high one
};

// What a slot's ranges come to: score = dot * key_step + (sum of q) * key_base, where
// dot has c - 8.
struct Slot {
  float key_step, key_base, value_step, value_middle;
};

template <int kDim, int kSets>
struct Shared {
  union {
    Stage<kDim> stage[kWarps][Stage<kDim>::kCount];
    float out[kWarps][8 * kSets][kDim];  // once the stages are done
  };
  alignas(16) Slot slot[kWarps][kSlots];
  float top[kWarps][8 * kSets], sum[kWarps][8 * kSets];
};

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
  const T step = from_float<T>((high - low) / 15.0f);
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

template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t word) {
  const T* v = reinterpret_cast<const T*>(&word);
  return make_float2(to_float(v[0]), to_float(v[1]));
}

// c - 8 in float16 of the codes at bits 0 to 3 (low), or 4 to 7, of both halves of a
// word: next to 1024, whose low bits they are, and that taken off again. Exact.
__device__ __forceinline__ uint32_t centred_low(uint32_t word) {  // (1024 + c) - 1032
  uint32_t y;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"((word & 0x000f000fu) | 0x64006400u), "r"(0xe408e408u));
  return y;
}
__device__ __forceinline__ uint32_t centred_high(uint32_t word) {  // (1024 + 16 c) / 16 - 72
  uint32_t y;
  asm("fma.rn.f16x2 %0, %1, %2, %3;"
      : "=r"(y)
      : "r"((word & 0x00f000f0u) | 0x64006400u), "r"(0x2c002c00u), "r"(0xd480d480u));
  return y;
}
// Codes 0 to 3 of both halves of a word as four pairs.
__device__ __forceinline__ void spread(uint32_t word, uint32_t (&pair)[4]) {
  const uint32_t next = word >> 8;
  pair[0] = centred_low(word);
  pair[1] = centred_high(word);
  pair[2] = centred_low(next);
  pair[3] = centred_high(next);
}

// c += a b, 16 x 16 by 16 x 8.
__device__ __forceinline__ void multiply(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of pairs, a row in four lanes, turned around.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int kWords>
__device__ __forceinline__ void read_words(const unsigned char* p, uint32_t (&w)[kWords]) {
  static_assert(kWords == 1 || kWords == 2 || kWords == 4);
  if constexpr (kWords == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
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

// kSets: of 8 heads. kMasked: with validity of the slots. kAligned: rows of codes are
// whole 16-byte words.
template <class T, int kDim, int kSets, bool kMasked, bool kAligned>
__global__ void __launch_bounds__(kThreads, kSets == 1 ? 4 : kDim == 64 ? 4 : 3)
    step_kernel(gs_window_attention_step_4bit_args a) {
  using S = Shared<kDim, kSets>;
  constexpr int kRow = Stage<kDim>::kRow, kStages = Stage<kDim>::kCount;
  constexpr int kKeyWords = kDim / 32;    // a lane's words of a key's row, of four lanes
  constexpr int kValueWords = kDim / 64;  // of a value's, of eight
  constexpr int kHeads = 8 * kSets;
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  S& s = *reinterpret_cast<S*>(shared_bytes);
  chain_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const uint32_t rank = cluster_rank(), blocks = cluster_size();
  const int group = a.heads / a.kv_heads, pieces = (group + kHeads - 1) / kHeads;
  const int64_t item = blockIdx.x / blocks;
  const int piece = static_cast<int>(item % pieces);
  const int kv_head = static_cast<int>(item / pieces % a.kv_heads);
  const int64_t b = item / pieces / a.kv_heads;
  const int head0 = kv_head * group + piece * kHeads;
  const int heads = min(kHeads, group - piece * kHeads);
  const int64_t position = a.positions[b];
  const bool idle = position < 0;
  const int slot = idle ? -1
                        : static_cast<int>(position < a.first
                                               ? position
                                               : a.first + (position - a.first) %
                                                               (a.slots - a.first));
  const int count = idle ? 0 : static_cast<int>(min(position + 1, int64_t{a.slots}));
  const int row_bytes = a.dim / 2;
  const int64_t row0 = (b * a.kv_heads + kv_head) * a.slots;
  uint8_t* const codes[2] = {a.k_codes + row0 * row_bytes, a.v_codes + row0 * row_bytes};
  uint32_t* const range[2] = {static_cast<uint32_t*>(a.k_range) + row0,
                              static_cast<uint32_t*>(a.v_range) + row0};
  uint8_t* const slots_valid = kMasked ? a.cache_valid + b * a.slots : nullptr;
  const bool token_valid = !kMasked || !a.valid || a.valid[b];

  // This warp's turns of 32 slots: me, me + all, ...
  const int me = static_cast<int>(rank) * kWarps + warp, all = static_cast<int>(blocks) * kWarps;
  const int turns = max(0, ((count + kSlots - 1) / kSlots - me + all - 1) / all);
  const auto base_of = [&](int t) { return (me + t * all) * kSlots; };
  const auto load = [&](int t) {
    if (t < turns) {
      Stage<kDim>& st = s.stage[warp][t % kStages];
      const int base = base_of(t);
      const int last = count - 1 - base;  // slots behind it are that one again
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const uint8_t* const from = codes[side] + int64_t{base} * row_bytes;
        if constexpr (kAligned) {
          // Four lanes (64 channels: two) have a row's 16-byte words.
          constexpr int kLanes = kDim / 32;
          const int word = 16 * (lane % kLanes);
          if (word < row_bytes)
#pragma unroll
            for (int r = 0; r < kLanes; ++r) {
              const int row = lane / kLanes + 32 / kLanes * r;
              cp_async16(st.codes[side] + row * kRow + word, from + min(row, last) * row_bytes + word);
            }
        } else {
          for (int w = 0; w < row_bytes; w += 4)
            cp_async4(st.codes[side] + lane * kRow + w, from + min(lane, last) * row_bytes + w);
        }
        cp_async4(&st.range[side][lane], range[side] + base + min(lane, last));
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const auto seen_in = [&](int t) {  // whether the lane's slot of a turn may be seen
    if (t >= turns) return false;
    const int at = base_of(t) + lane;
    if (at >= count) return false;
    return !kMasked || (at == slot ? token_valid : slots_valid[at] != 0);
  };
#pragma unroll
  for (int t = 0; t < kStages - 1; ++t) load(t);
  bool seen_next = seen_in(0);

  // The warp whose turn has the new token's slot rounds its rows.
  const int slot_turn = idle ? -1 : slot / kSlots;
  const bool owner = slot_turn >= 0 && slot_turn % all == me;
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
  // channel goes to 2^10.
  uint32_t q[kSets][kKeyWords][4];
  // Of the lane's columns, heads 2j and 2j + 1: what takes their dots and sums of q to
  // scores in base 2.
  float dot_scale[kSets][2], base_scale[kSets][2];
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
      for (int k = 0; k < 8; ++k) {
        total += x[w][k];
        largest = max_nan(largest, fabsf(x[w][k]));
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    }
    const uint32_t exponent = max(__float_as_uint(largest) & 0x7f800000u, 11u << 23);
    const float up = __uint_as_float((264u << 23) - exponent);
    const float down = __uint_as_float((254u << 23) - __float_as_uint(up));
#pragma unroll
    for (int w = 0; w < kKeyWords; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        q[r][w][e] = tc::pack2<__half>(x[w][e] * up, x[w][e + 4] * up);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int from = 4 * (2 * j + e);
      dot_scale[r][e] = __shfl_sync(0xffffffffu, down, from) * (a.scale * kLog2e);
      base_scale[r][e] = __shfl_sync(0xffffffffu, total, from) * (a.scale * kLog2e);
    }
  }
  float out[kSets][kValueWords][4][4] = {};
  float top[kSets][2], sum[kSets][2] = {}, middle_sum[kSets][2] = {};
#pragma unroll
  for (int r = 0; r < kSets; ++r) top[r][0] = top[r][1] = -INFINITY;
  // Value steps are taken relative to a power of two above the largest so far.
  uint32_t unit = 0;  // its bits
  float per_unit = 1.0f;

  // Slots in the order of the products' rows: row n of 8 is slot n / 2 + 4 (n % 2), so that
  // a lane's four slots of V, j, 4 + j, 8 + j and 12 + j, and its neighbours', lie next to one
  // another.
  const int key_row = (g >> 1) + 4 * (g & 1);
  for (int t = 0; t < turns; ++t) {
    load(t + kStages - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    Stage<kDim>& st = s.stage[warp][t % kStages];
    const int base = base_of(t);
    const bool seen = seen_next;
    seen_next = seen_in(t + 1);
    if (owner && base == slot_turn * kSlots) {
      const int side = lane >> 4, word = lane & 15;
      if (8 * word < a.dim)
        *reinterpret_cast<uint32_t*>(st.codes[side] + (slot - base) * kRow + 4 * word) = fresh.codes;
      if (word == 0) st.range[side][slot - base] = fresh.range;
      __syncwarp();
    }
    // A slot a lane: its ranges, zeros where it is not seen.
    const uint32_t visible = __ballot_sync(0xffffffffu, seen);
    {
      const float2 key = unpack2<T>(seen ? st.range[0][lane] : 0);
      const float2 value = unpack2<T>(seen ? st.range[1][lane] : 0);
      const uint32_t largest =
          __reduce_max_sync(0xffffffffu, __float_as_uint(value.x) & 0x7fffffffu);
      if (largest >= unit) {  // the same for the whole warp
        const uint32_t next = min(largest & 0x7f800000u, 0x7e000000u) + 0x00800000u;
        const float shrink = unit ? __uint_as_float(unit) / __uint_as_float(next) : 0.0f;
#pragma unroll
        for (int r = 0; r < kSets; ++r)
#pragma unroll
          for (int h = 0; h < kValueWords; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int c = 0; c < 4; ++c) out[r][h][i][c] *= shrink;
        unit = next;
        per_unit = __uint_as_float(0x7f000000u - next);
      }
      s.slot[warp][lane] = {key.x, fmaf(0.5f, key.x, key.y), value.x * per_unit,
                            fmaf(0.5f, value.x, value.y)};
    }
    __syncwarp();
    Slot of[4];  // the lane's slots as rows of the scores: key_row, + 8, + 16, + 24
#pragma unroll
    for (int i = 0; i < 4; ++i) of[i] = s.slot[warp][key_row + 8 * i];
    float x[kSets][2][4] = {};
#pragma unroll
    for (int half = 0; half < 2; ++half) {  // 16 slots
      uint32_t low[kKeyWords], high[kKeyWords];
      read_words<kKeyWords>(st.codes[0] + (16 * half + key_row) * kRow + 4 * kKeyWords * j, low);
      read_words<kKeyWords>(st.codes[0] + (16 * half + 8 + key_row) * kRow + 4 * kKeyWords * j, high);
#pragma unroll
      for (int w = 0; w < kKeyWords; ++w) {
        uint32_t p0[4], p8[4];
        spread(low[w], p0);
        spread(high[w], p8);
#pragma unroll
        for (int r = 0; r < kSets; ++r) {
          multiply(x[r][half], p0[0], p8[0], p0[1], p8[1], q[r][w][0], q[r][w][1]);
          multiply(x[r][half], p0[2], p8[2], p0[3], p8[3], q[r][w][2], q[r][w][3]);
        }
      }
    }
    uint32_t weight[kSets][4];  // of the slots of[i], both heads, then turned around
#pragma unroll
    for (int r = 0; r < kSets; ++r) {
      float score[4][2], next[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          score[i][e] = fmaf(x[r][i >> 1][2 * (i & 1) + e] * dot_scale[r][e], of[i].key_step,
                             base_scale[r][e] * of[i].key_base);
      if (visible != 0xffffffffu)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(visible >> (key_row + 8 * i) & 1)) score[i][0] = score[i][1] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) next[e] = fmaxf(next[e], score[i][e]);
      if (__any_sync(0xffffffffu, next[0] > top[r][0] + kSlack || next[1] > top[r][1] + kSlack)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1)
            next[e] = fmaxf(next[e], __shfl_xor_sync(0xffffffffu, next[e], o));
          if (next[e] > top[r][e] + kSlack) {
            const float shrink = tc::exp2_approx(top[r][e] - next[e]);
            top[r][e] = next[e];
            sum[r][e] *= shrink;
            middle_sum[r][e] *= shrink;
#pragma unroll
            for (int h = 0; h < kValueWords; ++h)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                out[r][h][i][e] *= shrink;
                out[r][h][i][2 + e] *= shrink;
              }
          }
        }
      }
      float shift[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) shift[e] = top[r][e] == -INFINITY ? 0.0f : kLift - top[r][e];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float p[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[e] = tc::exp2_approx(score[i][e] + shift[e]);
          sum[r][e] += p[e];
          middle_sum[r][e] = fmaf(p[e], of[i].value_middle, middle_sum[r][e]);
        }
        weight[r][i] = transposed(
            tc::pack2<__half>(p[0] * of[i].value_step, p[1] * of[i].value_step));
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t word[4][kValueWords];  // of the slots j, 4 + j, 8 + j, 12 + j
#pragma unroll
      for (int i = 0; i < 4; ++i)
        read_words<kValueWords>(
            st.codes[1] + (16 * half + 4 * i + j) * kRow + 4 * kValueWords * g, word[i]);
#pragma unroll
      for (int h = 0; h < kValueWords; ++h) {
        uint32_t a0[4], a1[4], a2[4], a3[4];  // channels 0 to 3 and 4 to 7, two slots each
        spread(__byte_perm(word[0][h], word[1][h], 0x5410), a0);
        spread(__byte_perm(word[0][h], word[1][h], 0x7632), a1);
        spread(__byte_perm(word[2][h], word[3][h], 0x5410), a2);
        spread(__byte_perm(word[2][h], word[3][h], 0x7632), a3);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int r = 0; r < kSets; ++r)
            multiply(out[r][h][e], a0[e], a1[e], a2[e], a3[e], weight[r][2 * half],
                     weight[r][2 * half + 1]);
      }
    }
    __syncwarp();  // all lanes are done with the stage that the next turn fills
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // the stages' place is free for the outputs

  // The warp's columns to shared memory: row g of product (h, e) is channel 8 (kValueWords g
  // + h) + e, row g + 8 channel e + 4.
  const float unit_size = __uint_as_float(unit);
#pragma unroll
  for (int r = 0; r < kSets; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int head = 8 * r + 2 * j + e;
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        sum[r][e] += __shfl_xor_sync(0xffffffffu, sum[r][e], o);
        middle_sum[r][e] += __shfl_xor_sync(0xffffffffu, middle_sum[r][e], o);
      }
      if (g == 0) {
        s.top[warp][head] = top[r][e];
        s.sum[warp][head] = sum[r][e];
      }
#pragma unroll
      for (int h = 0; h < kValueWords; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          s.out[warp][head][8 * (kValueWords * g + h) + i] =
              fmaf(out[r][h][i & 3][2 * (i >> 2) + e], unit_size, middle_sum[r][e]);
    }
  __syncthreads();
  // The warps joined into the first one's place.
  for (int c = threadIdx.x; c < heads * kDim; c += kThreads) {
    const int h = c / kDim, d = c % kDim;
    float whole = -INFINITY, o = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) whole = fmaxf(whole, s.top[w][h]);
    const float shift = whole == -INFINITY ? 0.0f : whole;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      o = fmaf(s.out[w][h][d], tc::exp2_approx(s.top[w][h] - shift), o);
    s.out[0][h][d] = o;
  }
  __syncthreads();
  if (threadIdx.x < heads) {
    const int h = threadIdx.x;
    float whole = -INFINITY, total = 0.0f;
    for (int w = 0; w < kWarps; ++w) whole = fmaxf(whole, s.top[w][h]);
    const float shift = whole == -INFINITY ? 0.0f : whole;
    for (int w = 0; w < kWarps; ++w)
      total = fmaf(s.sum[w][h], tc::exp2_approx(s.top[w][h] - shift), total);
    s.top[0][h] = whole;
    s.sum[0][h] = total;
  }
  cluster_sync();
  // The blocks joined, each block a part of the outputs.
  for (int c = static_cast<int>(rank) * kThreads + threadIdx.x; c < heads * kDim;
       c += static_cast<int>(blocks) * kThreads) {
    const int h = c / kDim, d = c % kDim;
    float whole = -INFINITY, total = 0.0f, o = 0.0f;
    for (uint32_t r = 0; r < blocks; ++r) whole = fmaxf(whole, read_block(&s.top[0][h], r));
    const float shift = whole == -INFINITY ? 0.0f : whole;
    for (uint32_t r = 0; r < blocks; ++r) {
      const float w = tc::exp2_approx(read_block(&s.top[0][h], r) - shift);
      total = fmaf(read_block(&s.sum[0][h], r), w, total);
      o = fmaf(read_block(&s.out[0][h][d], r), w, o);
    }
    if (d < a.dim)
      static_cast<T*>(a.out)[(b * a.heads + head0 + h) * a.dim + d] =
          from_float<T>(total == 0.0f ? 0.0f : o / total);
  }
  cluster_sync();  // the others have read this block's shared memory
}

// Blocks of a cluster: enough that every multiprocessor has several, as far as every
// warp still gets a turn.
int step_blocks(const gs_window_attention_step_4bit_args& a, int64_t items) {
  int blocks = 1;
  while (blocks < 16 && items * blocks < 4 * kSmCount && blocks * kWarps * kSlots < a.slots)
    blocks *= 2;
  return blocks;
}

template <class T, int kDim, int kSets, bool kMasked, bool kAligned>
int32_t step(const gs_window_attention_step_4bit_args& a, cudaStream_t stream) {
  const int64_t items = a.batch * a.kv_heads * ceil_div(a.heads / a.kv_heads, 8 * kSets);
  const int blocks = step_blocks(a, items);
  if (items * blocks > INT32_MAX) return GS_ERR_CAPACITY;
  constexpr size_t kShared = sizeof(Shared<kDim, kSets>);
  GS_TRY((allow_shared<step_kernel<T, kDim, kSets, kMasked, kAligned>>(kShared, true)));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = blocks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = static_cast<unsigned>(items * blocks);
  config.blockDim = kThreads;
  config.dynamicSmemBytes = kShared;
  config.stream = stream;
  config.attrs = attr;
  config.numAttrs = 2;
  cudaLaunchKernelEx(&config, step_kernel<T, kDim, kSets, kMasked, kAligned>, a);
  return check_launch();
}

bool strided16(const void* p, int64_t stride, int64_t head_stride) {
  return is_aligned(p, 16) && stride % 8 == 0 && head_stride % 8 == 0;
}

}  // namespace

int32_t launch_window_attention_step_4bit(const gs_window_attention_step_4bit_args& a,
                                          cudaStream_t stream) {
  if (a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.heads > 65535 || a.dim < 8 ||
      a.dim % 8)
    return GS_ERR_INVALID_ARGUMENT;
  if (a.dim > kMaxDim || (a.dtype != GS_BFLOAT16 && a.dtype != GS_FLOAT16))
    return GS_ERR_UNSUPPORTED;
  if (a.batch < 0 || a.first < 0 || a.slots <= a.first ||
      a.batch > GS_MAX_SEQUENCE_TOKENS / a.slots || !(a.scale > 0.0f && a.scale < INFINITY))
    return GS_ERR_INVALID_ARGUMENT;
  if (a.batch == 0) return GS_OK;
  if (!a.q || !a.k || !a.v || !a.k_codes || !a.v_codes || !a.k_range || !a.v_range ||
      !a.positions || !a.out || (a.valid && !a.cache_valid))
    return GS_ERR_INVALID_ARGUMENT;
  if (!strided16(a.q, a.q_stride, a.q_head_stride) ||
      !strided16(a.k, a.k_stride, a.k_head_stride) ||
      !strided16(a.v, a.v_stride, a.v_head_stride) || !is_aligned(a.k_codes, 16) ||
      !is_aligned(a.v_codes, 16) || !is_aligned(a.k_range, 16) || !is_aligned(a.v_range, 16) ||
      !is_aligned(a.out, 16) || !is_aligned(a.positions, 8))
    return GS_ERR_MISALIGNED;
  const auto typed = [&](auto t) {
    using T = decltype(t);
    const auto shaped = [&](auto masked, auto aligned) {
      constexpr bool kMasked = decltype(masked)::value, kAligned = decltype(aligned)::value;
      if (a.heads / a.kv_heads <= 8)
        return a.dim <= 64 ? step<T, 64, 1, kMasked, kAligned>(a, stream)
                           : step<T, 128, 1, kMasked, kAligned>(a, stream);
      return a.dim <= 64 ? step<T, 64, 2, kMasked, kAligned>(a, stream)
                         : step<T, 128, 2, kMasked, kAligned>(a, stream);
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
