// A linear layer with its epilogue, and its gradients.
//
//   z = x W^T + b,  y = act(z) + residual
//   dz = grad_y act'(z),  dx = dz W,  dW = dz^T x,  db = sum of dz over the rows
//
// One product kernel makes all three products D = A B^T on the tensor cores: tiles of
// 128 x kN a block, operands by TMA, sums in tensor memory. x W^T contracts along the
// channels of both operands, dz W along W's rows, dz^T x along the rows of both (an
// operand's descriptor says which, nothing is transposed).
//
// What bounds a product, and what it takes, forward unless said otherwise:
//   long contractions: the tensor cores. 65,536 x 1024 -> 4096: 360 us, 1.53 PFLOP/s, 0.91
//     of the rate of a long bare product in a burst; with gelu 400, with its slopes 456. In
//     a training pass the power limit lowers the clock: 490 to 640 us, and 365 to 480 each
//     for dx and dW, with the tensor cores active for 84 to 88 % of the time.
//   short ones: the results, 268 MB of 131,072 x 64 or 128 -> 1024 in 57 us (the epilogue
//     without its stores: 49). From 256 channels 80 us, as dx of 131,101 x 1024 from 256: the
//     loads take longer under the stores' traffic (53 without stores; 74 to 78 without half of
//     the products, or B's loads, or x in L2, or a stage more).
//   activations: gelu makes 137 us of these 80, with its slopes 156: two instructions an
//     element of the kind that a multiprocessor makes 16 a clock of, and a long chain. relu
//     80 and 109.
//   the general epilogue (Form::kAny): its decisions. gelu onto a float residual 239 us,
//     slopes in float 208; results of 1021 columns, which no TMA store takes, 341.
//   few rows: the loads' latency, and a launch. 96 x 2048 -> 8192: 14 us for 34 MB of
//     weights that are not in L2; 1 x 256 -> 1024: 5 us.
#include <algorithm>

#include "tensorcore.cuh"

namespace gs {
namespace {

using namespace tc;

// ---------------------------------------------------------------- activations

// act'(z) is kept in 16 bits, as (slope + 1/6) 49152: slopes lie in [-0.13, 1.13], so
// the error is 1.02e-5 at most, where float16's would be 2.4e-4 next to 1 and add
// to the rounding of dz, which has 11 bits in float16 itself. 0 and 1 are exact, and NaN,
// whose low bits are all ones, is the code that no slope has. (A float32 bias's gradient
// is a sum of unrounded dz: for it slopes can be kept as floats.)
constexpr float kSlopeScale = 49152.0f, kSlopeZero = 8192.0f, kTwo23 = 8388608.0f;
__device__ __forceinline__ uint32_t slope_codes(float2 slopes) {
  // The sums' low bits are the nearest whole numbers.
  const float2 x = fma2(slopes, make_float2(kSlopeScale, kSlopeScale),
                        make_float2(kTwo23 + kSlopeZero, kTwo23 + kSlopeZero));
  return __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x5410);
}
__device__ __forceinline__ float slope_value(uint32_t code) {
  return code == 0xffffu ? NAN : (__uint_as_float(0x4b000000u | code) - (kTwo23 + kSlopeZero)) * (1.0f / kSlopeScale);
}

__device__ __forceinline__ float reciprocal_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// act(z) in z, act'(z) in slope; two floats an instruction where there is one.
//
// gelu: with t = |z|, the normal distribution's upper tail is e^(-t^2/2) R(t), R smooth
// (Mills' ratio over sqrt(2 pi)); R = u P(u) with u = 1 / (1 + 0.3 t) and P the polynomial
// of degree 7 with the least relative error for t up to 14, 1.6e-7. The density that
// the slope needs is the same exponential.
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
template <int kCount>
__device__ __forceinline__ void activate(int kind, float2 (&z)[kCount], float2 (&slope)[kCount]) {
  if (kind == GS_RELU) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      slope[i] = make_float2(z[i].x > 0.0f ? 1.0f : 0.0f, z[i].y > 0.0f ? 1.0f : 0.0f);
      z[i] = make_float2(z[i].x < 0.0f ? 0.0f : z[i].x, z[i].y < 0.0f ? 0.0f : z[i].y);  // NaN stays
    }
  } else if (kind == GS_GELU) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const float2 t = make_float2(fabsf(z[i].x), fabsf(z[i].y));
      const float2 d = fma2(t, both(0.3f), both(1.0f));
      const float2 u = make_float2(reciprocal_approx(d.x), reciprocal_approx(d.y));
      const float2 x = mul2(mul2(z[i], z[i]), both(-0.72134752f));
      const float2 e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
      float2 p = fma2(both(0.0356748066842556f), u, both(-0.15720321238040924f));
      p = fma2(p, u, both(0.20635370910167694f));
      p = fma2(p, u, both(-0.053683821111917496f));
      p = fma2(p, u, both(0.12856172025203705f));
      p = fma2(p, u, both(0.09991347044706345f));
      p = fma2(p, u, both(0.12075395882129669f));
      p = fma2(p, u, both(0.11962930113077164f));
      const float2 tail = mul2(mul2(p, u), e);
      // What lies below z: the tail, or 1 less it. Not by 0.5 +- (0.5 - tail): small tails
      // keep their digits.
      const float2 rest = fma2(tail, both(-1.0f), both(1.0f));
      const float2 below = make_float2(z[i].x < 0.0f ? tail.x : rest.x,
                                       z[i].y < 0.0f ? tail.y : rest.y);
      slope[i] = fma2(mul2(z[i], both(0.39894228f)), e, below);
      z[i] = mul2(z[i], below);
    }
  } else if (kind == GS_SILU) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const float2 x = mul2(z[i], both(-1.44269504f));
      const float2 d = add2(make_float2(exp2_approx(x.x), exp2_approx(x.y)), both(1.0f));
      const float2 gate = make_float2(reciprocal_approx(d.x), reciprocal_approx(d.y));
      z[i] = mul2(z[i], gate);
      slope[i] = fma2(z[i], fma2(gate, both(-1.0f), both(1.0f)), gate);
    }
  }
}

__device__ __forceinline__ float read_as(const void* p, int dtype, int64_t i) {
  return dtype == GS_FLOAT32    ? static_cast<const float*>(p)[i]
         : dtype == GS_BFLOAT16 ? to_float(static_cast<const __nv_bfloat16*>(p)[i])
                                : to_float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void write_as(void* p, int dtype, int64_t i, float x) {
  if (dtype == GS_FLOAT32) static_cast<float*>(p)[i] = x;
  else if (dtype == GS_BFLOAT16) static_cast<__nv_bfloat16*>(p)[i] = from_float<__nv_bfloat16>(x);
  else static_cast<__half*>(p)[i] = from_float<__half>(x);
}

// ------------------------------------------------------------- product kernel

// Set when a bounded wait ran out (linear_status).
__device__ uint32_t g_timeout;

constexpr int kRows = 128;   // of a tile
constexpr int kDepth = 64;   // of a stage: 128 bytes of channels, or 64 rows
constexpr int kEpilogueWarps = 8;
constexpr int kGatherWarps = 8;  // of 16 rows: a tile's are all on their way at once
constexpr int product_threads(bool gather) {
  return 32 * (kEpilogueWarps + 2 + (gather ? kGatherWarps : 0));
}
constexpr int kChunkBytes = 4096;  // of the epilogue: 32 rows of 128 bytes

// What becomes of the sums D(m, n).
struct Epilogue {
  int64_t rows;  // D's extents
  int32_t columns;
  void* out;
  int64_t out_stride;
  int32_t out_dtype;
  // the forward's
  int32_t activation, bias_dtype;
  const void *bias, *residual;
  int64_t residual_stride;
  void* slope;
  int64_t slope_stride;
  bool slope_float;
  // Whether `out` and the residual lie as TMA takes them (rows of whole 16-byte words).
  bool tiled;
};

// The maps of what the epilogue reads and writes, in its chunks.
struct EpilogueMaps {
  CUtensorMap out, residual, slope;
};

// What an epilogue has to do, where the kernel is built for it: code that decides as it
// goes takes twice the instructions. kAny decides: it writes what TMA does not take, and does
// what none of the others is built for (a 16-bit residual, an activation before a float
// result, slopes in float, a float result without a residual in the forward).
enum class Form {
  kAny,
  kNarrow,    // 16-bit result
  kActive,    // 16-bit result of an activation
  kTraining,  // the same, and its slopes in 16 bits
  kWide,      // float result (sums to be joined)
  kStream,    // float result added to a residual
};

// Items are (split, row tile, column tile), the last one fastest: blocks that work at the
// same time share rows of A, and write whole rows of the result.
struct Plan {
  int32_t row_tiles, column_tiles, splits;
  int32_t steps;            // of kDepth, in the whole contraction
  int32_t steps_per_split;
  int64_t split_rows;       // rows of `out` from one split's sums to the next one's
};

// A block's (or a pair's) items: its own, and every one that many blocks further.
struct Walk {
  int32_t split, row, column;  // tiles
  int32_t split_step, row_step, column_step;
  __device__ Walk(const Plan& p, int blocks) {
    const auto cut = [&](uint32_t item, int32_t& s, int32_t& r, int32_t& c) {
      c = item % p.column_tiles;
      item /= p.column_tiles;
      r = item % p.row_tiles;
      s = item / p.row_tiles;
    };
    cut(blockIdx.x / blocks, split, row, column);
    cut(gridDim.x / blocks, split_step, row_step, column_step);
  }
  __device__ bool more(const Plan& p) const { return split < p.splits; }
  __device__ void advance(const Plan& p) {
    column += column_step;
    row += row_step;
    split += split_step;
    if (column >= p.column_tiles) column -= p.column_tiles, ++row;
    if (row >= p.row_tiles) row -= p.row_tiles, ++split;
  }
  __device__ int first_step(const Plan& p) const { return split * p.steps_per_split; }
  __device__ int steps(const Plan& p) const {
    return min(p.steps_per_split, p.steps - first_step(p));
  }
};

// kPair: two blocks share a tile of 2 kRows x kN.
template <int kN, bool kPair>
struct ProductShared {
  static constexpr int kBRows = kPair ? kN / 2 : kN;  // of B here
  static constexpr int kABytes = kRows * kDepth * 2, kBBytes = kBRows * kDepth * 2;
  // As many as fit: narrow tiles are for few rows, whose time is the loads' latency.
  static constexpr int kStages = kN == 256 ? (kPair ? 4 : 3) : kN == 128 ? 4 : kN == 64 ? 6 : 7;
  alignas(1024) unsigned char a[kStages][kABytes];
  alignas(1024) unsigned char b[kStages][kBBytes];
  alignas(1024) unsigned char out[kEpilogueWarps][2][kChunkBytes];
  // Columns of a 16-bit chunk: rows of 128 bytes (TMA takes about as long for rows of 64),
  // unless the tile is too narrow to give all warps chunks of them.
  static constexpr int kWide = kN >= 128 ? 64 : 32;
  float bias[kEpilogueWarps][kN];
  uint64_t full[kStages], empty[kStages], ready[2], drained[2], residual[kEpilogueWarps][2];
  uint32_t tensor;
};

// Where word 0 of a thread's row of a chunk is, in rows of 128 bytes or of 64; word w is
// there with its number flipped into bits 4 and up. So TMA's swizzle has it: words are
// exchanged so that eight rows' same words lie in different banks.
template <int kBytes>
__device__ __forceinline__ uint32_t row_of_chunk(uint32_t chunk, int row) {
  return kBytes == 128 ? chunk + row * 128 + ((row & 7) << 4) : chunk + row * 64 + ((row >> 1 & 3) << 4);
}
__device__ __forceinline__ void put_word(uint32_t at, uint32_t a, uint32_t b, uint32_t c,
                                         uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ uint4 get_word(uint32_t at) {
  uint4 w;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
               : "r"(at)
               : "memory");
  return w;
}
__device__ __forceinline__ void store_box(const CUtensorMap* map, int x, int row, uint32_t src) {
  asm volatile(
      "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(x), "r"(row), "r"(src)
      : "memory");
}
__device__ __forceinline__ void commit_stores() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Until all stores but the last kPending have read their shared memory.
template <int kPending>
__device__ __forceinline__ void wait_stores_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void wait_stores_done() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// The epilogue's warps: a row a thread, 32 columns at a time. Chunks of 32 floats' or
// kWide 16-bit columns pass through shared memory, from which TMA writes them; the
// residual's come by TMA to the place of the results, a chunk ahead if two fit. Where
// rows are no whole 16-byte words, a warp writes 32 columns of one row at a time instead.
template <class T, int kN, Form kForm, bool kPair>
__device__ bool epilogue(const Plan& plan, const Epilogue& e, const EpilogueMaps& maps,
                         ProductShared<kN, kPair>& s, uint32_t tensor, int warp, int lane) {
  constexpr int kWide = ProductShared<kN, kPair>::kWide, kNarrowBytes = kWide * 2;
  // The block's rows of a tile.
  constexpr int kTileRows = kPair ? 2 * kRows : kRows;
  const int row_in_tile = 32 * (warp & 3) + (kPair ? kRows * static_cast<int>(pair_rank()) : 0);
  constexpr int kParts = kWide / 32;  // steps of 32 columns of a 16-bit chunk
  constexpr bool kAny = kForm == Form::kAny;
  const bool wide = kAny ? e.out_dtype == GS_FLOAT32 : kForm == Form::kWide || kForm == Form::kStream;
  const bool add = kAny ? e.residual != nullptr : kForm == Form::kStream;
  const bool active = kAny || kForm == Form::kActive || kForm == Form::kTraining;
  const bool slopes = kAny ? e.slope != nullptr : kForm == Form::kTraining;
  const bool slope_float = kAny && e.slope_float;
  const bool by_tma = !kAny || e.tiled;
  const bool two = !slopes;  // two chunks in turn; with slopes, one and its slopes
  const uint32_t staged = shared_address(s.out[warp]);
  float* const biases = s.bias[warp];
  const int c0 = (warp >> 2) * kParts;  // the warp's first step; then every other chunk's
  const auto next_step = [&](int c) { return (c + 1) % kParts ? c + 1 : c + 1 + kParts; };
  struct Place {
    Walk walk;
    int c;
  };
  const auto column_of = [&](const Place& p) { return p.walk.column * kN + 32 * p.c; };
  const auto row_of = [&](const Place& p) { return p.walk.row * kTileRows + row_in_tile; };
  // The place, or the warp's next one, that has columns and starts a chunk.
  const auto chunk_from = [&](Place p) {
    while (p.walk.more(plan) && (p.c >= kN / 32 || column_of(p) >= e.columns)) {
      p.walk.advance(plan);
      p.c = c0;
    }
    return p;
  };
  const auto load_residual = [&](const Place& p, uint32_t use) {
    if (!p.walk.more(plan)) return;
    const uint32_t at = two ? use & 1 : 0;
    const uint32_t bar = shared_address(&s.residual[warp][at]);
    barrier_expect(bar, wide ? kChunkBytes : 32 * kNarrowBytes);
    load_box(staged + at * kChunkBytes, &maps.residual, column_of(p), row_of(p), bar);
  };
  bool good = true;
  uint32_t use = 0;  // chunks done
  Walk walk(plan, kPair ? 2 : 1);
  if (by_tma && add && lane == 0) load_residual(chunk_from({walk, c0}), 0);
  int bias_column = -1;
  for (uint32_t count = 0; walk.more(plan); walk.advance(plan), ++count) {
    const uint32_t buffer = count & 1;
    const int n0 = walk.column * kN;
    if (e.bias && n0 != bias_column) {
      __syncwarp();
      for (int i = lane; i < kN; i += 32)
        biases[i] = n0 + i < e.columns ? read_as(e.bias, e.bias_dtype, n0 + i) : 0.0f;
      __syncwarp();
      bias_column = n0;
    }
    const int row = walk.row * kTileRows + row_in_tile;
    const int64_t out_row = walk.split * plan.split_rows + row;
    good = good && barrier_wait_warp(shared_address(&s.ready[buffer]), count >> 1 & 1);
    fence_after_sync();
    const uint32_t sums = tensor + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + buffer * kN;
#pragma unroll 1
    for (int c = c0; c < kN / 32; c = next_step(c)) {
      const int n = n0 + 32 * c;
      if (n >= e.columns) break;
      float2 z[16], slope[16];
      load_columns32(sums + 32 * c, reinterpret_cast<float(&)[32]>(z));
      wait_loads();
      if (!good)
#pragma unroll
        for (float2& x : z) x = both(NAN);
      if (e.bias)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 b = *reinterpret_cast<const float4*>(biases + 32 * c + 4 * i);
          z[2 * i] = add2(z[2 * i], make_float2(b.x, b.y));
          z[2 * i + 1] = add2(z[2 * i + 1], make_float2(b.z, b.w));
        }
      if (active) activate(e.activation, z, slope);
      const int part = c % kParts;  // of a 16-bit chunk
      if (by_tma) {
        const uint32_t at = two ? use & 1 : 0, chunk = staged + at * kChunkBytes;
        const uint32_t slope_chunk = staged + kChunkBytes;
        if (wide || part == 0) {
          if (lane == 0) {
            if (two && !add) wait_stores_read<1>();
            else wait_stores_read<0>();
            if (add && two) load_residual(chunk_from({walk, wide ? next_step(c) : c + 2 * kParts}), use + 1);
          }
          if (add)
            good = good && barrier_wait_warp(shared_address(&s.residual[warp][at]),
                                             (two ? use >> 1 : use) & 1);
          __syncwarp();
        }
        if (wide) {
          const uint32_t to = row_of_chunk<128>(chunk, lane);
          if (add)
#pragma unroll
            for (int w = 0; w < 8; ++w) {
              const uint4 r = get_word(to ^ w << 4);
              z[2 * w] = add2(z[2 * w], make_float2(__uint_as_float(r.x), __uint_as_float(r.y)));
              z[2 * w + 1] = add2(z[2 * w + 1],
                                  make_float2(__uint_as_float(r.z), __uint_as_float(r.w)));
            }
#pragma unroll
          for (int w = 0; w < 8; ++w)
            put_word(to ^ w << 4, __float_as_uint(z[2 * w].x), __float_as_uint(z[2 * w].y),
                     __float_as_uint(z[2 * w + 1].x), __float_as_uint(z[2 * w + 1].y));
        } else {
          const uint32_t to = row_of_chunk<kNarrowBytes>(chunk, lane) ^ part << 6;
          if (add)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint4 r = get_word(to ^ w << 4);
              const T* v = reinterpret_cast<const T*>(&r);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                z[4 * w + k] = add2(z[4 * w + k],
                                    make_float2(to_float(v[2 * k]), to_float(v[2 * k + 1])));
            }
          uint32_t word[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) word[i] = pack2<T>(z[i].x, z[i].y);
#pragma unroll
          for (int w = 0; w < 4; ++w)
            put_word(to ^ w << 4, word[4 * w], word[4 * w + 1], word[4 * w + 2], word[4 * w + 3]);
        }
        if (slopes && slope_float) {
          if (!wide && part > 0) {  // the slopes of the chunk's part before
            if (lane == 0) wait_stores_read<0>();
            __syncwarp();
          }
          const uint32_t to = row_of_chunk<128>(slope_chunk, lane);
#pragma unroll
          for (int w = 0; w < 8; ++w)
            put_word(to ^ w << 4, __float_as_uint(slope[2 * w].x), __float_as_uint(slope[2 * w].y),
                     __float_as_uint(slope[2 * w + 1].x), __float_as_uint(slope[2 * w + 1].y));
        } else if (slopes) {
          const uint32_t to = row_of_chunk<kNarrowBytes>(slope_chunk, lane) ^ part << 6;
          uint32_t word[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) word[i] = slope_codes(slope[i]);
#pragma unroll
          for (int w = 0; w < 4; ++w)
            put_word(to ^ w << 4, word[4 * w], word[4 * w + 1], word[4 * w + 2], word[4 * w + 3]);
        }
        const bool ends = part == kParts - 1 || n + 32 >= e.columns;  // a 16-bit chunk
        if (wide || ends || slope_float) {
          fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            if (row < e.rows) {
              if (wide) store_box(&maps.out, n, static_cast<int>(out_row), chunk);
              else if (ends) store_box(&maps.out, n - 32 * part, static_cast<int>(out_row), chunk);
              if (slopes && slope_float) store_box(&maps.slope, n, row, slope_chunk);
              else if (slopes && ends) store_box(&maps.slope, n - 32 * part, row, slope_chunk);
            }
            commit_stores();
            if (add && !two && (wide || ends)) {
              wait_stores_read<0>();
              load_residual(chunk_from({walk, wide ? next_step(c) : c - part + 2 * kParts}), use + 1);
            }
          }
          if (wide || ends) ++use;
        }
      } else {
        float* const square = reinterpret_cast<float*>(s.out[warp]);
        const auto store = [&](const float2(&x)[16], auto&& put) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            square[32 * lane + (2 * i ^ lane)] = x[i].x;
            square[32 * lane + ((2 * i + 1) ^ lane)] = x[i].y;
          }
          __syncwarp();
          if (n + lane < e.columns)
            for (int r = 0; r < 32 && row + r < e.rows; ++r) put(r, square[32 * r + (lane ^ r)]);
        };
        store(z, [&](int r, float y) {
          if (add) y += read_as(e.residual, e.out_dtype, (row + r) * e.residual_stride + n + lane);
          write_as(e.out, e.out_dtype, (out_row + r) * e.out_stride + n + lane, y);
        });
        if (slopes)
          store(slope, [&](int r, float x) {
            const int64_t to = (row + r) * e.slope_stride + n + lane;
            if (slope_float) static_cast<float*>(e.slope)[to] = x;
            else static_cast<uint16_t*>(e.slope)[to] = static_cast<uint16_t>(slope_codes(both(x)));
          });
      }
    }
    fence_before_sync();
    __syncwarp();
    if (lane == 0) {
      const uint32_t bar = shared_address(&s.drained[buffer]);
      if constexpr (kPair) barrier_arrive_cluster(of_first_block(bar));
      else barrier_arrive(bar);
    }
  }
  if (lane == 0) wait_stores_done();
  if (!good)
    for (uint64_t& bar : s.residual[warp]) barrier_settle(shared_address(&bar));
  return good;
}

// An operand: a [rows, channels] array of 16-bit elements.
struct Operand {
  const void* data;
  int64_t rows, channels, stride;
};

// Rows of A that TMA does not take (no whole 16-byte words): a warp loads a row's 64
// channels at a time, two a lane, and puts them where TMA would have. All its rows of a
// stage are requested before the stage before is put down, so that their latency passes
// while that one waits for its place. No copy of A is made for it: that took a third of
// the time of a forward whose bound is its result (500,000 x 59 -> 256: 90 us a pass with
// one, 69 so; 72 without requests ahead).
constexpr int kGatherRows = kRows / kGatherWarps;
struct Gathered {
  uint32_t word[kGatherRows];
  uint32_t more;  // an odd row's 64th channel lies in a 33rd word: row i's is lane i's
};
// 1 if row i of the rows at `data` starts in the middle of a 4-byte word.
__device__ __forceinline__ int odd_row(const uint16_t* data, int64_t stride, int i) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(data) >> 1 ^ (i & stride)) & 1);
}
__device__ __forceinline__ const uint16_t* gathered_from(const Operand& a, int64_t row0, int k0) {
  return static_cast<const uint16_t*>(a.data) + row0 * a.stride + k0;
}
__device__ __forceinline__ Gathered gather_rows(const Operand& a, int64_t row0, int k0, int lane) {
  const int valid = static_cast<int>(min(int64_t{kDepth}, a.channels - k0));
  const uint16_t* const data = gathered_from(a, row0, k0);
  const int rows = static_cast<int>(min(int64_t{kGatherRows}, a.rows - row0));
  const auto words = [&](int i) {
    return reinterpret_cast<const uint32_t*>(data + i * a.stride - odd_row(data, a.stride, i));
  };
  Gathered g;
#pragma unroll
  for (int i = 0; i < kGatherRows; ++i)
    g.word[i] = i < rows && 2 * lane < valid + odd_row(data, a.stride, i) ? __ldg(words(i) + lane) : 0;
  g.more = lane < rows && odd_row(data, a.stride, lane) && valid == kDepth ? __ldg(words(lane) + 32) : 0;
  return g;
}
__device__ __forceinline__ void put_rows(const Gathered& g, const Operand& a, int64_t row0, int k0,
                                         uint32_t tile, int lane) {
  const int valid = static_cast<int>(min(int64_t{kDepth}, a.channels - k0));
  const uint16_t* const data = gathered_from(a, row0, k0);
#pragma unroll
  for (int i = 0; i < kGatherRows; ++i) {  // eight rows' swizzle starts over with the warp's rows
    uint32_t next = __shfl_down_sync(0xffffffffu, g.word[i], 1);
    const uint32_t last = __shfl_sync(0xffffffffu, g.more, i);
    if (lane == 31) next = last;
    uint32_t two = odd_row(data, a.stride, i) ? __byte_perm(g.word[i], next, 0x5432) : g.word[i];
    if (2 * lane + 1 >= valid) two = 2 * lane < valid ? two & 0xffffu : 0;
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(tile + i * 128 + ((lane >> 2 ^ (i & 7)) << 4) +
                                                 (lane & 3) * 4),
                 "r"(two)
                 : "memory");
  }
}

// D = A B^T, tile by tile: a block an SM that goes on to its next item, so that its loads
// and products of the next tile run under the epilogue of this one (two sets of sums in
// tensor memory). One warp loads, one issues the products, eight make the epilogue.
// kRowsA, kRowsB: the operand's contraction runs along its rows. kGather: A's rows by
// gather_rows.
template <class T, int kN, bool kRowsA, bool kRowsB, Form kForm, bool kPair, bool kGather>
__global__ void __launch_bounds__(product_threads(kGather), 1)
    product_kernel(Plan plan, Epilogue e, Operand a_rows,
                   const __grid_constant__ CUtensorMap a_map,
                   const __grid_constant__ CUtensorMap b_map,
                   const __grid_constant__ EpilogueMaps maps) {
  using Shared = ProductShared<kN, kPair>;
  constexpr int kStages = Shared::kStages;
  extern __shared__ __align__(1024) unsigned char shared_bytes[];
  Shared& s = *reinterpret_cast<Shared*>(shared_bytes);
  chain_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 32 * kEpilogueWarps) {
    for (int i = 0; i < kStages; ++i) {
      barrier_init(shared_address(&s.full[i]), kGather ? 1 + kGatherWarps : 1);
      barrier_init(shared_address(&s.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      barrier_init(shared_address(&s.ready[i]), 1);
      barrier_init(shared_address(&s.drained[i]), kPair ? 2 * kEpilogueWarps : kEpilogueWarps);
      for (int w = 0; w < kEpilogueWarps; ++w) barrier_init(shared_address(&s.residual[w][i]), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
  }
  if (warp == kEpilogueWarps + 1) {
    if constexpr (kPair) tensor_alloc_pair<2 * kN>(shared_address(&s.tensor));
    else tensor_alloc<2 * kN>(shared_address(&s.tensor));
  }
  fence_before_sync();
  __syncthreads();
  if constexpr (kPair) pair_sync();  // both blocks' barriers are ready
  fence_after_sync();
  const uint32_t tensor = s.tensor;
  const int rank = kPair ? static_cast<int>(pair_rank()) : 0;
  bool good = true;
  Walk walk(plan, kPair ? 2 : 1);

  if (warp == kEpilogueWarps) {  // loads
    if (lane == 0) {
      uint32_t turn = 0;  // stages used so far
      for (; walk.more(plan) && good; walk.advance(plan)) {
        const int m0 = (kPair ? 2 * walk.row + rank : walk.row) * kRows;
        const int n0 = walk.column * kN + rank * Shared::kBRows;
        const int first = walk.first_step(plan), steps = walk.steps(plan);
        for (int k = 0; k < steps; ++k, ++turn) {
          const uint32_t stage = turn % kStages, round = turn / kStages;
          if (round > 0) good = barrier_wait(shared_address(&s.empty[stage]), (round - 1) & 1);
          if (!good) break;
          uint32_t bar = shared_address(&s.full[stage]);
          const uint32_t a = shared_address(s.a[stage]), b = shared_address(s.b[stage]);
          const int k0 = (first + k) * kDepth;
          if (rank == 0)
            barrier_expect(bar, (kPair ? 2 : 1) * ((kGather ? 0 : Shared::kABytes) + Shared::kBBytes));
          if constexpr (kPair) bar = of_first_block(bar);
          const auto load = [&](uint32_t to, const CUtensorMap* map, int x, int r) {
            if constexpr (kPair) load_box_pair(to, map, x, r, bar);
            else load_box(to, map, x, r, bar);
          };
          if constexpr (kRowsA)
            for (int i = 0; i < kRows / 64; ++i)
              load(a + i * kDepth * 128, &a_map, m0 + 64 * i, k0);
          else if constexpr (!kGather)
            load(a, &a_map, k0, m0);
          if constexpr (kRowsB)
            for (int i = 0; i < Shared::kBRows / 64; ++i)
              load(b + i * kDepth * 128, &b_map, n0 + 64 * i, k0);
          else
            load(b, &b_map, k0, n0);
        }
      }
      if constexpr (kPair)  // the first block's products no longer signal to this one
        for (uint32_t last = turn > kStages ? turn - kStages : 0; last < turn && good; ++last)
          good = barrier_wait(shared_address(&s.empty[last % kStages]), last / kStages & 1);
    }
    __syncwarp();
  } else if (warp == kEpilogueWarps + 1) {  // products
    const uint32_t elected = elect_lane();
    const uint32_t kind = (kPair ? product_kind_pair<T>(kN, kRowsB) : product_kind<T>(kN, kRowsB)) |
                          (kRowsA ? 1u << 15 : 0u);
    const uint32_t a_word = kRowsA ? rows_word<kDepth>(shared_address(s.a[0]))
                                   : channels_word<kRows>(shared_address(s.a[0]));
    const uint32_t b_word = kRowsB ? rows_word<kDepth>(shared_address(s.b[0]))
                                   : channels_word<Shared::kBRows>(shared_address(s.b[0]));
    uint32_t turn = 0;
    for (uint32_t count = 0; rank == 0 && walk.more(plan) && good; walk.advance(plan), ++count) {
      const uint32_t buffer = count & 1, round = count >> 1;
      const int steps = walk.steps(plan);
      if (round > 0)
        good = barrier_wait_warp(shared_address(&s.drained[buffer]), (round - 1) & 1);
      fence_after_sync();
      for (int k = 0; k < steps && good; ++k, ++turn) {
        const uint32_t stage = turn % kStages;
        good = barrier_wait_warp(shared_address(&s.full[stage]), turn / kStages & 1);
        if (!good) break;
        fence_after_sync();
        const uint32_t a = a_word + stage * (Shared::kABytes >> 4);
        const uint32_t b = b_word + stage * (Shared::kBBytes >> 4);
#pragma unroll
        for (int i = 0; i < kDepth / 16; ++i) {
          const uint32_t a_step = a + (kRowsA ? rows_step(i) : channels_step<kRows>(i));
          const uint32_t b_step = b + (kRowsB ? rows_step(i) : channels_step<Shared::kBRows>(i));
          if constexpr (kPair)
            multiply_pair(elected, tensor + buffer * kN, a_step, b_step, kind, k > 0 || i > 0);
          else
            multiply(elected, tensor + buffer * kN, a_step, b_step, kind, k > 0 || i > 0);
        }
        if constexpr (kPair) commit_pair(elected, shared_address(&s.empty[stage]));
        else commit(elected, shared_address(&s.empty[stage]));
      }
      if (good) {
        if constexpr (kPair) commit_pair(elected, shared_address(&s.ready[buffer]));
        else commit(elected, shared_address(&s.ready[buffer]));
      }
    }
  } else if (kGather && warp >= kEpilogueWarps + 2) {
    const int rows_in_tile = kGatherRows * (warp - kEpilogueWarps - 2);
    struct Place {
      Walk walk;
      int k;  // of the item's steps
    };
    const auto row_of = [&](const Place& p) { return int64_t{p.walk.row} * kRows + rows_in_tile; };
    const auto depth_of = [&](const Place& p) { return (p.walk.first_step(plan) + p.k) * kDepth; };
    Place here = {walk, 0};
    Gathered now = gather_rows(a_rows, row_of(here), depth_of(here), lane);
    for (uint32_t turn = 0; here.walk.more(plan) && good; ++turn) {
      Place next = here;
      if (++next.k == here.walk.steps(plan)) {
        next.walk.advance(plan);
        next.k = 0;
      }
      Gathered ahead = now;
      if (next.walk.more(plan)) ahead = gather_rows(a_rows, row_of(next), depth_of(next), lane);
      const uint32_t stage = turn % kStages, round = turn / kStages;
      if (round > 0) good = barrier_wait_warp(shared_address(&s.empty[stage]), (round - 1) & 1);
      if (!good) break;
      put_rows(now, a_rows, row_of(here), depth_of(here), shared_address(s.a[stage]) + rows_in_tile * 128,
               lane);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) barrier_arrive(shared_address(&s.full[stage]));
      here = next;
      now = ahead;
    }
  } else {
    good = epilogue<T, kN, kForm, kPair>(plan, e, maps, s, tensor, warp, lane);
  }
  if (!good) {  // let what is in flight land
    for (uint64_t& bar : s.full) barrier_settle(shared_address(&bar));
    for (uint64_t& bar : s.empty) barrier_settle(shared_address(&bar));
    for (uint64_t& bar : s.ready) barrier_settle(shared_address(&bar));
    if (lane == 0) atomicExch(&g_timeout, 1u);
  }
  fence_before_sync();
  __syncthreads();
  if constexpr (kPair) pair_sync();  // neither block needs the other's memory any more
  fence_after_sync();
  if (warp == kEpilogueWarps + 1) {
    if constexpr (kPair) tensor_free_pair<2 * kN>(tensor);
    else tensor_free<2 * kN>(tensor);
  }
}

int32_t encode_operand(CUtensorMap* map, int32_t dtype, const Operand& o, int box_rows) {
  const cuuint64_t size[2] = {static_cast<cuuint64_t>(o.channels), static_cast<cuuint64_t>(o.rows)};
  const cuuint64_t stride[1] = {static_cast<cuuint64_t>(o.stride) * 2};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
  return encode(map, dtype, o.data, 2, size, stride, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// A [rows, columns] array in the epilogue's chunks.
int32_t encode_chunks(CUtensorMap* map, int32_t dtype, const void* data, int64_t rows,
                      int64_t columns, int64_t row_stride, int narrow_columns) {
  const cuuint64_t size[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)};
  const cuuint64_t stride[1] = {static_cast<cuuint64_t>(row_stride) * element_size(dtype)};
  const cuuint32_t box_columns = dtype == GS_FLOAT32 ? 32 : narrow_columns, box[2] = {box_columns, 32};
  return encode(map, dtype, data, 2, size, stride, box,
                box_columns * element_size(dtype) == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                                         : CU_TENSOR_MAP_SWIZZLE_64B);
}

bool tma_rows(const void* data, int64_t stride, int32_t dtype, int64_t columns) {
  return is_aligned(data, 16) && stride * element_size(dtype) % 16 == 0 && stride >= columns;
}

template <class T, int kN, bool kRowsA, bool kRowsB, Form kForm, bool kPair, bool kGather>
int32_t launch_product(int32_t dtype, const Operand& a, const Operand& b, const Plan& plan,
                       const Epilogue& e, cudaStream_t stream) {
  CUtensorMap a_map, b_map;
  if (!kGather) GS_TRY(encode_operand(&a_map, dtype, a, kRowsA ? kDepth : kRows));
  using Shared = ProductShared<kN, kPair>;
  GS_TRY(encode_operand(&b_map, dtype, b, kRowsB ? kDepth : Shared::kBRows));
  EpilogueMaps maps;
  if (e.tiled) {
    const int64_t out_rows = plan.splits > 1 ? plan.splits * plan.split_rows : e.rows;
    constexpr int kWide = Shared::kWide;
    GS_TRY(encode_chunks(&maps.out, e.out_dtype, e.out, out_rows, e.columns, e.out_stride, kWide));
    if (e.residual)
      GS_TRY(encode_chunks(&maps.residual, e.out_dtype, e.residual, e.rows, e.columns,
                           e.residual_stride, kWide));
    if (e.slope)  // bfloat16 stands for any 16 bits
      GS_TRY(encode_chunks(&maps.slope, e.slope_float ? GS_FLOAT32 : GS_BFLOAT16, e.slope, e.rows,
                           e.columns, e.slope_stride, kWide));
  }
  constexpr size_t kShared = sizeof(Shared);
  constexpr int kBlocks = kPair ? 2 : 1;
  GS_TRY((allow_shared<product_kernel<T, kN, kRowsA, kRowsB, kForm, kPair, kGather>>(kShared)));
  const int64_t items = int64_t{plan.row_tiles} * plan.column_tiles * plan.splits;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kBlocks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = static_cast<unsigned>(kBlocks * std::min<int64_t>(items, kSmCount / kBlocks));
  config.blockDim = product_threads(kGather);
  config.dynamicSmemBytes = kShared;
  config.stream = stream;
  config.attrs = attr;
  config.numAttrs = kPair ? 2 : 1;
  cudaLaunchKernelEx(&config, product_kernel<T, kN, kRowsA, kRowsB, kForm, kPair, kGather>, plan, e,
                     a, a_map, b_map, maps);
  return check_launch();
}

// The form that an epilogue has.
Form form_of(const Epilogue& e) {
  if (!e.tiled) return Form::kAny;
  const bool active = e.activation != GS_IDENTITY;
  if (e.out_dtype == GS_FLOAT32)
    return active || e.slope ? Form::kAny : e.residual ? Form::kStream : Form::kWide;
  if (e.residual || (e.slope && e.slope_float)) return Form::kAny;
  return !active ? Form::kNarrow : e.slope ? Form::kTraining : Form::kActive;
}

int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

constexpr int kPairDepth = 512;

// A tile: its columns, and whether a pair of blocks shares one of 2 kRows.
struct ProductTile {
  int columns;
  bool pair;
  int rows() const { return pair ? 2 * kRows : kRows; }
  int workers() const { return pair ? kSmCount / 2 : kSmCount; }
};

Plan plan_of(int64_t rows, int64_t columns, int64_t depth, ProductTile tile, int splits) {
  Plan p = {};
  p.row_tiles = static_cast<int32_t>(ceil_div(rows, tile.rows()));
  p.column_tiles = static_cast<int32_t>(ceil_div(columns, tile.columns));
  p.steps = static_cast<int32_t>(ceil_div(depth, kDepth));
  p.steps_per_split = static_cast<int32_t>(ceil_div(p.steps, splits));
  p.splits = static_cast<int32_t>(ceil_div(p.steps, p.steps_per_split));
  p.split_rows = int64_t{p.row_tiles} * tile.rows();
  return p;
}

// The tile with which the multiprocessors' last turn ends first. A turn takes a tile's
// columns and about 32 more for its start and end; a pair's takes three quarters as long
// for its columns, whose half it stages, where the contraction is long enough that the
// products and not the results bound it (131,101 x 256: contracting 1024, 93 us against 98;
// 131,101 x 1024: contracting 256, 90 against 78).
ProductTile tile_of(int64_t rows, int64_t columns, int64_t depth, int least, bool pairs = true) {
  ProductTile best = {};
  int64_t best_time = 0;
  const auto consider = [&](ProductTile t, int64_t turn) {
    const int64_t tiles = int64_t{ceil_div(rows, t.rows())} * ceil_div(columns, t.columns);
    const int64_t time = (tiles + t.workers() - 1) / t.workers() * turn;
    if (!best.columns || time < best_time) best = t, best_time = time;
  };
  if (pairs && depth >= kPairDepth) consider({256, true}, 192 + 32);
  for (int n = 256; n >= least; n /= 2) consider({n, false}, n + 32);
  return best;
}

// D = A B^T by `e`, in such tiles. The gradients' products have 16-bit results
// or sums to be joined only.
template <class T, bool kRowsA, bool kRowsB, bool kGather = false>
int32_t run_product(int32_t dtype, const Operand& a, const Operand& b, const Plan& plan, ProductTile tile,
                    const Epilogue& e, cudaStream_t stream) {
  const auto formed = [&](auto columns, auto pair) {
    constexpr int kN = decltype(columns)::value;
    constexpr bool kPair = decltype(pair)::value;
    const auto launch = [&](auto form) {
      return launch_product<T, kN, kRowsA, kRowsB, decltype(form)::value, kPair, kGather>(
          dtype, a, b, plan, e, stream);
    };
    // What is not built for these operands (a float result without a residual, forward) is
    // the general form's.
    switch (form_of(e)) {
      case Form::kNarrow: return launch(std::integral_constant<Form, Form::kNarrow>{});
      case Form::kWide:
        if constexpr (kRowsA && kRowsB) return launch(std::integral_constant<Form, Form::kWide>{});
        break;
      case Form::kActive:
        if constexpr (!kRowsB) return launch(std::integral_constant<Form, Form::kActive>{});
        break;
      case Form::kTraining:
        if constexpr (!kRowsB) return launch(std::integral_constant<Form, Form::kTraining>{});
        break;
      case Form::kStream:
        if constexpr (!kRowsB) return launch(std::integral_constant<Form, Form::kStream>{});
        break;
      case Form::kAny: break;
    }
    return launch(std::integral_constant<Form, Form::kAny>{});
  };
  if constexpr (!kGather)
    if (tile.pair) return formed(std::integral_constant<int, 256>{}, std::true_type{});
  switch (tile.columns) {
    case 256: return formed(std::integral_constant<int, 256>{}, std::false_type{});
    case 128: return formed(std::integral_constant<int, 128>{}, std::false_type{});
    case 64: return formed(std::integral_constant<int, 64>{}, std::false_type{});
    case 32:
      if constexpr (!kRowsB) return formed(std::integral_constant<int, 32>{}, std::false_type{});
  }
  return GS_ERR_UNSUPPORTED;
}

// ------------------------------------------------- the gradient of the sums

constexpr int kSlopeThreads = 256;
constexpr int kSlopeBlocks = 6 * kSmCount;

// How the work is cut: blocks of `lanes` words of eight columns, by strips of rows.
struct Strips {
  int32_t lanes, column_blocks;
  int64_t rows, count;  // of a strip; strips
};

// Eight floats of a row at `p`, of which `valid` exist.
template <bool kWhole, class G>
__device__ __forceinline__ void load_row(const G* p, int valid, float (&x)[8]) {
  if constexpr (!kWhole) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = k < valid ? to_float(p[k]) : 0.0f;
  } else if constexpr (sizeof(G) == 4) {
    float lo[4], hi[4];
    load_pack<4>(p, lo);
    load_pack<4>(p + 4, hi);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = lo[k], x[4 + k] = hi[k];
  } else {
    load_pack<8>(p, x);
  }
}

enum class Slopes { kNone, kCodes, kFloats };

// dz = grad_y act'(z) rounded to the operands' type, and each strip's sums of its columns
// (of what was not rounded). Rounded because it is an operand of two products: to keep what
// the rounding takes, each would be made twice, of dz's upper and lower bits, for gradients
// that are rounded to the same type themselves (a training pass's errors against 64 bits 2.4e-3 and 3.0e-4 in
// bfloat16 and float16, with dz in float 1.7e-3 and 2.1e-4). A thread has eight columns of every so many rows, and loads
// several rows before it works on the first: memory is the bound (65,536 x 4096 in
// float16: 280 us for 1.6 GB, 5.8 TB/s; 131,101 x 256 of a float gradient: 30 us for 200
// MB, 6.7 TB/s). kWhole: rows are whole 16-byte words.
template <class T, class G, Slopes kSlopes, bool kWhole>
__global__ void __launch_bounds__(kSlopeThreads, 3)
    slope_kernel(gs_linear_args a, Strips cut, int64_t stride, T* __restrict__ dz,
                 float* __restrict__ sums) {
  chain_wait();
  __shared__ float joined[kSlopeThreads][8 + 1];
  const int lane = threadIdx.x % cut.lanes, first = threadIdx.x / cut.lanes;
  const int step = kSlopeThreads / cut.lanes;
  const int64_t column = (blockIdx.y * int64_t{cut.lanes} + lane) * 8;
  const int valid = static_cast<int>(min(int64_t{8}, a.outputs - column));
  const int64_t row0 = blockIdx.x * cut.rows, end = min(row0 + cut.rows, a.rows);
  const G* __restrict__ const grad = static_cast<const G*>(a.grad_y) + column;
  float sum[8] = {};
  if (valid > 0) {
    constexpr bool kLong = sizeof(G) == 4, kExact = kSlopes == Slopes::kFloats;
    constexpr int kBatch = !kWhole ? 2 : kLong && kExact ? 3 : kLong || kExact ? 4 : 6;
    for (int64_t m0 = row0 + first; m0 < end; m0 += kBatch * step) {
      Pack<G, 8> g[kBatch];
      uint4 codes[kBatch];
      float exact[kBatch][8];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int64_t m = min(m0 + i * step, end - 1);
        if constexpr (kWhole) {
          if constexpr (sizeof(G) == 4) {
            reinterpret_cast<uint4*>(&g[i])[0] = __ldcs(reinterpret_cast<const uint4*>(grad + m * a.outputs));
            reinterpret_cast<uint4*>(&g[i])[1] = __ldcs(reinterpret_cast<const uint4*>(grad + m * a.outputs) + 1);
          } else {
            reinterpret_cast<uint4&>(g[i]) = __ldcs(reinterpret_cast<const uint4*>(grad + m * a.outputs));
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            g[i].v[k] = k < valid ? grad[m * a.outputs + k] : from_float<G>(0.0f);
        }
        if constexpr (kSlopes == Slopes::kCodes)
          codes[i] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.slope) +
                                                           m * stride + column));
        if constexpr (kSlopes == Slopes::kFloats)
          load_row<true>(static_cast<const float*>(a.slope) + m * stride + column, 8, exact[i]);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int64_t m = m0 + i * step;
        if (m >= end) break;
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = to_float(g[i].v[k]);
        if constexpr (kSlopes == Slopes::kCodes) {
          const uint32_t words[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float slope = slope_value(__byte_perm(words[k >> 1], 0, k & 1 ? 0x4432 : 0x4410));
            x[k] = kWhole || k < valid ? x[k] * slope : 0.0f;
          }
        }
        if constexpr (kSlopes == Slopes::kFloats)
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = kWhole || k < valid ? x[k] * exact[i][k] : 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] += x[k];
        if (dz) store_pack<8>(dz + m * stride + column, x);
      }
    }
  }
  if (!sums) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) joined[threadIdx.x][k] = sum[k];
  __syncthreads();
  for (int i = threadIdx.x; i < cut.lanes * 8; i += kSlopeThreads) {
    const int64_t c = blockIdx.y * int64_t{cut.lanes} * 8 + i;
    if (c >= a.outputs) break;
    float total = 0.0f;
    for (int r = 0; r < step; ++r) total += joined[r * cut.lanes + i / 8][i % 8];
    sums[blockIdx.x * int64_t{a.outputs} + c] = total;
  }
}

// What is left of the weight's and the bias's gradients, one launch: the splits' sums in
// order, rounded to the result's type, four columns a thread; and, in the first blocks,
// the strips' sums of 8 columns, in one order: 32 groups of strips, then the groups. A
// launch and the strips' latency, 5 us (256 x 1024 of 18 splits).
constexpr int kJoinThreads = 256, kBiasColumns = 8;
struct Joins {
  // the bias's: blocks, and strips of `outputs` sums
  int32_t bias_blocks, outputs, bias_dtype;
  int64_t strips;
  const float* sums;
  void* bias;
  // the weight's
  int32_t splits, rows, columns;
  int64_t part_size;
  const float* parts;
  void* weight;
};
template <class T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(Joins j) {
  chain_wait();
  if (blockIdx.x < j.bias_blocks) {
    __shared__ float groups[32][9];
    const int column = blockIdx.x * kBiasColumns + (threadIdx.x & 7), group = threadIdx.x >> 3;
    float sum = 0.0f;
    if (column < j.outputs)
#pragma unroll 8
      for (int64_t i = group; i < j.strips; i += 32) sum += j.sums[i * j.outputs + column];
    groups[group][threadIdx.x & 7] = sum;
    __syncthreads();
    if (group == 0 && column < j.outputs) {
      for (int g = 1; g < 32; ++g) sum += groups[g][threadIdx.x & 7];
      write_as(j.bias, j.bias_dtype, column, sum);
    }
    return;
  }
  const int64_t at = (blockIdx.x - j.bias_blocks) * int64_t{kJoinThreads} + threadIdx.x;
  const int words = (j.columns + 3) / 4;
  if (at >= int64_t{j.rows} * words) return;
  float4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int i = 0; i < j.splits; ++i) {
    const float4 x = reinterpret_cast<const float4*>(j.parts + i * j.part_size)[at];
    sum.x += x.x;
    sum.y += x.y;
    sum.z += x.z;
    sum.w += x.w;
  }
  const int column = static_cast<int>(at % words) * 4;
  T* const to = static_cast<T*>(j.weight) + at / words * j.columns + column;
  const float x[4] = {sum.x, sum.y, sum.z, sum.w};
  if (j.columns % 4 == 0) {
    store_pack<4>(to, x);
  } else {
    for (int k = 0; k < 4 && column + k < j.columns; ++k) to[k] = from_float<T>(x[k]);
  }
}

// Rows of 16-bit elements at any 2-byte address, to rows of whole 16-byte words: a
// word a thread, from the four or five 4-byte words that its elements lie in. 500,000 rows
// of 59: 25 us for 123 MB, 4.9 TB/s.
__global__ void __launch_bounds__(256)
    align_kernel(int64_t rows, int channels, const uint16_t* __restrict__ from, int64_t from_stride,
                 uint4* __restrict__ to, int words) {
  chain_wait();
  const int64_t total = rows * words;
  for (int64_t i = blockIdx.x * int64_t{256} + threadIdx.x; i < total; i += int64_t{gridDim.x} * 256) {
    const int64_t row = i / words;
    const int channel = static_cast<int>(i - row * words) * 8;
    const int valid = min(8, channels - channel);
    const uint16_t* const p = from + row * from_stride + channel;
    const bool odd = (reinterpret_cast<uintptr_t>(p) & 2) != 0;
    const uint32_t* const w = reinterpret_cast<const uint32_t*>(p - odd);
    const int last = valid + odd;  // elements from w on
    uint32_t x[5];
#pragma unroll
    for (int k = 0; k < 5; ++k) x[k] = 2 * k < last ? w[k] : 0;
    uint32_t y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      y[k] = odd ? __byte_perm(x[k], x[k + 1], 0x5432) : x[k];
      if (2 * k + 1 >= valid) y[k] = 2 * k < valid ? y[k] & 0xffffu : 0;
    }
    to[i] = make_uint4(y[0], y[1], y[2], y[3]);
  }
}

// --------------------------------------------------------------------- host

int32_t check_args(const gs_linear_args& a) {
  if (a.rows < 0 || a.rows > GS_MAX_SEQUENCE_TOKENS || a.inputs < 1 ||
      a.inputs > GS_MAX_LINEAR_FEATURES || a.outputs < 1 || a.outputs > GS_MAX_LINEAR_FEATURES ||
      a.activation < GS_IDENTITY || a.activation > GS_SILU)
    return GS_ERR_INVALID_ARGUMENT;
  if (a.dtype != GS_BFLOAT16 && a.dtype != GS_FLOAT16) return GS_ERR_UNSUPPORTED;
  for (int32_t t : {a.bias_dtype, a.residual_dtype})
    if (t != a.dtype && t != GS_FLOAT32) return GS_ERR_INVALID_ARGUMENT;
  if (!a.weight || (a.rows > 0 && !a.x)) return GS_ERR_INVALID_ARGUMENT;
  if (a.x_stride < 0 || a.weight_stride < a.inputs) return GS_ERR_INVALID_ARGUMENT;
  if (!is_aligned(a.x, 2) || !is_aligned(a.weight, 16) || a.weight_stride % 8)
    return GS_ERR_MISALIGNED;
  return GS_OK;
}

// Whether TMA takes x.
bool aligned_x(const gs_linear_args& a) {
  return is_aligned(a.x, 16) && a.x_stride % 8 == 0 && a.x_stride >= a.inputs;
}

template <class F>
int32_t with_sixteen_bit(int32_t dtype, F&& f) {
  return dtype == GS_BFLOAT16 ? f(__nv_bfloat16{}) : f(__half{});
}

int64_t slope_stride(const gs_linear_args& a) { return round_up(a.outputs, 8); }

// The backward's workspace: dz (where grad_y cannot be read in its place, and more than the
// bias's gradient is wanted), the strips' sums of dz, the splits' sums of dz^T x (where there
// are several splits: one writes the gradient itself).
struct BackwardPlan {
  bool own_dz;
  Strips strips;
  ProductTile weight_tile, x_tile;
  Plan weight, x;
  uint64_t dz, sums, parts, size;  // byte offsets, and the whole
};

Strips strips_of(int64_t rows, int64_t columns) {
  Strips s = {};
  s.lanes = 1;
  while (s.lanes < 32 && s.lanes * 8 < columns) s.lanes *= 2;
  s.column_blocks = static_cast<int32_t>(ceil_div(columns, s.lanes * 8));
  const int64_t step = kSlopeThreads / s.lanes;
  const int64_t strips = ceil_div(kSlopeBlocks, s.column_blocks);
  s.rows = round_up(ceil_div(rows, strips), 4 * step);  // four rows a thread at least
  s.count = ceil_div(rows, s.rows);
  return s;
}

BackwardPlan backward_plan(const gs_linear_args& a) {
  BackwardPlan p = {};
  if (a.rows == 0) return p;
  p.own_dz = a.activation != GS_IDENTITY || a.residual_dtype != a.dtype || a.outputs % 8 != 0;
  p.strips = strips_of(a.rows, a.outputs);
  // The weight's gradient has few tiles and a long contraction: split so that the items
  // are about one a multiprocessor.
  p.weight_tile = {256, a.rows >= kPairDepth && a.outputs > kRows && a.inputs > 128};
  while (p.weight_tile.columns > 64 && p.weight_tile.columns / 2 >= a.inputs)
    p.weight_tile.columns /= 2;
  const int64_t tiles = int64_t{ceil_div(a.outputs, p.weight_tile.rows())} *
                        ceil_div(a.inputs, p.weight_tile.columns);
  const int64_t splits = p.weight_tile.workers() / tiles;
  p.weight = plan_of(a.outputs, a.inputs, a.rows, p.weight_tile,
                     static_cast<int>(splits < 1 ? 1 : splits));
  p.x_tile = tile_of(a.rows, a.inputs, a.outputs, 64);
  p.x = plan_of(a.rows, a.inputs, a.outputs, p.x_tile, 1);
  uint64_t at = 0;
  const auto take = [&](uint64_t bytes) {
    const uint64_t from = at;
    at += (bytes + 255) / 256 * 256;
    return from;
  };
  const bool bias_only = a.grad_bias && !a.grad_x && !a.grad_weight;
  p.dz = take(p.own_dz && !bias_only ? static_cast<uint64_t>(a.rows) * slope_stride(a) * 2 : 0);
  p.sums = take(static_cast<uint64_t>(p.strips.count) * a.outputs * 4);
  p.parts = take(p.weight.splits == 1 ? 0
                                      : static_cast<uint64_t>(p.weight.splits) *
                                            p.weight.split_rows * round_up(a.inputs, 4) * 4);
  p.size = at;
  return p;
}

}  // namespace

uint64_t linear_workspace_size(const gs_linear_args& a) {
  return check_args(a) == GS_OK ? backward_plan(a).size : 0;
}

int32_t launch_align_rows(int64_t rows, int64_t channels, const void* from, int64_t from_stride,
                          void* to, cudaStream_t stream) {
  if (rows < 0 || rows > GS_MAX_SEQUENCE_TOKENS || channels < 1 ||
      channels > GS_MAX_LINEAR_FEATURES || from_stride < 0)
    return GS_ERR_INVALID_ARGUMENT;
  if (rows == 0) return GS_OK;
  if (!from || !to) return GS_ERR_INVALID_ARGUMENT;
  if (!is_aligned(from, 2) || !is_aligned(to, 16)) return GS_ERR_MISALIGNED;
  const int words = static_cast<int>((channels + 7) / 8);
  const int64_t blocks = (rows * words + 255) / 256;
  launch_chained(align_kernel, static_cast<unsigned>(blocks < 16 * kSmCount ? blocks : 16 * kSmCount),
                 256, stream, rows, static_cast<int>(channels), static_cast<const uint16_t*>(from),
                 from_stride, static_cast<uint4*>(to), words);
  return check_launch();
}

int32_t linear_status(cudaStream_t stream) { return take_timeout(g_timeout, stream); }

int32_t launch_linear(const gs_linear_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (a.rows == 0) return GS_OK;
  if (!a.y) return GS_ERR_INVALID_ARGUMENT;
  const size_t element = element_size(a.residual_dtype);
  if (!is_aligned(a.y, element) || !is_aligned(a.residual, element) ||
      !is_aligned(a.bias, element_size(a.bias_dtype)) || !is_aligned(a.slope, 16))
    return GS_ERR_MISALIGNED;
  Epilogue e = {};
  e.rows = a.rows;
  e.columns = a.outputs;
  e.out = a.y;
  e.out_stride = a.outputs;
  e.out_dtype = a.residual_dtype;
  e.activation = a.activation;
  e.bias = a.bias;
  e.bias_dtype = a.bias_dtype;
  e.residual = a.residual;
  e.residual_stride = a.residual_stride;
  e.slope = a.activation == GS_IDENTITY ? nullptr : a.slope;
  e.slope_stride = slope_stride(a);
  e.slope_float = a.slope_float != 0;
  e.tiled = tma_rows(a.y, a.outputs, a.residual_dtype, a.outputs) &&
            (!a.residual ||
             tma_rows(a.residual, a.residual_stride, a.residual_dtype, a.outputs));
  const bool gather = !aligned_x(a);
  const ProductTile tile = tile_of(a.rows, a.outputs, a.inputs, 32, !gather);
  const Plan plan = plan_of(a.rows, a.outputs, a.inputs, tile, 1);
  const Operand x = {a.x, a.rows, a.inputs, a.x_stride};
  const Operand weight = {a.weight, a.outputs, a.inputs, a.weight_stride};
  return with_sixteen_bit(a.dtype, [&](auto t) {
    using T = decltype(t);
    return gather ? run_product<T, false, false, true>(a.dtype, x, weight, plan, tile, e, stream)
                  : run_product<T, false, false>(a.dtype, x, weight, plan, tile, e, stream);
  });
}

int32_t launch_linear_backward(const gs_linear_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (a.rows > 0 && (!a.grad_y || !a.workspace || (a.activation != GS_IDENTITY && !a.slope)))
    return GS_ERR_INVALID_ARGUMENT;
  if (!aligned_x(a) || !is_aligned(a.grad_y, 16) || !is_aligned(a.slope, 16) ||
      !is_aligned(a.workspace, 256) || !is_aligned(a.grad_x, 2) || !is_aligned(a.grad_weight, 8) ||
      !is_aligned(a.grad_bias, element_size(a.bias_dtype)))
    return GS_ERR_MISALIGNED;
  const BackwardPlan p = backward_plan(a);
  if (a.workspace_size < p.size) return GS_ERR_CAPACITY;
  if (a.rows == 0) {
    if (a.grad_weight)
      GS_CUDA_TRY(cudaMemsetAsync(a.grad_weight, 0, int64_t{a.inputs} * a.outputs * 2, stream));
    if (a.grad_bias)
      GS_CUDA_TRY(cudaMemsetAsync(a.grad_bias, 0, int64_t{a.outputs} * element_size(a.bias_dtype),
                                  stream));
    return GS_OK;
  }
  unsigned char* const work = static_cast<unsigned char*>(a.workspace);
  float* const sums = a.grad_bias ? reinterpret_cast<float*>(work + p.sums) : nullptr;
  float* const parts = reinterpret_cast<float*>(work + p.parts);
  void* const dz = p.own_dz ? work + p.dz : const_cast<void*>(a.grad_y);
  const bool products = a.grad_x || a.grad_weight;
  const Operand dz_operand = {dz, a.rows, a.outputs, p.own_dz ? slope_stride(a) : a.outputs};
  return with_sixteen_bit(a.dtype, [&](auto t) {
    using T = decltype(t);
    if ((p.own_dz && products) || sums) {
      const dim3 grid(static_cast<unsigned>(p.strips.count), p.strips.column_blocks);
      T* const to = p.own_dz && products ? static_cast<T*>(dz) : nullptr;
      const auto launch = [&](auto g, auto slopes, auto whole) {
        using G = decltype(g);
        launch_chained(slope_kernel<T, G, decltype(slopes)::value, decltype(whole)::value>, grid,
                       kSlopeThreads, stream, a, p.strips, slope_stride(a), to, sums);
      };
      const auto with_whole = [&](auto g, auto slopes) {
        if (a.outputs % 8 == 0) launch(g, slopes, std::true_type{});
        else launch(g, slopes, std::false_type{});
      };
      const auto with_slopes = [&](auto g) {
        if (a.activation == GS_IDENTITY)
          with_whole(g, std::integral_constant<Slopes, Slopes::kNone>{});
        else if (a.slope_float)
          with_whole(g, std::integral_constant<Slopes, Slopes::kFloats>{});
        else
          with_whole(g, std::integral_constant<Slopes, Slopes::kCodes>{});
      };
      if (a.residual_dtype == GS_FLOAT32) with_slopes(float{});
      else with_slopes(T{});
      GS_TRY(check_launch());
    }
    Joins j = {};
    if (a.grad_bias) {
      j.bias_blocks = ceil_div(a.outputs, kBiasColumns);
      j.outputs = a.outputs;
      j.bias_dtype = a.bias_dtype;
      j.strips = p.strips.count;
      j.sums = sums;
      j.bias = a.grad_bias;
    }
    if (a.grad_x) {
      Epilogue e = {};
      e.rows = a.rows;
      e.columns = a.inputs;
      e.out = a.grad_x;
      e.out_stride = a.inputs;
      e.out_dtype = a.dtype;
      e.tiled = tma_rows(a.grad_x, a.inputs, a.dtype, a.inputs);
      GS_TRY((run_product<T, false, true>(a.dtype, dz_operand,
                                          {a.weight, a.outputs, a.inputs, a.weight_stride}, p.x,
                                          p.x_tile, e, stream)));
    }
    if (a.grad_weight) {
      Epilogue e = {};
      const bool whole = p.weight.splits == 1;  // no sums to join
      e.rows = a.outputs;
      e.columns = a.inputs;
      e.out = whole ? a.grad_weight : parts;
      e.out_stride = whole ? a.inputs : round_up(a.inputs, 4);
      e.out_dtype = whole ? a.dtype : GS_FLOAT32;
      e.tiled = tma_rows(e.out, e.out_stride, e.out_dtype, a.inputs);
      GS_TRY((run_product<T, true, true>(a.dtype, dz_operand,
                                         {a.x, a.rows, a.inputs, a.x_stride}, p.weight, p.weight_tile,
                                         e, stream)));
      if (!whole) {
        j.splits = p.weight.splits;
        j.rows = a.outputs;
        j.columns = a.inputs;
        j.part_size = p.weight.split_rows * round_up(a.inputs, 4);
        j.parts = parts;
        j.weight = a.grad_weight;
      }
    }
    const int64_t words = int64_t{j.rows} * ceil_div(j.columns, 4);
    if (const unsigned blocks = j.bias_blocks + ceil_div(words, kJoinThreads)) {
      launch_chained(join_kernel<T>, blocks, kJoinThreads, stream, j);
      GS_TRY(check_launch());
    }
    return static_cast<int32_t>(GS_OK);
  });
}

}  // namespace gs
