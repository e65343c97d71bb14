// Attention in a sliding window with a few first tokens that stay visible, over
// a packed batch of sequences; forward, backward, and one new token against a
// cache.
//
// Query i of a sequence of n tokens sees key j if the key is valid, j <= i +
// right, and j >= i - left or j < first. With s_ij = scale q_i . k_j,
//
//   p_ij = exp(s_ij - L_i),  L_i = log sum_j exp(s_ij),  o_i = sum_j p_ij v_j
//
// over the keys it sees, and o_i = 0, L_i = -inf where it sees none. Backward,
// with g_i the gradient of o_i and D_i = g_i . o_i:
//
//   e_ij = p_ij (g_i . v_j - D_i)
//   dq_i = scale sum_j e_ij k_j,  dk_j = scale sum_i e_ij q_i,  dv_j = sum_i p_ij g_i
//
// where a key's sums also run over the query heads that share it. Scores,
// exponentials, sums and accumulators are float; p and e are rounded to the inputs'
// type for their products, as the tensor cores take them, and D comes from the rounded
// outputs. Keys that no query sees, and queries that see none, never reach a sum, so
// what they hold (infinities, NaN) does not matter.

#include <algorithm>
#include <cmath>

#include "tensorcore.cuh"

namespace gs {

int32_t launch_window_attention(const gs_window_attention_args& a, cudaStream_t stream);
int32_t launch_window_attention_backward(const gs_window_attention_args& a, cudaStream_t stream);
int32_t launch_window_attention_step(const gs_window_attention_step_args& a, cudaStream_t stream);
int32_t window_attention_status(cudaStream_t stream);
uint64_t window_attention_workspace_size(const gs_window_attention_args& a);

namespace {

constexpr int kTile = GS_SEQUENCE_TILE;  // queries (or keys) of a block
constexpr int kMaxDim = 128;

// -------------------------------------------------- whole sequences, forward
//
// One block: two tiles of 128 queries of one head, walked over the tiles of
// kKeys keys that they see: first the tiles of first tokens that lie before the
// block's window, then the window. A group of four warps holds a tile of
// queries, one a thread; a ninth warp loads, a tenth issues the products.
//
//   scores  S = Q K^T            tensor memory, 128 x kKeys floats a group
//   P = exp2(S scale log2 e - m) each thread its row; 16 bits, over S
//   O (+)= P V                   tensor memory, 128 x dim floats a group
//
// While one group takes its exponentials, the tensor cores work for the other,
// and both read the same keys and values. m is the row's running maximum, but
// moves only when it has grown by more than 2^8: until then P stays at most
// 2^8 and O need not be rescaled.
//
// What bounds it: 16 exponentials a clock and multiprocessor at 64 channels (a
// 128 x 128 tile takes 1024 clocks of them, 512 of products), both at 128
// (1024 each); then the chain product, exponentials, product of a step, which
// two groups cover only in part. Two blocks a multiprocessor at 64 channels.
// Measured: 500,000 tokens, 4 heads of 64, 1041 keys seen: 990 us, 540 TFLOP/s,
// the exponentials' pipe 58% and the tensor cores 45% of the time busy; 131,072
// tokens, 8 heads of 128, 1029 keys: 822 us, 650 TFLOP/s. A block of nine tiles
// spends a sixth of its time before the first exponential and after the last.

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.0f;  // log2 of the growth that m lets pass
// log2 of what P is stored times. float16 cuts off what is below 2^-25, which a wide
// window may have many of: it gets what its range has left above 2^kSlack.
template <class T>
constexpr float kLift = std::is_same_v<T, __half> ? 7.0f : 0.0f;

// A wait ran out (never in a working kernel): set for
// gs_window_attention_status, the block's results are not valid.
__device__ uint32_t g_timeout;

// A row's result: NaN where a wait ran out, whatever the row has seen until then, and
// `empty` where there was nothing to see.
constexpr float row_value(bool good, bool none, float value, float empty) {
  return !good ? NAN : none ? empty : value;
}
static_assert(row_value(false, true, 0.0f, 0.0f) != row_value(false, true, 0.0f, 0.0f) &&
                  row_value(false, false, 1.0f, 0.0f) != row_value(false, false, 1.0f, 0.0f) &&
                  row_value(true, true, NAN, 0.0f) == 0.0f && row_value(true, false, 1.0f, 0.0f) == 1.0f,
              "a wait that ran out shows");

// After a wait that ran out, by the warp that issues products: those that it has issued
// read shared and write tensor memory until they are complete.
__device__ __forceinline__ void drain(uint64_t* bar) {
  tc::commit(tc::elect_lane(), tc::shared_address(bar));
  tc::barrier_settle(tc::shared_address(bar));
  __syncwarp();
}

// 32 bits with those under `n` set.
__device__ __forceinline__ uint32_t below32(int n) {
  return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
}

// `x` as a position that comparisons within a sequence cannot tell from it.
__device__ __forceinline__ int position(int64_t x) {
  return static_cast<int>(max(int64_t{-1}, min(x, int64_t{INT32_MAX})));
}

// First tile of sequence b.
__device__ __forceinline__ int64_t first_tile_of(const gs_window_attention_args& a, int64_t b) {
  return a.tile_starts ? __ldg(a.tile_starts + b) : (b ? a.num_tiles : 0);
}
// Runs of `length` tiles: sequence b's take the numbers from floor(first tile of
// b / length) + b on, which no two sequences share (some stay empty).
__device__ __forceinline__ int64_t run_of(int64_t first_tile, int64_t sequence, int length) {
  return first_tile / length + sequence;
}
// The sequence whose runs include number `run`.
__device__ __forceinline__ int64_t sequence_of_run(const gs_window_attention_args& a, int64_t run,
                                                   int length) {
  int64_t b = 0, above = a.tile_starts ? a.sequences : 1;
  while (above - b > 1) {  // the last one whose runs start at or before it
    const int64_t middle = (b + above) / 2;
    if (run_of(first_tile_of(a, middle), middle, length) <= run) b = middle;
    else above = middle;
  }
  return b;
}

// Which of 32 keys from position `start` on query i sees, if those under `end`
// are valid.
__device__ __forceinline__ uint32_t window_bits(const gs_window_attention_args& a, int i,
                                                int start, int end) {
  const int high = min(position(int64_t{i} + a.right + 1), end);
  const int low = position(int64_t{i} - a.left);
  return below32(high - start) & (~below32(low - start) | below32(a.first - start));
}

// Zeroes the rows of a loaded tile (kRows rows, kDim channels) whose bit is not
// set, so that what they hold (another sequence's rows, NaN of invalid keys)
// cannot reach a sum through a weight of zero.
template <int kDim, int kRows, int kThreadCount>
__device__ __forceinline__ void zero_rows(unsigned char* tile, const uint32_t (&keep)[kRows / 32],
                                          int tid) {
  constexpr int kPerRow = kThreadCount / kRows;  // threads of a row
  constexpr int kWordsEach = 8 / kPerRow;
  const int row = tid / kPerRow;
  uint32_t bits = keep[0];
#pragma unroll
  for (int c = 1; c < kRows / 32; ++c)
    if (row >= 32 * c) bits = keep[c];
  if (bits >> (row & 31) & 1) return;
#pragma unroll
  for (int box = 0; box < kDim / 64; ++box)
#pragma unroll
    for (int w = 0; w < kWordsEach; ++w)
      *reinterpret_cast<uint4*>(tile + box * (kRows * 128) + row * 128 +
                                ((tid % kPerRow) * kWordsEach + w) * 16) = make_uint4(0, 0, 0, 0);
}

// A block's results go through shared memory, where a thread puts its row's words
// and from where rows are written side by side (2 to 4% of the kernels' time, next
// to sixteen bytes, half a sector, a row and instruction).
template <class T, int kDim>
__device__ __forceinline__ void put_word(unsigned char* rows, int row, int word,
                                         const float (&v)[8]) {
  store_pack<8>(reinterpret_cast<T*>(rows + row * (2 * kDim) + (word ^ (row & 7)) * 16), v);
}
// Rows `from` to `to` of the tile; row 0 of the array is at `out`.
template <class T, int kDim, int kThreadCount>
__device__ __forceinline__ void write_rows(const unsigned char* rows, T* out, int64_t stride,
                                           int from, int to, int dim, int thread) {
  constexpr int kLanes = kDim / 8;
  const int word = thread % kLanes;
  if (8 * word >= dim) return;
  constexpr int kStep = kThreadCount / kLanes, kAtOnce = kTile / kStep < 8 ? kTile / kStep : 8;
#pragma unroll
  for (int base = 0; base < kTile; base += kAtOnce * kStep) {
    uint4 x[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int row = base + k * kStep + thread / kLanes;
      x[k] = *reinterpret_cast<const uint4*>(rows + row * (2 * kDim) + (word ^ (row & 7)) * 16);
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int row = base + k * kStep + thread / kLanes;
      if (row >= from && row < to) *reinterpret_cast<uint4*>(out + row * stride + 8 * word) = x[k];
    }
  }
}

// The tiles of keys that a run of kGroups tiles of queries walks over, as
// positions in the sequence, and each group's part of them.
template <int kKeys, int kGroups>
struct KeyWalk {
  int n, i, low, head, head_tiles, tiles;
  int from[kGroups], to[kGroups], high[kGroups];  // of the window's tiles; past its last key
  __device__ __forceinline__ KeyWalk(const gs_window_attention_args& a, const Tile& tile) {
    n = tile.end - tile.begin;
    i = tile.start - tile.begin;
    low = max(0, position(int64_t{i} - a.left));
    head = min(a.first, low);
    head_tiles = (head + kKeys - 1) / kKeys;
    tiles = head_tiles;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int first = i + g * kTile, last = min(first + kTile, n) - 1;
      high[g] = min(position(int64_t{last} + a.right + 1), n);
      // First tokens that reach into the window's tiles are seen by every group.
      from[g] = a.first > low ? 0 : (max(low, position(int64_t{first} - a.left)) - low) / kKeys;
      to[g] = first < n ? (high[g] - low + kKeys - 1) / kKeys : 0;
      if (first < n) tiles = head_tiles + to[g];
    }
  }
  __device__ __forceinline__ int start(int t) const {
    return t < head_tiles ? t * kKeys : low + (t - head_tiles) * kKeys;
  }
  // Keys of tile t that may be seen at all: those under this position.
  __device__ __forceinline__ int end(int t) const { return t < head_tiles ? head : n; }
  // How many tiles a group walks over, and the number of its step s.
  __device__ __forceinline__ int steps(int g) const {
    return i + g * kTile < n ? head_tiles + to[g] - from[g] : 0;
  }
  __device__ __forceinline__ int tile_of(int g, int s) const {
    return s < head_tiles ? s : s + from[g];
  }
  // Whether group g walks over tile t.
  __device__ __forceinline__ bool walks(int g, int t) const {
    return i + g * kTile < n &&
           (t < head_tiles || (t - head_tiles >= from[g] && t - head_tiles < to[g]));
  }
  // Whether group g is the last to read tile t: at the same step the second of
  // two groups is, else the first, which is behind in the window.
  __device__ __forceinline__ bool last_reader(int g, int t) const {
    const int other = 1 - g;
    return !walks(other, t) || (t < head_tiles || from[1] == 0 ? g == 1 : g == 0);
  }
  // How many sets of 32 keys of tile t group g needs.
  __device__ __forceinline__ int sets(int g, int t) const {
    const int keys = min(kKeys, (t < head_tiles ? head : high[g]) - start(t));
    return (keys + 31) / 32;
  }
};

template <int kDim>
struct ForwardShape {
  // At 64 channels two blocks share a multiprocessor, 16 warps for the
  // exponentials; at 128 one block fills it.
  static constexpr int kKeys = kDim == 64 ? 64 : 128;
  static constexpr int kBlocks = kDim == 64 ? 2 : 1;
  static constexpr int kColumns = kDim == 64 ? 256 : 512;
  static constexpr int kGroupColumns = kKeys + kDim;  // S, then O
  // At 128 a row of S does not fit a thread's 168 registers: the groups take 56 of
  // each thread of a third group of warps (two of them idle), 2% faster.
  static constexpr int kThreads = 2 * kTile + (kDim == 64 ? 64 : 128);
  static constexpr int kLaunched = 168, kWide = 224, kNarrow = 56;
  static_assert(2 * kWide + kNarrow <= 3 * kLaunched, "more would be waited for without end");
};

template <int kDim>
struct ForwardShared {
  // The second group is kTile / kKeys tiles ahead of the first.
  static constexpr int kStages = kDim == 64 ? 4 : 2;
  static constexpr int kKeys = ForwardShape<kDim>::kKeys;
  static constexpr int kQueryBytes = kTile * kDim * 2, kTileBytes = kKeys * kDim * 2;
  alignas(1024) unsigned char q[2][kQueryBytes];
  unsigned char k[kStages][kTileBytes];
  unsigned char v[kStages][kTileBytes];
  uint64_t q_full[2], k_full[kStages], v_full[kStages];  // loads
  uint64_t k_empty[kStages], v_empty[kStages];  // both groups' products with a tile are complete
  uint64_t scores[2];                           // S of a group's step is complete
  uint64_t weights[2];                          // P is written (128 arrivals)
  uint64_t summed[2];                           // all of a group's sums are complete
  uint64_t drained;                             // a wait ran out: the products that were issued
  uint32_t tensor;
};

template <class T, int kDim>
__global__ void __launch_bounds__(ForwardShape<kDim>::kThreads, ForwardShape<kDim>::kBlocks)
    attention_kernel(gs_window_attention_args a, const __grid_constant__ CUtensorMap q_map,
                     const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap v_map) {
  using namespace tc;
  using Shape = ForwardShape<kDim>;
  using Shared = ForwardShared<kDim>;
  constexpr int kKeys = Shape::kKeys, kStages = Shared::kStages, kSets = kKeys / 32;
  extern __shared__ __align__(1024) unsigned char shared_bytes[];
  Shared& s = *reinterpret_cast<Shared*>(shared_bytes);
  chain_wait();
  const int warp = threadIdx.x >> 5;
  const int head = blockIdx.x % a.heads, kv_head = head / (a.heads / a.kv_heads);
  const int64_t run = blockIdx.x / a.heads;
  const int64_t sequence = sequence_of_run(a, run, 2);
  const int64_t tile0 = first_tile_of(a, sequence);
  const int64_t index = tile0 + 2 * (run - run_of(tile0, sequence, 2));
  if (index >= first_tile_of(a, sequence + 1)) return;
  const Tile tile = tile_at(a.tiles, index, static_cast<int32_t>(a.tokens), kTile);
  const KeyWalk<kKeys, 2> walk(a, tile);
  const auto load = [&](unsigned char* dst, uint64_t* bar, const CUtensorMap* map, int h, int row,
                        int rows) {
    const uint32_t b = shared_address(bar), d = shared_address(dst);
    barrier_expect(b, rows * kDim * 2);
    for (int x = 0; x < kDim / 64; ++x) load_box(d + x * rows * 128, map, 64 * x, h, row, b);
  };
  if (threadIdx.x == 8 * 32) {
    for (int g = 0; g < 2; ++g) {
      barrier_init(shared_address(&s.q_full[g]), 1);
      barrier_init(shared_address(&s.scores[g]), 1);
      barrier_init(shared_address(&s.weights[g]), kTile);
      barrier_init(shared_address(&s.summed[g]), 1);
    }
    barrier_init(shared_address(&s.drained), 1);
    for (int i = 0; i < kStages; ++i) {
      barrier_init(shared_address(&s.k_full[i]), 1);
      barrier_init(shared_address(&s.v_full[i]), 1);
      barrier_init(shared_address(&s.k_empty[i]), 1);
      barrier_init(shared_address(&s.v_empty[i]), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
    // The first loads do not wait for the others to be ready.
    load(s.q[0], &s.q_full[0], &q_map, head, tile.start, kTile);
    load(s.k[0], &s.k_full[0], &k_map, kv_head, tile.begin + walk.start(0), kKeys);
    if (walk.steps(1) > 0)
      load(s.q[1], &s.q_full[1], &q_map, head, tile.start + kTile, kTile);
    load(s.v[0], &s.v_full[0], &v_map, kv_head, tile.begin + walk.start(0), kKeys);
  }
  if (warp == 9) tensor_alloc<Shape::kColumns>(shared_address(&s.tensor));
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tensor = s.tensor;
  bool good = true;

  if constexpr (kDim == 128)
    if (warp >= 8) registers_down<Shape::kNarrow>();
  if (warp == 8) {  // loads
    if ((threadIdx.x & 31) == 0) {
      for (int t = 1; t < walk.tiles && good; ++t) {
        const int stage = t % kStages, turn = t / kStages;
        if (turn > 0) good = barrier_wait(shared_address(&s.k_empty[stage]), (turn - 1) & 1);
        if (!good) break;
        load(s.k[stage], &s.k_full[stage], &k_map, kv_head, tile.begin + walk.start(t), kKeys);
        if (turn > 0) good = barrier_wait(shared_address(&s.v_empty[stage]), (turn - 1) & 1);
        if (!good) break;
        load(s.v[stage], &s.v_full[stage], &v_map, kv_head, tile.begin + walk.start(t), kKeys);
      }
    }
    __syncwarp();
  } else if (warp == 9) {  // products
    const int lane = threadIdx.x & 31;
    const uint32_t elected = elect_lane();
    const int dim_steps = (a.dim + 15) / 16;
    const uint32_t sum_kind = product_kind<T>(dim_steps * 16, true);
    const uint32_t score_kind = product_kind<T>(0, false);
    const uint32_t q = channels_word<kTile>(shared_address(s.q[0]));
    const uint32_t k = channels_word<kKeys>(shared_address(s.k[0]));
    const uint32_t v = rows_word<kKeys>(shared_address(s.v[0]));
    const int steps[2] = {walk.steps(0), walk.steps(1)};
    // One thread's arithmetic on what a step needs would take longer than the
    // step's products, so the lanes do it for 32 steps at a time. Eight bits of a
    // plan are for the values of a step, eight for the keys of the next one:
    // stage, parity of its load, whether to wait for the load (the tile's first
    // reader) and to release it (its last reader); then the sets of both.
    const auto tile_plan = [&](int g, int t) {
      const bool last = walk.last_reader(g, t), first = !last || !walk.walks(1 - g, t);
      return static_cast<uint32_t>(t % kStages | ((t / kStages) & 1) << 4 | first << 5 | last << 6);
    };
    const auto plan_of = [&](int g, int step) {
      uint32_t plan = 0;
      if (step >= 0 && step < steps[g]) {
        const int t = walk.tile_of(g, step);
        plan = tile_plan(g, t) | static_cast<uint32_t>(walk.sets(g, t)) << 16;
      }
      if (step + 1 < steps[g]) {
        const int t = walk.tile_of(g, step + 1);
        plan |= tile_plan(g, t) << 8 | static_cast<uint32_t>(walk.sets(g, t)) << 20;
      }
      return plan;
    };
    const auto wait_for = [&](uint64_t* bars, uint32_t plan) {
      if (plan & 32)
        good = good && barrier_wait_warp(shared_address(&bars[plan & 15]), plan >> 4 & 1);
    };
    const auto release = [&](uint64_t* bars, uint32_t plan) {
      if (plan & 64) commit(elected, shared_address(&bars[plan & 15]));
    };
    const auto issue_scores = [&](auto number, uint32_t plan) {
      constexpr int g = decltype(number)::value;
      const uint32_t keys = k + (plan >> 8 & 15) * (Shared::kTileBytes >> 4);
      const uint32_t kind = score_kind | (plan >> 20 & 15) << 19;  // 32 columns a set
#pragma unroll
      for (int i = 0; i < kDim / 16; ++i)
        if (i < dim_steps)
          multiply(elected, tensor + g * Shape::kGroupColumns,
                   q + g * (Shared::kQueryBytes >> 4) + channels_step<kTile>(i),
                   keys + channels_step<kKeys>(i), kind, i > 0);
      commit(elected, shared_address(&s.scores[g]));
    };
    const auto run_step = [&](auto number, int step, uint32_t plan) {
      constexpr int g = decltype(number)::value;
      if (step >= steps[g]) return;
      const bool more = step + 1 < steps[g];
      wait_for(s.v_full, plan);
      if (more) wait_for(s.k_full, plan >> 8);
      good = good && barrier_wait_warp(shared_address(&s.weights[g]), step & 1);
      if (good) {
        fence_after_sync();
        constexpr uint32_t column = g * Shape::kGroupColumns;
        const uint32_t values = v + (plan & 15) * (Shared::kTileBytes >> 4);
        const uint32_t count = plan >> 15 & 30;  // two steps of 16 keys a set
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i)
          if (i < count)
            multiply_tensor(elected, tensor + column + kKeys, tensor + column + 8 * i,
                            values + rows_step(i), sum_kind, step > 0 || i > 0);
        if (more) issue_scores(number, plan);  // in order behind the product that reads P
        else commit(elected, shared_address(&s.summed[g]));
        release(s.v_empty, plan);
        if (more) release(s.k_empty, plan >> 8);
      }
    };
    const auto start = [&](auto number) {
      constexpr int g = decltype(number)::value;
      if (steps[g] == 0) return;
      const uint32_t plan = plan_of(g, -1);
      wait_for(s.k_full, plan >> 8);
      good = good && barrier_wait_warp(shared_address(&s.q_full[g]), 0);
      if (good) {
        issue_scores(number, plan);
        release(s.k_empty, plan >> 8);
      }
    };
    using First = std::integral_constant<int, 0>;
    using Second = std::integral_constant<int, 1>;
    start(First{});
    start(Second{});
    const int most = max(steps[0], steps[1]);
    for (int base = 0; base < most && good; base += 32) {
      const uint32_t first = plan_of(0, base + lane), second = plan_of(1, base + lane);
      for (int step = base; step < min(base + 32, most) && good; ++step) {
        run_step(First{}, step, __shfl_sync(0xffffffffu, first, step - base));
        run_step(Second{}, step, __shfl_sync(0xffffffffu, second, step - base));
      }
    }
    __syncwarp();
  } else if (warp < 8) {
    if constexpr (kDim == 128) registers_up<Shape::kWide>();
    const int group = warp >> 2, row = threadIdx.x & (kTile - 1);
    const uint32_t scores = tensor + group * Shape::kGroupColumns +
                            (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t sums = scores + kKeys;
    const int i_first = walk.i + group * kTile, i = i_first + row;
    const float scale = a.scale * kLog2e;
    float top = -INFINITY, sum = 0.0f;
    const int steps = walk.steps(group);
    // Every query of the group sees every valid key of a tile that lies from
    // `from` (or under `first`) to `to`.
    const int from = position(int64_t{i_first} + kTile - 1 - a.left);
    const int to = min(position(int64_t{i_first} + a.right + 1), walk.n);
    for (int step = 0; step < steps; ++step) {
      const int t = walk.tile_of(group, step), start = walk.start(t), end = walk.end(t);
      bool whole = t < walk.head_tiles
                       ? start + kKeys <= end
                       : start + kKeys <= to && (start >= from || start + kKeys <= a.first);
      bool all = whole;  // the keys are all valid
      uint32_t keep[kSets];
      if (a.valid || !whole) {
        all = true;
#pragma unroll
        for (int c = 0; c < kSets; ++c) keep[c] = below32(end - start - 32 * c);
        if (a.valid) {
          const uint8_t* at = a.valid + tile.begin;
          uint8_t valid[kSets];  // all on their way at once
#pragma unroll
          for (int c = 0; c < kSets; ++c)
            valid[c] = __ldg(at + min(start + static_cast<int>(threadIdx.x & 31) + 32 * c, end - 1));
#pragma unroll
          for (int c = 0; c < kSets; ++c) keep[c] &= __ballot_sync(0xffffffffu, valid[c] != 0);
        }
#pragma unroll
        for (int c = 0; c < kSets; ++c) all = all && keep[c] == ~0u;
        whole = whole && all;
      }
      good = good && barrier_wait_warp(shared_address(&s.scores[group]), step & 1);
      if (!good) break;
      fence_after_sync();
      // All columns, also where the products made fewer: what is not seen is
      // masked, and straight code is worth more than a few exponentials.
      float x[kSets][32];
#pragma unroll
      for (int c = 0; c < kSets; ++c) load_columns32(scores + 32 * c, x[c]);
      wait_loads();
      if (!whole) {
#pragma unroll
        for (int c = 0; c < kSets; ++c) {
          const uint32_t bits = keep[c] & window_bits(a, i, start + 32 * c, end);
          if (!__all_sync(0xffffffffu, bits == ~0u)) {
#pragma unroll
            for (int e = 0; e < 32; ++e) x[c][e] = bits >> e & 1 ? x[c][e] : -INFINITY;
          }
        }
      }
      float high[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) high[k] = fmaxf(x[0][k], x[0][k + 8]);
#pragma unroll
      for (int c = 0; c < kSets; ++c)
#pragma unroll
        for (int e = c == 0 ? 16 : 0; e < 32; e += 16)
#pragma unroll
          for (int k = 0; k < 8; ++k) high[k] = max3(high[k], x[c][e + k], x[c][e + k + 8]);
      const float next = max3(max3(high[0], high[1], high[2]), max3(high[3], high[4], high[5]),
                              fmaxf(high[6], high[7])) * scale;
      // Sums of earlier tiles are complete: this tile's S came behind them.
      const bool grow = next > top + kSlack || (top == -INFINITY && next > top);
      if (__any_sync(0xffffffffu, grow)) {
        const float shrink = grow ? exp2_approx(top - next) : 1.0f;
        if (grow) top = next;
        sum *= shrink;
        if (step > 0) {
#pragma unroll 1
          for (int c = 0; c < kDim; c += 16) {
            float o[16];
            load_columns16(sums + c, o);
            wait_loads();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= shrink;
            store_columns16(sums + c, o);
          }
        }
      }
      // Where nothing is seen yet any finite shift will do: exp2(-inf) is 0.
      const float down = top == -INFINITY ? 0.0f : kLift<T> - top;
      const float2 shift = make_float2(down, down), factor = make_float2(scale, scale);
      float2 part[2] = {};
#pragma unroll
      for (int c = 0; c < kSets; ++c) {
        uint32_t packed[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 y = fma2(make_float2(x[c][2 * e], x[c][2 * e + 1]), factor, shift);
          const float2 p = make_float2(exp2_approx(y.x), exp2_approx(y.y));
          part[e & 1] = add2(part[e & 1], p);
          packed[e] = pack2<T>(p.x, p.y);
        }
        store_columns16(scores + 16 * c, packed);
      }
      sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
      if (!all) {
        const int stage = t % kStages;
        good = barrier_wait_warp(shared_address(&s.v_full[stage]), (t / kStages) & 1);
        if (!good) break;
        zero_rows<kDim, kKeys, kTile>(s.v[stage], keep, row);
        fence_async_shared();
      }
      wait_stores();
      fence_before_sync();
      barrier_arrive(shared_address(&s.weights[group]));
    }
    if (steps > 0) {
      if (good) good = barrier_wait_warp(shared_address(&s.summed[group]), 0);
      fence_after_sync();
      const int64_t token = int64_t{tile.start} + group * kTile + row;
      const bool write = token < tile.end;
      const float inverse = 1.0f / sum;
      unsigned char* rows = s.q[group];  // the products with the queries are complete
#pragma unroll
      for (int c = 0; c < kDim; c += 32) {
        float o[32];
        load_columns32(sums + c, o);
        wait_loads();
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = row_value(good, sum == 0.0f, o[e + k] * inverse, 0.0f);
          put_word<T, kDim>(rows, row, (c + e) / 8, v);
        }
      }
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(kTile) : "memory");
      write_rows<T, kDim, kTile>(
          rows, static_cast<T*>(a.out) + ((token - row) * a.heads + head) * a.dim,
          int64_t{a.heads} * a.dim, 0, static_cast<int>(tile.end - (token - row)), a.dim, row);
      if (write && a.lse)
        a.lse[head * a.tokens + token] =
            row_value(good, sum == 0.0f, (top - kLift<T> + log2f(sum)) * kLn2, -INFINITY);
    }
  }
  fence_before_sync();
  if (__syncthreads_or(!good)) {
    if (warp == 8 && (threadIdx.x & 31) == 0) {
      atomicExch(&g_timeout, 1u);
      for (uint64_t& b : s.q_full) barrier_settle(shared_address(&b));
      for (uint64_t& b : s.k_full) barrier_settle(shared_address(&b));
      for (uint64_t& b : s.v_full) barrier_settle(shared_address(&b));
    }
    if (warp == 9) drain(&s.drained);
  }
  if (warp == 9) tensor_free<Shape::kColumns>(tensor);
}

int64_t sequences_of(const gs_window_attention_args& a) { return a.tile_starts ? a.sequences : 1; }

template <class T, int kDim>
int32_t forward(const gs_window_attention_args& a, cudaStream_t stream) {
  using Shape = ForwardShape<kDim>;
  constexpr int kKeys = Shape::kKeys;
  CUtensorMap q, k, v;
  GS_TRY(tc::encode_heads(&q, a.dtype, a.q, a.tokens, a.heads, a.dim, a.q_stride, a.q_head_stride,
                          kTile));
  GS_TRY(tc::encode_heads(&k, a.dtype, a.k, a.tokens, a.kv_heads, a.dim, a.k_stride,
                          a.k_head_stride, kKeys));
  GS_TRY(tc::encode_heads(&v, a.dtype, a.v, a.tokens, a.kv_heads, a.dim, a.v_stride,
                          a.v_head_stride, kKeys));
  constexpr size_t kShared = sizeof(ForwardShared<kDim>);
  GS_TRY((allow_shared<attention_kernel<T, kDim>>(kShared, false,
                                                  kDim == 64 ? 0 : Shape::kLaunched)));
  const int64_t blocks = (a.num_tiles / 2 + sequences_of(a)) * a.heads;
  if (blocks > INT32_MAX) return GS_ERR_CAPACITY;
  launch_chained_shared(attention_kernel<T, kDim>, static_cast<unsigned>(blocks),
                        Shape::kThreads, kShared, stream, a, q, k, v);
  return check_launch();
}

// ------------------------------------------------- whole sequences, backward
//
// Two kernels of one shape: a block holds 128 rows of two operands (queries and
// their gradients, or keys and values) and walks over tiles of the other two,
// recomputing the scores,
//
//   S = rows0 tile0^T,  G = rows1 tile1^T          (tensor memory, floats)
//   P = exp2(S scale log2 e - L),  E = P (G - D)   (16 bits)
//   queries: dQ += E tile0;   keys: dK += E tile0, dV += P tile1
//
// so that every sum has one owner and one order: no atomics, and the query
// heads that share a key-value head are summed where its keys are. Seven products
// instead of the five of a kernel that adds to dQ from many blocks.
//
// Eight warps hold half a row a thread, a ninth loads, a tenth issues the
// products. One of 128 x 128 x 16 takes 64 clocks, and one of 64 columns no fewer,
// because shared memory delivers the 128 rows no faster: hence tiles of 128 rows
// at 128 channels (64 took 8% longer). To keep the tensor cores busy, S of the next
// tile follows as soon as this one's has been read (queries) or used (keys), while
// the warps work on G, and G of the next while they work on S. Sixteen warps were
// no faster.
//
// What bounds them is a tile's chain S, P, G, E, sum, of which one block's tiles
// overlap in part. Measured: 131,072 tokens, 8 heads (4 of keys) of 128, 1029 keys
// seen: queries 1078 us (750 TFLOP/s of products, the tensor cores busy for 43%
// of the time), keys 1250 us (860 TFLOP/s, 55%).

// First tokens are seen by all later queries, so the block of their keys would
// walk the whole sequence. It walks its window like the others; the queries
// further on are cut into chunks with a block each, and a last kernel adds the
// chunks' sums in order (131,072 tokens in 8 sequences: 8 us).

template <int kDim, bool kKeyRows>
struct BackwardShape {
  // Tiles of operand 0 wait for the sums, those of operand 1 no longer than for
  // G: at 128 channels there is room for three of the one and two of the other.
  static constexpr int kStages0 = kDim == 64 ? 4 : 3, kStages1 = kDim == 64 ? 3 : 2;
  // Rows of a tile. At 64 channels exponentials bound the kernels before products
  // do: two blocks a multiprocessor with smaller tiles take turns (one block with
  // tiles of 128 rows was 9% slower).
  static constexpr int kRows = kDim == 64 ? 64 : 128, kSets = kRows / 32;
  static constexpr int kBlocks = kDim == 64 ? 2 : 1, kColumns = kDim == 64 ? 256 : 512;
  static constexpr int kBytes = kTile * kDim * 2, kTileBytes = kRows * kDim * 2;
  // Columns of tensor memory. E lies over G, and the keys' P over S; the queries
  // have room for G twice.
  static constexpr int kGrad = kRows, kGrads = kKeyRows ? 1 : 2;
  static constexpr int kSum = kGrad + kGrads * kRows;
};

template <int kDim, bool kKeyRows>
struct BackwardShared {
  using Shape = BackwardShape<kDim, kKeyRows>;
  static constexpr int kStages0 = Shape::kStages0, kStages1 = Shape::kStages1;
  alignas(1024) unsigned char rows[2][Shape::kBytes];
  unsigned char tiles0[kStages0][Shape::kTileBytes];
  unsigned char tiles1[kStages1][Shape::kTileBytes];
  union {
    float row[kStages1][2][Shape::kRows];  // keys: -L and -D of a tile's queries
    struct {                               // queries: D, the squared norm of the gradient
      float part[kTile], norm[kTile];
    };
  };
  float grow, back;  // keys: E's factor over P's, and what scales dK back
  bool none[kStages1];  // keys: some of the tile's rows see nothing, or are not the sequence's
  uint64_t rows_full, full0[kStages0], full1[kStages1];  // loads
  uint64_t empty[kStages0];                              // a tile's sums are complete
  uint64_t scores, grads[2];  // S, G of a tile are complete
  uint64_t read;     // S is read (queries), P is written (keys): 256 arrivals
  // E is written (256 arrivals). The queries' next S and G do not wait for it, so
  // a warp may be a tile ahead of another: even and odd tiles have one each.
  uint64_t weights[2];
  uint64_t done;     // all sums are complete
  uint64_t drained;  // a wait ran out: the products that were issued are complete
  uint32_t tensor;
};

constexpr int kComputeThreads = 256;
constexpr int kLoadWarp = kComputeThreads / 32, kProductWarp = kLoadWarp + 1;
constexpr int kBackwardThreads = kComputeThreads + 64;

// Where step k of 16 of a tile's weights lies: 32 columns' weights are
// written over the first of them.
__device__ __forceinline__ constexpr uint32_t weight_column(int k) {
  return (k >> 1) * 32 + (k & 1) * 8;
}

// A tile of an operand, by one thread.
template <int kDim, bool kKeyRows>
__device__ __forceinline__ void load_tile(unsigned char* dst, uint64_t* full,
                                          const CUtensorMap* map, int2 at) {
  using Shape = BackwardShape<kDim, kKeyRows>;
  const uint32_t bar = tc::shared_address(full);
  tc::barrier_expect(bar, Shape::kTileBytes);
  for (int x = 0; x < kDim / 64; ++x)
    tc::load_box(tc::shared_address(dst) + x * Shape::kRows * 128, map, 64 * x, at.x, at.y, bar);
}

// The warp that loads what backward_setup has not. `place(t)` names the head and row of tile
// t; `rows(t, lane)` loads what else a tile needs and `keep(t, stage, ...)` puts it
// to shared memory, all lanes taking part; it goes with operand 1. False: a wait ran out.
template <int kDim, bool kKeyRows, class Place, class Rows, class Keep>
__device__ __forceinline__ bool load_tiles(BackwardShared<kDim, kKeyRows>& s, int tiles,
                                           const CUtensorMap* tile_map0,
                                           const CUtensorMap* tile_map1, const Place& place,
                                           const Rows& rows, const Keep& keep) {
  using namespace tc;
  using Shape = BackwardShape<kDim, kKeyRows>;
  constexpr int kStages0 = Shape::kStages0, kStages1 = Shape::kStages1;
  const int lane = threadIdx.x & 31;
  bool good = true;
  // The tile that had the place before has been summed up.
  const auto wait_for = [&](int t) {
    if (t >= 0)
      good = good && barrier_wait_warp(shared_address(&s.empty[t % kStages0]), (t / kStages0) & 1);
  };
  auto ahead = rows(0, lane);
  for (int t = 0; t < tiles; ++t) {
    // What the first tile needs comes first: the others' boxes would hold it up.
    if (t == 1)
      good = barrier_wait_warp(shared_address(&s.rows_full), 0) &&
             barrier_wait_warp(shared_address(&s.full1[0]), 0);
    const auto values = ahead;
    if (t + 1 < tiles) ahead = rows(t + 1, lane);
    const int stage0 = t % kStages0, stage1 = t % kStages1;
    wait_for(t - kStages0);
    if (!good) break;
    const int2 at = place(t);
    if (lane == 0 && t > 0)
      load_tile<kDim, kKeyRows>(s.tiles0[stage0], &s.full0[stage0], tile_map0, at);
    __syncwarp();
    // Queries: only G read the tile that had operand 1's place before, and G of a tile
    // is complete with the sum of the tile before it. (Waiting for G itself would be
    // wrong if this warp fell two of its phases behind: their parity is the same.)
    static_assert(kKeyRows || kStages0 == kStages1 + 1, "wait_for(t - kStages0) covers it");
    if constexpr (kKeyRows) wait_for(t - kStages1);
    else if (t == kStages1) wait_for(0);
    if (!good) break;
    keep(t, stage1, lane, values);
    __syncwarp();  // lane 0 has arrived at the first tile's barrier already
    if (lane > 0)
      barrier_arrive(shared_address(&s.full1[stage1]));
    else if (t > 0)
      load_tile<kDim, kKeyRows>(s.tiles1[stage1], &s.full1[stage1], tile_map1, at);
    __syncwarp();
  }
  __syncwarp();
  return good;
}

// The warp that issues the products (one elected lane of it). `sets(t)` says how many
// sets of 32 rows tile t needs. False: a wait ran out.
template <class T, int kDim, bool kKeyRows, class Sets>
__device__ __forceinline__ bool issue_products(BackwardShared<kDim, kKeyRows>& s, int dim,
                                               int tiles, const Sets& sets) {
  using namespace tc;
  using Shape = BackwardShape<kDim, kKeyRows>;
  constexpr int kStages0 = Shape::kStages0, kStages1 = Shape::kStages1;
  constexpr int kRows = Shape::kRows;
  constexpr uint32_t kWords = Shape::kBytes >> 4, kTileWords = Shape::kTileBytes >> 4;
  const uint32_t tensor = s.tensor;
  const uint32_t elected = elect_lane();
  const int steps = (dim + 15) / 16;
  const uint32_t score_kind = product_kind<T>(0, false);
  const uint32_t sum_kind = product_kind<T>((dim + 15) / 16 * 16, true);
  const uint32_t rows = channels_word<kTile>(shared_address(s.rows[0]));
  const uint32_t tiles0 = shared_address(s.tiles0[0]), tiles1 = shared_address(s.tiles1[0]);
  // S (operand 0) or G (operand 1) of the tile in a stage.
  const auto issue_scores = [&](int operand, int stage, int count, uint32_t column,
                                uint64_t* ready) {
    const uint32_t a = rows + operand * kWords;
    const uint32_t b = channels_word<kRows>(operand ? tiles1 : tiles0) + stage * kTileWords;
    const uint32_t kind = score_kind | static_cast<uint32_t>(count) << 19;  // 32 columns a set
#pragma unroll
    for (int i = 0; i < kDim / 16; ++i)
      if (i < steps)
        multiply(elected, tensor + column, a + channels_step<kTile>(i), b + channels_step<kRows>(i), kind,
                 i > 0);
    commit(elected, shared_address(ready));
  };
  // A sum from the weights at `column` and operand `operand` of a stage.
  const auto issue_sum = [&](int operand, int stage, int count, uint32_t column, uint32_t sum,
                             bool add) {
    const uint32_t b = rows_word<kRows>(operand ? tiles1 : tiles0) + stage * kTileWords;
#pragma unroll
    for (int i = 0; i < kRows / 16; ++i)
      if (i < 2 * count)
        multiply_tensor(elected, tensor + sum, tensor + column + weight_column(i), b + rows_step(i),
                        sum_kind, add || i > 0);
  };
  bool good = barrier_wait_warp(shared_address(&s.rows_full), 0) &&
              barrier_wait_warp(shared_address(&s.full0[0]), 0) &&
              barrier_wait_warp(shared_address(&s.full1[0]), 0);
  int count = sets(0);
  if (good) {
    issue_scores(0, 0, count, 0, &s.scores);
    issue_scores(1, 0, count, Shape::kGrad, &s.grads[0]);
  }
  int stage0 = 0, stage1 = 0;  // of tile t
  int next0 = 0, parity0 = 0, next1 = 0, parity1 = 0;  // of tile t + 1
  for (int t = 0; t < tiles && good; ++t) {
    const bool more = t + 1 < tiles;
    if (++next0 == kStages0) {
      next0 = 0;
      parity0 ^= 1;
    }
    if (++next1 == kStages1) {
      next1 = 0;
      parity1 ^= 1;
    }
    const int next_count = more ? sets(t + 1) : 0;
    const uint32_t grad = Shape::kGrad + (kKeyRows ? 0 : (t & 1) * kRows);
    const uint32_t next_grad = Shape::kGrad + (kKeyRows ? 0 : ((t + 1) & 1) * kRows);
    uint64_t* next_ready = &s.grads[kKeyRows ? 0 : (t + 1) & 1];
    if (more) good = barrier_wait_warp(shared_address(&s.full0[next0]), parity0);
    if (more && !kKeyRows)
      good = good && barrier_wait_warp(shared_address(&s.full1[next1]), parity1);
    good = good && barrier_wait_warp(shared_address(&s.read), t & 1);
    if (good) {
      fence_after_sync();
      if constexpr (kKeyRows) issue_sum(1, stage1, count, 0, Shape::kSum + kDim, t > 0);
      // In order behind the sum that reads P (keys), with S read (queries).
      if (more) {
        issue_scores(0, next0, next_count, 0, &s.scores);
        // The other half of G was last read by the sum of the tile before.
        if constexpr (!kKeyRows) issue_scores(1, next1, next_count, next_grad, next_ready);
      }
    }
    if (more && kKeyRows)
      good = good && barrier_wait_warp(shared_address(&s.full1[next1]), parity1);
    good = good && barrier_wait_warp(shared_address(&s.weights[t & 1]), (t >> 1) & 1);
    if (good) {
      fence_after_sync();
      issue_sum(0, stage0, count, grad, Shape::kSum, t > 0);
      commit(elected, shared_address(more ? &s.empty[stage0] : &s.done));
      if constexpr (kKeyRows)
        if (more) issue_scores(1, next1, next_count, next_grad, next_ready);
    }
    stage0 = next0;
    stage1 = next1;
    count = next_count;
  }
  __syncwarp();
  return good;
}

// The end of a block, all threads: tensor memory is given back, after a wait that ran
// out behind what is still in flight.
template <int kDim, bool kKeyRows>
__device__ __forceinline__ void backward_end(BackwardShared<kDim, kKeyRows>& s, int warp,
                                             uint32_t tensor, bool good) {
  using namespace tc;
  fence_before_sync();
  if (__syncthreads_or(!good)) {
    if (threadIdx.x == 32 * kLoadWarp) {
      atomicExch(&g_timeout, 1u);
      barrier_settle(shared_address(&s.rows_full));
      for (uint64_t& b : s.full0) barrier_settle(shared_address(&b));
      for (uint64_t& b : s.full1) barrier_settle(shared_address(&b));
    }
    if (warp == kProductWarp) drain(&s.drained);
  }
  if (warp == kProductWarp)
    tensor_free<BackwardShape<kDim, kKeyRows>::kColumns>(tensor);
}

// Barriers and tensor memory; the block's rows and the first tile are on their way
// before the other warps are ready.
template <int kDim, bool kKeyRows>
__device__ __forceinline__ void backward_setup(BackwardShared<kDim, kKeyRows>& s, int warp,
                                               const CUtensorMap* row_map0,
                                               const CUtensorMap* row_map1, int row_head, int row,
                                               const CUtensorMap* tile_map0,
                                               const CUtensorMap* tile_map1, int2 first) {
  using namespace tc;
  using Shape = BackwardShape<kDim, kKeyRows>;
  if (threadIdx.x == 32 * kLoadWarp) {
    barrier_init(shared_address(&s.rows_full), 1);
    for (uint64_t& b : s.full0) barrier_init(shared_address(&b), 1);
    for (uint64_t& b : s.full1) barrier_init(shared_address(&b), 32);
    for (uint64_t& b : s.empty) barrier_init(shared_address(&b), 1);
    barrier_init(shared_address(&s.scores), 1);
    for (uint64_t& b : s.grads) barrier_init(shared_address(&b), 1);
    barrier_init(shared_address(&s.read), kComputeThreads);
    for (uint64_t& b : s.weights) barrier_init(shared_address(&b), kComputeThreads);
    barrier_init(shared_address(&s.done), 1);
    barrier_init(shared_address(&s.drained), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
    const uint32_t bar = shared_address(&s.rows_full);
    barrier_expect(bar, 2 * Shape::kBytes);
    for (int x = 0; x < kDim / 64; ++x)
      load_box(shared_address(s.rows[0]) + x * kTile * 128, row_map0, 64 * x, row_head, row, bar);
    load_tile<kDim, kKeyRows>(s.tiles0[0], &s.full0[0], tile_map0, first);
    for (int x = 0; x < kDim / 64; ++x)
      load_box(shared_address(s.rows[1]) + x * kTile * 128, row_map1, 64 * x, row_head, row, bar);
    load_tile<kDim, kKeyRows>(s.tiles1[0], &s.full1[0], tile_map1, first);
  }
  if (warp == kProductWarp) tensor_alloc<Shape::kColumns>(shared_address(&s.tensor));
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
}

// float16 loses bits below 2^-14, where a wide window's weights are, and ends at
// 65504, which E passes under a loss scale. So P, at most 1, is stored times 2^p (about
// the window's width), and E times 2^e, with e from what bounds it:
//
//   |E_ij| <= |G_ij - D_i| <= |g_i| |v_j| + |D_i|,  |D_i| <= |g_i| max_j |v_j|
//
// over the keys that query i sees. The exponent brings the bound to between 2^14 and
// 2^15: a query's from its gradient's norm and the largest norm of a value in its block's
// tiles, a block of keys' from its values and the largest norm and D of its queries. The
// sums are scaled back by the same power of two. Rows that are not finite are left out
// of the maxima: what they reach is not finite whatever the scale. bfloat16 needs
// neither factor: it has the floats' range.
constexpr int kScaleLimit = 40;
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }
// e for a bound of at most `bound`.
__device__ __forceinline__ int weight_exponent(float bound) {
  const int log = (__float_as_int(bound) >> 23) - 127;  // bound < 2^(log + 1)
  return max(-kScaleLimit, min(14 - log, kScaleLimit));
}
__device__ __forceinline__ float finite_or_zero(float x) { return x < INFINITY ? x : 0.0f; }

template <class T>
constexpr bool kScaled = std::is_same_v<T, __half>;

// p, for the keys' kernel.
int weight_power(const gs_window_attention_args& a) {
  int p = 0;
  if (a.dtype == GS_FLOAT16) {
    const int64_t seen =
        std::min(a.tokens, int64_t{a.left} + int64_t{a.right} + 1 + int64_t{a.first});
    while (p < 15 && int64_t{2} << p <= seen) ++p;
  }
  return p;
}

// float16's maxima: of the squared norms of a tile's values [tile, kv head], and of the
// squared norm of the gradient and |D| of 32 queries [set of 32, head].
struct Peaks {
  float* values;
  float2* queries;
};
constexpr int kTileSets = kTile / 32;

// The squared norms of values: a block a tile and key-value head. Bound by memory and a
// launch; with the exponents' work a pass of 16,384 tokens, 8 heads of 64, takes 245 us
// instead of 229, one of 65,536 tokens, 8 heads (4) of 128, 1700 instead of 1650.
constexpr int kPeakThreads = 256;
template <class T, int kDim>
__global__ void __launch_bounds__(kPeakThreads) value_peak_kernel(gs_window_attention_args a,
                                                                  float* peaks) {
  chain_wait();
  __shared__ float s_peak[kPeakThreads / 32];
  constexpr int kLanes = kDim / 8, kStep = kPeakThreads / kLanes, kSteps = kTile / kStep;
  const int kv_head = blockIdx.x % a.kv_heads;
  const Tile tile =
      tile_at(a.tiles, blockIdx.x / a.kv_heads, static_cast<int32_t>(a.tokens), kTile);
  const int word = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const bool used = 8 * word < a.dim;
  const T* v = static_cast<const T*>(a.v) + kv_head * a.v_head_stride + (used ? 8 * word : 0);
  Pack<T, 8> x[kSteps];
  uint8_t valid[kSteps];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int64_t token = min(int64_t{tile.start} + row + k * kStep, int64_t{tile.end} - 1);
    x[k] = *reinterpret_cast<const Pack<T, 8>*>(v + token * a.v_stride);
    valid[k] = a.valid ? __ldg(a.valid + token) : 1;
  }
  float peak = 0.0f;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    float square = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) square = fmaf(to_float(x[k].v[e]), to_float(x[k].v[e]), square);
    if (!used) square = 0.0f;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) square += __shfl_xor_sync(0xffffffffu, square, o);
    if (valid[k]) peak = fmaxf(peak, finite_or_zero(square));
  }
  peak = warp_max(peak);
  if ((threadIdx.x & 31) == 0) s_peak[threadIdx.x >> 5] = peak;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPeakThreads / 32; ++w) peak = fmaxf(peak, s_peak[w]);
    peaks[blockIdx.x] = peak;
  }
}

__device__ __forceinline__ int lane_id() { return threadIdx.x & 31; }
__device__ __forceinline__ void sync_compute() {
  asm volatile("bar.sync 1, %0;" ::"n"(kComputeThreads) : "memory");
}

// D, the sums of gradient times output, of the tile's queries, by the compute warps:
// kDim / 8 lanes read a row of the outputs side by side; the gradients are in shared
// memory. False: they did not come.
template <class T, int kDim>
__device__ __forceinline__ bool row_products(const gs_window_attention_args& a, const Tile& tile,
                                             int head, BackwardShared<kDim, false>& s) {
  constexpr int kLanes = kDim / 8, kRows = 32 / kLanes;  // of a warp's step
  constexpr int kSteps = kTile / (kComputeThreads / 32) / kRows;
  const int lane = threadIdx.x & 31, word = lane % kLanes;
  const int first = (threadIdx.x >> 5) * kSteps * kRows + lane / kLanes;
  // Every lane loads, from a row and word that exist: loads that are branched around
  // came one after the other (22,000 clocks until D was known, 8000 now).
  const bool used = 8 * word < a.dim;
  const T* out = static_cast<const T*>(a.out) + (used ? 8 * word : 0);
  uint4 o[kSteps];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int64_t token = min(tile.start + first + k * kRows, tile.end - 1);
    o[k] = *reinterpret_cast<const uint4*>(out + (token * a.heads + head) * a.dim);
  }
  if (!tc::barrier_wait_warp(tc::shared_address(&s.rows_full), 0)) return false;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int row = first + k * kRows;
    float g[8], d = 0.0f, square = 0.0f;
    load_pack<8>(reinterpret_cast<const T*>(s.rows[1] + word / 8 * (kTile * 128) + row * 128 +
                                            ((word ^ row) & 7) * 16),
                 g);
    const Pack<T, 8>& values = reinterpret_cast<const Pack<T, 8>&>(o[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) d = fmaf(g[e], to_float(values.v[e]), d);
    if (!used) d = 0.0f;
#pragma unroll
    for (int x = kLanes / 2; x > 0; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
    if (word == 0) s.part[row] = d;
    if constexpr (kScaled<T>) {  // channels past the last are zeros
#pragma unroll
      for (int e = 0; e < 8; ++e) square = fmaf(g[e], g[e], square);
#pragma unroll
      for (int x = kLanes / 2; x > 0; x >>= 1)
        square += __shfl_xor_sync(0xffffffffu, square, x);
      if (word == 0) s.norm[row] = square;
    }
  }
  return true;
}

// log2 of a row's sum of exponentials, and where there is none (a row that sees
// nothing, a row past the end) what makes its weights 0.
__device__ __forceinline__ float weight_shift(float lse) {
  return lse == -INFINITY ? INFINITY : lse * kLog2e;
}

// dq, and D_i into `delta` for the keys' kernel.
template <class T, int kDim>
__global__ void __launch_bounds__(kBackwardThreads, BackwardShape<kDim, false>::kBlocks)
    grad_query_kernel(gs_window_attention_args a, float* delta, Peaks peaks,
                      const __grid_constant__ CUtensorMap q_map,
                      const __grid_constant__ CUtensorMap g_map,
                      const __grid_constant__ CUtensorMap k_map,
                      const __grid_constant__ CUtensorMap v_map) {
  using namespace tc;
  using Shape = BackwardShape<kDim, false>;
  using Shared = BackwardShared<kDim, false>;
  extern __shared__ __align__(1024) unsigned char shared_bytes[];
  Shared& s = *reinterpret_cast<Shared*>(shared_bytes);
  chain_wait();
  const int warp = threadIdx.x >> 5;
  const int head = blockIdx.x % a.heads, kv_head = head / (a.heads / a.kv_heads);
  const Tile tile =
      tile_at(a.tiles, blockIdx.x / a.heads, static_cast<int32_t>(a.tokens), kTile);
  constexpr int kKeys = Shape::kRows, kSets = Shape::kSets, kHalfSets = kSets / 2;
  const KeyWalk<kKeys, 1> walk(a, tile);
  backward_setup(s, warp, &q_map, &g_map, head, tile.start, &k_map, &v_map,
                 make_int2(kv_head, tile.begin + walk.start(0)));
  const uint32_t tensor = s.tensor;
  bool good = true;
  if (warp == kLoadWarp) {
    good = load_tiles<kDim, false>(
        s, walk.tiles, &k_map, &v_map,
        [&](int t) { return make_int2(kv_head, tile.begin + walk.start(t)); },
        [](int, int) { return 0; }, [](int, int, int, int) {});
  } else if (warp == kProductWarp) {
    good = issue_products<T, kDim, false>(s, a.dim, walk.tiles,
                                          [&](int t) { return walk.sets(0, t); });
  } else {
    const int half = warp >> 2, row = threadIdx.x & (kTile - 1);
    const uint32_t mine = tensor + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const int i_first = walk.i, i = i_first + row;
    const bool live = tile.start + row < tile.end;
    const int64_t slot = head * a.tokens + tile.start + row;
    const float shift = live ? weight_shift(a.lse[slot]) : INFINITY;
    const int64_t index = blockIdx.x / a.heads;  // the tile's number
    float value_peak = 0.0f;
    if constexpr (kScaled<T>) {  // of the tiles that hold the walk's keys
      const int low = walk.low / kTile, count = (walk.high[0] - 1) / kTile - low + 1;
      const float* of = peaks.values + (index - i_first / kTile) * a.kv_heads + kv_head;
      for (int k = threadIdx.x & 31; k < count + (walk.head_tiles > 0); k += 32)
        value_peak = fmaxf(value_peak, of[int64_t{k < count ? low + k : 0} * a.kv_heads]);
    }
    good = row_products<T, kDim>(a, tile, head, s);
    sync_compute();
    const float d = live ? s.part[row] : 0.0f;
    if (live && half == 0) delta[slot] = d;
    float up = 1.0f, back = a.scale;
    if constexpr (kScaled<T>) {
      const float norm = live ? s.norm[row] : 0.0f;
      const int e = weight_exponent(2.0f * sqrtf(norm * warp_max(value_peak)));
      up = power_of_two(e);
      back *= power_of_two(-e);
      if (half == 0) {
        const bool counts = shift != INFINITY;
        const float2 peak = make_float2(warp_max(counts ? finite_or_zero(norm) : 0.0f),
                                        warp_max(counts ? finite_or_zero(fabsf(d)) : 0.0f));
        if ((threadIdx.x & 31) == 0)
          peaks.queries[(index * kTileSets + warp) * a.heads + head] = peak;
      }
    }
    const float scale = a.scale * kLog2e;
    // Every query sees every valid key of a tile that lies from `from` (or under
    // `first`) to `to`.
    const int from = position(int64_t{i_first} + kTile - 1 - a.left);
    const int to = min(position(int64_t{i_first} + a.right + 1), walk.n);
    const float2 factor = make_float2(scale, scale), down = make_float2(-shift, -shift);
    const float2 grow = make_float2(up, up), less = make_float2(-d * up, -d * up);
    const uint32_t scores = mine + 32 * kHalfSets * half;
    // Whether the lane's keys of tile t are valid, a tile ahead.
    bool valid[kSets];
    const auto load_valid = [&](int t) {
      if (!a.valid || t >= walk.tiles) return;
      const int start = walk.start(t) + (threadIdx.x & 31), end = walk.end(t);
#pragma unroll
      for (int c = 0; c < kSets; ++c)
        valid[c] = __ldg(a.valid + tile.begin + min(start + 32 * c, end - 1)) &&
                   start + 32 * c < end;
    };
    load_valid(0);
    for (int t = 0; t < walk.tiles && good; ++t) {
      const int start = walk.start(t), end = walk.end(t);
      // What no query sees has no products either.
      const int sets = walk.sets(0, t) - kHalfSets * half;
      bool whole = t < walk.head_tiles
                       ? start + kKeys <= end
                       : start + kKeys <= to && (start >= from || start + kKeys <= a.first);
      bool all = whole;
      uint32_t keep[kSets], bits[kHalfSets];
      if (a.valid || !whole) {
        all = true;
#pragma unroll
        for (int c = 0; c < kSets; ++c) {
          keep[c] = a.valid ? __ballot_sync(0xffffffffu, valid[c]) : below32(end - start - 32 * c);
          all = all && keep[c] == ~0u;
        }
        whole = whole && all;
#pragma unroll
        for (int h = 0; h < kHalfSets; ++h)
          bits[h] = (half ? keep[kHalfSets + h] : keep[h]) &
                    window_bits(a, i, start + 32 * (kHalfSets * half + h), end);
      }
      load_valid(t + 1);
      if (!(good = barrier_wait_warp(shared_address(&s.scores), t & 1))) break;
      fence_after_sync();
      float x[kHalfSets][32];
#pragma unroll
      for (int h = 0; h < kHalfSets; ++h)
        if (h < sets) load_columns32(scores + 32 * h, x[h]);
      wait_loads();
      fence_before_sync();
      barrier_arrive(shared_address(&s.read));
#pragma unroll
      for (int h = 0; h < kHalfSets; ++h)
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const float2 y = fma2(make_float2(x[h][c], x[h][c + 1]), factor, down);
          x[h][c] = exp2_approx(y.x);
          x[h][c + 1] = exp2_approx(y.y);
        }
      if (!(good = barrier_wait_warp(shared_address(&s.grads[t & 1]), (t >> 1) & 1))) break;
      fence_after_sync();
      const uint32_t grads = scores + Shape::kGrad + (t & 1) * kKeys;
#pragma unroll
      for (int h = 0; h < kHalfSets; ++h)
        if (h < sets) {
          float g[32];
          load_columns32(grads + 32 * h, g);
          wait_loads();
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float2 e = mul2(make_float2(x[h][c], x[h][c + 1]),
                                  fma2(make_float2(g[c], g[c + 1]), grow, less));
            g[c] = e.x;
            g[c + 1] = e.y;
          }
          if (!whole) {
#pragma unroll
            for (int c = 0; c < 32; ++c) g[c] = bits[h] >> c & 1 ? g[c] : 0.0f;
          }
          uint32_t packed[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) packed[c] = pack2<T>(g[2 * c], g[2 * c + 1]);
          store_columns16(grads + 32 * h, packed);
        }
      if (!all) {
        const int stage = t % Shape::kStages0;
        if (!(good =
                  barrier_wait_warp(shared_address(&s.full0[stage]), (t / Shape::kStages0) & 1)))
          break;
        zero_rows<kDim, kKeys, kComputeThreads>(s.tiles0[stage], keep, threadIdx.x);
        fence_async_shared();
      }
      wait_stores();
      fence_before_sync();
      barrier_arrive(shared_address(&s.weights[t & 1]));
    }
    if (good) good = barrier_wait_warp(shared_address(&s.done), 0);
    fence_after_sync();
    unsigned char* rows = s.rows[0];  // the products with the queries are complete
    float o[kDim / 2];
#pragma unroll
    for (int c = 0; c < kDim / 2; c += 32)
      load_columns32(mine + Shape::kSum + half * (kDim / 2) + c,
                     reinterpret_cast<float(&)[32]>(o[c]));
    wait_loads();
#pragma unroll
    for (int e = 0; e < kDim / 2; e += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = good ? o[e + k] * back : NAN;
      put_word<T, kDim>(rows, row, (half * (kDim / 2) + e) / 8, v);
    }
    sync_compute();
    write_rows<T, kDim, kComputeThreads>(
        rows, static_cast<T*>(a.grad_q) + (int64_t{tile.start} * a.heads + head) * a.dim,
        int64_t{a.heads} * a.dim, 0, tile.end - tile.start, a.dim, threadIdx.x);
  }
  backward_end(s, warp, tensor, good);
}

// The sums of first tokens' keys: `base` [sequence, kv head, first, 2 (dK, dV),
// dim] over their own windows, `part` [slot, ...] over the chunks of `tiles`
// tiles of later queries, numbered as runs of tiles are.
struct FirstSums {
  float* base;
  float* part;
  int tiles, slots;
};
// Whether some query of a sequence of n sees first tokens before its window.
__device__ __forceinline__ bool beyond_window(const gs_window_attention_args& a, int n) {
  return a.first > 0 && n > int64_t{a.left} + 1;
}

// dk and dv.
template <class T, int kDim>
__global__ void __launch_bounds__(kBackwardThreads, BackwardShape<kDim, true>::kBlocks)
    grad_key_kernel(gs_window_attention_args a, int power, const float* delta, Peaks peaks,
                    FirstSums sums,
                    const __grid_constant__ CUtensorMap k_map,
                    const __grid_constant__ CUtensorMap v_map,
                    const __grid_constant__ CUtensorMap q_map,
                    const __grid_constant__ CUtensorMap g_map) {
  using namespace tc;
  using Shape = BackwardShape<kDim, true>;
  using Shared = BackwardShared<kDim, true>;
  constexpr int kRows = Shape::kRows, kSets = Shape::kSets, kHalfSets = kSets / 2;
  extern __shared__ __align__(1024) unsigned char shared_bytes[];
  Shared& s = *reinterpret_cast<Shared*>(shared_bytes);
  chain_wait();
  const int warp = threadIdx.x >> 5, group = a.heads / a.kv_heads;
  const int kv_head = blockIdx.x % a.kv_heads;
  const int64_t item = blockIdx.x / a.kv_heads;
  const bool chunk = item < sums.slots;  // the long items come first
  Tile tile;
  int low, high;   // queries, as positions
  int64_t number;  // of the block's tile of keys
  if (chunk) {
    const int64_t b = sequence_of_run(a, item, sums.tiles);
    const int64_t tile0 = number = first_tile_of(a, b), tiles = first_tile_of(a, b + 1) - tile0;
    const int64_t index = (item - run_of(tile0, b, sums.tiles)) * sums.tiles;
    if (index >= tiles) return;
    tile = tile_at(a.tiles, tile0, static_cast<int32_t>(a.tokens), kTile);
    const int64_t n = tile.end - tile.begin;
    low = position(max(index * kTile, int64_t{a.left} + 1));
    high = static_cast<int>(min((index + sums.tiles) * kTile, n));
    if (low >= high) return;
  } else {
    number = item - sums.slots;
    tile = tile_at(a.tiles, number, static_cast<int32_t>(a.tokens), kTile);
    const int64_t n = tile.end - tile.begin, j = tile.start - tile.begin;
    low = max(0, position(j - a.right));
    high = static_cast<int>(min(n, min(j + kTile, n) + a.left));
  }
  const int n = tile.end - tile.begin;
  const int per_head = (high - low + kRows - 1) / kRows;
  const int tiles = per_head * group;
  backward_setup(s, warp, &k_map, &v_map, kv_head, tile.start, &q_map, &g_map,
                 make_int2(kv_head * group, tile.begin + low));
  const uint32_t tensor = s.tensor;
  bool good = true;
  if (warp == kLoadWarp) {
    float grow = 1.0f, value_peak = 0.0f;
    float2 peak[4] = {};  // of the lane's sets of 32 queries
    if constexpr (kScaled<T>) {
      const int set = low / 32, count = ((high - 1) / 32 - set + 1) * group;
      const float2* of = peaks.queries +
                         ((number - (tile.start - tile.begin) / kTile) * kTileSets + set) * a.heads +
                         kv_head * group;
      const auto at = [&](int k) {  // a number past the last names the last again
        k = min(k, count - 1);
        return of[int64_t{k / group} * a.heads + k % group];
      };
      value_peak = peaks.values[number * a.kv_heads + kv_head];
#pragma unroll
      for (int k = 0; k < 4; ++k) peak[k] = at(lane_id() + 32 * k);
      for (int k = lane_id() + 128; k < count; k += 32) {
        const float2 x = at(k);
        peak[0] = make_float2(fmaxf(peak[0].x, x.x), fmaxf(peak[0].y, x.y));
      }
    }
    // L and D of a tile's queries come along, negated.
    struct RowValues {
      float shift[kSets], delta[kSets];
    };
    good = load_tiles<kDim, true>(
        s, tiles, &q_map, &g_map,
        [&](int t) {
          return make_int2(kv_head * group + t / per_head,
                           tile.begin + low + (t % per_head) * kRows);
        },
        [&](int t, int lane) {
          RowValues v;
          const int i = low + (t % per_head) * kRows + lane;
          const int64_t at = (kv_head * group + t / per_head) * a.tokens + tile.begin;
          // Loads from rows that exist, all on their way at once.
#pragma unroll
          for (int k = 0; k < kSets; ++k) {
            const int64_t where = at + min(i + 32 * k, n - 1);
            v.shift[k] = a.lse[where];
            v.delta[k] = delta[where];
          }
          return v;
        },
        [&](int t, int stage, int lane, const RowValues& v) {
          if (kScaled<T> && t == 0) {  // the tile's values and the peaks were loaded side by side
            const float norm = warp_max(fmaxf(fmaxf(peak[0].x, peak[1].x),
                                              fmaxf(peak[2].x, peak[3].x)));
            const float d = warp_max(fmaxf(fmaxf(peak[0].y, peak[1].y),
                                           fmaxf(peak[2].y, peak[3].y)));
            const int e = weight_exponent(fmaf(1.001f, sqrtf(norm * value_peak), d));
            grow = power_of_two(e - power);
            if (lane == 0) {
              s.grow = grow;
              s.back = a.scale * power_of_two(-e);
            }
          }
          const int i = low + (t % per_head) * kRows + lane;
          bool none = false;
#pragma unroll
          for (int k = 0; k < kSets; ++k) {
            const bool in = i + 32 * k < n;
            none = none || !in || v.shift[k] == -INFINITY;
            s.row[stage][0][lane + 32 * k] =
                in ? power - weight_shift(v.shift[k]) : -INFINITY;
            s.row[stage][1][lane + 32 * k] = in ? -v.delta[k] * grow : 0.0f;
          }
          none = __any_sync(0xffffffffu, none);
          if (lane == 0) s.none[stage] = none;
        });
  } else if (warp == kProductWarp) {
    good = issue_products<T, kDim, true>(s, a.dim, tiles, [&](int t) {
      return min(kSets, (high - low - (t % per_head) * kRows + 31) / 32);
    });
  } else {
    const int half = warp >> 2, row = threadIdx.x & (kTile - 1);
    const uint32_t mine = tensor + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const int j_first = tile.start - tile.begin, j = j_first + row;
    const bool live = j < n && (!chunk || j < a.first);
    const bool seen = live && (!a.valid || a.valid[tile.start + row]);
    const bool any_seen = __any_sync(0xffffffffu, seen), all_seen = __all_sync(0xffffffffu, seen);
    // The queries that see key j: those from `from` to `to`. All of the block's keys
    // are seen by the queries from `all_from` to `all_to`.
    const int from = chunk ? position(int64_t{j} + a.left + 1) : position(int64_t{j} - a.right);
    const int to = chunk ? high : min(high, position(int64_t{j} + a.left + 1));
    const int all_from = position(int64_t{j_first} + kTile - 1 - a.right);
    const int all_to = chunk ? 0 : min(high, position(int64_t{j_first} + a.left + 1));
    const float scale = a.scale * kLog2e;
    const float2 factor = make_float2(scale, scale);
    const uint32_t scores = mine + 32 * kHalfSets * half, grads = scores + Shape::kGrad;
    int stage0 = 0, stage1 = 0, parity1 = 0, index = 0;
    for (int t = 0; t < tiles; ++t) {
      const int start = low + index * kRows, first = start + 32 * kHalfSets * half;
      // Sets of 32 queries of this half; what lies past the last has no products.
      const int sets = min(kHalfSets, (high - first + 31) >> 5);
      const bool whole = all_seen && start >= all_from && start + kRows <= all_to;
      uint32_t bits[kHalfSets];
      if (!whole) {
#pragma unroll
        for (int h = 0; h < kHalfSets; ++h)
          bits[h] = seen ? below32(to - first - 32 * h) & ~below32(from - first - 32 * h) : 0;
      }
      if (!(good = barrier_wait_warp(shared_address(&s.scores), t & 1) &&
                   barrier_wait_warp(shared_address(&s.full1[stage1]), parity1)))
        break;
      fence_after_sync();
      const bool none = !whole && s.none[stage1];
      float x[kHalfSets][32];
      if (any_seen) {
#pragma unroll
        for (int h = 0; h < kHalfSets; ++h)
          if (h < sets) load_columns32(scores + 32 * h, x[h]);
        wait_loads();
      }
      const float4* shifts = reinterpret_cast<const float4*>(s.row[stage1][0] + 32 * kHalfSets * half);
#pragma unroll
      for (int h = 0; h < kHalfSets; ++h)
        if (h < sets) {
          uint32_t packed[16];
          if (any_seen) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const float4 l = shifts[8 * h + c];
              float* p = &x[h][4 * c];
              const float2 y0 = fma2(make_float2(p[0], p[1]), factor, make_float2(l.x, l.y));
              const float2 y1 = fma2(make_float2(p[2], p[3]), factor, make_float2(l.z, l.w));
              p[0] = exp2_approx(y0.x);
              p[1] = exp2_approx(y0.y);
              p[2] = exp2_approx(y1.x);
              p[3] = exp2_approx(y1.y);
            }
            if (!whole) {
#pragma unroll
              for (int c = 0; c < 32; ++c) x[h][c] = bits[h] >> c & 1 ? x[h][c] : 0.0f;
            }
#pragma unroll
            for (int c = 0; c < 16; ++c) packed[c] = pack2<T>(x[h][2 * c], x[h][2 * c + 1]);
          } else {
#pragma unroll
            for (int c = 0; c < 16; ++c) packed[c] = 0;
          }
          store_columns16(scores + 32 * h, packed);
        }
      // No gradient flows through a query that sees nothing: what it and its gradient
      // hold must not meet its weights of zero, nor what the next sequence's rows do.
      if (none) {
        uint32_t keep[kSets];
#pragma unroll
        for (int c = 0; c < kSets; ++c)
          keep[c] = __ballot_sync(0xffffffffu, s.row[stage1][0][lane_id() + 32 * c] != -INFINITY);
        zero_rows<kDim, kRows, kComputeThreads>(s.tiles0[stage0], keep, threadIdx.x);
        zero_rows<kDim, kRows, kComputeThreads>(s.tiles1[stage1], keep, threadIdx.x);
        fence_async_shared();
      }
      wait_stores();
      fence_before_sync();
      barrier_arrive(shared_address(&s.read));
      if (!(good = barrier_wait_warp(shared_address(&s.grads[0]), t & 1))) break;
      fence_after_sync();
      const float up = kScaled<T> ? s.grow : 1.0f;
      const float2 grow = make_float2(up, up);
      const float4* deltas = reinterpret_cast<const float4*>(s.row[stage1][1] + 32 * kHalfSets * half);
#pragma unroll
      for (int h = 0; h < kHalfSets; ++h)
        if (h < sets) {
          uint32_t packed[16];
          if (any_seen) {
            float g[32];
            load_columns32(grads + 32 * h, g);
            wait_loads();
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const float4 d = deltas[8 * h + c];
              float* e = &g[4 * c];
              const float* p = &x[h][4 * c];
              const float2 e0 = mul2(make_float2(p[0], p[1]),
                                     fma2(make_float2(e[0], e[1]), grow, make_float2(d.x, d.y)));
              const float2 e1 = mul2(make_float2(p[2], p[3]),
                                     fma2(make_float2(e[2], e[3]), grow, make_float2(d.z, d.w)));
              e[0] = e0.x;
              e[1] = e0.y;
              e[2] = e1.x;
              e[3] = e1.y;
            }
            if (!whole) {
#pragma unroll
              for (int c = 0; c < 32; ++c) g[c] = bits[h] >> c & 1 ? g[c] : 0.0f;
            }
#pragma unroll
            for (int c = 0; c < 16; ++c) packed[c] = pack2<T>(g[2 * c], g[2 * c + 1]);
          } else {
#pragma unroll
            for (int c = 0; c < 16; ++c) packed[c] = 0;
          }
          store_columns16(grads + 32 * h, packed);
        }
      wait_stores();
      fence_before_sync();
      barrier_arrive(shared_address(&s.weights[t & 1]));
      if (++index == per_head) index = 0;
      if (++stage0 == Shape::kStages0) stage0 = 0;
      if (++stage1 == Shape::kStages1) {
        stage1 = 0;
        parity1 ^= 1;
      }
    }
    if (good) good = barrier_wait_warp(shared_address(&s.done), 0);
    fence_after_sync();
    // First tokens that later queries see too: floats for the sum of the chunks.
    const int summed = beyond_window(a, n) ? a.first : 0;
    const int64_t where = chunk ? item : tile.sequence;
    float* sum = (chunk ? sums.part : sums.base) +
                 ((where * a.kv_heads + kv_head) * a.first + j) * 2 * a.dim;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float o[kDim / 2];
#pragma unroll
      for (int c = 0; c < kDim / 2; c += 32)
        load_columns32(mine + Shape::kSum + which * kDim + half * (kDim / 2) + c,
                       reinterpret_cast<float(&)[32]>(o[c]));
      wait_loads();
      const float factor = which ? power_of_two(-power) : kScaled<T> ? s.back : a.scale;
#pragma unroll
      for (int e = 0; e < kDim / 2; e += 8) {
        const int c = half * (kDim / 2) + e;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = good ? o[e + k] * factor : NAN;
        put_word<T, kDim>(s.rows[which], row, c / 8, v);
        if (live && j < summed && c < a.dim) store_pack<8>(sum + which * a.dim + c, v);
      }
    }
    if (!chunk) {
      sync_compute();
      for (int which = 0; which < 2; ++which)
        write_rows<T, kDim, kComputeThreads>(
            s.rows[which],
            static_cast<T*>(which ? a.grad_v : a.grad_k) +
                (int64_t{tile.start} * a.kv_heads + kv_head) * a.dim,
            int64_t{a.kv_heads} * a.dim, summed - j_first, n - j_first, a.dim, threadIdx.x);
    }
  }
  backward_end(s, warp, tensor, good);
}

// dk and dv of first tokens: their window's sum and the chunks' in order, a
// block a token and key-value head; the chunks are shared out to kParts rows of
// threads, whose sums are added in order.
constexpr int kParts = 4;
template <class T>
__global__ void __launch_bounds__(2 * kMaxDim * kParts) first_sum_kernel(
    gs_window_attention_args a, FirstSums sums) {
  chain_wait();
  __shared__ float s_part[kParts][2 * kMaxDim];
  const int j = blockIdx.x % a.first;
  const int kv_head = blockIdx.x / a.first % a.kv_heads;
  const int64_t b = blockIdx.x / (int64_t{a.first} * a.kv_heads);
  const int64_t tile0 = first_tile_of(a, b), tiles = first_tile_of(a, b + 1) - tile0;
  if (tiles == 0) return;
  const Tile tile = tile_at(a.tiles, tile0, static_cast<int32_t>(a.tokens), kTile);
  const int64_t n = tile.end - tile.begin;
  if (j >= n || !beyond_window(a, static_cast<int>(n))) return;
  const int c = threadIdx.x % (2 * kMaxDim), part = threadIdx.x / (2 * kMaxDim);
  const int64_t row = (int64_t{kv_head} * a.first + j) * 2 * a.dim + c;
  const int64_t stride = int64_t{a.kv_heads} * a.first * 2 * a.dim;
  const int64_t slot = run_of(tile0, b, sums.tiles);
  const int64_t length = int64_t{sums.tiles} * kTile;
  const int64_t from = (int64_t{a.left} + 1) / length, to = (n + length - 1) / length;
  float sum = 0.0f;
  if (c < 2 * a.dim) {
    if (part == 0) sum = sums.base[b * stride + row];
#pragma unroll 8
    for (int64_t k = from + part; k < to; k += kParts) sum += sums.part[(slot + k) * stride + row];
  }
  s_part[part][c] = sum;
  __syncthreads();
  if (part == 0 && c < 2 * a.dim) {
    for (int p = 1; p < kParts; ++p) sum += s_part[p][c];
    const int64_t at = (int64_t{tile.begin + j} * a.kv_heads + kv_head) * a.dim;
    if (c < a.dim) static_cast<T*>(a.grad_k)[at + c] = from_float<T>(sum);
    else static_cast<T*>(a.grad_v)[at + c - a.dim] = from_float<T>(sum);
  }
}

// D of every row, to a 256-byte boundary.
int64_t delta_floats(const gs_window_attention_args& a) {
  return (a.tokens * a.heads + 63) / 64 * 64;
}

// float16's maxima: floats of those of the queries, and of all of them to a 256-byte
// boundary.
int64_t query_peak_floats(const gs_window_attention_args& a) {
  return a.num_tiles * kTileSets * a.heads * 2;
}
int64_t peak_floats(const gs_window_attention_args& a) {
  if (a.dtype != GS_FLOAT16) return 0;
  return (query_peak_floats(a) + a.num_tiles * a.kv_heads + 63) / 64 * 64;
}

// A chunk is about as long as a window's walk, so that its block takes about as
// long as the others.
int64_t chunk_tiles(const gs_window_attention_args& a) {
  const int64_t window =
      std::min(a.tokens, int64_t{a.left}) + std::min(a.tokens, int64_t{a.right});
  return std::max<int64_t>(8, (window + kTile - 1) / kTile + 1);
}
int64_t chunk_slots(const gs_window_attention_args& a) {
  return a.first > 0 ? a.num_tiles / chunk_tiles(a) + sequences_of(a) : 0;
}

template <class T, int kDim>
int32_t backward(const gs_window_attention_args& a, cudaStream_t stream) {
  CUtensorMap rows[4], tiles[4];  // q, grad_out, k, v
  const void* const base[4] = {a.q, a.grad_out, a.k, a.v};
  const int64_t stride[4] = {a.q_stride, int64_t{a.heads} * a.dim, a.k_stride, a.v_stride};
  const int64_t head_stride[4] = {a.q_head_stride, a.dim, a.k_head_stride, a.v_head_stride};
  for (int m = 0; m < 4; ++m) {
    const int64_t heads = m < 2 ? a.heads : a.kv_heads;
    constexpr int kRows = BackwardShape<kDim, true>::kRows;
    GS_TRY(tc::encode_heads(&rows[m], a.dtype, base[m], a.tokens, heads, a.dim, stride[m],
                            head_stride[m], kTile));
    if constexpr (kRows == kTile) tiles[m] = rows[m];
    else
      GS_TRY(tc::encode_heads(&tiles[m], a.dtype, base[m], a.tokens, heads, a.dim, stride[m],
                              head_stride[m], kRows));
  }
  float* delta = static_cast<float*>(a.workspace);
  float* maxima = delta + delta_floats(a);
  const Peaks peaks = {maxima + query_peak_floats(a), reinterpret_cast<float2*>(maxima)};
  FirstSums sums;
  sums.tiles = static_cast<int>(chunk_tiles(a));
  sums.slots = static_cast<int>(chunk_slots(a));
  sums.base = maxima + peak_floats(a);
  sums.part = sums.base + sequences_of(a) * a.kv_heads * a.first * 2 * a.dim;
  constexpr size_t kQueryShared = sizeof(BackwardShared<kDim, false>);
  constexpr size_t kKeyShared = sizeof(BackwardShared<kDim, true>);
  GS_TRY((allow_shared<grad_query_kernel<T, kDim>>(kQueryShared)));
  GS_TRY((allow_shared<grad_key_kernel<T, kDim>>(kKeyShared)));
  const int64_t key_blocks = (a.num_tiles + sums.slots) * a.kv_heads;
  const int64_t first_blocks = sequences_of(a) * a.kv_heads * a.first;
  if (key_blocks > INT32_MAX || first_blocks > INT32_MAX) return GS_ERR_CAPACITY;
  if constexpr (kScaled<T>) {
    launch_chained(value_peak_kernel<T, kDim>, static_cast<unsigned>(a.num_tiles * a.kv_heads),
                   kPeakThreads, stream, a, peaks.values);
    GS_TRY(check_launch());
  }
  launch_chained_shared(grad_query_kernel<T, kDim>, static_cast<unsigned>(a.num_tiles * a.heads),
                        kBackwardThreads, kQueryShared, stream, a, delta, peaks, rows[0], rows[1],
                        tiles[2], tiles[3]);
  GS_TRY(check_launch());
  launch_chained_shared(grad_key_kernel<T, kDim>, static_cast<unsigned>(key_blocks),
                        kBackwardThreads, kKeyShared, stream, a, weight_power(a), delta, peaks, sums, rows[2],
                        rows[3],
                        tiles[0], tiles[1]);
  GS_TRY(check_launch());
  if (first_blocks > 0)
    launch_chained(first_sum_kernel<T>, static_cast<unsigned>(first_blocks), 2 * kMaxDim * kParts,
                   stream, a, sums);
  return check_launch();
}

// ------------------------------------------------- one new token a stream
//
// The cache is read once: that is the bound (96 streams of 4100 slots, 4
// key-value heads of 128: 806 MB in 139 us, 5.8 TB/s; one stream takes 9 us, the
// latency of a launch, a load and the join). A cluster of blocks shares the
// slots of a stream and key-value head, up to 16 query heads (more: more
// clusters). TMA brings tiles of 64 slots to shared memory some tiles ahead,
// which keeps over 100 KB in flight a multiprocessor (loads straight to
// registers, 12 warps: 4.3 TB/s); a warp takes 16 slots of each and reads
// them in the shape of its matrix products:
//
//   scores [heads x slots] = q K^T: a lane's 16 bytes of a key row are its
//     parts of two products, with q's channels permuted alike;
//   out [heads x dim] += P V: a lane's 16 bytes of two value rows, interleaved,
//     are its parts of eight products, one channel of eight to each; the scores'
//     places in the registers are the ones that P needs.
//
// The warps' maxima, sums and outputs are joined in order, in the block and then
// across the cluster through distributed shared memory: one launch, no
// workspace, no atomics.

constexpr int kStepWarps = 4;
constexpr int kStepThreads = 32 * kStepWarps;
constexpr int kStepSlots = 16;  // a warp's slots of a tile
constexpr int kStepTile = kStepWarps * kStepSlots;
constexpr int kStepStages = 3;

template <int kDim, int kHalves>
struct StepShared {
  static constexpr int kTileBytes = kStepTile * kDim * 2;
  union {
    struct {
      alignas(1024) unsigned char k[kStepStages][kTileBytes];
      unsigned char v[kStepStages][kTileBytes];
    };
    float out[kStepWarps][8 * kHalves][kDim];  // once the tiles are done
  };
  float top[kStepWarps][8 * kHalves], sum[kStepWarps][8 * kHalves];
  uint64_t full[kStepStages], empty[kStepStages];
};

// Sixteen bytes, number `word`, of a row of a loaded tile.
__device__ __forceinline__ uint4 tile_word(const unsigned char* tile, int row, int word) {
  return *reinterpret_cast<const uint4*>(tile + (word >> 3) * (kStepTile * 128) + row * 128 +
                                         (((word & 7) ^ (row & 7)) << 4));
}

// c += a b for kHalves halves of 8 rows; with one, the rows of the second are
// zeros that need no registers.
template <class T, int kHalves>
__device__ __forceinline__ void warp_product(float (&half)[kHalves][2],
                                             const uint32_t (&rows)[kHalves][2], uint32_t b0,
                                             uint32_t b1) {
  float c[4] = {half[0][0], half[0][1], 0.0f, 0.0f};
  uint32_t a[4] = {rows[0][0], 0, rows[0][1], 0};
  if constexpr (kHalves == 2) {
    c[2] = half[1][0]; c[3] = half[1][1];
    a[1] = rows[1][0]; a[3] = rows[1][1];
  }
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  half[0][0] = c[0];
  half[0][1] = c[1];
  if constexpr (kHalves == 2) {
    half[1][0] = c[2];
    half[1][1] = c[3];
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// A float at the same place of another block's shared memory.
__device__ __forceinline__ float read_block(const float* p, uint32_t rank) {
  uint32_t there;
  float x;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(there)
               : "r"(tc::shared_address(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(there) : "memory");
  return x;
}

// kMasked: with validity of the slots (3% more time).
template <class T, int kDim, int kHalves, bool kMasked>
__global__ void __launch_bounds__(kStepThreads, kDim == 64 ? 4 : 2)
    attention_step_kernel(gs_window_attention_step_args a, const __grid_constant__ CUtensorMap k_map,
                          const __grid_constant__ CUtensorMap v_map) {
  using Shared = StepShared<kDim, kHalves>;
  extern __shared__ __align__(1024) unsigned char shared_bytes[];
  Shared& s = *reinterpret_cast<Shared*>(shared_bytes);
  chain_wait();
  constexpr int kChunks = kDim / 32;  // of a key row, two products each
  constexpr int kParts = kDim / 64;   // of a value row, eight products each
  constexpr int kStepHeads = 8 * kHalves;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const uint32_t rank = cluster_rank(), blocks = cluster_size();
  const int group = a.heads / a.kv_heads, pieces = (group + kStepHeads - 1) / kStepHeads;
  const int64_t item = blockIdx.x / blocks;
  const int piece = static_cast<int>(item % pieces);
  const int kv_head = static_cast<int>(item / pieces % a.kv_heads);
  const int64_t b = item / pieces / a.kv_heads;
  const int head0 = kv_head * group + piece * kStepHeads;
  const int heads = min(kStepHeads, group - piece * kStepHeads);
  const int64_t position = a.positions[b];
  const bool idle = position < 0;
  const int64_t slot = idle                 ? -1
                       : position < a.first ? position
                                            : a.first + (position - a.first) % (a.slots - a.first);
  const int count = idle ? 0 : static_cast<int>(min(position + 1, int64_t{a.slots}));
  const int64_t row = int64_t{a.kv_heads} * a.dim;
  T* cache_k = static_cast<T*>(a.cache_k) + b * a.slots * row + kv_head * a.dim;
  T* cache_v = static_cast<T*>(a.cache_v) + b * a.slots * row + kv_head * a.dim;
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride + kv_head * a.k_head_stride;
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride + kv_head * a.v_head_stride;
  // The new token's slot is read by nobody: its rows and its validity come from the
  // arguments.
  uint8_t* const slots_valid = kMasked ? a.cache_valid + b * a.slots : nullptr;
  const bool token_valid = !kMasked || !a.valid || a.valid[b];
  if (kMasked && !idle && rank == 0 && piece == 0 && kv_head == 0 && threadIdx.x == 0)
    slots_valid[slot] = token_valid;
  if (!idle && rank == 0 && piece == 0)
    for (int c = threadIdx.x; c < a.dim; c += kStepThreads) {
      cache_k[slot * row + c] = k[c];
      cache_v[slot * row + c] = v[c];
    }

  // q's rows g (and g + 8), in the order of the key rows' products.
  uint32_t q[kChunks][2][kHalves][2];
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
#pragma unroll
    for (int r = 0; r < kHalves; ++r) {
      uint4 word = make_uint4(0, 0, 0, 0);
      if (g + 8 * r < heads && 32 * c + 8 * j < a.dim)
        word = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.q_stride +
                                               (head0 + g + 8 * r) * a.q_head_stride + 32 * c +
                                               8 * j);
      q[c][0][r][0] = word.x;
      q[c][0][r][1] = word.y;
      q[c][1][r][0] = word.z;
      q[c][1][r][1] = word.w;
    }
  const float scale = a.scale * kLog2e;
  float out[kParts][8][kHalves][2] = {};
  float top[kHalves], sum[kHalves] = {};
#pragma unroll
  for (int r = 0; r < kHalves; ++r) top[r] = -INFINITY;

  // This block's tiles of the stream's slots: rank, rank + blocks, ...
  const int tiles = max(0, ((count + kStepTile - 1) / kStepTile - static_cast<int>(rank) +
                            static_cast<int>(blocks) - 1) /
                               static_cast<int>(blocks));
  const auto base_of = [&](int t) {
    return (static_cast<int>(rank) + t * static_cast<int>(blocks)) * kStepTile;
  };
  const auto load_tile = [&](int t) {
    const int stage = t % kStepStages;
    const uint32_t bar = tc::shared_address(&s.full[stage]);
    const int first = static_cast<int>(b * a.slots) + base_of(t);
    tc::barrier_expect(bar, 2 * Shared::kTileBytes);
    for (int x = 0; x < kDim / 64; ++x) {
      tc::load_box(tc::shared_address(s.k[stage]) + x * kStepTile * 128, &k_map, 64 * x, kv_head,
                   first, bar);
      tc::load_box(tc::shared_address(s.v[stage]) + x * kStepTile * 128, &v_map, 64 * x, kv_head,
                   first, bar);
    }
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStepStages; ++i) {
      tc::barrier_init(tc::shared_address(&s.full[i]), 1);
      tc::barrier_init(tc::shared_address(&s.empty[i]), kStepWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tc::fence_async_shared();
    for (int t = 0; t < kStepStages && t < tiles; ++t) load_tile(t);
  }
  __syncthreads();
  bool good = true;
  for (int t = 0; t < tiles; ++t) {
    const int stage = t % kStepStages;
    // The tile before last's stage gets its next tile once all warps are done
    // with it, which by now they mostly are.
    if (threadIdx.x == 0 && t >= 1 && t - 1 + kStepStages < tiles) {
      good = good && tc::barrier_wait(tc::shared_address(&s.empty[(t - 1) % kStepStages]),
                                      ((t - 1) / kStepStages) & 1);
      if (good) load_tile(t - 1 + kStepStages);
    }
    const int row0 = warp * kStepSlots, base = base_of(t) + row0;
    // Which of the lane's slots, 2j, 2j+1, 2j+8 and 2j+9, may be seen.
    bool seen[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int at = base + 2 * j + (m & 1) + 8 * (m >> 1);
      seen[m] = at < count;
      if (kMasked && seen[m]) seen[m] = at == slot ? token_valid : slots_valid[at] != 0;
    }
    good = __all_sync(0xffffffffu, good) &&
           tc::barrier_wait_warp(tc::shared_address(&s.full[stage]), (t / kStepStages) & 1);
    if (!good) break;
    // Keys base + g and base + 8 + g; values of the slots 2j, 2j+1, 2j+8, 2j+9.
    uint4 key[2][kChunks];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) key[n][c] = tile_word(s.k[stage], row0 + 8 * n + g, 4 * c + j);
      if (base + 8 * n + g == slot)
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          key[n][c] = 32 * c + 8 * j < a.dim
                          ? *reinterpret_cast<const uint4*>(k + 32 * c + 8 * j)
                          : make_uint4(0, 0, 0, 0);
    }
    float x[2][kHalves][2] = {};  // scores of the slots 8n + 2j, 8n + 2j + 1
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        warp_product<T, kHalves>(x[n], q[c][0], key[n][c].x, key[n][c].y);
        warp_product<T, kHalves>(x[n], q[c][1], key[n][c].z, key[n][c].w);
      }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int r = 0; r < kHalves; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (!seen[2 * n + e]) x[n][r][e] = -INFINITY;
    uint32_t p[kHalves][2];
#pragma unroll
    for (int r = 0; r < kHalves; ++r) {
      float next = fmaxf(fmaxf(x[0][r][0], x[0][r][1]), fmaxf(x[1][r][0], x[1][r][1]));
      next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, 1));
      next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, 2)) * scale;
      const bool grow = next > top[r] + kSlack || (top[r] == -INFINITY && next > top[r]);
      if (__any_sync(0xffffffffu, grow)) {
        const float shrink = grow ? tc::exp2_approx(top[r] - next) : 1.0f;
        if (grow) top[r] = next;
        sum[r] *= shrink;
#pragma unroll
        for (int h = 0; h < kParts; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            out[h][i][r][0] *= shrink;
            out[h][i][r][1] *= shrink;
          }
      }
      const float shift = top[r] == -INFINITY ? 0.0f : kLift<T> - top[r];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float p0 = tc::exp2_approx(fmaf(x[n][r][0], scale, shift));
        const float p1 = tc::exp2_approx(fmaf(x[n][r][1], scale, shift));
        sum[r] += p0 + p1;
        p[r][n] = tc::pack2<T>(p0, p1);
      }
    }
#pragma unroll
    for (int h = 0; h < kParts; ++h) {
      uint4 value[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int r = 2 * j + (n & 1) + 8 * (n >> 1);
        value[n] = tile_word(s.v[stage], row0 + r, 8 * h + g);
        // What an empty slot, or one left out, holds must not meet its weight of zero.
        if (base + r == slot && 64 * h + 8 * g < a.dim)
          value[n] = *reinterpret_cast<const uint4*>(v + 64 * h + 8 * g);
        if (!seen[n]) value[n] = make_uint4(0, 0, 0, 0);
      }
      const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&value[0]);
      const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&value[1]);
      const uint32_t* v8 = reinterpret_cast<const uint32_t*>(&value[2]);
      const uint32_t* v9 = reinterpret_cast<const uint32_t*>(&value[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        warp_product<T, kHalves>(out[h][2 * i], p, __byte_perm(v0[i], v1[i], 0x5410),
                                 __byte_perm(v8[i], v9[i], 0x5410));
        warp_product<T, kHalves>(out[h][2 * i + 1], p, __byte_perm(v0[i], v1[i], 0x7632),
                                 __byte_perm(v8[i], v9[i], 0x7632));
      }
    }
    __syncwarp();
    if (lane == 0) tc::barrier_arrive(tc::shared_address(&s.empty[stage]));
  }
  if (!good) {  // let what is in flight land, and show that the result is not valid
    for (uint64_t& bar : s.full) tc::barrier_settle(tc::shared_address(&bar));
    for (float& x : sum) x = NAN;
    if (lane == 0) atomicExch(&g_timeout, 1u);
  }
  __syncthreads();  // the tiles' place is free for the outputs

  // The warp's rows to shared memory: product i's column n is channel 8n + i of
  // its part.
#pragma unroll
  for (int r = 0; r < kHalves; ++r) {
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
    if (j == 0) {
      s.top[warp][g + 8 * r] = top[r];
      s.sum[warp][g + 8 * r] = sum[r];
    }
#pragma unroll
    for (int h = 0; h < kParts; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          s.out[warp][g + 8 * r][64 * h + 8 * (2 * j + e) + i] = out[h][i][r][e];
  }
  __syncthreads();
  // The warps joined into the first one's place.
  for (int c = threadIdx.x; c < heads * kDim; c += kStepThreads) {
    const int h = c / kDim, d = c % kDim;
    float whole = -INFINITY, o = 0.0f;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) whole = fmaxf(whole, s.top[w][h]);
    const float shift = whole == -INFINITY ? 0.0f : whole;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w)
      o = fmaf(s.out[w][h][d], tc::exp2_approx(s.top[w][h] - shift), o);
    s.out[0][h][d] = o;
  }
  __syncthreads();
  if (threadIdx.x < heads) {
    const int h = threadIdx.x;
    float whole = -INFINITY, total = 0.0f;
    for (int w = 0; w < kStepWarps; ++w) whole = fmaxf(whole, s.top[w][h]);
    const float shift = whole == -INFINITY ? 0.0f : whole;
    for (int w = 0; w < kStepWarps; ++w)
      total = fmaf(s.sum[w][h], tc::exp2_approx(s.top[w][h] - shift), total);
    s.top[0][h] = whole;
    s.sum[0][h] = total;
  }
  cluster_sync();
  // The blocks joined, each block a part of the outputs.
  for (int c = static_cast<int>(rank) * kStepThreads + threadIdx.x; c < heads * kDim;
       c += static_cast<int>(blocks) * kStepThreads) {
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

// Blocks of a cluster: enough that every multiprocessor has several blocks, as
// far as each warp still gets slots (96 streams of 4100 slots: 138 us with
// clusters of 2, 148 us with 4).
int step_blocks(const gs_window_attention_step_args& a, int64_t items) {
  int blocks = 1;
  while (blocks < 16 && items * blocks < 4 * kSmCount &&
         2 * blocks * kStepTile <= a.slots)
    blocks *= 2;
  return blocks;
}

template <class T, int kDim, int kHalves, bool kMasked>
int32_t step(const gs_window_attention_step_args& a, cudaStream_t stream) {
  const int64_t items = a.batch * a.kv_heads * ceil_div(a.heads / a.kv_heads, 8 * kHalves);
  const int blocks = step_blocks(a, items);
  if (items * blocks > INT32_MAX) return GS_ERR_CAPACITY;
  CUtensorMap k, v;
  const int64_t row = int64_t{a.kv_heads} * a.dim;
  GS_TRY(tc::encode_heads(&k, a.dtype, a.cache_k, a.batch * a.slots, a.kv_heads, a.dim, row, a.dim,
                          kStepTile));
  GS_TRY(tc::encode_heads(&v, a.dtype, a.cache_v, a.batch * a.slots, a.kv_heads, a.dim, row, a.dim,
                          kStepTile));
  constexpr size_t kShared = sizeof(StepShared<kDim, kHalves>);
  GS_TRY((allow_shared<attention_step_kernel<T, kDim, kHalves, kMasked>>(kShared, true)));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = blocks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = static_cast<unsigned>(items * blocks);
  config.blockDim = kStepThreads;
  config.dynamicSmemBytes = kShared;
  config.stream = stream;
  config.attrs = attr;
  config.numAttrs = 2;
  cudaLaunchKernelEx(&config, attention_step_kernel<T, kDim, kHalves, kMasked>, a, k, v);
  return check_launch();
}

bool sixteen_bit(int32_t dtype) { return dtype == GS_BFLOAT16 || dtype == GS_FLOAT16; }

bool strided16(const void* p, int64_t stride, int64_t head_stride) {
  return is_aligned(p, 16) && stride % 8 == 0 && head_stride % 8 == 0;
}

int32_t check_heads(int32_t heads, int32_t kv_heads, int32_t dim, int32_t dtype) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || heads > 65535 || dim < 8 || dim % 8)
    return GS_ERR_INVALID_ARGUMENT;
  return dim > kMaxDim || !sixteen_bit(dtype) ? GS_ERR_UNSUPPORTED : GS_OK;
}

int32_t check_args(const gs_window_attention_args& a) {
  GS_TRY(check_heads(a.heads, a.kv_heads, a.dim, a.dtype));
  if (a.tokens < 0 || a.tokens > GS_MAX_SEQUENCE_TOKENS || a.num_tiles < 0 || a.num_tiles > INT32_MAX / a.heads ||
      a.left < 0 || a.right < 0 || a.first < 0 || a.first > GS_MAX_FIRST_TOKENS ||
      !(a.scale > 0.0f && a.scale < INFINITY))
    return GS_ERR_INVALID_ARGUMENT;
  if (!is_aligned(a.tiles, 16)) return GS_ERR_MISALIGNED;
  if (!layout_holds(a.tokens, a.sequences, a.num_tiles, a.tiles, a.tile_starts))
    return GS_ERR_INVALID_ARGUMENT;
  if (a.num_tiles == 0) return GS_OK;
  if (!a.q || !a.k || !a.v || !a.out) return GS_ERR_INVALID_ARGUMENT;
  if (!strided16(a.q, a.q_stride, a.q_head_stride) ||
      !strided16(a.k, a.k_stride, a.k_head_stride) ||
      !strided16(a.v, a.v_stride, a.v_head_stride) || !is_aligned(a.out, 16))
    return GS_ERR_MISALIGNED;
  return GS_OK;
}

// Calls f with a value of the 16-bit type that `dtype` names.
template <class F>
int32_t with_sixteen_bit(int32_t dtype, F&& f) {
  return dtype == GS_BFLOAT16 ? f(__nv_bfloat16{}) : f(__half{});
}

}  // namespace

uint64_t window_attention_workspace_size(const gs_window_attention_args& a) {
  const int64_t first =
      (sequences_of(a) + chunk_slots(a)) * a.kv_heads * a.first * 2 * a.dim;
  return sizeof(float) * static_cast<uint64_t>(delta_floats(a) + peak_floats(a) + first);
}

int32_t launch_window_attention(const gs_window_attention_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (a.num_tiles == 0) return GS_OK;
  return with_sixteen_bit(a.dtype, [&](auto t) {
    using T = decltype(t);
    return a.dim <= 64 ? forward<T, 64>(a, stream) : forward<T, 128>(a, stream);
  });
}

int32_t window_attention_status(cudaStream_t stream) { return take_timeout(g_timeout, stream); }

int32_t launch_window_attention_backward(const gs_window_attention_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (a.num_tiles == 0) return GS_OK;
  if (!a.lse || !a.grad_out || !a.grad_q || !a.grad_k || !a.grad_v || !a.workspace)
    return GS_ERR_INVALID_ARGUMENT;
  for (const void* p : {a.grad_out, static_cast<const void*>(a.grad_q),
                        static_cast<const void*>(a.grad_k), static_cast<const void*>(a.grad_v)})
    if (!is_aligned(p, 16)) return GS_ERR_MISALIGNED;
  if (!is_aligned(a.workspace, 256)) return GS_ERR_MISALIGNED;
  if (a.workspace_size < window_attention_workspace_size(a)) return GS_ERR_CAPACITY;
  return with_sixteen_bit(a.dtype, [&](auto t) {
    using T = decltype(t);
    return a.dim <= 64 ? backward<T, 64>(a, stream) : backward<T, 128>(a, stream);
  });
}

int32_t launch_window_attention_step(const gs_window_attention_step_args& a, cudaStream_t stream) {
  GS_TRY(check_heads(a.heads, a.kv_heads, a.dim, a.dtype));
  if (a.batch < 0 || a.first < 0 || a.slots <= a.first || a.batch > GS_MAX_SEQUENCE_TOKENS / a.slots ||
      !(a.scale > 0.0f && a.scale < INFINITY))
    return GS_ERR_INVALID_ARGUMENT;
  if (a.batch == 0) return GS_OK;
  if (!a.q || !a.k || !a.v || !a.cache_k || !a.cache_v || !a.positions || !a.out ||
      (a.valid && !a.cache_valid))
    return GS_ERR_INVALID_ARGUMENT;
  if (!strided16(a.q, a.q_stride, a.q_head_stride) ||
      !strided16(a.k, a.k_stride, a.k_head_stride) ||
      !strided16(a.v, a.v_stride, a.v_head_stride) || !is_aligned(a.cache_k, 16) ||
      !is_aligned(a.cache_v, 16) || !is_aligned(a.out, 16) || !is_aligned(a.positions, 8))
    return GS_ERR_MISALIGNED;
  return with_sixteen_bit(a.dtype, [&](auto t) {
    using T = decltype(t);
    const auto shaped = [&](auto masked) {
      constexpr bool kMasked = decltype(masked)::value;
      if (a.heads / a.kv_heads <= 8)
        return a.dim <= 64 ? step<T, 64, 1, kMasked>(a, stream)
                           : step<T, 128, 1, kMasked>(a, stream);
      return a.dim <= 64 ? step<T, 64, 2, kMasked>(a, stream)
                         : step<T, 128, 2, kMasked>(a, stream);
    };
    return a.cache_valid ? shaped(std::true_type{}) : shaped(std::false_type{});
  });
}

}  // namespace gs
