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
// exponentials, sums and accumulators are float. Keys that no query sees are
// never read into a sum, so what they hold (infinities, NaN) does not matter.

#include "tensorcore.cuh"

namespace gs {

int32_t launch_window_attention(const gs_window_attention_args& a, cudaStream_t stream);
int32_t launch_window_attention_backward(const gs_window_attention_args& a, cudaStream_t stream);
int32_t launch_window_attention_step(const gs_window_attention_step_args& a, cudaStream_t stream);
int32_t window_attention_status(cudaStream_t stream);
uint64_t window_attention_workspace_size(int64_t tokens, int64_t heads);

namespace {

constexpr int kTile = GS_SEQUENCE_TILE;  // queries (or keys) of a block
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 128;
constexpr int kWords = kMaxDim / 32;  // channels of a row that a lane sums

template <class T>
__device__ __forceinline__ float dot(const float* a, const T* b, int dim) {
  float s = 0.0f;
  for (int c = 0; c < dim; c += 8) {
    float x[8];
    load_pack<8>(b + c, x);
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fmaf(a[c + k], x[k], s);
  }
  return s;
}

template <class T>
__device__ __forceinline__ void stage_row(float* row, const T* p, int dim, int lane) {
  for (int c = lane; c < dim; c += 32) row[c] = to_float(p[c]);
  __syncwarp();
}

// acc += sum over the warp's 32 (weight, row) pairs, lanes over the channels.
template <class T>
__device__ __forceinline__ void add_rows(float (&acc)[kWords], float weight, const T* base,
                                         int64_t stride, int64_t row, int dim, int lane) {
  for (int l = 0; l < 32; ++l) {
    const float w = __shfl_sync(0xffffffffu, weight, l);
    const int64_t r = __shfl_sync(0xffffffffu, row, l);
    if (w == 0.0f) continue;
#pragma unroll
    for (int k = 0; k < kWords; ++k)
      if (lane + 32 * k < dim) acc[k] = fmaf(w, to_float(base[r * stride + lane + 32 * k]), acc[k]);
  }
}

template <class T>
__device__ __forceinline__ void store_row(T* p, const float (&acc)[kWords], float scale, int dim,
                                          int lane) {
#pragma unroll
  for (int k = 0; k < kWords; ++k)
    if (lane + 32 * k < dim) p[lane + 32 * k] = from_float<T>(acc[k] * scale);
}

// The keys a query sees, in at most two runs: first tokens before the window,
// and the window.
struct Runs {
  int low, high, head;
  __device__ __forceinline__ Runs(const gs_window_attention_args& a, int i, int n) {
    low = static_cast<int>(max(int64_t{0}, int64_t{i} - a.left));
    high = static_cast<int>(min(int64_t{n}, int64_t{i} + a.right + 1));
    head = min(a.first, low);
  }
  __device__ __forceinline__ int count() const { return head + high - low; }
  __device__ __forceinline__ int key(int index) const {
    return index < head ? index : low + index - head;
  }
};

// -------------------------------------------------- whole sequences, forward
//
// One block: kTile queries of one head, walked over the tiles of kKeys keys
// that they see: first the tiles of first tokens that lie before the block's
// window, then the window. Four warps hold a query a thread; a fifth warp's
// first thread loads the tiles and issues the products.
//
//   scores  S = Q K^T            tensor memory, 128 x 64 floats
//   P = exp2(S scale log2 e - m) each thread its row; 16 bits, over S
//   O (+)= P V                   tensor memory, 128 x dim floats
//
// m is the row's running maximum, but moves only when it has grown by more
// than 2^8: until then P stays at most 2^8, which both types hold with all
// their precision, and O need not be rescaled.

constexpr int kKeys = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.0f;  // log2 of the growth that m lets pass

// A wait ran out (never in a working kernel): set for
// gs_window_attention_status, the block's results are not valid.
__device__ uint32_t g_timeout;

// 64 bits with those under `n` set.
__device__ __forceinline__ uint64_t below(int64_t n) {
  return n <= 0 ? 0 : n >= 64 ? ~uint64_t{0} : (uint64_t{1} << n) - 1;
}

// The keys that a tile of queries walks over, as tiles of kKeys: positions in
// the sequence.
struct KeyWalk {
  int n, low, high, head, head_tiles, tiles;
  __device__ __forceinline__ KeyWalk(const gs_window_attention_args& a, const Tile& tile) {
    n = tile.end - tile.begin;
    const int64_t i = tile.start - tile.begin;
    const int64_t last = min(i + kTile, int64_t{n}) - 1;
    low = static_cast<int>(max(int64_t{0}, i - a.left));
    high = static_cast<int>(min(int64_t{n}, last + a.right + 1));
    head = min(a.first, low);
    head_tiles = (head + kKeys - 1) / kKeys;
    tiles = head_tiles + (high - low + kKeys - 1) / kKeys;
  }
  __device__ __forceinline__ int start(int t) const {
    return t < head_tiles ? t * kKeys : low + (t - head_tiles) * kKeys;
  }
  // Keys of tile t that may be seen at all: those under this position.
  __device__ __forceinline__ int end(int t) const { return t < head_tiles ? head : n; }
};

// Which of the keys at `start` query i sees, were all valid and in the tile.
__device__ __forceinline__ uint64_t window_bits(const gs_window_attention_args& a, int64_t i,
                                                int start, int end) {
  const int64_t high = min(i + a.right + 1, int64_t{end});
  return below(high - start) & (~below(i - a.left - start) | below(a.first - start));
}

// The valid keys among the 64 from row `row` on (bits from `rows` on are 0);
// every lane of the warp gets them.
__device__ __forceinline__ uint64_t valid_bits(const uint8_t* valid, int64_t row, int rows) {
  if (!valid) return below(rows);
  const int lane = threadIdx.x & 31;
  const bool low = lane < rows && __ldg(valid + row + lane);
  const bool high = lane + 32 < rows && __ldg(valid + row + lane + 32);
  return static_cast<uint64_t>(__ballot_sync(0xffffffffu, high)) << 32 |
         __ballot_sync(0xffffffffu, low);
}

// Zeroes the rows of a loaded tile (kDim channels, kRows = 64 rows) whose bit
// is not set, so that what they hold (another sequence's rows, NaN of invalid
// keys) cannot reach a sum through a weight of zero.
template <int kDim, int kThreadCount>
__device__ __forceinline__ void zero_rows(unsigned char* tile, uint64_t keep, int tid) {
  constexpr int kPerRow = kThreadCount / 64;  // threads of a row
  constexpr int kWordsEach = 8 / kPerRow;
  const int row = tid / kPerRow;
  if (keep >> row & 1) return;
#pragma unroll
  for (int box = 0; box < kDim / 64; ++box)
#pragma unroll
    for (int w = 0; w < kWordsEach; ++w)
      *reinterpret_cast<uint4*>(tile + box * 8192 + row * 128 +
                                ((tid % kPerRow) * kWordsEach + w) * 16) = make_uint4(0, 0, 0, 0);
}

template <int kDim>
struct ForwardShared {
  static constexpr int kKeyStages = 2, kValueStages = 2;
  static constexpr int kQueryBytes = kTile * kDim * 2, kTileBytes = kKeys * kDim * 2;
  alignas(1024) unsigned char q[kQueryBytes];
  unsigned char k[kKeyStages][kTileBytes];
  unsigned char v[kValueStages][kTileBytes];
  uint64_t q_full, k_full[kKeyStages], v_full[kValueStages];  // loads
  uint64_t scores;   // S of a tile is complete
  uint64_t weights;  // P of a tile is written (128 arrivals)
  uint64_t summed;   // O has a tile's sum
  uint32_t tensor;
};

template <class T, int kDim>
__global__ void __launch_bounds__(kTile + 32, kDim == 64 ? 4 : 2)
    attention_kernel(gs_window_attention_args a, const __grid_constant__ CUtensorMap q_map,
                     const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap v_map) {
  using namespace tc;
  using Shared = ForwardShared<kDim>;
  constexpr int kScoreColumn = 0, kOutColumn = kKeys;
  constexpr int kColumns = kDim == 64 ? 128 : 256;
  constexpr int kBoxes = kDim / 64;
  extern __shared__ __align__(1024) unsigned char shared_bytes[];
  Shared& s = *reinterpret_cast<Shared*>(shared_bytes);
  chain_wait();
  const int warp = threadIdx.x >> 5;
  const int head = blockIdx.x % a.heads, kv_head = head / (a.heads / a.kv_heads);
  const Tile tile =
      tile_at(a.tiles, blockIdx.x / a.heads, static_cast<int32_t>(a.tokens), kTile);
  const KeyWalk walk(a, tile);
  if (threadIdx.x == 0) {
    barrier_init(shared_address(&s.q_full), 1);
    for (uint64_t& b : s.k_full) barrier_init(shared_address(&b), 1);
    for (uint64_t& b : s.v_full) barrier_init(shared_address(&b), 1);
    barrier_init(shared_address(&s.scores), 1);
    barrier_init(shared_address(&s.weights), kTile);
    barrier_init(shared_address(&s.summed), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
  }
  if (warp == 4) tensor_alloc<kColumns>(shared_address(&s.tensor));
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tensor = s.tensor;
  bool good = true;

  if (warp == 4) {
    if ((threadIdx.x & 31) == 0) {
      const auto load = [&](unsigned char* dst, uint64_t* bar, const CUtensorMap* map, int h,
                            int row, int bytes, int box_bytes) {
        const uint32_t b = shared_address(bar), d = shared_address(dst);
        barrier_expect(b, bytes);
        for (int x = 0; x < kBoxes; ++x) load_box(d + x * box_bytes, map, 64 * x, h, row, b);
      };
      const auto load_keys = [&](int t) {
        load(s.k[t % Shared::kKeyStages], &s.k_full[t % Shared::kKeyStages], &k_map, kv_head,
             tile.begin + walk.start(t), Shared::kTileBytes, kKeys * 128);
      };
      const auto load_values = [&](int t) {
        load(s.v[t % Shared::kValueStages], &s.v_full[t % Shared::kValueStages], &v_map, kv_head,
             tile.begin + walk.start(t), Shared::kTileBytes, kKeys * 128);
      };
      load(s.q, &s.q_full, &q_map, head, tile.start, Shared::kQueryBytes, kTile * 128);
      for (int t = 0; t < Shared::kKeyStages && t < walk.tiles; ++t) load_keys(t);
      for (int t = 0; t < Shared::kValueStages && t < walk.tiles; ++t) load_values(t);

      const int steps = (a.dim + 15) / 16;
      const uint32_t score_kind = product_kind<T>(kKeys, false);
      const uint32_t sum_kind = product_kind<T>((a.dim + 15) / 16 * 16, true);
      const uint32_t q = shared_address(s.q);
      const auto issue_scores = [&](int t) {
        const int stage = t % Shared::kKeyStages;
        good = good && barrier_wait(shared_address(&s.k_full[stage]),
                                    (t / Shared::kKeyStages) & 1);
        const uint32_t k = shared_address(s.k[stage]);
        for (int i = 0; i < steps; ++i)
          multiply(tensor + kScoreColumn, along_channels<kTile>(q, i), along_channels<kKeys>(k, i),
                   score_kind, i > 0);
        commit(shared_address(&s.scores));
      };
      good = barrier_wait(shared_address(&s.q_full), 0);
      if (good) issue_scores(0);
      int t = 0;
      for (; t < walk.tiles && good; ++t) {
        good = barrier_wait(shared_address(&s.weights), t & 1);
        if (!good) break;
        fence_after_sync();
        // P(t) was written from S(t): the products that read K(t) are complete.
        if (t + Shared::kKeyStages < walk.tiles) load_keys(t + Shared::kKeyStages);
        const int stage = t % Shared::kValueStages;
        good = barrier_wait(shared_address(&s.v_full[stage]), (t / Shared::kValueStages) & 1);
        const uint32_t v = shared_address(s.v[stage]);
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i)
          multiply_tensor(tensor + kOutColumn, tensor + kScoreColumn + 8 * i,
                          along_rows<kKeys>(v, i), sum_kind, t > 0 || i > 0);
        commit(shared_address(&s.summed));
        // In order behind the product that reads P(t).
        if (t + 1 < walk.tiles) issue_scores(t + 1);
        // S(t) was complete behind the sum of t - 1: V(t - 1) is free.
        if (t >= 1 && t - 1 + Shared::kValueStages < walk.tiles)
          load_values(t - 1 + Shared::kValueStages);
      }
      if (!good) {
        // Let what is in flight land before the shared memory is given back.
        for (uint64_t& b : s.k_full)
          for (int p = 0; p < 2; ++p) barrier_wait(shared_address(&b), p);
        for (uint64_t& b : s.v_full)
          for (int p = 0; p < 2; ++p) barrier_wait(shared_address(&b), p);
        atomicExch(&g_timeout, 1u);
      }
    }
    __syncwarp();
  } else {
    const int row = threadIdx.x, lane = threadIdx.x & 31;
    const uint32_t mine = tensor + (static_cast<uint32_t>(warp * 32) << 16);
    const int64_t i = tile.start - tile.begin + row;  // the query's position
    const float scale = a.scale * kLog2e;
    float top = -INFINITY, sum = 0.0f;
    // The first and the last query of the block, for what all of them see.
    const int64_t i_first = tile.start - tile.begin, i_last = i_first + kTile - 1;
    for (int t = 0; t < walk.tiles; ++t) {
      const int start = walk.start(t), end = walk.end(t);
      const uint64_t keep =
          valid_bits(a.valid, int64_t{tile.begin} + start, min(end - start, kKeys));
      const bool whole = keep == ~uint64_t{0} && (t < walk.head_tiles ||
                                                  (start + kKeys <= i_first + a.right + 1 &&
                                                   (start >= i_last - a.left ||
                                                    start + kKeys <= a.first)));
      if (!(good = barrier_wait_warp(shared_address(&s.scores), t & 1))) break;
      fence_after_sync();
      float x[2][32];
      load_columns32(mine + kScoreColumn, x[0]);
      load_columns32(mine + kScoreColumn + 32, x[1]);
      wait_loads();
      if (!whole) {
        const uint64_t bits = keep & window_bits(a, i, start, end);
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          x[0][c] = bits >> c & 1 ? x[0][c] : -INFINITY;
          x[1][c] = bits >> (c + 32) & 1 ? x[1][c] : -INFINITY;
        }
      }
      float high[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        high[c & 1] = fmaxf(high[c & 1], x[0][c]);
        high[2 + (c & 1)] = fmaxf(high[2 + (c & 1)], x[1][c]);
      }
      const float next =
          fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3])) * scale;
      // Sums of earlier tiles are complete: this tile's S came behind them.
      const bool grow = next > top + kSlack || (top == -INFINITY && next > top);
      if (__any_sync(0xffffffffu, grow)) {
        const float shrink = grow ? exp2_approx(top - next) : 1.0f;
        if (grow) top = next;
        sum *= shrink;
        if (t > 0) {
#pragma unroll 1
          for (int c = 0; c < kDim; c += 16) {
            float o[16];
            load_columns16(mine + kOutColumn + c, o);
            wait_loads();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= shrink;
            store_columns16(mine + kOutColumn + c, o);
          }
        }
      }
      // Where nothing is seen yet any finite shift will do: exp2(-inf) is 0.
      const float shift = top == -INFINITY ? 0.0f : -top;
      float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      uint32_t packed[2][16];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float p0 = exp2_approx(fmaf(x[half][2 * c], scale, shift));
          const float p1 = exp2_approx(fmaf(x[half][2 * c + 1], scale, shift));
          part[2 * half] += p0;
          part[2 * half + 1] += p1;
          packed[half][c] = pack2<T>(p0, p1);
        }
        store_columns16(mine + kScoreColumn + 16 * half, packed[half]);
      }
      sum += (part[0] + part[1]) + (part[2] + part[3]);
      if (keep != ~uint64_t{0}) {
        const int stage = t % Shared::kValueStages;
        if (!(good = barrier_wait_warp(shared_address(&s.v_full[stage]),
                                  (t / Shared::kValueStages) & 1)))
          break;
        zero_rows<kDim, kTile>(s.v[stage], keep, row);
        fence_async_shared();
      }
      wait_stores();
      fence_before_sync();
      barrier_arrive(shared_address(&s.weights));
    }
    if (good) good = barrier_wait_warp(shared_address(&s.summed), (walk.tiles - 1) & 1);
    fence_after_sync();
    const bool write = tile.start + row < tile.end;
    const float inverse = 1.0f / sum;
    T* out = static_cast<T*>(a.out) + (int64_t{tile.start + row} * a.heads + head) * a.dim;
#pragma unroll
    for (int c = 0; c < kDim; c += 32) {
      float o[32];
      load_columns32(mine + kOutColumn + c, o);
      wait_loads();
#pragma unroll
      for (int e = 0; e < 32; e += 8)
        if (write && c + e < a.dim) {
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            v[k] = good ? (sum == 0.0f ? 0.0f : o[e + k] * inverse) : NAN;
          store_pack<8>(out + c + e, v);
        }
    }
    if (write && a.lse)
      a.lse[head * a.tokens + tile.start + row] =
          sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
    if (!good && lane == 0) atomicExch(&g_timeout, 1u);
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 4) tensor_free<kColumns>(tensor);
}

template <class T, int kDim>
int32_t forward(const gs_window_attention_args& a, cudaStream_t stream) {
  constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
  CUtensorMap q, k, v;
  GS_TRY(tc::encode_map(&q, kBf16, a.q, a.tokens, a.heads, a.dim, a.q_stride, a.q_head_stride,
                        kTile));
  GS_TRY(tc::encode_map(&k, kBf16, a.k, a.tokens, a.kv_heads, a.dim, a.k_stride, a.k_head_stride,
                        kKeys));
  GS_TRY(tc::encode_map(&v, kBf16, a.v, a.tokens, a.kv_heads, a.dim, a.v_stride, a.v_head_stride,
                        kKeys));
  constexpr size_t kShared = sizeof(ForwardShared<kDim>);
  GS_CUDA_TRY(cudaFuncSetAttribute(attention_kernel<T, kDim>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, kShared));
  launch_chained_shared(attention_kernel<T, kDim>, static_cast<unsigned>(a.num_tiles * a.heads),
                        kTile + 32, kShared, stream, a, q, k, v);
  return check_launch();
}

// dq, and D_i into `delta` for the keys' kernel.
template <class T>
__global__ void __launch_bounds__(kThreads) grad_query_kernel(gs_window_attention_args a,
                                                              float* delta) {
  chain_wait();
  __shared__ float s_row[kWarps][kMaxDim], s_grad[kWarps][kMaxDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Tile tile = tile_at(a.tiles, blockIdx.x, static_cast<int32_t>(a.tokens), kTile);
  const int head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
  const T* k = static_cast<const T*>(a.k) + kv_head * a.k_head_stride;
  const T* v = static_cast<const T*>(a.v) + kv_head * a.v_head_stride;
  const int last = min(tile.end, tile.start + kTile);
  for (int t = tile.start + warp; t < last; t += kWarps) {
    __syncwarp();
    const int64_t at = (int64_t{t} * a.heads + head) * a.dim;
    stage_row(s_row[warp], static_cast<const T*>(a.q) + t * a.q_stride + head * a.q_head_stride,
              a.dim, lane);
    stage_row(s_grad[warp], static_cast<const T*>(a.grad_out) + at, a.dim, lane);
    const T* out = static_cast<const T*>(a.out) + at;
    float d = 0.0f;
    for (int c = lane; c < a.dim; c += 32) d = fmaf(s_grad[warp][c], to_float(out[c]), d);
    d = warp_sum(d);
    const float lse = a.lse[head * a.tokens + t];
    if (lane == 0) delta[head * a.tokens + t] = d;
    const Runs runs(a, t - tile.begin, tile.end - tile.begin);
    float acc[kWords] = {};
    if (lse != -INFINITY)
      for (int base = 0; base < runs.count(); base += 32) {
        const bool in = base + lane < runs.count();
        const int64_t key = tile.begin + (in ? runs.key(base + lane) : 0);
        float e = 0.0f;
        if (in && (!a.valid || a.valid[key])) {
          const float p = expf(fmaf(dot(s_row[warp], k + key * a.k_stride, a.dim), a.scale, -lse));
          e = p * (dot(s_grad[warp], v + key * a.v_stride, a.dim) - d);
        }
        add_rows(acc, e, k, a.k_stride, key, a.dim, lane);
      }
    store_row(static_cast<T*>(a.grad_q) + at, acc, a.scale, a.dim, lane);
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) grad_key_kernel(gs_window_attention_args a,
                                                            const float* delta) {
  chain_wait();
  __shared__ float s_key[kWarps][kMaxDim], s_value[kWarps][kMaxDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Tile tile = tile_at(a.tiles, blockIdx.x, static_cast<int32_t>(a.tokens), kTile);
  const int kv_head = blockIdx.y, group = a.heads / a.kv_heads;
  const int last = min(tile.end, tile.start + kTile), n = tile.end - tile.begin;
  for (int t = tile.start + warp; t < last; t += kWarps) {
    __syncwarp();
    float dk[kWords] = {}, dv[kWords] = {};
    if (!a.valid || a.valid[t]) {
      stage_row(s_key[warp], static_cast<const T*>(a.k) + t * a.k_stride + kv_head * a.k_head_stride,
                a.dim, lane);
      stage_row(s_value[warp],
                static_cast<const T*>(a.v) + t * a.v_stride + kv_head * a.v_head_stride, a.dim,
                lane);
      const int64_t j = t - tile.begin;
      const int64_t from = max(int64_t{0}, j - a.right);
      const int64_t to = j < a.first ? n : min(int64_t{n}, j + a.left + 1);
      for (int h = kv_head * group; h < (kv_head + 1) * group; ++h) {
        const T* q = static_cast<const T*>(a.q) + h * a.q_head_stride;
        const T* g = static_cast<const T*>(a.grad_out) + int64_t{h} * a.dim;
        const int64_t g_stride = int64_t{a.heads} * a.dim;
        for (int64_t base = from; base < to; base += 32) {
          const bool in = base + lane < to;
          const int64_t row = tile.begin + (in ? base + lane : 0);
          float p = 0.0f, e = 0.0f;
          if (in) {
            const float lse = a.lse[h * a.tokens + row];
            p = expf(fmaf(dot(s_key[warp], q + row * a.q_stride, a.dim), a.scale, -lse));
            e = p * (dot(s_value[warp], g + row * g_stride, a.dim) - delta[h * a.tokens + row]);
          }
          add_rows(dk, e, q, a.q_stride, row, a.dim, lane);
          add_rows(dv, p, g, g_stride, row, a.dim, lane);
        }
      }
    }
    const int64_t at = (int64_t{t} * a.kv_heads + kv_head) * a.dim;
    store_row(static_cast<T*>(a.grad_k) + at, dk, a.scale, a.dim, lane);
    store_row(static_cast<T*>(a.grad_v) + at, dv, 1.0f, a.dim, lane);
  }
}

// One new token a stream against its cache of `slots` tokens: the first
// `first` tokens keep their slots, later ones take the others in turn. The new
// token's key and value come from the arguments; the block of a key-value
// head's first query head also writes them to their slot, which no block reads.
template <class T>
__global__ void __launch_bounds__(kThreads) attention_step_kernel(gs_window_attention_step_args a) {
  chain_wait();
  __shared__ float s_row[kMaxDim], s_acc[kWarps][kMaxDim], s_top[kWarps], s_sum[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t b = blockIdx.x;
  const int head = blockIdx.y, group = a.heads / a.kv_heads, kv_head = head / group;
  const int64_t position = a.positions[b];
  T* out = static_cast<T*>(a.out) + (b * a.heads + head) * a.dim;
  if (position < 0) {
    for (int c = threadIdx.x; c < a.dim; c += kThreads) out[c] = from_float<T>(0.0f);
    return;
  }
  const int64_t slot = position < a.first
                           ? position
                           : a.first + (position - a.first) % (a.slots - a.first);
  const int count = static_cast<int>(min(position + 1, int64_t{a.slots}));
  const int64_t row = int64_t{a.kv_heads} * a.dim;
  T* cache_k = static_cast<T*>(a.cache_k) + b * a.slots * row + kv_head * a.dim;
  T* cache_v = static_cast<T*>(a.cache_v) + b * a.slots * row + kv_head * a.dim;
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride + kv_head * a.k_head_stride;
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride + kv_head * a.v_head_stride;
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride + head * a.q_head_stride;
  if (head % group == 0)
    for (int c = threadIdx.x; c < a.dim; c += kThreads) {
      cache_k[slot * row + c] = k[c];
      cache_v[slot * row + c] = v[c];
    }
  for (int c = threadIdx.x; c < a.dim; c += kThreads) s_row[c] = to_float(q[c]);
  __syncthreads();
  float top = -INFINITY, sum = 0.0f, acc[kWords] = {};
  for (int base = 32 * warp; base < count; base += kThreads) {
    const bool in = base + lane < count;
    float s = -INFINITY;
    if (in) s = dot(s_row, base + lane == slot ? k : cache_k + (base + lane) * row, a.dim) * a.scale;
    const float next = fmaxf(top, warp_max(s));
    const float p = in ? expf(s - next) : 0.0f, shrink = expf(top - next);
    top = next;
    sum = fmaf(sum, shrink, warp_sum(p));
#pragma unroll
    for (int c = 0; c < kWords; ++c) acc[c] *= shrink;
    for (int l = 0; l < min(32, count - base); ++l) {
      const float w = __shfl_sync(0xffffffffu, p, l);
      const T* value = base + l == slot ? v : cache_v + (base + l) * row;
#pragma unroll
      for (int c = 0; c < kWords; ++c)
        if (lane + 32 * c < a.dim) acc[c] = fmaf(w, to_float(value[lane + 32 * c]), acc[c]);
    }
  }
  if (lane == 0) {
    s_top[warp] = top;
    s_sum[warp] = sum;
  }
#pragma unroll
  for (int c = 0; c < kWords; ++c) s_acc[warp][lane + 32 * c] = acc[c];
  __syncthreads();
  float whole = -INFINITY, total = 0.0f;
  for (int w = 0; w < kWarps; ++w) whole = fmaxf(whole, s_top[w]);
  for (int w = 0; w < kWarps; ++w) total = fmaf(s_sum[w], expf(s_top[w] - whole), total);
  for (int c = threadIdx.x; c < a.dim; c += kThreads) {
    float o = 0.0f;
    for (int w = 0; w < kWarps; ++w) o = fmaf(s_acc[w][c], expf(s_top[w] - whole), o);
    out[c] = from_float<T>(o / total);
  }
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
  if (a.tokens < 0 || a.tokens > INT32_MAX || a.num_tiles < 0 || a.num_tiles > INT32_MAX / a.heads ||
      a.left < 0 || a.right < 0 || a.first < 0 || a.first > GS_MAX_FIRST_TOKENS ||
      !(a.scale > 0.0f && a.scale < INFINITY))
    return GS_ERR_INVALID_ARGUMENT;
  if (!a.tiles && a.num_tiles != (a.tokens + kTile - 1) / kTile) return GS_ERR_INVALID_ARGUMENT;
  if (!is_aligned(a.tiles, 16)) return GS_ERR_MISALIGNED;
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

uint64_t window_attention_workspace_size(int64_t tokens, int64_t heads) {
  return sizeof(float) * static_cast<uint64_t>(tokens) * heads;
}

int32_t launch_window_attention(const gs_window_attention_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (a.num_tiles == 0) return GS_OK;
  return with_sixteen_bit(a.dtype, [&](auto t) {
    using T = decltype(t);
    return a.dim <= 64 ? forward<T, 64>(a, stream) : forward<T, 128>(a, stream);
  });
}

int32_t window_attention_status(cudaStream_t stream) {
  uint32_t timeout = 0;
  const uint32_t clear = 0;
  GS_CUDA_TRY(cudaMemcpyFromSymbolAsync(&timeout, g_timeout, sizeof(timeout), 0,
                                        cudaMemcpyDeviceToHost, stream));
  GS_CUDA_TRY(cudaMemcpyToSymbolAsync(g_timeout, &clear, sizeof(clear), 0,
                                      cudaMemcpyHostToDevice, stream));
  GS_CUDA_TRY(cudaStreamSynchronize(stream));
  return timeout ? GS_ERR_TIMEOUT : GS_OK;
}

int32_t launch_window_attention_backward(const gs_window_attention_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (a.num_tiles == 0) return GS_OK;
  if (!a.lse || !a.grad_out || !a.grad_q || !a.grad_k || !a.grad_v || !a.workspace)
    return GS_ERR_INVALID_ARGUMENT;
  for (const void* p : {a.grad_out, static_cast<const void*>(a.grad_q),
                        static_cast<const void*>(a.grad_k), static_cast<const void*>(a.grad_v)})
    if (!is_aligned(p, 16)) return GS_ERR_MISALIGNED;
  if (a.workspace_size < window_attention_workspace_size(a.tokens, a.heads))
    return GS_ERR_CAPACITY;
  float* delta = static_cast<float*>(a.workspace);
  return with_sixteen_bit(a.dtype, [&](auto t) {
    using T = decltype(t);
    launch_chained(grad_query_kernel<T>, dim3(a.num_tiles, a.heads), kThreads, stream, a, delta);
    GS_TRY(check_launch());
    launch_chained(grad_key_kernel<T>, dim3(a.num_tiles, a.kv_heads), kThreads, stream, a,
                   static_cast<const float*>(delta));
    return check_launch();
  });
}

int32_t launch_window_attention_step(const gs_window_attention_step_args& a, cudaStream_t stream) {
  GS_TRY(check_heads(a.heads, a.kv_heads, a.dim, a.dtype));
  if (a.batch < 0 || a.batch > INT32_MAX || a.first < 0 || a.slots <= a.first ||
      !(a.scale > 0.0f && a.scale < INFINITY))
    return GS_ERR_INVALID_ARGUMENT;
  if (a.batch == 0) return GS_OK;
  if (!a.q || !a.k || !a.v || !a.cache_k || !a.cache_v || !a.positions || !a.out)
    return GS_ERR_INVALID_ARGUMENT;
  if (!strided16(a.q, a.q_stride, a.q_head_stride) ||
      !strided16(a.k, a.k_stride, a.k_head_stride) ||
      !strided16(a.v, a.v_stride, a.v_head_stride) || !is_aligned(a.cache_k, 16) ||
      !is_aligned(a.cache_v, 16) || !is_aligned(a.out, 16) || !is_aligned(a.positions, 8))
    return GS_ERR_MISALIGNED;
  return with_sixteen_bit(a.dtype, [&](auto t) {
    using T = decltype(t);
    launch_chained(attention_step_kernel<T>, dim3(a.batch, a.heads), kThreads, stream, a);
    return check_launch();
  });
}

}  // namespace gs
