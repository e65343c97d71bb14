// The gated linear recurrence along a packed batch of sequences,
//
//   h_t = k_t h_{t-1} + a_t x_t,   a_t = sigmoid(gate_t),  k_t = 1 - a_t,
//
// channel by channel: alpha compositing's "over" with a learned opacity, walked
// along the tokens. Backward, with g_t the gradient of h_t = y_t and the message
// u_t = k_t (g_t + u_{t+1}) that token t hands to token t-1 (u after the last
// token: the gradient of the last state),
//
//   l_t = g_t + u_{t+1},  dx_t = a_t l_t,  dgate_t = l_t (x_t - h_{t-1}) a_t k_t,
//
// and u_1 is the gradient of the initial state. Both directions are chains of
// maps s -> A s + B, which compose associatively, so the sequence is cut into
// tiles of kTile tokens: one kernel folds each tile to its (A, B), one scans the
// tiles of each sequence for the state that enters each tile, one walks the
// tiles from those states. Inside a tile, each warp holds kTokens tokens of 32
// lanes' channels in registers and the warps' folds are joined in order in
// shared memory. Every order is fixed, so results repeat bit for bit.
//
// States, products and gates are float; the states that enter the tiles are
// kept in float for the backward, which recomputes h from them instead of
// reading the rounded y.

#include "sequence.cuh"

namespace gs {

int32_t launch_gated_scan(const gs_gated_scan_args& a, cudaStream_t stream);
int32_t launch_gated_scan_backward(const gs_gated_scan_args& a, cudaStream_t stream);
int32_t launch_gated_scan_step(int64_t batch, int32_t channels, int32_t dtype, const void* x,
                               int64_t x_stride, const void* gate, int64_t gate_stride,
                               float* state, void* y, cudaStream_t stream);
uint64_t gated_scan_workspace_size(int64_t num_tiles, int64_t channels);

namespace {

constexpr int kTile = GS_SEQUENCE_TILE;
constexpr int kTokens = 8;               // tokens a thread holds
constexpr int kWarps = kTile / kTokens;  // warps of a tile's block
constexpr int kThreads = 32 * kWarps;
constexpr int kScanWarps = 16;  // warps that share a sequence's tiles in the tile scan

// a = sigmoid(gate) and k = 1 - a, both with small relative error: the smaller
// of the two is e / (1 + e) with e = exp(-|gate|), never a difference.
__device__ __forceinline__ void open_gate(float gate, float& a, float& k) {
  const float e = __expf(-fabsf(gate));
  const float large = __fdividef(1.0f, 1.0f + e), small = e * large;
  a = gate >= 0.0f ? large : small;
  k = gate >= 0.0f ? small : large;
}

// A map s -> a s + b.
struct Affine {
  float a, b;
};

// What a block works on: a tile of tokens and 32 V channels, V to a lane.
template <int V>
struct Place {
  Tile tile;
  int64_t index;  // of the tile
  int channel;    // the lane's first
  int first, count;  // the warp's tokens in the tile's sequence
  bool live;         // the lane has channels
  __device__ __forceinline__ Place(const gs_gated_scan_args& a, bool reverse) {
    const int columns = (a.channels + 32 * V - 1) / (32 * V);
    index = blockIdx.x / columns;
    if (reverse) index = a.num_tiles - 1 - index;
    channel = (static_cast<int>(blockIdx.x % columns) * 32 + (threadIdx.x & 31)) * V;
    live = channel < a.channels;
    tile = tile_at(a.tiles, index, static_cast<int32_t>(a.tokens), kTile);
    first = tile.start + static_cast<int>(threadIdx.x >> 5) * kTokens;
    count = min(kTokens, min(tile.end, tile.start + kTile) - first);
    if (!live) count = 0;
  }
};

template <class T, int V>
__device__ __forceinline__ void load_tokens(const T* p, int64_t stride, int first, int channel,
                                            int count, float (&x)[kTokens][V]) {
#pragma unroll
  for (int t = 0; t < kTokens; ++t)
    if (t < count) load_pack<V>(p + (first + t) * stride + channel, x[t]);
}

// Joins the warps' folds in order (from the last warp if `reverse`): returns
// the map of what comes before the calling warp, and in `whole` the tile's.
template <int V, bool reverse>
__device__ __forceinline__ void join(const Affine (&mine)[V], Affine (&before)[V],
                                     Affine (&whole)[V], Affine (*shared)[32 * V]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int v = 0; v < V; ++v) shared[warp][v * 32 + lane] = mine[v];
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Affine sum = {1.0f, 0.0f};
    before[v] = sum;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int at = reverse ? kWarps - 1 - w : w;
      if (at == warp) before[v] = sum;
      const Affine f = shared[at][v * 32 + lane];
      sum = {f.a * sum.a, fmaf(f.a, sum.b, f.b)};
    }
    whole[v] = sum;
  }
}

// Folds every tile: forward the map of the state through it, backward the map
// of the message through it (from its end to its start).
template <class T, int V, bool kBackward>
__global__ void __launch_bounds__(kThreads) fold_kernel(gs_gated_scan_args a, Affine* folds) {
  chain_wait();
  __shared__ Affine s_fold[kWarps][32 * V];
  const Place<V> p(a, false);
  float x[kTokens][V], gate[kTokens][V];
  load_tokens<T, V>(static_cast<const T*>(a.gate), a.gate_stride, p.first, p.channel, p.count, gate);
  load_tokens<T, V>(static_cast<const T*>(kBackward ? a.grad_y : a.x),
                    kBackward ? int64_t{a.channels} : a.x_stride, p.first, p.channel, p.count, x);
  Affine mine[V], before[V], whole[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    mine[v] = {1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      const int t = kBackward ? kTokens - 1 - i : i;
      if (t < p.count) {
        float al, k;
        open_gate(gate[t][v], al, k);
        mine[v].b = kBackward ? k * (x[t][v] + mine[v].b) : fmaf(k, mine[v].b, al * x[t][v]);
        mine[v].a *= k;
      }
    }
  }
  join<V, kBackward>(mine, before, whole, s_fold);
  if (threadIdx.x < 32 && p.live)
#pragma unroll
    for (int v = 0; v < V; ++v) folds[p.index * a.channels + p.channel + v] = whole[v];
}

// The states (backward: messages) that enter the tiles, one block a sequence
// and 32 channels: each warp folds its share of the sequence's tiles, the
// shares are joined in order, each warp walks its share again.
template <bool kBackward>
__global__ void __launch_bounds__(32 * kScanWarps) tile_scan_kernel(gs_gated_scan_args a,
                                                                    const Affine* folds,
                                                                    float* entering) {
  chain_wait();
  __shared__ Affine s_fold[kScanWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int columns = (a.channels + 31) / 32;
  const int64_t sequence = blockIdx.x / columns;
  const int channel = static_cast<int>(blockIdx.x % columns) * 32 + lane;
  const bool live = channel < a.channels;
  const int64_t begin = a.tile_starts ? __ldg(a.tile_starts + sequence) : 0;
  const int64_t end = a.tile_starts ? __ldg(a.tile_starts + sequence + 1) : a.num_tiles;
  const int64_t share = (end - begin + kScanWarps - 1) / kScanWarps;
  const int64_t from = min(end, begin + warp * share), to = min(end, from + share);
  const auto tile_of = [&](int64_t i) { return kBackward ? begin + end - 1 - i : i; };
  Affine sum = {1.0f, 0.0f};
  if (live)
#pragma unroll 4
    for (int64_t i = from; i < to; ++i) {
      const Affine f = folds[tile_of(i) * a.channels + channel];
      sum = {f.a * sum.a, fmaf(f.a, sum.b, f.b)};
    }
  s_fold[warp][lane] = sum;
  __syncthreads();
  if (!live) return;
  const int64_t slot = sequence * a.channels + channel;
  const float* start = kBackward ? a.grad_last : a.initial;
  float state = start ? start[slot] : 0.0f;
  for (int w = 0; w < warp; ++w) state = fmaf(s_fold[w][lane].a, state, s_fold[w][lane].b);
#pragma unroll 4
  for (int64_t i = from; i < to; ++i) {
    const int64_t at = tile_of(i) * a.channels + channel;
    const Affine f = folds[at];
    entering[at] = state;
    state = fmaf(f.a, state, f.b);
  }
  float* final = kBackward ? a.grad_initial : a.last;
  if (warp == kScanWarps - 1 && final) final[slot] = state;
}

// The walk from the entering states. Tiles go from the last to the first: the
// fold just before read them from the first to the last, so the end of its
// inputs is what L2 still holds.
template <class T, int V>
__global__ void __launch_bounds__(kThreads) walk_kernel(gs_gated_scan_args a) {
  chain_wait();
  __shared__ Affine s_fold[kWarps][32 * V];
  const Place<V> p(a, true);
  float x[kTokens][V], gate[kTokens][V];
  load_tokens<T, V>(static_cast<const T*>(a.gate), a.gate_stride, p.first, p.channel, p.count, gate);
  load_tokens<T, V>(static_cast<const T*>(a.x), a.x_stride, p.first, p.channel, p.count, x);
  Affine mine[V], before[V], whole[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    mine[v] = {1.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < kTokens; ++t)
      if (t < p.count) {
        float al;
        open_gate(gate[t][v], al, gate[t][v]);
        x[t][v] *= al;
        mine[v] = {mine[v].a * gate[t][v], fmaf(gate[t][v], mine[v].b, x[t][v])};
      }
  }
  join<V, false>(mine, before, whole, s_fold);
  if (!p.live) return;
  float state[V];
#pragma unroll
  for (int v = 0; v < V; ++v)
    state[v] = fmaf(before[v].a, a.entering[p.index * a.channels + p.channel + v], before[v].b);
  T* y = static_cast<T*>(a.y);
#pragma unroll
  for (int t = 0; t < kTokens; ++t)
    if (t < p.count) {
#pragma unroll
      for (int v = 0; v < V; ++v) state[v] = fmaf(gate[t][v], state[v], x[t][v]);
      store_pack<V>(y + int64_t{p.first + t} * a.channels + p.channel, state);
    }
}

template <class T, int V>
__global__ void __launch_bounds__(kThreads) walk_back_kernel(gs_gated_scan_args a,
                                                             const float* messages) {
  chain_wait();
  __shared__ Affine s_fold[2][kWarps][32 * V];
  const Place<V> p(a, true);
  float x[kTokens][V], gate[kTokens][V], g[kTokens][V], open[kTokens][V];
  load_tokens<T, V>(static_cast<const T*>(a.gate), a.gate_stride, p.first, p.channel, p.count, gate);
  load_tokens<T, V>(static_cast<const T*>(a.x), a.x_stride, p.first, p.channel, p.count, x);
  load_tokens<T, V>(static_cast<const T*>(a.grad_y), int64_t{a.channels}, p.first, p.channel,
                    p.count, g);
  Affine ahead[V], back[V], before[V], after[V], whole[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    ahead[v] = back[v] = {1.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < kTokens; ++t)
      if (t < p.count) {
        open_gate(gate[t][v], open[t][v], gate[t][v]);
        ahead[v].b = fmaf(gate[t][v], ahead[v].b, open[t][v] * x[t][v]);
        ahead[v].a *= gate[t][v];
      }
#pragma unroll
    for (int t = kTokens - 1; t >= 0; --t)
      if (t < p.count) back[v].b = gate[t][v] * (g[t][v] + back[v].b);
    back[v].a = ahead[v].a;
  }
  join<V, false>(ahead, before, whole, s_fold[0]);
  join<V, true>(back, after, whole, s_fold[1]);
  if (!p.live) return;
  const int64_t slot = p.index * a.channels + p.channel;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float state = fmaf(before[v].a, a.entering[slot + v], before[v].b);
    float message = fmaf(after[v].a, messages[slot + v], after[v].b);
    // forward: x_t becomes x_t - h_{t-1}
#pragma unroll
    for (int t = 0; t < kTokens; ++t)
      if (t < p.count) {
        const float push = open[t][v] * x[t][v];
        x[t][v] -= state;
        state = fmaf(gate[t][v], state, push);
      }
    // back: x_t becomes dgate_t and g_t becomes dx_t
#pragma unroll
    for (int t = kTokens - 1; t >= 0; --t)
      if (t < p.count) {
        const float l = g[t][v] + message;
        message = gate[t][v] * l;
        g[t][v] = open[t][v] * l;
        x[t][v] *= message * open[t][v];
      }
  }
  T* grad_x = static_cast<T*>(a.grad_x);
  T* grad_gate = static_cast<T*>(a.grad_gate);
#pragma unroll
  for (int t = 0; t < kTokens; ++t)
    if (t < p.count) {
      const int64_t at = int64_t{p.first + t} * a.channels + p.channel;
      store_pack<V>(grad_x + at, g[t]);
      store_pack<V>(grad_gate + at, x[t]);
    }
}

template <class T>
__global__ void __launch_bounds__(256) scan_step_kernel(int64_t count, int channels, const T* x,
                                                        int64_t x_stride, const T* gate,
                                                        int64_t gate_stride, float* state, T* y) {
  chain_wait();
  const int64_t i = int64_t{blockIdx.x} * 256 + threadIdx.x;
  if (i >= count) return;
  const int64_t row = i / channels;
  const int c = static_cast<int>(i - row * channels);
  float al, k;
  open_gate(to_float(gate[row * gate_stride + c]), al, k);
  const float h = fmaf(k, state[i], al * to_float(x[row * x_stride + c]));
  state[i] = h;
  y[i] = from_float<T>(h);
}

int32_t check_args(const gs_gated_scan_args& a) {
  if (a.tokens < 0 || a.tokens > INT32_MAX || a.channels < 1 || a.sequences < 1 ||
      a.num_tiles < 0 || a.dtype < GS_FLOAT32 || a.dtype > GS_FLOAT16)
    return GS_ERR_INVALID_ARGUMENT;
  if (a.tile_starts ? (a.num_tiles > 0 && !a.tiles)
                    : (a.tiles || a.sequences != 1 ||
                       a.num_tiles != (a.tokens + kTile - 1) / kTile))
    return GS_ERR_INVALID_ARGUMENT;
  if (!is_aligned(a.tiles, 16)) return GS_ERR_MISALIGNED;
  const int64_t columns = (int64_t{a.channels} + 31) / 32;
  if (columns * (a.num_tiles > a.sequences ? a.num_tiles : a.sequences) > INT32_MAX)
    return GS_ERR_CAPACITY;
  if (a.num_tiles > 0 && (!a.x || !a.gate || !a.entering || !a.workspace))
    return GS_ERR_INVALID_ARGUMENT;
  if (a.workspace_size < gated_scan_workspace_size(a.num_tiles, a.channels))
    return GS_ERR_CAPACITY;
  return GS_OK;
}

// Two 16-bit channels a lane make a warp's row of a tile a full 128-byte line;
// they need even strides and 4-byte aligned arrays. Otherwise one channel a lane.
template <class T>
bool two_channels(const gs_gated_scan_args& a) {
  if (sizeof(T) == 4 || a.channels % 2 || a.x_stride % 2 || a.gate_stride % 2) return false;
  for (const void* p : {a.x, a.gate, a.grad_y, static_cast<const void*>(a.y),
                        static_cast<const void*>(a.grad_x), static_cast<const void*>(a.grad_gate)})
    if (!is_aligned(p, 4)) return false;
  return true;
}

template <class T, int V>
int32_t forward(const gs_gated_scan_args& a, cudaStream_t stream) {
  Affine* folds = static_cast<Affine*>(a.workspace);
  const unsigned blocks = ceil_div(a.channels, 32 * V) * static_cast<unsigned>(a.num_tiles);
  const unsigned chains = ceil_div(a.channels, 32) * static_cast<unsigned>(a.sequences);
  if (blocks) {
    launch_chained(fold_kernel<T, V, false>, blocks, kThreads, stream, a, folds);
    GS_TRY(check_launch());
  }
  launch_chained(tile_scan_kernel<false>, chains, 32 * kScanWarps, stream, a, folds, a.entering);
  GS_TRY(check_launch());
  if (blocks) launch_chained(walk_kernel<T, V>, blocks, kThreads, stream, a);
  return check_launch();
}

template <class T, int V>
int32_t backward(const gs_gated_scan_args& a, cudaStream_t stream) {
  Affine* folds = static_cast<Affine*>(a.workspace);
  float* messages = reinterpret_cast<float*>(folds + a.num_tiles * a.channels);
  const unsigned blocks = ceil_div(a.channels, 32 * V) * static_cast<unsigned>(a.num_tiles);
  const unsigned chains = ceil_div(a.channels, 32) * static_cast<unsigned>(a.sequences);
  if (blocks) {
    launch_chained(fold_kernel<T, V, true>, blocks, kThreads, stream, a, folds);
    GS_TRY(check_launch());
  }
  launch_chained(tile_scan_kernel<true>, chains, 32 * kScanWarps, stream, a, folds, messages);
  GS_TRY(check_launch());
  if (blocks) launch_chained(walk_back_kernel<T, V>, blocks, kThreads, stream, a, messages);
  return check_launch();
}

}  // namespace

uint64_t gated_scan_workspace_size(int64_t num_tiles, int64_t channels) {
  return (sizeof(Affine) + sizeof(float)) * static_cast<uint64_t>(num_tiles) * channels;
}

int32_t launch_gated_scan(const gs_gated_scan_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (!a.last || (a.num_tiles > 0 && !a.y)) return GS_ERR_INVALID_ARGUMENT;
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2)
      if (two_channels<T>(a)) return forward<T, 2>(a, stream);
    return forward<T, 1>(a, stream);
  });
}

int32_t launch_gated_scan_backward(const gs_gated_scan_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (a.num_tiles > 0 && (!a.grad_y || !a.grad_x || !a.grad_gate)) return GS_ERR_INVALID_ARGUMENT;
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2)
      if (two_channels<T>(a)) return backward<T, 2>(a, stream);
    return backward<T, 1>(a, stream);
  });
}

int32_t launch_gated_scan_step(int64_t batch, int32_t channels, int32_t dtype, const void* x,
                               int64_t x_stride, const void* gate, int64_t gate_stride,
                               float* state, void* y, cudaStream_t stream) {
  if (batch < 0 || channels < 1) return GS_ERR_INVALID_ARGUMENT;
  const int64_t count = batch * channels;
  if (count == 0) return GS_OK;
  if (!x || !gate || !state || !y) return GS_ERR_INVALID_ARGUMENT;
  if (count / 256 >= INT32_MAX) return GS_ERR_CAPACITY;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    launch_chained(scan_step_kernel<T>, ceil_div(count, 256), 256, stream, count, channels,
                   static_cast<const T*>(x), x_stride, static_cast<const T*>(gate), gate_stride,
                   state, static_cast<T*>(y));
    return check_launch();
  });
}

}  // namespace gs
