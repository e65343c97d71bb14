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
// tiles from those states. Inside a tile, each thread holds kTokens tokens of
// its channels in registers and the threads' folds are joined in order in
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
constexpr int kTokens = 8;                // tokens a thread holds
constexpr int kGroups = kTile / kTokens;  // threads that share a channel of a tile
constexpr int kScanThreads = 1024;

// e = exp(-gate), a = sigmoid(gate) = 1 / (1 + e); k = 1 - a is e a, with the
// same relative error however small it is. The exponent is cut where a is far
// below any gate's use, so that e stays finite.
__device__ __forceinline__ float open_gate(float gate, float& e) {
  constexpr float kMinusLog2e = -1.4426950408889634f;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fminf(gate * kMinusLog2e, 100.0f)));
  return __fdividef(1.0f, 1.0f + e);
}

// A map s -> a s + b.
struct Affine {
  float a, b;
};
__device__ __forceinline__ Affine then(Affine first, Affine second) {
  return {second.a * first.a, fmaf(second.a, first.b, second.b)};
}

// What a block works on: a tile of tokens and kLanes V channels, V to a thread;
// kGroups threads of kTokens tokens each share a channel.
template <int V>
struct Place {
  static constexpr int kLanes = V == 1 ? 32 : 16;
  static constexpr int kChannels = kLanes * V;
  static constexpr int kThreads = kLanes * kGroups;
  Tile tile;
  int64_t index;     // of the tile
  int channel;       // the thread's first
  int group;
  int first, count;  // the thread's tokens
  bool live;         // the thread has channels
  __device__ __forceinline__ Place(const gs_gated_scan_args& a, bool reverse) {
    const int columns = (a.channels + kChannels - 1) / kChannels;
    index = blockIdx.x / columns;
    if (reverse) index = a.num_tiles - 1 - index;
    channel = (static_cast<int>(blockIdx.x % columns) * kLanes + threadIdx.x % kLanes) * V;
    live = channel < a.channels;
    group = threadIdx.x / kLanes;
    tile = tile_at(a.tiles, index, static_cast<int32_t>(a.tokens), kTile);
    first = tile.start + group * kTokens;
    count = live ? min(kTokens, min(tile.end, tile.start + kTile) - first) : 0;
  }
};

// The thread's tokens of one array; what it does not have reads as `missing`.
template <class T, int V>
__device__ __forceinline__ void load_tokens(const void* p, int64_t stride, const Place<V>& at,
                                            float missing, float (&x)[kTokens][V]) {
  const T* q = static_cast<const T*>(p) + at.first * stride + at.channel;
#pragma unroll
  for (int t = 0; t < kTokens; ++t) {
#pragma unroll
    for (int v = 0; v < V; ++v) x[t][v] = missing;
    if (t < at.count) load_pack<V>(q + t * stride, x[t]);
  }
}
constexpr float kShut = -INFINITY;  // a missing token's gate: the identity map

// Joins the groups' maps in order (from the last group if `reverse`): one
// thread a channel composes them, leaving in the group's place the map of all
// before it, and returns the whole tile's (in the first kChannels threads).
template <int V, bool reverse>
__device__ __forceinline__ Affine join(Affine (*maps)[Place<V>::kChannels]) {
  Affine sum = {1.0f, 0.0f};
  __syncthreads();
  if (threadIdx.x < Place<V>::kChannels) {
    Affine f[kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) f[g] = maps[g][threadIdx.x];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int at = reverse ? kGroups - 1 - g : g;
      maps[at][threadIdx.x] = sum;
      sum = then(sum, f[at]);
    }
  }
  __syncthreads();
  return sum;
}

// Folds every tile: forward the map of the state through it, backward the map
// of the message through it (from its end to its start). h + a (x - h) and
// A - a A save forming k.
template <class T, int V, bool kBackward>
__global__ void __launch_bounds__(Place<V>::kThreads) fold_kernel(gs_gated_scan_args a,
                                                                  Affine* folds) {
  chain_wait();
  __shared__ Affine s_maps[kGroups][Place<V>::kChannels];
  const Place<V> p(a, false);
  float x[kTokens][V], gate[kTokens][V];
  load_tokens<T>(a.gate, a.gate_stride, p, kShut, gate);
  if constexpr (kBackward) load_tokens<T>(a.grad_y, a.channels, p, 0.0f, x);
  else load_tokens<T>(a.x, a.x_stride, p, 0.0f, x);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Affine f = {1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      const int t = kBackward ? kTokens - 1 - i : i;
      float e;
      const float al = open_gate(gate[t][v], e);
      if constexpr (kBackward) {
        const float l = x[t][v] + f.b;
        f.b = fmaf(-al, l, l);
      } else {
        f.b = fmaf(al, x[t][v] - f.b, f.b);
      }
      f.a = fmaf(-al, f.a, f.a);
    }
    s_maps[p.group][threadIdx.x % Place<V>::kLanes * V + v] = f;
  }
  const Affine whole = join<V, kBackward>(s_maps);
  const int channel = p.channel / Place<V>::kChannels * Place<V>::kChannels + threadIdx.x;
  if (threadIdx.x < Place<V>::kChannels && channel < a.channels)
    folds[p.index * a.channels + channel] = whole;
}

// The states (backward: messages) that enter the tiles, a block a sequence and
// kChannels channels: each of kScanThreads / kChannels groups of threads folds
// its share of the sequence's tiles, the shares are joined in order, each group
// walks its share again.
template <bool kBackward, int kChannels>
__global__ void __launch_bounds__(kScanThreads) tile_scan_kernel(gs_gated_scan_args a,
                                                                 const Affine* folds,
                                                                 float* entering) {
  chain_wait();
  constexpr int kShares = kScanThreads / kChannels;
  __shared__ Affine s_fold[kShares][kChannels];
  const int lane = threadIdx.x % kChannels, part = threadIdx.x / kChannels;
  const int columns = (a.channels + kChannels - 1) / kChannels;
  const int64_t sequence = blockIdx.x / columns;
  const int channel = static_cast<int>(blockIdx.x % columns) * kChannels + lane;
  const bool live = channel < a.channels;
  const int64_t begin = a.tile_starts ? __ldg(a.tile_starts + sequence) : 0;
  const int64_t end = a.tile_starts ? __ldg(a.tile_starts + sequence + 1) : a.num_tiles;
  const int64_t share = (end - begin + kShares - 1) / kShares;
  const int64_t from = min(end, begin + part * share), to = min(end, from + share);
  const auto tile_of = [&](int64_t i) { return kBackward ? begin + end - 1 - i : i; };
  Affine sum = {1.0f, 0.0f};
  if (live)
#pragma unroll 8
    for (int64_t i = from; i < to; ++i) sum = then(sum, folds[tile_of(i) * a.channels + channel]);
  s_fold[part][lane] = sum;
  __syncthreads();
  const int64_t slot = sequence * a.channels + channel;
  if (part == 0 && live) {
    // The state that enters each share takes the place of its map.
    const float* start = kBackward ? a.grad_last : a.initial;
    float state = start ? start[slot] : 0.0f;
#pragma unroll 8
    for (int w = 0; w < kShares; ++w) {
      const Affine f = s_fold[w][lane];
      s_fold[w][lane].b = state;
      state = fmaf(f.a, state, f.b);
    }
    float* final = kBackward ? a.grad_initial : a.last;
    if (final) final[slot] = state;
  }
  __syncthreads();
  if (!live) return;
  float state = s_fold[part][lane].b;
#pragma unroll 8
  for (int64_t i = from; i < to; ++i) {
    const int64_t at = tile_of(i) * a.channels + channel;
    const Affine f = folds[at];
    entering[at] = state;
    state = fmaf(f.a, state, f.b);
  }
}

// The walk from the entering states. Tiles go from the last to the first: the
// fold just before read them from the first to the last, so the end of its
// inputs is what L2 still holds.
template <class T, int V>
__global__ void __launch_bounds__(Place<V>::kThreads) walk_kernel(gs_gated_scan_args a) {
  chain_wait();
  __shared__ Affine s_maps[kGroups][Place<V>::kChannels];
  const Place<V> p(a, true);
  float x[kTokens][V], gate[kTokens][V], state[V];
  load_tokens<T>(a.gate, a.gate_stride, p, kShut, gate);
  load_tokens<T>(a.x, a.x_stride, p, 0.0f, x);
  if (p.live) load_pack<V>(a.entering + p.index * a.channels + p.channel, state);
  const int lane = threadIdx.x % Place<V>::kLanes * V;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Affine f = {1.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      float e;
      gate[t][v] = open_gate(gate[t][v], e);
      f.b = fmaf(gate[t][v], x[t][v] - f.b, f.b);
      f.a = fmaf(-gate[t][v], f.a, f.a);
    }
    s_maps[p.group][lane + v] = f;
  }
  join<V, false>(s_maps);
  if (!p.live) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const Affine f = s_maps[p.group][lane + v];
    state[v] = fmaf(f.a, state[v], f.b);
  }
  T* y = static_cast<T*>(a.y) + int64_t{p.first} * a.channels + p.channel;
#pragma unroll
  for (int t = 0; t < kTokens; ++t)
    if (t < p.count) {
#pragma unroll
      for (int v = 0; v < V; ++v) state[v] = fmaf(gate[t][v], x[t][v] - state[v], state[v]);
      store_pack<V>(y + int64_t{t} * a.channels, state);
    }
}

template <class T, int V>
__global__ void __launch_bounds__(Place<V>::kThreads) walk_back_kernel(gs_gated_scan_args a,
                                                                       const float* messages) {
  chain_wait();
  __shared__ Affine s_ahead[kGroups][Place<V>::kChannels], s_back[kGroups][Place<V>::kChannels];
  const Place<V> p(a, true);
  float x[kTokens][V], al[kTokens][V], g[kTokens][V], keep[kTokens][V], state[V], message[V];
  load_tokens<T>(a.gate, a.gate_stride, p, kShut, al);
  load_tokens<T>(a.x, a.x_stride, p, 0.0f, x);
  load_tokens<T>(a.grad_y, a.channels, p, 0.0f, g);
  if (p.live) {
    load_pack<V>(a.entering + p.index * a.channels + p.channel, state);
    load_pack<V>(messages + p.index * a.channels + p.channel, message);
  }
  const int lane = threadIdx.x % Place<V>::kLanes * V;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Affine ahead = {1.0f, 0.0f}, back = {1.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      float e;
      al[t][v] = open_gate(al[t][v], e);
      keep[t][v] = e * al[t][v];
      ahead.b = fmaf(al[t][v], x[t][v] - ahead.b, ahead.b);
      ahead.a *= keep[t][v];
    }
#pragma unroll
    for (int t = kTokens - 1; t >= 0; --t) back.b = keep[t][v] * (g[t][v] + back.b);
    back.a = ahead.a;
    s_ahead[p.group][lane + v] = ahead;
    s_back[p.group][lane + v] = back;
  }
  join<V, false>(s_ahead);
  join<V, true>(s_back);
  if (!p.live) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const Affine ahead = s_ahead[p.group][lane + v], back = s_back[p.group][lane + v];
    float h = fmaf(ahead.a, state[v], ahead.b);
    float u = fmaf(back.a, message[v], back.b);
    // forward: x_t becomes x_t - h_{t-1}
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      x[t][v] -= h;
      h = fmaf(al[t][v], x[t][v], h);
    }
    // back: x_t becomes dgate_t and g_t becomes dx_t
#pragma unroll
    for (int t = kTokens - 1; t >= 0; --t) {
      const float l = g[t][v] + u;
      u = keep[t][v] * l;
      g[t][v] = al[t][v] * l;
      x[t][v] *= u * al[t][v];
    }
  }
  const int64_t at = int64_t{p.first} * a.channels + p.channel;
  T* grad_x = static_cast<T*>(a.grad_x) + at;
  T* grad_gate = static_cast<T*>(a.grad_gate) + at;
#pragma unroll
  for (int t = 0; t < kTokens; ++t)
    if (t < p.count) {
      store_pack<V>(grad_x + int64_t{t} * a.channels, g[t]);
      store_pack<V>(grad_gate + int64_t{t} * a.channels, x[t]);
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
  float e;
  const float al = open_gate(to_float(gate[row * gate_stride + c]), e);
  const float h = fmaf(al, to_float(x[row * x_stride + c]) - state[i], state[i]);
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
  const int64_t columns = (int64_t{a.channels} + 7) / 8;
  if (columns * (a.num_tiles > a.sequences ? a.num_tiles : a.sequences) > INT32_MAX)
    return GS_ERR_CAPACITY;
  if (a.num_tiles > 0 && (!a.x || !a.gate || !a.entering || !a.workspace))
    return GS_ERR_INVALID_ARGUMENT;
  if (a.workspace_size < gated_scan_workspace_size(a.num_tiles, a.channels))
    return GS_ERR_CAPACITY;
  return GS_OK;
}

// Four channels a thread (8 or 16 bytes a load) need rows and arrays aligned to
// them; otherwise one.
template <class T>
bool four_channels(const gs_gated_scan_args& a) {
  if (a.channels % 4 || a.x_stride % 4 || a.gate_stride % 4) return false;
  for (const void* p : {a.x, a.gate, a.grad_y, static_cast<const void*>(a.y),
                        static_cast<const void*>(a.grad_x), static_cast<const void*>(a.grad_gate)})
    if (!is_aligned(p, 4 * sizeof(T))) return false;
  return is_aligned(a.entering, 16) && is_aligned(a.workspace, 16);
}

template <bool kBackward>
int32_t scan_tiles(const gs_gated_scan_args& a, const Affine* folds, float* entering,
                   cudaStream_t stream) {
  // Long sequences: fewer channels a block, so that more threads share the
  // tiles (7813 tiles of 64 channels: 2 blocks of 32 channels took 116 us).
  const bool narrow = a.num_tiles / a.sequences > 256;
  const unsigned blocks =
      ceil_div(a.channels, narrow ? 8 : 32) * static_cast<unsigned>(a.sequences);
  if (narrow)
    launch_chained(tile_scan_kernel<kBackward, 8>, blocks, kScanThreads, stream, a, folds,
                   entering);
  else
    launch_chained(tile_scan_kernel<kBackward, 32>, blocks, kScanThreads, stream, a, folds,
                   entering);
  return check_launch();
}

template <class T, int V>
int32_t forward(const gs_gated_scan_args& a, cudaStream_t stream) {
  Affine* folds = static_cast<Affine*>(a.workspace);
  constexpr int kThreads = Place<V>::kThreads;
  const unsigned blocks =
      ceil_div(a.channels, Place<V>::kChannels) * static_cast<unsigned>(a.num_tiles);
  if (blocks) {
    launch_chained(fold_kernel<T, V, false>, blocks, kThreads, stream, a, folds);
    GS_TRY(check_launch());
  }
  GS_TRY(scan_tiles<false>(a, folds, a.entering, stream));
  if (blocks) launch_chained(walk_kernel<T, V>, blocks, kThreads, stream, a);
  return check_launch();
}

template <class T, int V>
int32_t backward(const gs_gated_scan_args& a, cudaStream_t stream) {
  Affine* folds = static_cast<Affine*>(a.workspace);
  float* messages = reinterpret_cast<float*>(folds + a.num_tiles * a.channels);
  constexpr int kThreads = Place<V>::kThreads;
  const unsigned blocks =
      ceil_div(a.channels, Place<V>::kChannels) * static_cast<unsigned>(a.num_tiles);
  if (blocks) {
    launch_chained(fold_kernel<T, V, true>, blocks, kThreads, stream, a, folds);
    GS_TRY(check_launch());
  }
  GS_TRY(scan_tiles<true>(a, folds, messages, stream));
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
    return four_channels<T>(a) ? forward<T, 4>(a, stream) : forward<T, 1>(a, stream);
  });
}

int32_t launch_gated_scan_backward(const gs_gated_scan_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (a.num_tiles > 0 && (!a.grad_y || !a.grad_x || !a.grad_gate)) return GS_ERR_INVALID_ARGUMENT;
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return four_channels<T>(a) ? backward<T, 4>(a, stream) : backward<T, 1>(a, stream);
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
