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
// tiles of kTile tokens and those into spans of a few tiles: one kernel folds each span to
// its (A, B), one scans the spans of each sequence for the state that enters
// each, one walks the spans from those states. Inside a tile, each thread holds kTokens tokens of
// its channels in registers and the threads' folds are joined in order in
// shared memory. Every order is fixed, so results repeat bit for bit.
//
// What bounds it: memory; the fold's second reading of gate and x (of gate and
// grad_y on the way back) is the price of a sequence split without blocks that
// wait for one another. Walks go the other way round from folds, so that part of
// it comes from L2. Measured at 1,000,000 tokens of 64 16-bit channels (128 MB an
// array): fold 46 us (5.6 TB/s), walk 69 us (5.6 TB/s), back 47 and 110 us (5.8
// TB/s), the scans of the spans' maps 10 us each.
//
// States, products and gates are float; the states that enter the tiles are
// kept in float for the backward, which recomputes h from them instead of
// reading the rounded y.

#include <algorithm>

#include "tensorcore.cuh"

namespace gs {

int32_t launch_gated_scan(const gs_gated_scan_args& a, cudaStream_t stream);
int32_t launch_gated_scan_backward(const gs_gated_scan_args& a, cudaStream_t stream);
int32_t launch_gated_scan_step(int64_t batch, int32_t channels, int32_t dtype, const void* x,
                               int64_t x_stride, const void* gate, int64_t gate_stride,
                               float* state, void* y, cudaStream_t stream);
uint64_t gated_scan_workspace_size(const gs_gated_scan_args& a);
int32_t gated_scan_status(cudaStream_t stream);

namespace {

constexpr int kTile = GS_SEQUENCE_TILE;
constexpr int kTokens = 8;                // tokens a thread holds
constexpr int kGroups = kTile / kTokens;  // threads that share a channel of a tile

constexpr float kMinusLog2e = -1.4426950408889634f;
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 both(float x) { return {x, x}; }
__device__ __forceinline__ float2 minus(float2 a, float2 b) {
  return tc::fma2(b, both(-1.0f), a);
}

// Two gates at a time, as is all arithmetic here: the instructions that a pass
// issued took longer than its memory did. -a = -sigmoid(gate) = 1 / (-1 - e),
// e = exp(-gate); e may be infinite, a NaN stays one.
__device__ __forceinline__ float2 minus_gate(float2 gate) {
  const float2 t = tc::mul2(gate, both(kMinusLog2e));
  const float2 d =
      tc::fma2({tc::exp2_approx(t.x), tc::exp2_approx(t.y)}, both(-1.0f), both(-1.0f));
  return {reciprocal(d.x), reciprocal(d.y)};
}
// a, and k = 1 - a as e a, with the same relative error however small it is. e is
// cut at 2^100 so that it stays finite; 2^-100 less, a shut gate's a is nothing.
__device__ __forceinline__ float2 open_gate(float2 gate, float2& keep) {
  const float2 t = tc::mul2(gate, both(kMinusLog2e));
  const auto cut = [](float x) {
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(100.0f));
    return tc::exp2_approx(y);
  };
  const float2 e = {cut(t.x), cut(t.y)}, d = tc::add2(e, both(1.0f));
  const float2 a = {reciprocal(d.x), reciprocal(d.y)};
  keep = tc::mul2(e, a);
  return tc::add2(a, both(-0x1p-100f));
}

// N channels of a thread, in pairs. (A last one alone has a pair of its own.)
template <int N>
constexpr int kPairs = (N + 1) / 2;
template <int N, class T>
__device__ __forceinline__ void store_pairs(T* p, const float2 (&x)[kPairs<N>]) {
  Pack<T, N> a;
#pragma unroll
  for (int v = 0; v < N; ++v) a.v[v] = from_float<T>(v % 2 ? x[v / 2].y : x[v / 2].x);
  *reinterpret_cast<Pack<T, N>*>(p) = a;
}
// A word of shared memory: two values of 16 bits, or one.
template <class T>
__device__ __forceinline__ float2 from_word(uint32_t w) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  else
    return __half22float2(reinterpret_cast<const __half2&>(w));
}

// A map s -> a s + b.
struct alignas(8) Affine {
  float a, b;
};
template <int N>
struct Affines {  // those of N channels
  float2 a[kPairs<N>], b[kPairs<N>];
  __device__ __forceinline__ Affines() {
#pragma unroll
    for (int v = 0; v < kPairs<N>; ++v) a[v] = both(1.0f), b[v] = both(0.0f);
  }
  __device__ __forceinline__ void put(Affine* maps) const {
#pragma unroll
    for (int v = 0; v < N / 2; ++v)
      reinterpret_cast<float4*>(maps)[v] = {a[v].x, b[v].x, a[v].y, b[v].y};
    if constexpr (N % 2) maps[N - 1] = {a[N / 2].x, b[N / 2].x};
  }
};
// The values that `pass` left in the maps.
template <int N>
__device__ __forceinline__ void take(const Affine* maps, float2 (&x)[kPairs<N>]) {
#pragma unroll
  for (int v = 0; v < N; ++v) (v % 2 ? x[v / 2].y : x[v / 2].x) = maps[v].b;
  if constexpr (N % 2) x[N / 2].y = 0.0f;
}
__device__ __forceinline__ Affine then(Affine first, Affine second) {
  return {second.a * first.a, fmaf(second.a, first.b, second.b)};
}

// Sequences are walked in spans of `length` tiles, one block and one composed
// map a span. Sequence b's spans take the slots from floor(first tile of b /
// length) + b on, which no two sequences share.
struct Spans {
  int length, slots;
  __device__ __forceinline__ int64_t slot_of(int64_t first_tile, int64_t sequence) const {
    return first_tile / length + sequence;
  }
};
__device__ __forceinline__ int64_t first_tile_of(const gs_gated_scan_args& a, int64_t b) {
  return a.tile_starts ? __ldg(a.tile_starts + b) : (b ? a.num_tiles : 0);
}

// What a block works on: a span's tiles and kChannels channels, V to a thread,
// kLanes threads side by side; kGroups threads of kTokens tokens each share a
// channel of a tile.
template <int V, int kLanes>
struct Place {
  static constexpr int kChannels = kLanes * V;
  int64_t slot, tile;  // the span's slot, its first tile
  int tiles;           // 0: the slot is empty
  int row, end;        // the first tile's first row, the sequence's end
  int block_channel;   // the block's first channel
  __device__ __forceinline__ Place(const gs_gated_scan_args& a, const Spans& spans, bool reverse) {
    const int columns = (a.channels + kChannels - 1) / kChannels;
    slot = blockIdx.x / columns;
    if (reverse) slot = spans.slots - 1 - slot;
    block_channel = static_cast<int>(blockIdx.x % columns) * kChannels;
    int64_t b = 0, above = a.tile_starts ? a.sequences : 1;
    while (above - b > 1) {  // the last sequence whose slots start at or before this one
      const int64_t middle = (b + above) / 2;
      if (spans.slot_of(first_tile_of(a, middle), middle) <= slot) b = middle;
      else above = middle;
    }
    const int64_t tile0 = first_tile_of(a, b), count = first_tile_of(a, b + 1) - tile0;
    const int64_t offset = (slot - spans.slot_of(tile0, b)) * spans.length;
    tile = tile0 + offset;
    tiles = static_cast<int>(max(int64_t{0}, min(int64_t{spans.length}, count - offset)));
    if (tiles > 0) {
      const Tile t = tile_at(a.tiles, tile, static_cast<int32_t>(a.tokens), kTile);
      row = t.start;
      end = t.end;
    }
  }
  __device__ __forceinline__ int lane() const { return threadIdx.x % kLanes; }
  __device__ __forceinline__ int group() const { return threadIdx.x / kLanes; }
  __device__ __forceinline__ int channel() const { return block_channel + lane() * V; }
  // The thread's first row of the span's tile i, and how many rows it has there.
  __device__ __forceinline__ int first(int i) const { return row + i * kTile + group() * kTokens; }
  __device__ __forceinline__ int count(int i) const {
    return max(0, min(kTokens, end - first(i)));
  }
};

// Where a block's tiles come from. With whole 16-byte words a row the tensor
// memory accelerator copies boxes of 128 bytes of channels and a tile's rows to
// shared memory, a tile ahead of the walk; a thread then reads 8 bytes a row.
// (Loads straight to registers left a block waiting for most of its time:
// 2.0 TB/s.) The other arrays are loaded a channel a thread.
constexpr int kBoxBytes = 128 * kTile;
constexpr int kStages = 2;
constexpr float kShut = -INFINITY;  // a missing token's gate: the identity map

__device__ uint32_t g_timeout;  // a wait ran out: for gs_gated_scan_status

template <int kArrays>
struct Boxes {
  alignas(128) unsigned char data[kStages][kArrays][kBoxBytes];
  uint64_t full[kStages];
};

template <class T, int kArrays>
struct BoxSource {
  static constexpr int kLanes = 16, V = 8 / sizeof(T);
  using At = Place<V, kLanes>;
  Boxes<kArrays>& s;
  const CUtensorMap* const maps;
  const At& at;
  bool backward, good = true;
  __device__ __forceinline__ BoxSource(unsigned char* shared, const CUtensorMap* m, const At& p,
                                       bool back)
      : s(*reinterpret_cast<Boxes<kArrays>*>(shared)), maps(m), at(p), backward(back) {
    if (threadIdx.x == 0) {
      for (uint64_t& b : s.full) tc::barrier_init(tc::shared_address(&b), 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      tc::fence_async_shared();
      for (int step = 0; step < kStages && step < at.tiles; ++step) request(step);
    }
    __syncthreads();
  }
  // Step `step` of the walk works on the span's tile:
  __device__ __forceinline__ int tile_of(int step) const {
    return backward ? at.tiles - 1 - step : step;
  }
  __device__ __forceinline__ void request(int step) {
    const uint32_t bar = tc::shared_address(&s.full[step % kStages]);
    tc::barrier_expect(bar, kArrays * kBoxBytes);
#pragma unroll
    for (int k = 0; k < kArrays; ++k)
      tc::load_box(tc::shared_address(s.data[step % kStages][k]), maps + k, at.block_channel,
                   at.row + tile_of(step) * kTile, bar);
  }
  __device__ __forceinline__ void wait(int step) {
    good = good && tc::barrier_wait_warp(tc::shared_address(&s.full[step % kStages]),
                                         (step / kStages) & 1);
  }
  // Called by all once every thread has read step `step` and a barrier has passed.
  __device__ __forceinline__ void release(int step) {
    if (threadIdx.x == 0 && step + kStages < at.tiles && good) {
      tc::fence_async_shared();
      request(step + kStages);
    }
  }
  // Array 0 is the gate.
  template <int kArray>
  __device__ __forceinline__ void read(int step, int t, float2 (&x)[kPairs<V>]) const {
    const int r = at.group() * kTokens + t;
    uint2 w = *reinterpret_cast<const uint2*>(s.data[step % kStages][kArray] + r * 128 +
                                              at.lane() * 8);
    constexpr uint32_t kMissing = kArray                              ? 0u
                                  : std::is_same_v<T, float>          ? 0xff800000u
                                  : std::is_same_v<T, __nv_bfloat16> ? 0xff80ff80u
                                                                      : 0xfc00fc00u;
    if (t >= at.count(tile_of(step))) w = {kMissing, kMissing};
    if constexpr (std::is_same_v<T, float>) {
      x[0] = {__uint_as_float(w.x), __uint_as_float(w.y)};
    } else {
      x[0] = from_word<T>(w.x);
      x[1] = from_word<T>(w.y);
    }
  }
  // At the end: whether all waits came back; if not, copies still in flight land first.
  __device__ __forceinline__ void finish() {
    if (good) return;
    for (uint64_t& b : s.full) tc::barrier_settle(tc::shared_address(&b));
    if (threadIdx.x == 0) atomicExch(&g_timeout, 1u);
  }
};

// The same from global memory, a channel a thread.
template <class T, int kArrays>
struct PlainSource {
  static constexpr int kLanes = 32, V = 1;
  using At = Place<V, kLanes>;
  const T* base[kArrays];
  int64_t stride[kArrays];
  const At& at;
  bool backward;
  static constexpr bool good = true;
  const bool live;
  __device__ __forceinline__ PlainSource(const gs_gated_scan_args& a, const void* const (&p)[kArrays],
                                         const int64_t (&strides)[kArrays], const At& place,
                                         bool back)
      : at(place), backward(back), live(place.channel() < a.channels) {
#pragma unroll
    for (int k = 0; k < kArrays; ++k) {
      base[k] = static_cast<const T*>(p[k]);
      stride[k] = strides[k];
    }
  }
  __device__ __forceinline__ int tile_of(int step) const {
    return backward ? at.tiles - 1 - step : step;
  }
  __device__ __forceinline__ void wait(int) {}
  __device__ __forceinline__ void release(int) {}
  __device__ __forceinline__ void finish() {}
  template <int kArray>
  __device__ __forceinline__ void read(int step, int t, float2 (&x)[1]) const {
    const int i = tile_of(step);
    x[0].x = live && t < at.count(i)
                 ? to_float(base[kArray][(at.first(i) + t) * stride[kArray] + at.channel()])
                 : (kArray ? 0.0f : kShut);
    x[0].y = 0.0f;
  }
};

// The thread that joins a channel's groups: composes their maps in order.
template <int kChannels, bool kReverse>
__device__ __forceinline__ Affine compose(const Affine (*maps)[kChannels], Affine sum) {
  Affine f[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) f[g] = maps[kReverse ? kGroups - 1 - g : g][threadIdx.x];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) sum = then(sum, f[g]);
  return sum;
}
// The same for a value that passes through them: what enters each group takes
// the place of its map (in `b`).
template <int kChannels, bool kReverse>
__device__ __forceinline__ float pass(Affine (*maps)[kChannels], int channel, float value) {
  Affine f[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) f[g] = maps[kReverse ? kGroups - 1 - g : g][channel];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    maps[kReverse ? kGroups - 1 - g : g][channel].b = value;
    value = fmaf(f[g].a, value, f[g].b);
  }
  return value;
}

// Folds every span: forward the map of the state through it, backward the map
// of the message through it (from its end to its start). h - (-a) (x - h) and
// A + (-a) A save forming k. Arrays: gate, and x or grad_y.
template <class Source, bool kBackward>
__device__ __forceinline__ void fold(const gs_gated_scan_args& a, const typename Source::At& at,
                                     Source& source, Affine* folds) {
  constexpr int V = Source::V, kChannels = Source::At::kChannels;
  __shared__ alignas(16) Affine s_maps[kGroups][kChannels];
  Affine span = {1.0f, 0.0f};
  for (int step = 0; step < at.tiles; ++step) {
    Affines<V> f;
    source.wait(step);
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      const int t = kBackward ? kTokens - 1 - i : i;
      float2 gate[kPairs<V>], x[kPairs<V>];
      source.template read<0>(step, t, gate);
      source.template read<1>(step, t, x);
#pragma unroll
      for (int v = 0; v < kPairs<V>; ++v) {
        const float2 al = minus_gate(gate[v]);
        if constexpr (kBackward) {
          const float2 l = tc::add2(x[v], f.b[v]);
          f.b[v] = tc::fma2(al, l, l);
        } else {
          f.b[v] = tc::fma2(al, minus(f.b[v], x[v]), f.b[v]);
        }
        f.a[v] = tc::fma2(al, f.a[v], f.a[v]);
      }
    }
    f.put(&s_maps[at.group()][at.lane() * V]);
    __syncthreads();
    source.release(step);
    if (threadIdx.x < kChannels) span = compose<kChannels, kBackward>(s_maps, span);
    __syncthreads();
  }
  const int channel = at.block_channel + threadIdx.x;
  if (threadIdx.x < kChannels && channel < a.channels)
    folds[at.slot * a.channels + channel] = source.good ? span : Affine{NAN, NAN};
  source.finish();
}

// The walk from the entering states. Arrays: gate, x.
template <class T, class Source>
__device__ __forceinline__ void walk(const gs_gated_scan_args& a, const typename Source::At& at,
                                     Source& source, const float* states) {
  constexpr int V = Source::V, kChannels = Source::At::kChannels;
  __shared__ alignas(16) Affine s_maps[kGroups][kChannels];
  const int joined = at.block_channel + threadIdx.x;  // the channel that the thread joins
  const bool joins = threadIdx.x < kChannels && joined < a.channels;
  float carry = joins ? states[at.slot * a.channels + joined] : 0.0f;
  T* y = static_cast<T*>(a.y) + at.channel();
  const bool live = at.channel() < a.channels;
  for (int step = 0; step < at.tiles; ++step) {
    float2 x[kTokens][kPairs<V>], al[kTokens][kPairs<V>];  // al: -a
    Affines<V> f;
    source.wait(step);
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      source.template read<0>(step, t, al[t]);
      source.template read<1>(step, t, x[t]);
#pragma unroll
      for (int v = 0; v < kPairs<V>; ++v) {
        al[t][v] = minus_gate(al[t][v]);
        f.b[v] = tc::fma2(al[t][v], minus(f.b[v], x[t][v]), f.b[v]);
        f.a[v] = tc::fma2(al[t][v], f.a[v], f.a[v]);
      }
    }
    f.put(&s_maps[at.group()][at.lane() * V]);
    __syncthreads();
    source.release(step);
    if (threadIdx.x < kChannels) {
      if (!source.good) carry = NAN;
      if (joins) a.entering[(at.tile + step) * a.channels + joined] = carry;
      carry = pass<kChannels, false>(s_maps, threadIdx.x, carry);
    }
    __syncthreads();
    float2 h[kPairs<V>];
    take<V>(&s_maps[at.group()][at.lane() * V], h);
    const int first = at.first(step), count = live ? at.count(step) : 0;
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
#pragma unroll
      for (int v = 0; v < kPairs<V>; ++v) h[v] = tc::fma2(al[t][v], minus(h[v], x[t][v]), h[v]);
      if (t < count) store_pairs<V>(y + int64_t{first + t} * a.channels, h);
    }
  }
  source.finish();
}

// The walk back from the entering messages. Arrays: gate, x, grad_y.
template <class T, class Source>
__device__ __forceinline__ void walk_back(const gs_gated_scan_args& a,
                                          const typename Source::At& at, Source& source,
                                          const float* messages) {
  constexpr int V = Source::V, kChannels = Source::At::kChannels;
  __shared__ alignas(16) Affine s_ahead[kGroups][kChannels], s_back[kGroups][kChannels];
  // One thread a channel passes the state on, another one the message.
  const int joined = at.block_channel + threadIdx.x % kChannels;
  const bool forward = threadIdx.x < kChannels;
  const bool joins = threadIdx.x < 2 * kChannels && joined < a.channels;
  float carry = joins && !forward ? messages[at.slot * a.channels + joined] : 0.0f;
  const bool live = at.channel() < a.channels;
  for (int step = 0; step < at.tiles; ++step) {
    const int i = at.tiles - 1 - step;
    if (joins && forward) carry = a.entering[(at.tile + i) * a.channels + joined];
    float2 x[kTokens][kPairs<V>], al[kTokens][kPairs<V>], keep[kTokens][kPairs<V>];
    Affines<V> ahead, back;
    source.wait(step);
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      source.template read<0>(step, t, al[t]);
      source.template read<1>(step, t, x[t]);
#pragma unroll
      for (int v = 0; v < kPairs<V>; ++v) {
        al[t][v] = open_gate(al[t][v], keep[t][v]);
        ahead.b[v] = tc::fma2(al[t][v], minus(x[t][v], ahead.b[v]), ahead.b[v]);
        ahead.a[v] = tc::mul2(ahead.a[v], keep[t][v]);
      }
    }
#pragma unroll
    for (int t = kTokens - 1; t >= 0; --t) {
      float2 g[kPairs<V>];
      source.template read<2>(step, t, g);
#pragma unroll
      for (int v = 0; v < kPairs<V>; ++v)
        back.b[v] = tc::mul2(keep[t][v], tc::add2(g[v], back.b[v]));
    }
#pragma unroll
    for (int v = 0; v < kPairs<V>; ++v) back.a[v] = ahead.a[v];
    ahead.put(&s_ahead[at.group()][at.lane() * V]);
    back.put(&s_back[at.group()][at.lane() * V]);
    __syncthreads();
    // The last step's gradients have been read for the second time by now.
    if (step > 0) source.release(step - 1);
    if (!source.good) carry = NAN;
    if (forward) pass<kChannels, false>(s_ahead, threadIdx.x, carry);
    else if (threadIdx.x < 2 * kChannels)
      carry = pass<kChannels, true>(s_back, threadIdx.x - kChannels, carry);
    __syncthreads();
    float2 h[kPairs<V>], u[kPairs<V>];
    take<V>(&s_ahead[at.group()][at.lane() * V], h);
    take<V>(&s_back[at.group()][at.lane() * V], u);
    const int count = live ? at.count(i) : 0;
    const int64_t offset = int64_t{at.first(i)} * a.channels + at.channel();
    T* grad_x = static_cast<T*>(a.grad_x) + offset;
    T* grad_gate = static_cast<T*>(a.grad_gate) + offset;
    // forward: x_t becomes x_t - h_{t-1}
#pragma unroll
    for (int t = 0; t < kTokens; ++t)
#pragma unroll
      for (int v = 0; v < kPairs<V>; ++v) {
        x[t][v] = minus(x[t][v], h[v]);
        h[v] = tc::fma2(al[t][v], x[t][v], h[v]);
      }
    // back: g becomes dx_t and x_t becomes dgate_t
#pragma unroll
    for (int t = kTokens - 1; t >= 0; --t) {
      float2 g[kPairs<V>];
      source.template read<2>(step, t, g);
#pragma unroll
      for (int v = 0; v < kPairs<V>; ++v) {
        const float2 l = tc::add2(g[v], u[v]);
        u[v] = tc::mul2(keep[t][v], l);
        g[v] = tc::mul2(al[t][v], l);
        x[t][v] = tc::mul2(x[t][v], tc::mul2(u[v], al[t][v]));
      }
      if (t < count) {
        store_pairs<V>(grad_x + int64_t{t} * a.channels, g);
        store_pairs<V>(grad_gate + int64_t{t} * a.channels, x[t]);
      }
    }
  }
  source.finish();
}

struct Maps {
  CUtensorMap gate, x, grad;
};

constexpr int kBoxThreads = 16 * kGroups, kPlainThreads = 32 * kGroups;

template <class T, bool kBackward>
__global__ void __launch_bounds__(kBoxThreads, 3)
    fold_boxes_kernel(gs_gated_scan_args a, Spans spans, Affine* folds,
                      const __grid_constant__ Maps maps) {
  chain_wait();
  extern __shared__ __align__(128) unsigned char s_boxes[];
  using Source = BoxSource<T, 2>;
  const typename Source::At at(a, spans, false);
  if (at.tiles == 0) return;
  Source source(s_boxes, &maps.gate, at, kBackward);
  fold<Source, kBackward>(a, at, source, folds);
}
template <class T, bool kBackward>
__global__ void __launch_bounds__(kPlainThreads)
    fold_kernel(gs_gated_scan_args a, Spans spans, Affine* folds) {
  chain_wait();
  using Source = PlainSource<T, 2>;
  const typename Source::At at(a, spans, false);
  if (at.tiles == 0) return;
  Source source(a, {a.gate, kBackward ? a.grad_y : a.x},
                {a.gate_stride, kBackward ? int64_t{a.channels} : a.x_stride}, at, kBackward);
  fold<Source, kBackward>(a, at, source, folds);
}

// Walks go over the spans from the last to the first: the fold just before
// read them from the first to the last, so the end of its inputs is what L2
// still holds.
template <class T>
__global__ void __launch_bounds__(kBoxThreads, 2)
    walk_boxes_kernel(gs_gated_scan_args a, Spans spans, const float* states,
                      const __grid_constant__ Maps maps) {
  chain_wait();
  extern __shared__ __align__(128) unsigned char s_boxes[];
  using Source = BoxSource<T, 2>;
  const typename Source::At at(a, spans, true);
  if (at.tiles == 0) return;
  Source source(s_boxes, &maps.gate, at, false);
  walk<T>(a, at, source, states);
}
template <class T>
__global__ void __launch_bounds__(kPlainThreads)
    walk_kernel(gs_gated_scan_args a, Spans spans, const float* states) {
  chain_wait();
  using Source = PlainSource<T, 2>;
  const typename Source::At at(a, spans, true);
  if (at.tiles == 0) return;
  Source source(a, {a.gate, a.x}, {a.gate_stride, a.x_stride}, at, false);
  walk<T>(a, at, source, states);
}

template <class T>
__global__ void __launch_bounds__(kBoxThreads, 2)
    walk_back_boxes_kernel(gs_gated_scan_args a, Spans spans, const float* messages,
                           const __grid_constant__ Maps maps) {
  chain_wait();
  extern __shared__ __align__(128) unsigned char s_boxes[];
  using Source = BoxSource<T, 3>;
  const typename Source::At at(a, spans, true);
  if (at.tiles == 0) return;
  Source source(s_boxes, &maps.gate, at, true);
  walk_back<T>(a, at, source, messages);
}
template <class T>
__global__ void __launch_bounds__(kPlainThreads)
    walk_back_kernel(gs_gated_scan_args a, Spans spans, const float* messages) {
  chain_wait();
  using Source = PlainSource<T, 3>;
  const typename Source::At at(a, spans, true);
  if (at.tiles == 0) return;
  Source source(a, {a.gate, a.x, a.grad_y}, {a.gate_stride, a.x_stride, int64_t{a.channels}}, at,
                true);
  walk_back<T>(a, at, source, messages);
}

// The states (backward: messages) that enter the spans, a block a sequence and
// kChannels channels: each of kScanThreads / kChannels groups of threads folds
// its share of the sequence's spans, the shares are joined in order, each group
// walks its share again.
template <bool kBackward, int kChannels, int kScanThreads>
__global__ void __launch_bounds__(kScanThreads) span_scan_kernel(gs_gated_scan_args a, Spans spans,
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
  const int64_t tile0 = first_tile_of(a, sequence);
  const int64_t tiles = first_tile_of(a, sequence + 1) - tile0;
  const int64_t begin = spans.slot_of(tile0, sequence);
  const int64_t end = begin + (tiles + spans.length - 1) / spans.length;
  const int64_t share = (end - begin + kShares - 1) / kShares;
  const int64_t from = min(end, begin + part * share), to = min(end, from + share);
  const auto slot_of = [&](int64_t i) { return kBackward ? begin + end - 1 - i : i; };
  // A few maps at a time, loaded before the first is used.
  constexpr int kAtOnce = kChannels == 8 ? 8 : 2;
  const auto load = [&](int64_t i, Affine (&f)[kAtOnce]) {
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      f[k] = folds[slot_of(min(i + k, to - 1)) * a.channels + channel];
  };
  Affine sum = {1.0f, 0.0f}, f[kAtOnce];
  if (live)
    for (int64_t i = from; i < to; i += kAtOnce) {
      load(i, f);
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k)
        if (i + k < to) sum = then(sum, f[k]);
    }
  s_fold[part][lane] = sum;
  __syncthreads();
  const int64_t slot = sequence * a.channels + channel;
  if (part == 0 && live) {
    // The state that enters each share takes the place of its map.
    const float* start = kBackward ? a.grad_last : a.initial;
    float state = start ? start[slot] : 0.0f;
    constexpr int kTurn = kShares < 16 ? kShares : 16;
    for (int base = 0; base < kShares; base += kTurn) {
      Affine g[kTurn];
#pragma unroll
      for (int w = 0; w < kTurn; ++w) g[w] = s_fold[base + w][lane];
#pragma unroll
      for (int w = 0; w < kTurn; ++w) {
        s_fold[base + w][lane].b = state;
        state = fmaf(g[w].a, state, g[w].b);
      }
    }
    float* final = kBackward ? a.grad_initial : a.last;
    if (final) final[slot] = state;
  }
  __syncthreads();
  if (!live) return;
  float state = s_fold[part][lane].b;
  for (int64_t i = from; i < to; i += kAtOnce) {
    load(i, f);
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (i + k < to) {
        entering[slot_of(i + k) * a.channels + channel] = state;
        state = fmaf(f[k].a, state, f[k].b);
      }
  }
}

// One token: a state's 14 bytes (16-bit types) once. 512 x 2048 states: 6.5 us, of which
// 2.2 us of memory; the rest is a launch's latency.
template <class T>
__global__ void __launch_bounds__(256) scan_step_kernel(int64_t count, int channels, const T* x,
                                                        int64_t x_stride, const T* gate,
                                                        int64_t gate_stride, float* state, T* y) {
  chain_wait();
  const int64_t i = int64_t{blockIdx.x} * 256 + threadIdx.x;
  if (i >= count) return;
  const int64_t row = i / channels;
  const int c = static_cast<int>(i - row * channels);
  const float al = minus_gate(both(to_float(gate[row * gate_stride + c]))).x;
  const float h = fmaf(al, state[i] - to_float(x[row * x_stride + c]), state[i]);
  state[i] = h;
  y[i] = from_float<T>(h);
}

int32_t check_args(const gs_gated_scan_args& a) {
  if (a.tokens < 0 || a.tokens > GS_MAX_SEQUENCE_TOKENS || a.channels < 1 || a.sequences < 1 ||
      a.num_tiles < 0 || a.dtype < GS_FLOAT32 || a.dtype > GS_FLOAT16)
    return GS_ERR_INVALID_ARGUMENT;
  if (!layout_holds(a.tokens, a.sequences, a.num_tiles, a.tiles, a.tile_starts) ||
      (!a.tile_starts && a.sequences != 1))
    return GS_ERR_INVALID_ARGUMENT;
  if (!is_aligned(a.tiles, 16) || !is_aligned(a.workspace, 8)) return GS_ERR_MISALIGNED;
  const int64_t columns = (int64_t{a.channels} + 7) / 8;
  if (columns * (a.num_tiles + a.sequences) > INT32_MAX) return GS_ERR_CAPACITY;
  if (a.num_tiles > 0 && (!a.x || !a.gate || !a.entering || !a.workspace))
    return GS_ERR_INVALID_ARGUMENT;
  if (a.workspace_size < gated_scan_workspace_size(a))
    return GS_ERR_CAPACITY;
  return GS_OK;
}

// Boxes need whole 16-byte words: arrays, rows and strides.
template <class T>
bool whole_words(const gs_gated_scan_args& a) {
  constexpr int kWord = 16 / sizeof(T);
  if (a.channels % kWord || a.x_stride % kWord || a.gate_stride % kWord || a.x_stride <= 0 ||
      a.gate_stride <= 0)
    return false;
  for (const void* p : {a.x, a.gate, a.grad_y, static_cast<const void*>(a.y),
                        static_cast<const void*>(a.grad_x), static_cast<const void*>(a.grad_gate)})
    if (!is_aligned(p, 16)) return false;
  return true;
}

int64_t slots_of(const gs_gated_scan_args& a, int64_t length) {
  return a.num_tiles / length + (a.tile_starts ? a.sequences : 1);
}

// Long spans give a block a walk to load ahead in and leave few maps to scan;
// but first every multiprocessor gets its blocks, several times over. At most
// 8 tiles: longer ones gain nothing more.
template <class T>
Spans spans_of(const gs_gated_scan_args& a, bool boxes) {
  const int64_t items = a.num_tiles * ceil_div(a.channels, boxes ? 128 / sizeof(T) : 32);
  const int64_t length = std::clamp<int64_t>(items / (8 * kSmCount), 1, 8);
  return {static_cast<int>(length), static_cast<int>(slots_of(a, length))};
}

template <bool kBackward>
int32_t scan_spans(const gs_gated_scan_args& a, const Spans& spans, const Affine* folds,
                   float* entering, cudaStream_t stream) {
  // Long sequences: fewer channels a block and more threads share the spans
  // (1,000,000 x 64: 10 us; 100,003 x 1024 in 24 sequences: 5 us, with 1024 threads 11).
  const int64_t sequences = a.tile_starts ? a.sequences : 1;
  const bool narrow = spans.slots / sequences > 128;
  const unsigned blocks = ceil_div(a.channels, narrow ? 8 : 32) * static_cast<unsigned>(sequences);
  if (narrow)
    launch_chained(span_scan_kernel<kBackward, 8, 1024>, blocks, 1024, stream, a, spans, folds,
                   entering);
  else
    launch_chained(span_scan_kernel<kBackward, 32, 256>, blocks, 256, stream, a, spans, folds,
                   entering);
  return check_launch();
}

// The maps of the arrays that a pass loads: gate, then x and grad_y in the order
// given (backward's fold: gate, grad_y).
template <class T>
int32_t encode_maps(const gs_gated_scan_args& a, bool grad_first, Maps* maps) {
  GS_TRY(tc::encode_rows(&maps->gate, a.dtype, a.gate, a.tokens, a.channels, a.gate_stride, kTile));
  GS_TRY(tc::encode_rows(grad_first ? &maps->grad : &maps->x, a.dtype, a.x, a.tokens, a.channels,
                         a.x_stride, kTile));
  if (a.grad_y)
    GS_TRY(tc::encode_rows(grad_first ? &maps->x : &maps->grad, a.dtype, a.grad_y, a.tokens,
                           a.channels, a.channels, kTile));
  return GS_OK;
}

template <class T>
int32_t forward(const gs_gated_scan_args& a, cudaStream_t stream) {
  const bool boxes = whole_words<T>(a);
  const Spans spans = spans_of<T>(a, boxes);
  Affine* folds = static_cast<Affine*>(a.workspace);
  float* states = reinterpret_cast<float*>(folds + int64_t{spans.slots} * a.channels);
  const unsigned blocks = a.num_tiles == 0 ? 0
                                           : ceil_div(a.channels, boxes ? 128 / sizeof(T) : 32) *
                                                 static_cast<unsigned>(spans.slots);
  constexpr size_t kShared = sizeof(Boxes<2>);
  Maps maps = {};
  if (blocks && boxes) {
    GS_TRY(encode_maps<T>(a, false, &maps));
    GS_TRY((allow_shared<fold_boxes_kernel<T, false>>(kShared)));
    GS_TRY((allow_shared<walk_boxes_kernel<T>>(kShared)));
    launch_chained_shared(fold_boxes_kernel<T, false>, blocks, kBoxThreads, kShared, stream, a,
                          spans, folds, maps);
  } else if (blocks) {
    launch_chained(fold_kernel<T, false>, blocks, kPlainThreads, stream, a, spans, folds);
  }
  GS_TRY(check_launch());
  GS_TRY(scan_spans<false>(a, spans, folds, states, stream));
  if (blocks && boxes)
    launch_chained_shared(walk_boxes_kernel<T>, blocks, kBoxThreads, kShared, stream, a, spans,
                          states, maps);
  else if (blocks)
    launch_chained(walk_kernel<T>, blocks, kPlainThreads, stream, a, spans, states);
  return check_launch();
}

template <class T>
int32_t backward(const gs_gated_scan_args& a, cudaStream_t stream) {
  const bool boxes = whole_words<T>(a);
  const Spans spans = spans_of<T>(a, boxes);
  Affine* folds = static_cast<Affine*>(a.workspace);
  float* messages = reinterpret_cast<float*>(folds + int64_t{spans.slots} * a.channels);
  const unsigned blocks = a.num_tiles == 0 ? 0
                                           : ceil_div(a.channels, boxes ? 128 / sizeof(T) : 32) *
                                                 static_cast<unsigned>(spans.slots);
  if (blocks && boxes) {
    Maps maps = {};
    GS_TRY(encode_maps<T>(a, true, &maps));
    GS_TRY((allow_shared<fold_boxes_kernel<T, true>>(sizeof(Boxes<2>))));
    launch_chained_shared(fold_boxes_kernel<T, true>, blocks, kBoxThreads, sizeof(Boxes<2>),
                          stream, a, spans, folds, maps);
  } else if (blocks) {
    launch_chained(fold_kernel<T, true>, blocks, kPlainThreads, stream, a, spans, folds);
  }
  GS_TRY(check_launch());
  GS_TRY(scan_spans<true>(a, spans, folds, messages, stream));
  if (blocks && boxes) {
    Maps maps = {};
    GS_TRY(encode_maps<T>(a, false, &maps));
    GS_TRY((allow_shared<walk_back_boxes_kernel<T>>(sizeof(Boxes<3>))));
    launch_chained_shared(walk_back_boxes_kernel<T>, blocks, kBoxThreads, sizeof(Boxes<3>),
                          stream, a, spans, messages, maps);
  } else if (blocks) {
    launch_chained(walk_back_kernel<T>, blocks, kPlainThreads, stream, a, spans, messages);
  }
  return check_launch();
}

}  // namespace

// Maps and states of the spans, which are never more than with one tile each.
uint64_t gated_scan_workspace_size(const gs_gated_scan_args& a) {
  return (sizeof(Affine) + sizeof(float)) * static_cast<uint64_t>(slots_of(a, 1)) * a.channels;
}

int32_t gated_scan_status(cudaStream_t stream) { return take_timeout(g_timeout, stream); }

int32_t launch_gated_scan(const gs_gated_scan_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (!a.last || (a.num_tiles > 0 && !a.y)) return GS_ERR_INVALID_ARGUMENT;
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return forward<T>(a, stream);
  });
}

int32_t launch_gated_scan_backward(const gs_gated_scan_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a));
  if (a.num_tiles > 0 && (!a.grad_y || !a.grad_x || !a.grad_gate)) return GS_ERR_INVALID_ARGUMENT;
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return backward<T>(a, stream);
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
