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

#include "sequence.cuh"

namespace gs {

int32_t launch_window_attention(const gs_window_attention_args& a, cudaStream_t stream);
int32_t launch_window_attention_backward(const gs_window_attention_args& a, cudaStream_t stream);
int32_t launch_window_attention_step(const gs_window_attention_step_args& a, cudaStream_t stream);
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

template <class T>
__global__ void __launch_bounds__(kThreads) attention_kernel(gs_window_attention_args a) {
  chain_wait();
  __shared__ float s_row[kWarps][kMaxDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Tile tile = tile_at(a.tiles, blockIdx.x, static_cast<int32_t>(a.tokens), kTile);
  const int head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
  const T* k = static_cast<const T*>(a.k) + kv_head * a.k_head_stride;
  const T* v = static_cast<const T*>(a.v) + kv_head * a.v_head_stride;
  const int last = min(tile.end, tile.start + kTile);
  for (int t = tile.start + warp; t < last; t += kWarps) {
    __syncwarp();
    stage_row(s_row[warp], static_cast<const T*>(a.q) + t * a.q_stride + head * a.q_head_stride,
              a.dim, lane);
    const Runs runs(a, t - tile.begin, tile.end - tile.begin);
    float top = -INFINITY, sum = 0.0f, acc[kWords] = {};
    for (int base = 0; base < runs.count(); base += 32) {
      const bool in = base + lane < runs.count();
      const int64_t key = tile.begin + (in ? runs.key(base + lane) : 0);
      float s = -INFINITY;
      if (in && (!a.valid || a.valid[key]))
        s = dot(s_row[warp], k + key * a.k_stride, a.dim) * a.scale;
      // Nothing seen so far: any finite shift leaves exp(-inf) = 0, and a NaN score shows.
      const float next = fmaxf(top, warp_max(s)), shift = next == -INFINITY ? 0.0f : next;
      const float p = expf(s - shift), shrink = expf(top - shift);
      top = next;
      sum = fmaf(sum, shrink, warp_sum(p));
#pragma unroll
      for (int c = 0; c < kWords; ++c) acc[c] *= shrink;
      add_rows(acc, p, v, a.v_stride, key, a.dim, lane);
    }
    store_row(static_cast<T*>(a.out) + (int64_t{t} * a.heads + head) * a.dim, acc,
              sum == 0.0f ? 0.0f : 1.0f / sum, a.dim, lane);
    if (a.lse && lane == 0)
      a.lse[head * a.tokens + t] = sum == 0.0f ? -INFINITY : top + logf(sum);
  }
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
  if (a.tokens < 0 || a.tokens > INT32_MAX || a.num_tiles < 0 || a.num_tiles > INT32_MAX ||
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
    launch_chained(attention_kernel<T>, dim3(a.num_tiles, a.heads), kThreads, stream, a);
    return check_launch();
  });
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
