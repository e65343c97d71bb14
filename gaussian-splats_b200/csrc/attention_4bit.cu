// One new token a stream against a window's cache held in 4 bits: the step of
// attention.cu with rows of codes, x ~ (c - 7.5) step + middle, c in 0..15.
//
//   score_t = scale q . k_t,  p = softmax(score) over the slots that count,
//   out = sum p_t v_t
#include "tensorcore.cuh"

namespace gs {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxDim = 128;

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

template <class T>
__device__ __forceinline__ uint32_t code_of(float x, float step, float middle) {
  if (!(step > 0.0f && step < INFINITY)) return 8;
  const double place = rint((static_cast<double>(x) - middle) / static_cast<double>(step) + 7.5);
  return static_cast<uint32_t>(fmin(fmax(place, 0.0), 15.0));
}

template <class T>
__global__ void __launch_bounds__(kThreads) step_kernel(gs_window_attention_step_4bit_args a) {
  __shared__ float q[kMaxDim], weight[kThreads], parts[kThreads / 32];
  __shared__ uint8_t fresh[2][kMaxDim / 2];
  __shared__ T fresh_range[2][2];
  chain_wait();
  const int group = a.heads / a.kv_heads;
  const int64_t b = blockIdx.x / a.heads;
  const int head = blockIdx.x % a.heads, kv_head = head / group;
  const int thread = threadIdx.x, lane = thread & 31, warp = thread >> 5;
  const int64_t position = a.positions[b];
  T* const out = static_cast<T*>(a.out) + (b * a.heads + head) * a.dim;
  if (position < 0) {
    if (thread < a.dim) out[thread] = from_float<T>(0.0f);
    return;
  }
  const int64_t slot = position < a.first
                           ? position
                           : a.first + (position - a.first) % (a.slots - a.first);
  const int count = static_cast<int>(min(position + 1, int64_t{a.slots}));
  const int64_t row0 = (b * a.kv_heads + kv_head) * a.slots;
  const bool token_valid = !a.cache_valid || !a.valid || a.valid[b];
  const bool writes = head % group == 0;
  if (a.cache_valid && head == 0 && thread == 0) a.cache_valid[b * a.slots + slot] = token_valid;
  // The new token's rows as they are held.
  for (int side = 0; side < 2; ++side) {
    const T* x = side == 0
                     ? static_cast<const T*>(a.k) + b * a.k_stride + kv_head * a.k_head_stride
                     : static_cast<const T*>(a.v) + b * a.v_stride + kv_head * a.v_head_stride;
    if (warp == 0) {
      float high = -INFINITY, low = INFINITY;
      for (int c = lane; c < a.dim; c += 32) {
        high = max_nan(high, to_float(x[c]));
        low = min_nan(low, to_float(x[c]));
      }
      for (int o = 16; o > 0; o >>= 1) {
        high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, o));
        low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
      }
      const T step = from_float<T>((high - low) / 15.0f);
      const T middle = from_float<T>(0.5f * high + 0.5f * low);
      for (int c = lane; c < a.dim / 2; c += 32)
        fresh[side][c] = static_cast<uint8_t>(
            code_of<T>(to_float(x[2 * c]), to_float(step), to_float(middle)) |
            code_of<T>(to_float(x[2 * c + 1]), to_float(step), to_float(middle)) << 4);
      if (lane == 0) {
        fresh_range[side][0] = step;
        fresh_range[side][1] = middle;
      }
    }
  }
  if (thread < a.dim)
    q[thread] = to_float(static_cast<const T*>(a.q)[b * a.q_stride + head * a.q_head_stride + thread]) *
                a.scale;
  __syncthreads();
  if (writes)
    for (int side = 0; side < 2; ++side) {
      uint8_t* codes = (side == 0 ? a.k_codes : a.v_codes) + (row0 + slot) * (a.dim / 2);
      T* range = static_cast<T*>(side == 0 ? a.k_range : a.v_range) + (row0 + slot) * 2;
      if (thread < a.dim / 2) codes[thread] = fresh[side][thread];
      if (thread < 2) range[thread] = fresh_range[side][thread];
    }
  const auto row_of = [&](int side, int at) {
    return at == slot ? fresh[side]
                      : (side == 0 ? a.k_codes : a.v_codes) + (row0 + at) * (a.dim / 2);
  };
  const auto range_of = [&](int side, int at) {
    return at == slot ? fresh_range[side]
                      : static_cast<const T*>(side == 0 ? a.k_range : a.v_range) + (row0 + at) * 2;
  };
  float top = -INFINITY, sum = 0.0f, o = 0.0f;
  for (int base = 0; base < count; base += kThreads) {
    const int at = base + thread;
    float score = -INFINITY;
    if (at < count &&
        (!a.cache_valid || (at == slot ? token_valid : a.cache_valid[b * a.slots + at] != 0))) {
      const uint8_t* codes = row_of(0, at);
      const T* range = range_of(0, at);
      const float step = to_float(range[0]), middle = to_float(range[1]);
      score = 0.0f;
      for (int c = 0; c < a.dim / 2; ++c) {
        const uint32_t two = codes[c];
        score = fmaf(q[2 * c], fmaf(static_cast<float>(two & 15) - 7.5f, step, middle), score);
        score = fmaf(q[2 * c + 1], fmaf(static_cast<float>(two >> 4) - 7.5f, step, middle), score);
      }
    }
    __syncthreads();  // parts and weights of the tile before are read
    float high = warp_max(score);
    if (lane == 0) parts[warp] = high;
    weight[thread] = score;
    __syncthreads();
    for (float x : parts) high = fmaxf(high, x);
    const float next = fmaxf(top, high), shift = next == -INFINITY ? 0.0f : next;
    const float shrink = expf(top - shift);
    top = next;
    sum *= shrink;
    o *= shrink;
    const int tile = min(kThreads, count - base);
    for (int t = 0; t < tile; ++t) {
      if (weight[t] == -INFINITY) continue;  // what is left out must not meet its weight
      const float p = expf(weight[t] - shift);
      sum += p;
      if (thread < a.dim) {
        const uint32_t two = row_of(1, base + t)[thread / 2];
        const T* range = range_of(1, base + t);
        const float c = static_cast<float>(thread & 1 ? two >> 4 : two & 15);
        o = fmaf(p, fmaf(c - 7.5f, to_float(range[0]), to_float(range[1])), o);
      }
    }
  }
  if (thread < a.dim) out[thread] = from_float<T>(sum == 0.0f ? 0.0f : o / sum);
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
  if (a.batch * a.heads > INT32_MAX) return GS_ERR_CAPACITY;
  const unsigned blocks = static_cast<unsigned>(a.batch * a.heads);
  if (a.dtype == GS_BFLOAT16) launch_chained(step_kernel<__nv_bfloat16>, blocks, kThreads, stream, a);
  else launch_chained(step_kernel<__half>, blocks, kThreads, stream, a);
  return check_launch();
}

}  // namespace gs
