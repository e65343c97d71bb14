// Root-mean-square norm of a token's channels, with the residual's addition
// before it and, for serving, an 8-bit output with one scale a token.
//
//   z = x + r,  m = 1 / sqrt(mean(z^2) + eps),  y = z m w
//
// and, for the 8-bit output, s = max|y| / 448 (1 for a token of zeros) and
// q = y / s rounded to e4m3 (448 is e4m3's largest value). Backward, with g
// the gradient of y and h that of the sum z (the residual stream's own):
//
//   dz = m (g w - z m^2 mean(g w z)) + h,   dw = sum over tokens of g z m
//
// dz is the gradient of x and of r. Everything is computed in float. The
// forward norms the unrounded z; the backward reads z as it was stored (in
// the residual's type), which is what the next layer saw too.
//
// Bound by memory: a token's row is read and written once.

#include <cuda_fp8.h>

#include "sequence.cuh"

namespace gs {

int32_t launch_rms_norm(const gs_rms_norm_args& a, cudaStream_t stream);
int32_t launch_rms_norm_backward(const gs_rms_norm_args& a, cudaStream_t stream);
uint64_t rms_norm_workspace_size(int64_t rows, int64_t channels);

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBackwardBlocks = 2 * kSmCount;  // rows of partial weight gradients
constexpr float kE4m3Max = 448.0f;

__device__ __forceinline__ float load_weight(const void* w, int32_t dtype, int64_t c) {
  if (dtype == GS_FLOAT32) return __ldg(static_cast<const float*>(w) + c);
  if (dtype == GS_BFLOAT16) return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(w) + c));
  return __half2float(__ldg(static_cast<const __half*>(w) + c));
}

// The 8-bit code of z w / s' for s' = max|z w| / 448 (y / s without the m that
// cancels), from the product in double: a float chain z m w / s is off by a few
// units in the last place, which moves one value in some 10^5 across a rounding
// boundary of e4m3. The last conversion rounds a float that keeps, in its lowest
// bit, whether bits were cut off, so that the one rounding is to e4m3.
__device__ __forceinline__ uint8_t to_e4m3(double zw, double inverse) {
  const double v = zw * inverse;
  float f = __double2float_rz(v);
  if (static_cast<double>(f) != v && v == v) f = __int_as_float(__float_as_int(f) | 1);
  return __nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3);
}

// Any channel count and alignment: one warp a token, the row read again for
// each pass over it (from L1 after the first).
template <class T, class R>
__global__ void __launch_bounds__(kThreads) norm_kernel(gs_rms_norm_args a) {
  chain_wait();
  const int64_t row = int64_t{blockIdx.x} * kWarps + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const int lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const R* r = a.residual ? static_cast<const R*>(a.residual) + row * a.residual_stride : nullptr;
  float square = 0.0f;
  for (int c = lane; c < a.channels; c += 32) {
    const float z = to_float(x[c]) + (r ? to_float(r[c]) : 0.0f);
    if (a.sum) static_cast<R*>(a.sum)[row * a.channels + c] = from_float<R>(z);
    square = fmaf(z, z, square);
  }
  const float m = rsqrtf(warp_sum(square) / static_cast<float>(a.channels) + a.eps);
  double inverse = 0.0;
  const auto product = [&](int c) {
    const double z = static_cast<double>(to_float(x[c])) + (r ? to_float(r[c]) : 0.0f);
    return z * load_weight(a.weight, a.weight_dtype, c);
  };
  if (a.q) {
    float top = 0.0f;
    for (int c = lane; c < a.channels; c += 32)
      top = fmaxf(top, fabsf(static_cast<float>(product(c))));
    top = warp_max(top);
    if (top > 0.0f) inverse = kE4m3Max / static_cast<double>(top);
    if (lane == 0) a.scale[row] = top > 0.0f ? top * m / kE4m3Max : 1.0f;
  }
  for (int c = lane; c < a.channels; c += 32) {
    if (a.q) {
      a.q[row * a.channels + c] = to_e4m3(product(c), inverse);
    } else {
      const float z = to_float(x[c]) + (r ? to_float(r[c]) : 0.0f);
      static_cast<T*>(a.y)[row * a.channels + c] =
          from_float<T>(z * m * load_weight(a.weight, a.weight_dtype, c));
    }
  }
}

// Sums over a block; every thread gets both totals.
__device__ __forceinline__ float2 block_sum2(float2 v, float2* shared) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  float2 total = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    total.x += shared[w].x;
    total.y += shared[w].y;
  }
  return total;
}

// Any channel count and alignment: one block a token at a time. A channel's
// weight gradient is summed by the one thread that owns the channel, token
// after token, in shared memory; the block's sums go to its row of partials.
template <class T, class R>
__global__ void __launch_bounds__(kThreads) norm_backward_kernel(gs_rms_norm_args a,
                                                                 float* partials) {
  chain_wait();
  extern __shared__ float s_dw[];
  __shared__ float2 s_sum[kWarps];
  for (int c = threadIdx.x; c < a.channels; c += kThreads) s_dw[c] = 0.0f;
  const float inverse = 1.0f / static_cast<float>(a.channels);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const R* z = static_cast<const R*>(a.sum) + row * a.sum_stride;
    const T* g = static_cast<const T*>(a.grad_y) + row * a.channels;
    const R* h = a.grad_sum ? static_cast<const R*>(a.grad_sum) + row * a.channels : nullptr;
    float2 v = make_float2(0.0f, 0.0f);
    for (int c = threadIdx.x; c < a.channels; c += kThreads) {
      const float zc = to_float(z[c]);
      const float gw = to_float(g[c]) * load_weight(a.weight, a.weight_dtype, c);
      v.x = fmaf(zc, zc, v.x);
      v.y = fmaf(gw, zc, v.y);
    }
    v = block_sum2(v, s_sum);
    const float m = rsqrtf(v.x * inverse + a.eps);
    const float pull = v.y * inverse * m * m;
    for (int c = threadIdx.x; c < a.channels; c += kThreads) {
      const float zc = to_float(z[c]), gc = to_float(g[c]);
      const float gw = gc * load_weight(a.weight, a.weight_dtype, c);
      const float d = fmaf(m, fmaf(-zc, pull, gw), h ? to_float(h[c]) : 0.0f);
      static_cast<T*>(a.grad_x)[row * a.channels + c] = from_float<T>(d);
      if (a.grad_residual)
        static_cast<R*>(a.grad_residual)[row * a.channels + c] = from_float<R>(d);
      s_dw[c] = fmaf(gc, zc * m, s_dw[c]);
    }
  }
  for (int c = threadIdx.x; c < a.channels; c += kThreads)
    partials[int64_t{blockIdx.x} * a.channels + c] = s_dw[c];
}

// The weight gradient: the blocks' partial sums in block order, 32 channels a
// block, each warp an eighth of the rows.
template <class W>
__global__ void __launch_bounds__(kThreads) norm_weight_kernel(const float* partials, int blocks,
                                                               int channels, W* grad_weight) {
  chain_wait();
  __shared__ float s_part[kWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float sum = 0.0f;
  if (c < channels)
#pragma unroll 8
    for (int b = warp; b < blocks; b += kWarps) sum += partials[int64_t{b} * channels + c];
  s_part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && c < channels) {
    sum = 0.0f;
    for (int w = 0; w < kWarps; ++w) sum += s_part[w][lane];
    grad_weight[c] = from_float<W>(sum);
  }
}

int backward_blocks(int64_t rows) {
  return static_cast<int>(rows < kBackwardBlocks ? rows : kBackwardBlocks);
}

int32_t check_args(const gs_rms_norm_args& a, bool backward) {
  const auto valid = [](int32_t t) { return t >= GS_FLOAT32 && t <= GS_FLOAT16; };
  if (a.rows < 0 || a.channels < 1 || a.channels > GS_MAX_NORM_CHANNELS || !valid(a.dtype) ||
      !valid(a.residual_dtype) || !valid(a.weight_dtype) || !a.weight)
    return GS_ERR_INVALID_ARGUMENT;
  if (a.residual_dtype != a.dtype && a.residual_dtype != GS_FLOAT32) return GS_ERR_UNSUPPORTED;
  if (a.rows == 0) return GS_OK;
  if (backward) {
    if (!a.sum || !a.grad_y || !a.grad_x || !a.grad_weight || !a.workspace)
      return GS_ERR_INVALID_ARGUMENT;
    if (a.workspace_size < rms_norm_workspace_size(a.rows, a.channels)) return GS_ERR_CAPACITY;
  } else if (!a.x || (a.q ? !a.scale : !a.y)) {
    return GS_ERR_INVALID_ARGUMENT;
  }
  return GS_OK;
}

template <class T, class R>
int32_t forward(const gs_rms_norm_args& a, cudaStream_t stream) {
  launch_chained(norm_kernel<T, R>, ceil_div(a.rows, kWarps), kThreads, stream, a);
  return check_launch();
}

template <class T, class R>
int32_t backward(const gs_rms_norm_args& a, cudaStream_t stream) {
  float* partials = static_cast<float*>(a.workspace);
  const int blocks = backward_blocks(a.rows);
  const size_t shared = sizeof(float) * a.channels;
  GS_CUDA_TRY(cudaFuncSetAttribute(norm_backward_kernel<T, R>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   sizeof(float) * GS_MAX_NORM_CHANNELS));
  launch_chained_shared(norm_backward_kernel<T, R>, blocks, kThreads, shared, stream, a, partials);
  GS_TRY(check_launch());
  return with_dtype(a.weight_dtype, [&](auto w) {
    using W = decltype(w);
    launch_chained(norm_weight_kernel<W>, ceil_div(a.channels, 32), kThreads, stream, partials,
                   blocks, a.channels, static_cast<W*>(a.grad_weight));
    return check_launch();
  });
}

}  // namespace

uint64_t rms_norm_workspace_size(int64_t rows, int64_t channels) {
  return sizeof(float) * static_cast<uint64_t>(backward_blocks(rows)) * channels;
}

int32_t launch_rms_norm(const gs_rms_norm_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a, false));
  if (a.rows == 0) return GS_OK;
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return a.residual_dtype == a.dtype ? forward<T, T>(a, stream) : forward<T, float>(a, stream);
  });
}

int32_t launch_rms_norm_backward(const gs_rms_norm_args& a, cudaStream_t stream) {
  GS_TRY(check_args(a, true));
  if (a.rows == 0) {
    if (a.grad_weight)
      GS_CUDA_TRY(cudaMemsetAsync(a.grad_weight, 0,
                                  static_cast<size_t>(a.channels) * element_size(a.weight_dtype),
                                  stream));
    return GS_OK;
  }
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return a.residual_dtype == a.dtype ? backward<T, T>(a, stream) : backward<T, float>(a, stream);
  });
}

}  // namespace gs
