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
// forward norms the unrounded z, and so does the backward: it reads z as it was
// stored where that is a float (or x itself), and adds x and r again where a 16-bit
// sum would bring its rounding into every term (dw's error against the definition
// is then half as large again; the price is one more 16-bit array to read).
//
// Bound by memory: a token's row is read and written once. 262,144 tokens of 1024
// 16-bit channels on a 32-bit residual: forward 467 us (6.9 TB/s), backward 665 us
// (6.5 TB/s) and 6 us for the weight's sums; 16 tokens to 8 bits 4.5 us.

#include <cuda_fp8.h>

#include <algorithm>

#include "sequence.cuh"

namespace gs {

int32_t launch_rms_norm(const gs_rms_norm_args& a, cudaStream_t stream);
int32_t launch_rms_norm_backward(const gs_rms_norm_args& a, cudaStream_t stream);
uint64_t rms_norm_workspace_size(int64_t rows, int64_t channels);

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBackwardBlocks = 4 * kSmCount;  // rows of partial weight gradients
constexpr float kE4m3Max = 448.0f;

__device__ __forceinline__ float load_weight(const void* w, int32_t dtype, int64_t c) {
  if (dtype == GS_FLOAT32) return __ldg(static_cast<const float*>(w) + c);
  if (dtype == GS_BFLOAT16) return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(w) + c));
  return __half2float(__ldg(static_cast<const __half*>(w) + c));
}

__device__ __forceinline__ void load_weights(const void* w, int32_t dtype, int c, float (&x)[8]) {
  if (dtype == GS_FLOAT32) load_pack<8>(static_cast<const float*>(w) + c, x);
  else if (dtype == GS_BFLOAT16) load_pack<8>(static_cast<const __nv_bfloat16*>(w) + c, x);
  else load_pack<8>(static_cast<const __half*>(w) + c, x);
}

// The 8-bit code of z w / s' for s' = max|z w| / 448 (y / s without the m that
// cancels), from the product in double: a float chain z m w / s is off by a few
// units in the last place, which moves one value in some 10^5 across a rounding
// boundary of e4m3. The last conversion rounds a float that keeps, in its lowest
// bit, whether anything was cut off, so that the one rounding is to e4m3. Quotients
// of 16-bit inputs often lie halfway between two codes, where the rounding of
// `inverse` must not decide: it is 2^-50 too large, so that such a product is not below
// the halfway point, and what is less than 2^-40 above it (448 * 1.5 * 2^-50 at most)
// counts as nothing. The nearest other quotient of 16-bit inputs is 2^-37 away.
constexpr double kAbove = 1.0 + 0x1p-50;
__device__ __forceinline__ uint8_t to_e4m3(double zw, double inverse) {
  const double v = zw * inverse;
  float f = __double2float_rz(v);
  if (fabs(v - static_cast<double>(f)) > 0x1p-40) f = __int_as_float(__float_as_int(f) | 1);
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
    const double z = to_float(x[c]) + (r ? to_float(r[c]) : 0.0f);
    return z * load_weight(a.weight, a.weight_dtype, c);
  };
  if (a.q) {
    float top = 0.0f;
    for (int c = lane; c < a.channels; c += 32)
      top = fmaxf(top, fabsf(static_cast<float>(product(c))));
    top = warp_max(top);
    if (top > 0.0f) inverse = kE4m3Max / static_cast<double>(top) * kAbove;
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
__device__ __forceinline__ float block_max(float v, float2* shared) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5].x = v;
  __syncthreads();
  float top = shared[0].x;
#pragma unroll
  for (int w = 1; w < kWarps; ++w) top = fmaxf(top, shared[w].x);
  return top;
}

// Rows of whole, aligned 16-byte words: kLanes threads (a warp or the block)
// hold a token in registers, kIter words of 8 channels a thread, all loaded
// before the first is used, so the row is read once and a multiprocessor has
// tens of kilobytes in flight.
template <class T, class R, int kLanes, int kIter>
__global__ void __launch_bounds__(kThreads) norm_rows_kernel(gs_rms_norm_args a) {
  chain_wait();
  __shared__ float2 s_sum[kWarps];
  constexpr int kRows = kThreads / kLanes;
  const int64_t row = int64_t{blockIdx.x} * kRows + threadIdx.x / kLanes;
  if (row >= a.rows) return;
  const int lane = threadIdx.x % kLanes;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const R* r = a.residual ? static_cast<const R*>(a.residual) + row * a.residual_stride : nullptr;
  float z[kIter][8];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int c = (i * kLanes + lane) * 8;
    if (c < a.channels) load_pack<8>(x + c, z[i]);
  }
  if (r)
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int c = (i * kLanes + lane) * 8;
      float y[8];
      if (c < a.channels) {
        load_pack<8>(r + c, y);
#pragma unroll
        for (int k = 0; k < 8; ++k) z[i][k] += y[k];
      }
    }
  float square = 0.0f;
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int c = (i * kLanes + lane) * 8;
    if (c < a.channels) {
#pragma unroll
      for (int k = 0; k < 8; ++k) square = fmaf(z[i][k], z[i][k], square);
      if (a.sum) store_pack<8>(static_cast<R*>(a.sum) + row * a.channels + c, z[i]);
    }
  }
  square = kLanes == 32 ? warp_sum(square) : block_sum2(make_float2(square, 0.0f), s_sum).x;
  const float m = rsqrtf(square / static_cast<float>(a.channels) + a.eps);
  double inverse = 0.0;
  if (a.q) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int c = (i * kLanes + lane) * 8;
      if (c < a.channels) {
        float w[8];
        load_weights(a.weight, a.weight_dtype, c, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(z[i][k] * w[k]));
      }
    }
    top = kLanes == 32 ? warp_max(top) : block_max(top, s_sum);
    if (top > 0.0f) inverse = kE4m3Max / static_cast<double>(top) * kAbove;
    if (lane == 0) a.scale[row] = top > 0.0f ? top * m / kE4m3Max : 1.0f;
  }
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int c = (i * kLanes + lane) * 8;
    if (c >= a.channels) continue;
    float w[8];
    load_weights(a.weight, a.weight_dtype, c, w);
    if (a.q) {
      uint2 codes = make_uint2(0, 0);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        codes.x |= to_e4m3(static_cast<double>(z[i][k]) * w[k], inverse) << (8 * k);
        codes.y |= to_e4m3(static_cast<double>(z[i][k + 4]) * w[k + 4], inverse) << (8 * k);
      }
      *reinterpret_cast<uint2*>(a.q + row * a.channels + c) = codes;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = z[i][k] * m * w[k];
      store_pack<8>(static_cast<T*>(a.y) + row * a.channels + c, w);
    }
  }
}

// Any channel count and alignment: one block a token at a time. A channel's
// weight gradient is summed by the one thread that owns the channel, token
// after token, in shared memory; the block's sums go to its row of partials.
// kAgain: z is x + r again, else the stored sum.
template <class T, class R, bool kAgain>
__global__ void __launch_bounds__(kThreads) norm_backward_kernel(gs_rms_norm_args a,
                                                                 float* partials) {
  chain_wait();
  extern __shared__ float s_dw[];
  __shared__ float2 s_sum[kWarps];
  for (int c = threadIdx.x; c < a.channels; c += kThreads) s_dw[c] = 0.0f;
  const float inverse = 1.0f / static_cast<float>(a.channels);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const R* sum = kAgain ? nullptr : static_cast<const R*>(a.sum) + row * a.sum_stride;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const R* r = static_cast<const R*>(a.residual) + row * a.residual_stride;
    const auto z = [&](int c) {
      if constexpr (kAgain) return to_float(x[c]) + to_float(r[c]);
      else return to_float(sum[c]);
    };
    const T* g = static_cast<const T*>(a.grad_y) + row * a.channels;
    const R* h = a.grad_sum ? static_cast<const R*>(a.grad_sum) + row * a.channels : nullptr;
    float2 v = make_float2(0.0f, 0.0f);
    for (int c = threadIdx.x; c < a.channels; c += kThreads) {
      const float zc = z(c);
      const float gw = to_float(g[c]) * load_weight(a.weight, a.weight_dtype, c);
      v.x = fmaf(zc, zc, v.x);
      v.y = fmaf(gw, zc, v.y);
    }
    v = block_sum2(v, s_sum);
    const float m = rsqrtf(v.x * inverse + a.eps);
    const float pull = v.y * inverse * m * m;
    for (int c = threadIdx.x; c < a.channels; c += kThreads) {
      const float zc = z(c), gc = to_float(g[c]);
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

// Sums over a group of kLanes threads of the block; `turn` alternates between
// two sets of slots, so that one barrier a row is enough.
template <int kLanes>
__device__ __forceinline__ float2 group_sum2(float2 v, float2 (*shared)[kWarps], int turn) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  if constexpr (kLanes > 32) {
    constexpr int kGroupWarps = kLanes / 32;
    const int warp = threadIdx.x >> 5, group = threadIdx.x / kLanes;
    if ((threadIdx.x & 31) == 0) shared[turn][warp] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(kLanes) : "memory");
    v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kGroupWarps; ++w) {
      v.x += shared[turn][group * kGroupWarps + w].x;
      v.y += shared[turn][group * kGroupWarps + w].y;
    }
  }
  return v;
}

// Rows of whole, aligned 16-byte words: a group of kLanes threads holds a
// token, kIter words of 8 channels a thread, and the weight gradients of their
// channels from token to token; a block's groups add theirs up in order. One
// or two words a thread keep a thread at 64 registers, so that 32 warps a
// multiprocessor cover the loads (a warp a token of 1024 channels took 160
// registers, 8 warps, and 963 us for 262,144 tokens). kAgain spills a few words at 64
// registers; three blocks instead of four without spills took 967 us for a pass of
// 262,144 x 1024 bf16 on a bf16 residual, four 801 (712 with the stored sum).
template <class T, class R, bool kAgain, int kLanes, int kIter>
__global__ void __launch_bounds__(kThreads, 4 / kIter)
    norm_rows_backward_kernel(gs_rms_norm_args a, float* partials) {
  chain_wait();
  extern __shared__ float s_dw[];
  __shared__ float2 s_sum[2][kWarps];
  int turn = 0;
  constexpr int kRows = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const float inverse = 1.0f / static_cast<float>(a.channels);
  float dw[kIter][8] = {};
  for (int64_t row = int64_t{blockIdx.x} * kRows + group; row < a.rows;
       row += int64_t{gridDim.x} * kRows) {
    const R* z_row = kAgain ? static_cast<const R*>(a.residual) + row * a.residual_stride
                            : static_cast<const R*>(a.sum) + row * a.sum_stride;
    const T* x_row = static_cast<const T*>(a.x) + row * a.x_stride;
    const int64_t at = row * a.channels;
    Pack<R, 8> z[kIter], h[kIter];  // kAgain: r in z's place
    Pack<T, 8> g[kIter], x[kIter];
    const auto value = [&](int i, int k) {
      if constexpr (kAgain) return to_float(x[i].v[k]) + to_float(z[i].v[k]);
      else return to_float(z[i].v[k]);
    };
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int c = (i * kLanes + lane) * 8;
      if (c < a.channels) {
        z[i] = *reinterpret_cast<const Pack<R, 8>*>(z_row + c);
        if constexpr (kAgain) x[i] = *reinterpret_cast<const Pack<T, 8>*>(x_row + c);
        g[i] = *reinterpret_cast<const Pack<T, 8>*>(static_cast<const T*>(a.grad_y) + at + c);
        if (a.grad_sum)
          h[i] = *reinterpret_cast<const Pack<R, 8>*>(static_cast<const R*>(a.grad_sum) + at + c);
      }
    }
    float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int c = (i * kLanes + lane) * 8;
      if (c < a.channels) {
        float w[8];
        load_weights(a.weight, a.weight_dtype, c, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float zc = value(i, k);
          v.x = fmaf(zc, zc, v.x);
          v.y = fmaf(to_float(g[i].v[k]) * w[k], zc, v.y);
        }
      }
    }
    v = group_sum2<kLanes>(v, s_sum, turn);
    turn ^= 1;
    const float m = rsqrtf(v.x * inverse + a.eps);
    const float pull = v.y * inverse * m * m;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int c = (i * kLanes + lane) * 8;
      if (c >= a.channels) continue;
      float w[8];
      load_weights(a.weight, a.weight_dtype, c, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float zc = value(i, k), gc = to_float(g[i].v[k]);
        const float own = a.grad_sum ? to_float(h[i].v[k]) : 0.0f;
        w[k] = fmaf(m, fmaf(-zc, pull, gc * w[k]), own);
        dw[i][k] = fmaf(gc, zc * m, dw[i][k]);
      }
      store_pack<8>(static_cast<T*>(a.grad_x) + at + c, w);
      if (a.grad_residual) store_pack<8>(static_cast<R*>(a.grad_residual) + at + c, w);
    }
  }
  for (int owner = 0; owner < kRows; ++owner) {
    if (group == owner)
#pragma unroll
      for (int i = 0; i < kIter; ++i) {
        const int c = (i * kLanes + lane) * 8;
        if (c < a.channels)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float sum = owner ? s_dw[c + k] + dw[i][k] : dw[i][k];
            if (owner == kRows - 1) partials[int64_t{blockIdx.x} * a.channels + c + k] = sum;
            else s_dw[c + k] = sum;
          }
      }
    __syncthreads();
  }
}

// The weight gradient: the blocks' partial sums, 32 channels a block, each warp
// its share of the rows, the shares in order.
constexpr int kWeightWarps = 32;
template <class W>
__global__ void __launch_bounds__(32 * kWeightWarps) norm_weight_kernel(const float* partials, int blocks,
                                                               int channels, W* grad_weight) {
  chain_wait();
  __shared__ float s_part[kWeightWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float sum = 0.0f;
  if (c < channels)
#pragma unroll 8
    for (int b = warp; b < blocks; b += kWeightWarps) sum += partials[int64_t{b} * channels + c];
  s_part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && c < channels) {
    sum = 0.0f;
    for (int w = 0; w < kWeightWarps; ++w) sum += s_part[w][lane];
    grad_weight[c] = from_float<W>(sum);
  }
}

int backward_blocks(int64_t rows) {
  return static_cast<int>(rows < kBackwardBlocks ? rows : kBackwardBlocks);
}

// Whether the backward makes a 16-bit sum again from its parts.
bool adds_again(const gs_rms_norm_args& a) {
  return !a.sum && a.x && a.residual && a.dtype != GS_FLOAT32 && a.residual_dtype == a.dtype;
}

int32_t check_args(const gs_rms_norm_args& a, bool backward) {
  const auto valid = [](int32_t t) { return t >= GS_FLOAT32 && t <= GS_FLOAT16; };
  if (a.rows < 0 || a.channels < 1 || a.channels > GS_MAX_NORM_CHANNELS || !valid(a.dtype) ||
      !valid(a.residual_dtype) || !valid(a.weight_dtype) || !a.weight)
    return GS_ERR_INVALID_ARGUMENT;
  if (a.residual_dtype != a.dtype && a.residual_dtype != GS_FLOAT32) return GS_ERR_UNSUPPORTED;
  if (a.rows == 0) return GS_OK;
  if (backward) {
    if ((!a.sum && !adds_again(a)) || !a.grad_y || !a.grad_x || !a.grad_weight || !a.workspace)
      return GS_ERR_INVALID_ARGUMENT;
    if (a.workspace_size < rms_norm_workspace_size(a.rows, a.channels)) return GS_ERR_CAPACITY;
  } else if (!a.x || (a.q ? !a.scale : !a.y)) {
    return GS_ERR_INVALID_ARGUMENT;
  }
  return GS_OK;
}

template <int N>
using Number = std::integral_constant<int, N>;

// Calls f with the forward's (threads of a token, words of 8 channels a
// thread): a warp up to `warp_channels`, else the block.
template <class F>
int32_t with_forward_shape(int channels, int warp_channels, F&& f) {
  if (channels <= warp_channels) {
    if (channels <= 256) return f(Number<32>{}, Number<1>{});
    if (channels <= 512) return f(Number<32>{}, Number<2>{});
    if (channels <= 1024) return f(Number<32>{}, Number<4>{});
    return f(Number<32>{}, Number<8>{});
  }
  if (channels <= 2048) return f(Number<256>{}, Number<1>{});
  if (channels <= 4096) return f(Number<256>{}, Number<2>{});
  if (channels <= 8192) return f(Number<256>{}, Number<4>{});
  return f(Number<256>{}, Number<8>{});
}

// The same for the backward, up to 8192 channels: as few words a thread as a
// block can have.
template <class F>
int32_t with_backward_shape(int channels, F&& f) {
  if (channels <= 256) return f(Number<32>{}, Number<1>{});
  if (channels <= 512) return f(Number<64>{}, Number<1>{});
  if (channels <= 1024) return f(Number<128>{}, Number<1>{});
  if (channels <= 2048) return f(Number<256>{}, Number<1>{});
  if (channels <= 4096) return f(Number<256>{}, Number<2>{});
  return f(Number<256>{}, Number<4>{});
}

bool whole_words(const gs_rms_norm_args& a) {
  if (a.channels % 8 || a.x_stride % 8 || a.residual_stride % 8 || a.sum_stride % 8) return false;
  for (const void* p : {a.x, a.residual, a.weight, static_cast<const void*>(a.y),
                        static_cast<const void*>(a.sum), static_cast<const void*>(a.q), a.grad_y,
                        a.grad_sum, static_cast<const void*>(a.grad_x),
                        static_cast<const void*>(a.grad_residual)})
    if (!is_aligned(p, 16)) return false;
  return true;
}

template <class T, class R>
int32_t forward(const gs_rms_norm_args& a, cudaStream_t stream) {
  if (whole_words(a)) {
    // With fewer tokens than multiprocessors a token's latency is the call's:
    // the whole block shares it.
    const int warp_channels = a.rows <= kSmCount ? 256 : 2048;
    return with_forward_shape(a.channels, warp_channels, [&](auto lanes, auto iter) {
      constexpr int kLanes = decltype(lanes)::value, kIter = decltype(iter)::value;
      launch_chained(norm_rows_kernel<T, R, kLanes, kIter>, ceil_div(a.rows, kThreads / kLanes),
                     kThreads, stream, a);
      return check_launch();
    });
  }
  launch_chained(norm_kernel<T, R>, ceil_div(a.rows, kWarps), kThreads, stream, a);
  return check_launch();
}

template <class T, class R, bool kAgain>
int32_t backward(const gs_rms_norm_args& a, cudaStream_t stream) {
  float* partials = static_cast<float*>(a.workspace);
  int blocks = backward_blocks(a.rows);
  const size_t shared = sizeof(float) * a.channels;
  if (whole_words(a) && a.channels <= 8192) {
    GS_TRY(with_backward_shape(a.channels, [&](auto lanes, auto iter) {
      constexpr int kLanes = decltype(lanes)::value, kIter = decltype(iter)::value;
      blocks = std::min<int>(blocks, ceil_div(a.rows, kThreads / kLanes));
      launch_chained_shared(norm_rows_backward_kernel<T, R, kAgain, kLanes, kIter>, blocks, kThreads,
                            kLanes < kThreads ? shared : 0, stream, a, partials);
      return check_launch();
    }));
  } else {
    GS_TRY((allow_shared<norm_backward_kernel<T, R, kAgain>>(sizeof(float) *
                                                             GS_MAX_NORM_CHANNELS)));
    launch_chained_shared(norm_backward_kernel<T, R, kAgain>, blocks, kThreads, shared, stream, a,
                          partials);
    GS_TRY(check_launch());
  }
  return with_dtype(a.weight_dtype, [&](auto w) {
    using W = decltype(w);
    launch_chained(norm_weight_kernel<W>, ceil_div(a.channels, 32), 32 * kWeightWarps, stream, partials,
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
    if constexpr (!std::is_same_v<T, float>)
      if (adds_again(a)) return backward<T, T, true>(a, stream);
    return a.residual_dtype == a.dtype ? backward<T, T, false>(a, stream)
                                       : backward<T, float, false>(a, stream);
  });
}

}  // namespace gs
