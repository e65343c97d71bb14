// Shared pieces of the sequence operators (attention.cu, recurrence.cu, norm.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace gs {

// Element conversions: every operator computes in float and rounds once, on
// the store.
template <class T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(x);
  else return __half2float(x);
}
template <class T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(x);
  else return __float2half_rn(x);
}

// N consecutive elements at an address aligned to min(16, N * sizeof(T))
// bytes, in loads and stores of that width.
template <class T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
  T v[N];
};
template <int N, class T>
__device__ __forceinline__ void load_pack(const T* p, float (&x)[N]) {
  const Pack<T, N> a = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int k = 0; k < N; ++k) x[k] = to_float(a.v[k]);
}
template <int N, class T>
__device__ __forceinline__ void store_pack(T* p, const float (&x)[N]) {
  Pack<T, N> a;
#pragma unroll
  for (int k = 0; k < N; ++k) a.v[k] = from_float<T>(x[k]);
  *reinterpret_cast<Pack<T, N>*>(p) = a;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

inline int element_size(int32_t dtype) { return dtype == GS_FLOAT32 ? 4 : 2; }
inline bool is_aligned(const void* p, uintptr_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}

// Whether a batch's layout may be walked: a table with its sequences' first tiles,
// or neither and the tiles of one sequence.
inline bool layout_holds(int64_t tokens, int64_t sequences, int64_t num_tiles,
                         const int32_t* tiles, const int32_t* tile_starts) {
  if (tile_starts)
    return sequences >= 1 && sequences <= INT32_MAX / 2 && num_tiles <= INT32_MAX &&
           (num_tiles == 0 || tiles);
  return !tiles && num_tiles == (tokens + GS_SEQUENCE_TILE - 1) / GS_SEQUENCE_TILE;
}

// Calls f with a value of the element type that `dtype` names.
template <class F>
inline int32_t with_dtype(int32_t dtype, F&& f) {
  switch (dtype) {
    case GS_FLOAT32: return f(float{});
    case GS_BFLOAT16: return f(__nv_bfloat16{});
    case GS_FLOAT16: return f(__half{});
  }
  return GS_ERR_INVALID_ARGUMENT;
}

// Lets a kernel have `bytes` of dynamic shared memory (and clusters of 16 blocks),
// once a device: the attribute calls cost as much as a launch's other host work.
// `registers`: refuses a build that launches with fewer a thread, for a kernel whose
// warps share them out.
template <auto kKernel>
inline int32_t allow_shared(size_t bytes, bool wide_clusters = false, int registers = 0) {
  static std::atomic<uint64_t> done{0};
  int device;
  GS_CUDA_TRY(cudaGetDevice(&device));
  const uint64_t bit = uint64_t{1} << (device & 63);
  if (device < 64 && (done.load(std::memory_order_relaxed) & bit)) return GS_OK;
  GS_CUDA_TRY(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   static_cast<int>(bytes)));
  if (registers) {
    cudaFuncAttributes attributes;
    GS_CUDA_TRY(cudaFuncGetAttributes(&attributes, reinterpret_cast<const void*>(kKernel)));
    if (attributes.numRegs < registers) return GS_ERR_UNSUPPORTED;
  }
  if (wide_clusters)
    GS_CUDA_TRY(cudaFuncSetAttribute(kKernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  done.fetch_or(bit, std::memory_order_relaxed);
  return GS_OK;
}

// Reads and clears the flag that a kernel sets when a bounded wait ran out.
inline int32_t take_timeout(const uint32_t& flag, cudaStream_t stream) {
  uint32_t value = 0;
  const uint32_t clear = 0;
  GS_CUDA_TRY(cudaMemcpyFromSymbolAsync(&value, flag, sizeof(value), 0, cudaMemcpyDeviceToHost,
                                        stream));
  GS_CUDA_TRY(cudaMemcpyToSymbolAsync(flag, &clear, sizeof(clear), 0, cudaMemcpyHostToDevice,
                                      stream));
  GS_CUDA_TRY(cudaStreamSynchronize(stream));
  return value ? GS_ERR_TIMEOUT : GS_OK;
}

// One tile of a packed batch: rows [start, min(start + tile, end)) of the
// sequence that occupies rows [begin, end). A batch of one sequence needs no
// table: its tiles follow from the row count.
struct Tile {
  int32_t begin, end, start, sequence;
};
__device__ __forceinline__ Tile tile_at(const int32_t* table, int64_t index, int32_t rows,
                                        int32_t tile) {
  if (table) {
    const int4 t = __ldg(reinterpret_cast<const int4*>(table) + index);
    return {t.x, t.y, t.z, t.w};
  }
  return {0, rows, static_cast<int32_t>(index * tile), 0};
}

}  // namespace gs
