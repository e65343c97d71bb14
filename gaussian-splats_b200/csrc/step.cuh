// What the kernels of one new token a stream share (attention.cu, attention_4bit.cu):
// small products on whole warps, and clusters of blocks that join through distributed
// shared memory.
#pragma once

#include "tensorcore.cuh"

namespace gs {

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

}  // namespace gs
