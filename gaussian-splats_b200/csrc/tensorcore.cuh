// The 5th-generation tensor cores as attention.cu uses them: tiles loaded by
// TMA into 128-byte-swizzled shared memory, products issued by one thread
// (tcgen05.mma, 16-bit operands, float accumulators in tensor memory), results
// read back a row a thread.
#pragma once

#include <cuda.h>

#include "sequence.cuh"

namespace gs {
namespace tc {

__device__ __forceinline__ uint32_t shared_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// ------------------------------------------------------------------ barriers

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}

// Waits for the barrier's phase of this parity; false if it did not complete
// within the limit of tries, 1.5 us each: 1.6 s, far above any wait of a working
// kernel, which is at most a load or a few products long. A warp whose wait ran out
// waits no more, and the block's others run out behind it.
constexpr int kWaitLimit = 1 << 20;
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity,
                                             int limit = kWaitLimit) {
  for (int i = 0; i < limit; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}
// After a wait that ran out: time (25 ms) for what is still on its way to the
// barrier, whichever phase that is, before the shared memory is given back.
__device__ __forceinline__ void barrier_settle(uint32_t bar) {
  for (uint32_t parity = 0; parity < 2; ++parity) barrier_wait(bar, parity, 1 << 14);
}
// The same for all threads of a warp together.
__device__ __forceinline__ bool barrier_wait_warp(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, barrier_wait(bar, parity));
}

// Orders this thread's plain shared-memory writes before later reads of them
// by the tensor cores or TMA.
__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// ----------------------------------------------------------------------- TMA

// Loads the box at (x, head, row) of a [row, head, channel] array.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int head,
                                         int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(row), "r"(bar)
      : "memory");
}

// Loads the box at (x, row) of a [row, channel] array.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int row,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row), "r"(bar)
      : "memory");
}

// ------------------------------------------------------------- tensor memory

// Tensor memory is addressed as lane << 16 | column, 128 lanes of 512 32-bit
// columns; a warp reaches the 32 lanes of its place in its group of four.
template <int kColumns>
__device__ __forceinline__ void tensor_alloc(uint32_t shared_slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   shared_slot),
               "n"(kColumns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <int kColumns>
__device__ __forceinline__ void tensor_free(uint32_t address) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address),
               "n"(kColumns));
}
__device__ __forceinline__ void fence_before_sync() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after_sync() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// 32 columns of the warp's 32 lanes, a lane a thread. Reads are complete after
// wait_loads, writes after wait_stores.
__device__ __forceinline__ void load_columns32(uint32_t address, float (&x)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(address)
      : "memory");
}
__device__ __forceinline__ void load_columns16(uint32_t address, float (&x)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(address)
      : "memory");
}
template <class V>
__device__ __forceinline__ void store_columns16(uint32_t address, const V (&x)[16]) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(x);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(address),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void wait_loads() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void wait_stores() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// ------------------------------------------------------------------ products

// Tiles lie in shared memory as TMA's 128-byte swizzle writes boxes of 64
// channels: rows of 128 bytes, eight rows to a swizzled kilobyte, one box of
// kRows rows after the other along the channels. An operand's descriptor names
// where it starts, the stride between eight-row groups and, if the contraction
// runs along the rows, the stride between boxes. The one thread that issues the
// products is their bottleneck if it has to assemble descriptors (130 clocks a
// product, where a product takes 32 to 64), so it only adds to their low words:
// `channels_word` / `rows_word` of a tile, plus a constant for step k of 16 along
// the channels or along the rows.
template <int kRows>
__device__ __forceinline__ uint32_t channels_word(uint32_t tile) {
  return (tile >> 4) | 1u << 16;
}
template <int kRows>
__device__ __forceinline__ constexpr uint32_t channels_step(int k) {
  return static_cast<uint32_t>((k >> 2) * (kRows * 8) + (k & 3) * 2);
}
template <int kRows>
__device__ __forceinline__ uint32_t rows_word(uint32_t tile) {
  return (tile >> 4) | static_cast<uint32_t>(kRows * 8) << 16;
}
__device__ __forceinline__ constexpr uint32_t rows_step(int k) {
  return static_cast<uint32_t>(k * 128);
}
__device__ __forceinline__ uint64_t descriptor(uint32_t word) {
  constexpr uint32_t kHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(word), "r"(kHigh));
  return d;
}

// What a product of 128 rows and n columns is, for both operands of type T:
// float accumulators; `rows_b` if B's contraction runs along its rows.
template <class T>
__device__ __forceinline__ uint32_t product_kind(int n, bool rows_b) {
  const uint32_t type = std::is_same_v<T, __nv_bfloat16> ? 1 : 0;
  return 1u << 4 | type << 7 | type << 10 | (rows_b ? 1u << 16 : 0u) |
         static_cast<uint32_t>(n >> 3) << 17 | (128u >> 4) << 24;
}

// One lane of a warp that is converged here: 1 for it, 0 for the others. The
// whole warp goes through the code that issues products, with the instruction
// itself predicated to that lane: its operands are then the warp's and stay in
// uniform registers.
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t elected;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(elected));
  return elected;
}
// D (+)= A B^T with A and B in shared memory (low words of descriptors).
__device__ __forceinline__ void multiply(uint32_t elected, uint32_t d, uint32_t a, uint32_t b,
                                         uint32_t kind, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(descriptor(a)), "l"(descriptor(b)), "r"(kind), "r"(static_cast<uint32_t>(add)),
      "r"(elected)
      : "memory");
}
// D (+)= A B^T with A in tensor memory (two 16-bit values a column).
__device__ __forceinline__ void multiply_tensor(uint32_t elected, uint32_t d, uint32_t a,
                                                uint32_t b, uint32_t kind, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(descriptor(b)), "r"(kind), "r"(static_cast<uint32_t>(add)), "r"(elected)
      : "memory");
}
// The barrier's phase completes when the products issued so far have.
__device__ __forceinline__ void commit(uint32_t elected, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          bar),
      "r"(elected)
      : "memory");
}

// ---------------------------------------------------------------- arithmetic

// A group of four warps gives registers back or takes them, to kCount a thread; who
// takes waits for those that the block was launched with to become free.
template <int kCount>
__device__ __forceinline__ void registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCount));
}
template <int kCount>
__device__ __forceinline__ void registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kCount));
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// Two floats at a time in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(y))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
        "l"(reinterpret_cast<const uint64_t&>(c)));
  return y;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 y;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(y))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return y;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 y;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(y))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return y;
}
// Two floats rounded to the 16-bit type T, the first in the low half.
template <class T>
__device__ __forceinline__ uint32_t pack2(float low, float high) {
  uint32_t r;
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
  return r;
}

// ---------------------------------------------------------------------- host

// Encodes the map of an array of `axes` axes (innermost first, contiguous;
// strides in bytes from the second axis on) for boxes of `box`; what lies
// outside the array reads as zeros.
inline int32_t encode(CUtensorMap* map, int32_t dtype, const void* base, int axes,
                      const cuuint64_t* size, const cuuint64_t* stride, const cuuint32_t* box,
                      CUtensorMapSwizzle swizzle) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> found_before{nullptr};  // threads may come here side by side
  Encode call = found_before.load(std::memory_order_acquire);
  if (!call) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    GS_CUDA_TRY(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !f) return GS_ERR_UNSUPPORTED;
    call = reinterpret_cast<Encode>(f);
    found_before.store(call, std::memory_order_release);
  }
  const CUtensorMapDataType type = dtype == GS_FLOAT32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == GS_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint32_t step[3] = {1, 1, 1};
  for (int attempt = 0; attempt < 2; ++attempt) {
    const CUresult r = call(map, type, axes, const_cast<void*>(base), size, stride, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return GS_OK;
    if (r != CUDA_ERROR_INVALID_CONTEXT) break;
    // A thread that has made no runtime call yet (an autograd worker) has no
    // context for this driver call; selecting its device binds one.
    int device;
    GS_CUDA_TRY(cudaGetDevice(&device));
    GS_CUDA_TRY(cudaSetDevice(device));
  }
  return GS_ERR_INVALID_ARGUMENT;
}

// A [tokens, heads, dim] array of 16-bit elements in boxes of 64 channels and
// `rows` tokens of one head, swizzled as the products read them.
inline int32_t encode_heads(CUtensorMap* map, int32_t dtype, const void* base, int64_t tokens,
                            int64_t heads, int64_t dim, int64_t token_stride, int64_t head_stride,
                            int rows) {
  const cuuint64_t size[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(tokens)};
  const cuuint64_t stride[2] = {static_cast<cuuint64_t>(head_stride) * 2,
                                static_cast<cuuint64_t>(token_stride) * 2};
  const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(rows)};
  return encode(map, dtype, base, 3, size, stride, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// A [rows, channels] array in boxes of 128 bytes of channels and `box_rows` rows.
inline int32_t encode_rows(CUtensorMap* map, int32_t dtype, const void* base, int64_t rows,
                           int64_t channels, int64_t row_stride, int box_rows) {
  const int64_t element = element_size(dtype);
  const cuuint64_t size[2] = {static_cast<cuuint64_t>(channels), static_cast<cuuint64_t>(rows)};
  const cuuint64_t stride[1] = {static_cast<cuuint64_t>(row_stride * element)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / element),
                             static_cast<cuuint32_t>(box_rows)};
  return encode(map, dtype, base, 2, size, stride, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

}  // namespace tc
}  // namespace gs
