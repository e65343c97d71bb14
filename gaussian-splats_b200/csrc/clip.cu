// The global norm of many gradients, and clipping to it.
//
//   norm = sqrt(sum of g^2 over all elements of all tensors)
//   factor = min(1, max_norm / (norm + 1e-6)),  g <- factor g
//
// Bound: memory. The norm reads every element once; clipping reads and writes
// each once more, and nothing where the factor is 1. The tensors' addresses
// travel with the launch, so that many tensors are one kernel, without a table in
// device memory to fill first. The tensors are cut into chunks of 32 KB, which the
// blocks take in turn; a block's sum, and the sum over the blocks, are made in one
// order, so that results repeat bit for bit. The norm of 1.4 GB takes
// 200 us (7.1 TB/s), multiplying 472 MB 142 us (6.6 TB/s); with few gradients each
// kernel is its launch and one chunk's latency, 2 to 4 us.
//
// A thread's squares (128 bytes of elements) are added in float and that sum in
// double from there on. Squares leave float's range long before norms do, so a
// thread whose float sum is very small or large squares its elements in double.
#include "sequence.cuh"

namespace gs {
namespace {

constexpr int kThreads = 256;
constexpr int kVectors = 8;                             // 16-byte words a thread and chunk
constexpr int64_t kChunkWords = kThreads * kVectors;    // 32 KB
constexpr int kSmallTable = 80, kLargeTable = 1024;     // tensors of one launch: 1.7 KB, 21.5 KB
constexpr int kBlocks = 6 * kSmCount;                   // 3 of 6 resident at once (scaling: 2)
constexpr double kEps = 1e-6;

template <int kEntries>
struct Table {
  void* data[kEntries];
  int64_t count[kEntries];
  int32_t start[kEntries + 1];  // first chunk
  int32_t tensors;
  uint8_t dtype[kEntries];
};

// One chunk of a tensor: whole 16-byte words [first, last), and, for its first
// and last chunk, the elements in front of the words and behind them.
struct Chunk {
  unsigned char* words;
  int64_t first, last;
  unsigned char *head, *tail;
  int head_count, tail_count, dtype;
};

template <int kEntries>
__device__ Chunk chunk_at(const Table<kEntries>& t, int chunk) {
  int low = 0, high = t.tensors;  // the last tensor that starts at or before it
  while (high - low > 1) {
    const int middle = (low + high) / 2;
    if (t.start[middle] <= chunk) low = middle;
    else high = middle;
  }
  Chunk c;
  c.dtype = t.dtype[low];
  const int size = c.dtype == GS_FLOAT32 ? 4 : 2;
  unsigned char* const data = static_cast<unsigned char*>(t.data[low]);
  const int64_t bytes = t.count[low] * size;
  const int64_t misaligned = -reinterpret_cast<intptr_t>(data) & 15;
  const int64_t lead = misaligned < bytes ? misaligned : bytes;
  const int64_t words = (bytes - lead) / 16;
  const int64_t index = chunk - t.start[low];
  c.words = data + lead;
  c.first = index * kChunkWords;
  c.last = c.first + kChunkWords < words ? c.first + kChunkWords : words;
  c.head = data;
  c.head_count = index == 0 ? static_cast<int>(lead / size) : 0;
  c.tail = c.words + words * 16;
  c.tail_count = chunk + 1 == t.start[low + 1]
                     ? static_cast<int>((bytes - lead - words * 16) / size) : 0;
  return c;
}

template <class T>
__device__ __forceinline__ void unpack(const uint4& word, float (&x)[16 / sizeof(T)]) {
  const T* v = reinterpret_cast<const T*>(&word);
#pragma unroll
  for (int k = 0; k < static_cast<int>(16 / sizeof(T)); ++k) x[k] = to_float(v[k]);
}

template <class T>
__device__ double chunk_squares(const Chunk& c) {
  constexpr int kPer = 16 / sizeof(T);
  uint4 word[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int64_t at = c.first + threadIdx.x + i * kThreads;
    word[i] = at < c.last ? __ldg(reinterpret_cast<const uint4*>(c.words) + at)
                          : make_uint4(0, 0, 0, 0);
  }
  float parts[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    float x[kPer];
    unpack<T>(word[i], x);
    parts[i] = x[0] * x[0];
#pragma unroll
    for (int k = 1; k < kPer; ++k) parts[i] = fmaf(x[k], x[k], parts[i]);
  }
#pragma unroll
  for (int o = kVectors / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) parts[i] += parts[i + o];
  double sum;
  if (parts[0] >= 1e-30f && parts[0] <= 1e38f) {
    sum = parts[0];
  } else {
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      float x[kPer];
      unpack<T>(word[i], x);
#pragma unroll
      for (int k = 0; k < kPer; ++k) sum = fma(static_cast<double>(x[k]), x[k], sum);
    }
  }
  if (static_cast<int>(threadIdx.x) < c.head_count) {
    const double x = to_float(reinterpret_cast<const T*>(c.head)[threadIdx.x]);
    sum = fma(x, x, sum);
  }
  if (static_cast<int>(threadIdx.x) < c.tail_count) {
    const double x = to_float(reinterpret_cast<const T*>(c.tail)[threadIdx.x]);
    sum = fma(x, x, sum);
  }
  return sum;
}

template <class T>
__device__ void chunk_scale(const Chunk& c, float factor) {
  constexpr int kPer = 16 / sizeof(T);
  uint4* const words = reinterpret_cast<uint4*>(c.words);
  uint4 word[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int64_t at = c.first + threadIdx.x + i * kThreads;
    if (at < c.last) word[i] = words[at];
  }
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int64_t at = c.first + threadIdx.x + i * kThreads;
    if (at >= c.last) break;
    float x[kPer];
    unpack<T>(word[i], x);
#pragma unroll
    for (int k = 0; k < kPer; ++k) x[k] *= factor;
    store_pack<kPer>(reinterpret_cast<T*>(words + at), x);
  }
  const auto scale_one = [&](unsigned char* p) {
    T* const e = reinterpret_cast<T*>(p) + threadIdx.x;
    *e = from_float<T>(to_float(*e) * factor);
  };
  if (static_cast<int>(threadIdx.x) < c.head_count) scale_one(c.head);
  if (static_cast<int>(threadIdx.x) < c.tail_count) scale_one(c.tail);
}

// The sum of the block's values, in one order, in every thread.
__device__ double block_sum(double x) {
  __shared__ double parts[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = x;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) sum += parts[w];
  return sum;
}

template <int kEntries>
__global__ void __launch_bounds__(kThreads)
    square_sum_kernel(const __grid_constant__ Table<kEntries> table, double* partials) {
  chain_wait();
  double sum = 0.0;
  for (int chunk = blockIdx.x; chunk < table.start[table.tensors]; chunk += gridDim.x) {
    const Chunk c = chunk_at(table, chunk);
    if (c.dtype == GS_FLOAT32) sum += chunk_squares<float>(c);
    else if (c.dtype == GS_BFLOAT16) sum += chunk_squares<__nv_bfloat16>(c);
    else sum += chunk_squares<__half>(c);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

// The norm and the factor from the blocks' sums; every thread gets the factor.
__device__ float finish(const double* partials, int count, double max_norm, float* result) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) sum += partials[i];
  const double norm = sqrt(block_sum(sum));
  const double ratio = max_norm / (norm + kEps);
  const float factor = ratio >= 1.0 ? 1.0f : static_cast<float>(ratio);  // NaN stays
  if (result && threadIdx.x == 0) {
    result[0] = static_cast<float>(norm);
    result[1] = factor;
  }
  return factor;
}

__global__ void __launch_bounds__(kThreads)
    norm_kernel(const double* partials, int count, double max_norm, float* result) {
  chain_wait();
  finish(partials, count, max_norm, result);
}

// From the last chunk to the first: what the norm's kernel read last is still in L2.
template <int kEntries>
__global__ void __launch_bounds__(kThreads)
    scale_kernel(const __grid_constant__ Table<kEntries> table, const double* partials, int count,
                 double max_norm, float* result) {
  chain_wait();
  const float factor = finish(partials, count, max_norm, blockIdx.x == 0 ? result : nullptr);
  if (factor == 1.0f) return;
  const int chunks = table.start[table.tensors];
  for (int chunk = chunks - 1 - static_cast<int>(blockIdx.x); chunk >= 0; chunk -= gridDim.x) {
    const Chunk c = chunk_at(table, chunk);
    if (c.dtype == GS_FLOAT32) chunk_scale<float>(c, factor);
    else if (c.dtype == GS_BFLOAT16) chunk_scale<__nv_bfloat16>(c, factor);
    else chunk_scale<__half>(c, factor);
  }
}

int64_t launches_of(int64_t tensors) {
  return tensors <= kSmallTable ? 1 : (tensors + kLargeTable - 1) / kLargeTable;
}

// Chunks of a tensor: of its whole words behind the first 16-byte border, one at least.
int64_t chunks_of(const gs_gradient& g) {
  const int64_t words = g.count * element_size(g.dtype) / 16;
  return words <= kChunkWords ? 1 : (words + kChunkWords - 1) / kChunkWords;
}

// Calls f(table, blocks) for the tensors in launches of at most kEntries.
template <int kEntries, class F>
int32_t for_tables(int64_t tensors, const gs_gradient* list, F&& f) {
  Table<kEntries> table;
  for (int64_t first = 0; first < tensors; first += kEntries) {
    const int count = static_cast<int>(tensors - first < kEntries ? tensors - first : kEntries);
    int64_t chunks = 0;
    table.tensors = count;
    for (int i = 0; i < count; ++i) {
      const gs_gradient& g = list[first + i];
      table.data[i] = g.data;
      table.count[i] = g.count;
      table.dtype[i] = static_cast<uint8_t>(g.dtype);
      table.start[i] = static_cast<int32_t>(chunks);
      chunks += chunks_of(g);
      if (chunks > INT32_MAX - kBlocks) return GS_ERR_CAPACITY;
    }
    table.start[count] = static_cast<int32_t>(chunks);
    GS_TRY(f(table, static_cast<int>(chunks < kBlocks ? chunks : kBlocks)));
  }
  return GS_OK;
}

template <int kEntries>
int32_t run(int64_t tensors, const gs_gradient* list, double max_norm, bool scale, float* result,
            double* partials, cudaStream_t stream) {
  int blocks = 0;
  GS_TRY(for_tables<kEntries>(tensors, list, [&](const Table<kEntries>& table, int n) {
    launch_chained(square_sum_kernel<kEntries>, n, kThreads, stream, table, partials + blocks);
    blocks += n;
    return check_launch();
  }));
  if (!scale) {
    launch_chained(norm_kernel, 1, kThreads, stream, static_cast<const double*>(partials), blocks,
                   max_norm, result);
    return check_launch();
  }
  return for_tables<kEntries>(tensors, list, [&](const Table<kEntries>& table, int n) {
    launch_chained(scale_kernel<kEntries>, n, kThreads, stream, table,
                   static_cast<const double*>(partials), blocks, max_norm, result);
    return check_launch();
  });
}

}  // namespace

uint64_t clip_grad_norm_workspace_size(int64_t tensors) {
  return sizeof(double) * kBlocks * static_cast<uint64_t>(launches_of(tensors));
}

int32_t launch_clip_grad_norm(int64_t tensors, const gs_gradient* list, double max_norm,
                              bool scale, float* result, void* workspace, uint64_t workspace_size,
                              cudaStream_t stream) {
  if (tensors < 1 || tensors > (1 << 20) || !list || !result || !workspace || !(max_norm >= 0.0))
    return GS_ERR_INVALID_ARGUMENT;
  for (int64_t i = 0; i < tensors; ++i) {
    const gs_gradient& g = list[i];
    if (g.count < 0 || g.count > int64_t{1} << 40 || (g.count > 0 && !g.data) ||
        g.dtype < GS_FLOAT32 || g.dtype > GS_FLOAT16)
      return GS_ERR_INVALID_ARGUMENT;
    if (!is_aligned(g.data, element_size(g.dtype))) return GS_ERR_MISALIGNED;
  }
  if (!is_aligned(result, 4) || !is_aligned(workspace, 8)) return GS_ERR_MISALIGNED;
  if (workspace_size < clip_grad_norm_workspace_size(tensors)) return GS_ERR_CAPACITY;
  double* const partials = static_cast<double*>(workspace);
  return tensors <= kSmallTable
             ? run<kSmallTable>(tensors, list, max_norm, scale, result, partials, stream)
             : run<kLargeTable>(tensors, list, max_norm, scale, result, partials, stream);
}

}  // namespace gs
