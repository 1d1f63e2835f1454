// The bias of a learned table over distance buckets as a tensor
// (mn_relative_bias), and the table's gradient.
//
// bias[h, i, j] = table[bucket(j - i - start), h] depends on h and on the
// diagonal j - i alone, so both directions work with the queries + keys - 1
// diagonals: the forward writes each value from one lookup, the gradient adds
// up each diagonal over a chunk of rows (one thread per diagonal, its rows in
// order) and then the diagonals of each bucket, all in a fixed order.
#include <algorithm>

#include "packed.cuh"

namespace mn {
namespace rb {

constexpr int kThreads = 256;
constexpr int kRows = 64;  // rows of a chunk whose diagonals one block adds up

template <typename T>
__global__ void __launch_bounds__(kThreads) forward_kernel(int heads, int queries, int keys, int start, Borders bo,
                                                           const T* __restrict__ table, T* __restrict__ bias) {
  const int64_t n = (int64_t)heads * queries * keys;
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < n; e += (int64_t)gridDim.x * kThreads) {
    const int j = (int)(e % keys);
    const int64_t r = e / keys;
    const int i = (int)(r % queries), h = (int)(r / queries);
    bias[e] = table[bucket_of(bo, j - i - start) * heads + h];
  }
}

// part[chunk, h, diag]: the sum of dbias[h, i, i + diag - (queries - 1)] over
// the rows i of the chunk
template <typename T>
__global__ void __launch_bounds__(kThreads) diagonal_kernel(int heads, int queries, int keys, const T* __restrict__ dbias,
                                                            float* __restrict__ part) {
  const int diags = queries + keys - 1;
  const int g = blockIdx.x * kThreads + threadIdx.x, h = blockIdx.y, i0 = blockIdx.z * kRows;
  if (g >= diags) return;
  float x = 0.f;
  for (int i = i0; i < min(queries, i0 + kRows); ++i) {
    const int j = i + g - (queries - 1);
    if (j >= 0 && j < keys) x += to_f32(dbias[((int64_t)h * queries + i) * keys + j]);
  }
  part[((int64_t)blockIdx.z * heads + h) * diags + g] = x;
}

__global__ void __launch_bounds__(kThreads) bucket_kernel(int heads, int queries, int keys, int start, Borders bo, int chunks,
                                                          const float* __restrict__ part, float* __restrict__ dtable) {
  __shared__ float scratch[32];
  const int u = blockIdx.x, h = blockIdx.y, diags = queries + keys - 1;
  float x = 0.f;
  for (int g = threadIdx.x; g < diags; g += kThreads)
    if (bucket_of(bo, g - (queries - 1) - start) == u)
      for (int c = 0; c < chunks; ++c) x += part[((int64_t)c * heads + h) * diags + g];
  x = block_sum(x, scratch);
  if (threadIdx.x == 0) dtable[u * heads + h] = x;
}

static int chunks_of(int queries) { return (queries + kRows - 1) / kRows; }

static bool sizes_ok(int heads, int queries, int keys, int start) {
  return heads > 0 && queries >= 0 && keys >= 0 && queries < (1 << 30) && keys < (1 << 30) && start < (1 << 30) &&
         start > -(1 << 30);
}

}  // namespace rb
}  // namespace mn

using namespace mn;

extern "C" int mn_relative_bias(int heads, int queries, int keys, int query_start, int buckets, int two_sided,
                                int num_borders, const int32_t* borders, int dtype, const void* table, void* bias,
                                void* stream) {
  Borders bo;
  if (!rb::sizes_ok(heads, queries, keys, query_start) || dtype < 0 || dtype > 2) return MN_ERR_ARG;
  if (!make_borders(&bo, buckets, two_sided, num_borders, borders)) return MN_ERR_ARG;
  if (queries == 0 || keys == 0) return MN_OK;
  if (!table || !bias) return MN_ERR_ARG;
  cudaGetLastError();
  const int64_t n = (int64_t)heads * queries * keys;
  const unsigned grid = (unsigned)std::min<int64_t>((n + rb::kThreads - 1) / rb::kThreads, 148 * 32);
  auto st = static_cast<cudaStream_t>(stream);
  if (dtype == MN_F32)
    rb::forward_kernel<float><<<grid, rb::kThreads, 0, st>>>(heads, queries, keys, query_start, bo,
                                                            static_cast<const float*>(table), static_cast<float*>(bias));
  else
    rb::forward_kernel<uint16_t><<<grid, rb::kThreads, 0, st>>>(heads, queries, keys, query_start, bo,
                                                               static_cast<const uint16_t*>(table),
                                                               static_cast<uint16_t*>(bias));
  return cudaGetLastError() == cudaSuccess ? MN_OK : MN_ERR_LAUNCH;
}

extern "C" size_t mn_relative_bias_backward_workspace_bytes(int heads, int queries, int keys, int buckets) {
  (void)buckets;
  if (heads < 1 || queries < 1 || keys < 1) return 0;
  return (size_t)rb::chunks_of(queries) * heads * ((size_t)queries + keys - 1) * 4;
}

extern "C" int mn_relative_bias_backward(int heads, int queries, int keys, int query_start, int buckets, int two_sided,
                                         int num_borders, const int32_t* borders, int dtype, const void* dbias,
                                         float* dtable, void* workspace, size_t workspace_bytes, void* stream) {
  Borders bo;
  if (!rb::sizes_ok(heads, queries, keys, query_start) || dtype < 0 || dtype > 2 || !dtable) return MN_ERR_ARG;
  if (!make_borders(&bo, buckets, two_sided, num_borders, borders)) return MN_ERR_ARG;
  if (queries == 0 || keys == 0) return MN_ERR_ARG;
  if (!dbias) return MN_ERR_ARG;
  if (heads > 65535 || rb::chunks_of(queries) > 65535) return MN_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < mn_relative_bias_backward_workspace_bytes(heads, queries, keys, buckets))
    return MN_ERR_WORKSPACE;
  cudaGetLastError();
  float* part = static_cast<float*>(workspace);
  const int chunks = rb::chunks_of(queries), diags = queries + keys - 1;
  const dim3 grid((diags + rb::kThreads - 1) / rb::kThreads, heads, chunks);
  auto st = static_cast<cudaStream_t>(stream);
  if (dtype == MN_F32)
    rb::diagonal_kernel<float><<<grid, rb::kThreads, 0, st>>>(heads, queries, keys, static_cast<const float*>(dbias), part);
  else if (dtype == MN_F16)
    rb::diagonal_kernel<__half><<<grid, rb::kThreads, 0, st>>>(heads, queries, keys, static_cast<const __half*>(dbias), part);
  else
    rb::diagonal_kernel<__nv_bfloat16><<<grid, rb::kThreads, 0, st>>>(heads, queries, keys,
                                                                     static_cast<const __nv_bfloat16*>(dbias), part);
  rb::bucket_kernel<<<dim3(buckets, heads), rb::kThreads, 0, st>>>(heads, queries, keys, query_start, bo, chunks, part, dtable);
  return cudaGetLastError() == cudaSuccess ? MN_OK : MN_ERR_LAUNCH;
}
