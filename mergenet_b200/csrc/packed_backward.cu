// Gradients of the packed attention (mn_packed_attention_backward): one warp
// per query row and head (dq) or per key row and key head (dk, dv), the
// channels over the lanes.
#include "packed_tc.cuh"

namespace mn {
namespace pk {

constexpr int kThreads = 128;

template <typename T>
__device__ __forceinline__ void load_row(const T* p, int d, int lane, float (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = lane + 32 * i < d ? to_f32(p[lane + 32 * i]) : 0.f;
}
__device__ __forceinline__ float dot4(const float (&a)[4], const float (&b)[4]) {
  return warp_sum(a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3]);
}
template <typename T>
__device__ __forceinline__ void store_row(T* p, int d, int lane, const float (&x)[4], float f) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < d) p[lane + 32 * i] = from_f32<T>(x[i] * f);
}

// dq, each row's delta, and each row's sums of ds by bucket (part)
template <typename T>
__global__ void __launch_bounds__(kThreads) dq_kernel(mn_packed_args a, Borders bo, float* delta, float* part) {
  __shared__ float hist[kThreads / 32][64];
  const int lane = threadIdx.x & 31, wi = threadIdx.x >> 5;
  const int64_t w = (int64_t)blockIdx.x * (kThreads / 32) + wi;
  if (w >= (int64_t)a.tq * a.heads) return;
  const int t = (int)(w / a.heads), h = (int)(w % a.heads), g = a.heads / a.kv_heads, hk = h / g, d = a.head_dim;
  const int b = seq_of_row(a.cu_q, a.nseq, t);
  for (int i = lane; i < 64; i += 32) hist[wi][i] = 0.f;
  __syncwarp();
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, dl = 0.f;
  if (b < a.nseq) {
    const Seq s = load_seq(a.cu_q, a.cu_k, a.len_k, b, a.tq, a.tk);
    const int pos = t - s.q0 + s.nk - s.nq;
    const int end = a.causal ? min(s.nk, pos + 1) : s.nk;
    const float lse = a.lse[((int64_t)hk * a.tq + t) * g + h % g];
    float q[4], k[4], v[4], go[4], o[4];
    load_row(static_cast<const T*>(a.q) + t * a.q_st + h * a.q_sh, d, lane, q);
    load_row(static_cast<const T*>(a.dout) + t * a.do_st + h * a.do_sh, d, lane, go);
    load_row(static_cast<const T*>(a.out) + ((int64_t)t * a.heads + h) * d, d, lane, o);
    dl = dot4(go, o);
    for (int j = 0; j < end; ++j) {
      load_row(static_cast<const T*>(a.k) + (int64_t)(s.k0 + j) * a.k_st + hk * a.k_sh, d, lane, k);
      load_row(static_cast<const T*>(a.v) + (int64_t)(s.k0 + j) * a.v_st + hk * a.v_sh, d, lane, v);
      float x = dot4(q, k) * a.scale;
      int u = 0;
      if (a.bias_table) {
        u = bucket_of(bo, j - pos);
        x += load_any(a.bias_table, a.bias_dtype, u * a.heads + h);
      }
      const float ds = exp2f(x * kLog2e - lse) * (dot4(go, v) - dl);
      if (a.bias_table && lane == 0) hist[wi][u] += ds;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += ds * k[i];
    }
  }
  store_row(static_cast<T*>(a.dq) + ((int64_t)t * a.heads + h) * d, d, lane, acc, a.scale);
  if (lane == 0) delta[((int64_t)hk * a.tq + t) * g + h % g] = dl;
  __syncwarp();
  if (a.bias_table)
    for (int u = lane; u < a.buckets; u += 32) part[((int64_t)t * a.heads + h) * a.buckets + u] = hist[wi][u];
}

// dtable[u, h] = sum over t of part[t, h, u]: one block per (u, h)
__global__ void __launch_bounds__(kThreads) dbias_kernel(const float* part, int tq, int heads, int buckets, float* out) {
  __shared__ float scratch[32];
  const int u = blockIdx.x, h = blockIdx.y;
  float x = 0.f;
  for (int t = threadIdx.x; t < tq; t += kThreads) x += part[((int64_t)t * heads + h) * buckets + u];
  x = block_sum(x, scratch);
  if (threadIdx.x == 0) out[u * heads + h] = x;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) dkv_kernel(mn_packed_args a, Borders bo, const float* delta) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (w >= (int64_t)a.tk * a.kv_heads) return;
  const int row = (int)(w / a.kv_heads), hk = (int)(w % a.kv_heads), g = a.heads / a.kv_heads, d = a.head_dim;
  const int b = seq_of_row(a.cu_k, a.nseq, row);
  float dk[4] = {0.f, 0.f, 0.f, 0.f}, dv[4] = {0.f, 0.f, 0.f, 0.f};
  if (b < a.nseq) {
    const Seq s = load_seq(a.cu_q, a.cu_k, a.len_k, b, a.tq, a.tk);
    const int j = row - s.k0;
    if (j < s.nk) {
      float q[4], k[4], v[4], go[4];
      load_row(static_cast<const T*>(a.k) + row * a.k_st + hk * a.k_sh, d, lane, k);
      load_row(static_cast<const T*>(a.v) + row * a.v_st + hk * a.v_sh, d, lane, v);
      const int first = a.causal ? max(0, j - (s.nk - s.nq)) : 0;
      for (int i = first; i < s.nq; ++i) {
        const int t = s.q0 + i;
        for (int gg = 0; gg < g; ++gg) {
          const int h = hk * g + gg;
          load_row(static_cast<const T*>(a.q) + t * a.q_st + h * a.q_sh, d, lane, q);
          load_row(static_cast<const T*>(a.dout) + t * a.do_st + h * a.do_sh, d, lane, go);
          float x = dot4(q, k) * a.scale;
          if (a.bias_table)
            x += load_any(a.bias_table, a.bias_dtype, bucket_of(bo, j - i - (s.nk - s.nq)) * a.heads + h);
          const int64_t at = ((int64_t)hk * a.tq + t) * g + gg;
          const float p = exp2f(x * kLog2e - a.lse[at]);
          const float ds = p * (dot4(go, v) - delta[at]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            dk[e] += ds * q[e];
            dv[e] += p * go[e];
          }
        }
      }
    }
  }
  store_row(static_cast<T*>(a.dk) + ((int64_t)row * a.kv_heads + hk) * d, d, lane, dk, a.scale);
  store_row(static_cast<T*>(a.dv) + ((int64_t)row * a.kv_heads + hk) * d, d, lane, dv, 1.f);
}

static unsigned blocks(int64_t warps) { return (unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32)); }

}  // namespace pk
}  // namespace mn

using namespace mn;

extern "C" size_t mn_packed_attention_backward_workspace_bytes(const mn_packed_args* a) {
  if (!a || a->tq < 1 || a->heads < 1) return 0;
  return (size_t)a->tq * a->heads * 4 * (1 + (a->bias_table ? a->buckets : 0));
}

extern "C" int mn_packed_attention_backward(const mn_packed_args* args, void* workspace, size_t workspace_bytes, int* status,
                                            void* stream) {
  Borders bo;
  const int rc = pk::check(args, &bo, true);
  if (rc != MN_OK) return rc;
  (void)status;
  if (args->tq == 0 && args->tk == 0) return MN_OK;
  if (workspace_bytes < mn_packed_attention_backward_workspace_bytes(args) || (args->tq > 0 && !workspace))
    return MN_ERR_WORKSPACE;
  cudaGetLastError();
  auto st = static_cast<cudaStream_t>(stream);
  float* delta = static_cast<float*>(workspace);
  float* part = delta + (size_t)args->tq * args->heads;
  const unsigned nq = pk::blocks((int64_t)args->tq * args->heads), nk = pk::blocks((int64_t)args->tk * args->kv_heads);
  if (args->dtype == MN_F16) {
    if (nq) pk::dq_kernel<__half><<<nq, pk::kThreads, 0, st>>>(*args, bo, delta, part);
    if (nk) pk::dkv_kernel<__half><<<nk, pk::kThreads, 0, st>>>(*args, bo, delta);
  } else {
    if (nq) pk::dq_kernel<__nv_bfloat16><<<nq, pk::kThreads, 0, st>>>(*args, bo, delta, part);
    if (nk) pk::dkv_kernel<__nv_bfloat16><<<nk, pk::kThreads, 0, st>>>(*args, bo, delta);
  }
  if (args->bias_table)
    pk::dbias_kernel<<<dim3(args->buckets, args->heads), pk::kThreads, 0, st>>>(part, args->tq, args->heads, args->buckets,
                                                                              args->dbias);
  return cudaGetLastError() == cudaSuccess ? MN_OK : MN_ERR_LAUNCH;
}
