// Tensor-core plumbing shared by the packed attention's forward and backward:
// tensor maps of packed rows, tile lookup, bias values, waits.
#pragma once

#include <initializer_list>
#include <type_traits>

#include "packed.cuh"
#include "tc_common.cuh"
#include "tma.cuh"

namespace mn {
namespace pk {

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kHalfBytes = 128 * 128;  // 128 rows of 64 16-bit channels

template <typename ET>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// From 2^16 on (a step of fp32 is then 2^-7) a score is rounded on its own
// before the row's maximum is taken off it.  One multiply-add for both, with
// the maximum rounded and the score not, leaves an exponent of up to half a
// step: 2^16 and more at scores of 10^8, past fp16's range.
constexpr float kBig = 65536.f;
__device__ __forceinline__ bool is_big(float x) { return fabsf(x) > kBig && fabsf(x) < INFINITY; }
// An entry of the bias table in log2 units, held to +-2^17 but for the
// infinities: a mask's value hides a key as well from there as from -10^9, and
// the scores beside it, and their row's logarithm, keep steps of 2^-7.
__device__ __forceinline__ float table_value(const mn_packed_args& a, int bucket, int head) {
  const float v = load_any(a.bias_table, a.bias_dtype, (int64_t)bucket * a.heads + head);
  const float y = v * kLog2e;
  return fabsf(y) > 131072.f && fabsf(v) < INFINITY ? copysignf(131072.f, v) : y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float max32(const float* x, float m) {
  float a[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int e = 0; e < 32; e += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = max3(a[i], x[e + 2 * i], x[e + 2 * i + 1]);
  return fmaxf(max3(a[0], a[1], a[2]), a[3]);
}

// Wait for the phase with the given parity, bounded in time like
// tc::mbar_wait, which looks at the clock and at *err (a trip to the L2)
// before its second try; a hand-off between the warps of a tile is shorter
// than that trip, so here the first 64 tries go without.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, const int* err) {
  const uint32_t addr = tc::smem_u32(bar);
  for (int i = 0; i < 64; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return tc::mbar_wait(bar, parity, err);
}

// One lane of a converged warp, the same each time.  The compiler knows that a
// single thread passes, so the tensor-core instructions behind it are issued
// as they stand; behind `lane == 0` each took about 140 cycles (a product of
// 128 x 128 x 128 was issued in 1,150 cycles and executes in about 500).
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is));
  return is != 0;
}

// Register exchange between the warp groups of a CTA (a whole group executes
// it).  A taker waits until the givers' registers are free, so the shares may
// not exceed what the CTA was launched with: launch_regs() on the host checks
// the launch, a static_assert at each kernel the shares.
template <int N>
__device__ __forceinline__ void regs_take() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_give() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Tiles of `m` rows of every sequence share one index space without a prefix
// sum: sequence b's tiles begin at slot cu[b] / m + b.  A sequence of L rows
// has ceil(L / m) tiles and at least that many slots, at most one of them
// left empty.  Rows behind the last sequence are sequence n, with no keys.
__device__ __forceinline__ int slot_of_seq(const int32_t* cu, int b, int m, int rows) {
  return min(max(cu[b], 0), rows) / m + b;
}
inline int64_t tile_slots(int rows, int n, int m) { return (int64_t)rows / m + n + 1; }

// The sequence of tile slot `slot` of the query rows (of the key rows when
// KEYS), by a whole warp: the last sequence b in 0..n whose first slot is at or
// below it.  Sequence n is the rows behind the last one, which see nothing.
// 32 probes a step narrow the range to 32 sequences, whose offsets are then
// all read at once (a trip to memory a step; one for up to 32 sequences).
struct Found {
  Seq s;
  int local;  // the slot's place among the sequence's own
  int seq;    // its number (nseq: the rows behind the last one)
};
template <bool KEYS>
__device__ __forceinline__ Found seq_of_slot(const mn_packed_args& a, int m, int slot) {
  const int32_t* cu = KEYS ? a.cu_k : a.cu_q;
  const int rows = KEYS ? a.tk : a.tq, n = a.nseq, lane = threadIdx.x & 31;
  int lo = 0, hi = n + 1;  // the first slot of lo is at or below `slot`, that of hi is not
  while (hi - lo > 32) {
    const int step = (hi - lo + 31) / 32;
    const int b = lo + (lane + 1) * step;
    const bool le = b < hi && slot_of_seq(cu, b, m, rows) <= slot;
    const unsigned vote = __ballot_sync(MN_FULL_MASK, le);
    const int nlo = lo + (vote == 0 ? 0 : 32 - __clz(vote)) * step;  // offsets ascend
    hi = min(hi, nlo + step);
    lo = nlo;
  }
  const int b = min(lo + lane, hi - 1), e = min(b + 1, n);
  const int q0 = a.cu_q[b], q1 = a.cu_q[e], k0 = a.cu_k[b], k1 = a.cu_k[e], len = a.len_k && b < n ? a.len_k[b] : 0x7fffffff;
  Found f;
  f.s.q0 = min(max(q0, 0), a.tq);
  f.s.nq = (b < n ? min(max(q1, f.s.q0), a.tq) : a.tq) - f.s.q0;
  f.s.k0 = min(max(k0, 0), a.tk);
  f.s.slot = (b < n ? min(max(k1, f.s.k0), a.tk) : a.tk) - f.s.k0;
  f.s.nk = b < n ? min(max(len, 0), f.s.slot) : 0;
  const int first = (KEYS ? f.s.k0 : f.s.q0) / m + b;
  const unsigned vote = __ballot_sync(MN_FULL_MASK, first <= slot);
  const int src = vote == 0 ? 0 : 31 - __clz(vote);
  f.s.q0 = __shfl_sync(MN_FULL_MASK, f.s.q0, src);
  f.s.nq = __shfl_sync(MN_FULL_MASK, f.s.nq, src);
  f.s.k0 = __shfl_sync(MN_FULL_MASK, f.s.k0, src);
  f.s.slot = __shfl_sync(MN_FULL_MASK, f.s.slot, src);
  f.s.nk = __shfl_sync(MN_FULL_MASK, f.s.nk, src);
  f.local = slot - __shfl_sync(MN_FULL_MASK, first, src);
  f.seq = __shfl_sync(MN_FULL_MASK, b, src);
  return f;
}
// The same with the tiles in descending order of their work, so that the last
// CTAs to start are the shortest (in the sequences' own order the last of a
// few waves could begin with a long sequence: 64 caches of 700 to 8,192 keys
// 234 -> 228 us, training on 7 documents of 33 to 4,000 tokens 893 -> 842 us).  A warp holds up to
// kRanked sequences; the work of a tile is what it walks over: the keys of
// its sequence, or (KEYS) the queries that see its keys.
constexpr int kRanked = 255;
template <bool KEYS>
__device__ __forceinline__ Found ranked_slot(const mn_packed_args& a, int m, int slot) {
  constexpr int E = (kRanked + 1) / 32;
  const int n = a.nseq, lane = threadIdx.x & 31;
  int val[E], shift[E], used[E], tiles[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    val[e] = shift[e] = used[e] = tiles[e] = 0;
    const int b = lane + 32 * e;
    if (b <= n) {
      const int end = min(b + 1, n);
      const int q0 = min(max(a.cu_q[b], 0), a.tq), k0 = min(max(a.cu_k[b], 0), a.tk);
      const int nq = (b < n ? min(max(a.cu_q[end], q0), a.tq) : a.tq) - q0;
      const int sl = (b < n ? min(max(a.cu_k[end], k0), a.tk) : a.tk) - k0;
      const int nk = b == n ? 0 : a.len_k ? min(max(a.len_k[b], 0), sl) : sl;
      val[e] = KEYS ? nq : nk;
      shift[e] = nk - nq;
      tiles[e] = KEYS ? (sl + m - 1) / m : (nq + m - 1) / m;
      used[e] = KEYS ? (nk + m - 1) / m : tiles[e];
    }
  }
  // tiles of sequence e whose work is at least x
  auto count = [&](int e, int x) -> int {
    if (x <= 0) return tiles[e];
    if (val[e] < x) return 0;
    if (!KEYS || !a.causal) return used[e];
    const int spare = val[e] - x + shift[e];  // tile i is seen by val - max(0, i m - shift) queries
    return spare < 0 ? 0 : min(used[e], spare / m + 1);
  };
  auto total = [&](int x) -> int {
    int c = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) c += count(e, x);
    return __reduce_add_sync(MN_FULL_MASK, c);
  };
  Found f;
  f.s.q0 = f.s.nq = f.s.k0 = f.s.nk = f.s.slot = 0;
  f.local = -1;
  f.seq = n;
  if (slot >= total(0)) return f;
  int most = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) most = max(most, val[e]);
  int lo = 0, hi = __reduce_max_sync(MN_FULL_MASK, most) + 1;  // total(lo) > slot >= total(hi)
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (total(mid) > slot) lo = mid;
    else hi = mid;
  }
  int rest = slot - total(hi), mine = 0;  // its place among the tiles of work lo, by lane
#pragma unroll
  for (int e = 0; e < E; ++e) mine += count(e, lo) - count(e, hi);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(MN_FULL_MASK, incl, o);
    if (lane >= o) incl += t;
  }
  const int src = __ffs(__ballot_sync(MN_FULL_MASK, incl > rest)) - 1;
  int b = 0, at = rest - (incl - mine);
  bool found = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = count(e, lo) - count(e, hi);
    if (!found && at < c) {
      found = true;
      b = lane + 32 * e;
      f.local = count(e, hi) + at;
    }
    at -= c;
  }
  f.seq = b = __shfl_sync(MN_FULL_MASK, b, src);
  f.local = __shfl_sync(MN_FULL_MASK, f.local, src);
  const int end = min(b + 1, n);
  f.s.q0 = min(max(a.cu_q[b], 0), a.tq);
  f.s.nq = (b < n ? min(max(a.cu_q[end], f.s.q0), a.tq) : a.tq) - f.s.q0;
  f.s.k0 = min(max(a.cu_k[b], 0), a.tk);
  f.s.slot = (b < n ? min(max(a.cu_k[end], f.s.k0), a.tk) : a.tk) - f.s.k0;
  f.s.nk = b == n ? 0 : a.len_k ? min(max(a.len_k[b], 0), f.s.slot) : f.s.slot;
  return f;
}
// handed to the CTA through shared memory
__device__ __forceinline__ void put_found(volatile uint32_t* at, const Found& f) {
  if ((threadIdx.x & 31) == 0) {
    at[0] = f.s.q0; at[1] = f.s.nq; at[2] = f.s.k0; at[3] = f.s.nk; at[4] = f.s.slot; at[5] = f.local;
    at[6] = f.seq;
  }
}
__device__ __forceinline__ Found get_found(const volatile uint32_t* at) {
  Found f;
  f.s.q0 = at[0]; f.s.nq = at[1]; f.s.k0 = at[2]; f.s.nk = at[3]; f.s.slot = at[4]; f.local = at[5];
  f.seq = at[6];
  return f;
}

// 32 fp32 values of one row as ET, 16 bytes at a time, up to channel `d`
template <typename ET>
__device__ __forceinline__ void store32(ET* row, int c0, int d, const float* o, float f) {
  uint4* dst = reinterpret_cast<uint4*>(row + c0);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c0 + 8 * i < d)
      dst[i] = make_uint4(pack2<ET>(o[8 * i] * f, o[8 * i + 1] * f), pack2<ET>(o[8 * i + 2] * f, o[8 * i + 3] * f),
                          pack2<ET>(o[8 * i + 4] * f, o[8 * i + 5] * f), pack2<ET>(o[8 * i + 6] * f, o[8 * i + 7] * f));
}

__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(tc::smem_u32(bar))
      : "memory");
}

// Zero rows [from, to) of a tile of 128-byte rows in `halves` parts `stride`
// bytes apart (a whole warp), for operand rows that a product must not read:
// 0 times NaN is NaN.
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from, int to, int halves, uint32_t stride = kHalfBytes) {
  const int lane = threadIdx.x & 31, n = (to - from) * 8;
  for (int h = 0; h < halves; ++h)
    for (int i = lane; i < n; i += 32)
      *reinterpret_cast<uint4*>(tile + h * stride + from * 128 + i * 16) = make_uint4(0, 0, 0, 0);
  tc::fence_async_smem();
  __syncwarp();
}

// ------------------------------------------------------------------- host
// Tensor maps are encoded through the driver, which wants a current context;
// a host thread that has made no runtime call yet (an autograd worker) has
// none until its device is set.
inline bool bind_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}
// Query-side rows [rows, heads, d] as (d, g, key head, row) with boxes of 64
// channels x g heads x n rows: row n * g + i of the tile is head i of row n.
inline bool map_q(CUtensorMap* map, bool bf16, const void* p, int64_t st, int64_t sh, int rows, int heads, int kv_heads,
                  int d, int n) {
  const int g = heads / kv_heads;
  if (heads == 1) sh = (d + 7) / 8 * 8;  // a dimension of one row has any stride
  if (rows == 1) st = sh * heads;
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)g, (cuuint64_t)kv_heads, (cuuint64_t)rows};
  const cuuint64_t strides[3] = {(cuuint64_t)sh * 2, (cuuint64_t)sh * 2 * g, (cuuint64_t)st * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)g, 1, (cuuint32_t)n};
  return tma::encode(map, bf16, 4, p, dims, strides, box, true, true);
}
// Key-side rows [rows, kv_heads, d] with boxes of 64 channels x n rows
inline bool map_k(CUtensorMap* map, bool bf16, const void* p, int64_t st, int64_t sh, int rows, int kv_heads, int d, int n) {
  if (kv_heads == 1) sh = (d + 7) / 8 * 8;
  if (rows == 1) st = sh * kv_heads;
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)kv_heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)sh * 2, (cuuint64_t)st * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)n};
  return tma::encode(map, bf16, 3, p, dims, strides, box, true, true);
}
// Tensors and workspaces are read and written 16 bytes at a time (NULL is
// looked at where it matters).
inline bool aligned(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}
// what a tensor map of groups of g heads needs of a [rows, heads, d] tensor:
// strides of whole 16 bytes below 2^40 bytes (no tensor that fits the card has
// larger ones, but for dimensions of one, whose stride is not looked at)
inline bool rows_ok(const void* p, int64_t st, int64_t sh, int rows, int heads, int g) {
  auto fits = [](int64_t stride, int64_t most) { return stride > 0 && stride % 8 == 0 && stride < most; };
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || fits(st, int64_t(1) << 39)) &&
         (heads <= 1 || fits(sh, (int64_t(1) << 39) / g));
}
// The kernel was compiled to launch with at least `regs` registers a thread.
template <typename F>
inline bool launch_regs(F* func, int regs) {
  static std::mutex mu;
  static std::map<const void*, int> known;
  const void* key = reinterpret_cast<const void*>(func);
  std::lock_guard<std::mutex> lock(mu);
  auto it = known.find(key);
  if (it == known.end()) {
    cudaFuncAttributes at;
    if (cudaFuncGetAttributes(&at, func) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
    it = known.emplace(key, at.numRegs).first;
  }
  return it->second >= regs;
}
inline int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

int check(const mn_packed_args* a, Borders* bo, bool backward);  // packed_forward.cu

}  // namespace pk
}  // namespace mn
