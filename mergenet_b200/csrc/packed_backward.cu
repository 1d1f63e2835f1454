// Gradients of the packed attention (mn_packed_attention_backward), on the
// tensor cores:
//
//   p = 2^(x log2e - lse),  delta = dout . out,  ds = p (dout V^T - delta)
//   dq = scale ds K,  dk = scale ds^T Q,  dv = p^T dout
//   dtable[u, h] = sum of ds over the pairs of bucket u
//
// Two kernels, each recomputing p and ds: dq walks the keys of a query tile,
// dk and dv walk the query tiles of a key tile.  Seven products instead of
// the five of a single kernel, but every sum stays in one CTA's tensor
// memory: no atomics, a fixed order, no fp32 dq in memory.  Both keep p and
// ds in tensor memory as the 16-bit left operand of the next product (the
// key-side kernel works on transposed scores, S^T = K Q^T, so that p^T and
// ds^T have the keys in the lanes), so they never pass through shared memory.
//
// Tiles are those of the forward: 128 rows of (token, head of the group), so
// the gradients of a shared key head are summed over its query heads by the
// same products.  W threads share a row of a block's columns (4 * W compute
// warps); one warp issues the MMAs and one loads.  Four to a row keep the
// special-function unit busier than two: four warps to a scheduler.
//
// Blocks are 128 columns at 128 channels and 64 up to 64 channels, where two
// CTAs then share an SM and one's start and end run under the other's work
// (32 images of 197-785 tokens: 291 -> 271 us a step).
// What bounds a block is the compute warps' own chain: scores from tensor
// memory, exponentials (1,024 cycles of the special-function unit for 128 x
// 128), ds, both as 16-bit operands back; about 2,400 cycles against 1,536 of
// products for dq.  In the key-side kernel tensor memory holds both
// accumulators and one S at 128 channels; p and ds both go over dP, so that the
// next scores need not wait for p to be read (p over S instead: 3,700 cycles a
// tile against 2,048 of products; dk and dv of 7 documents 350 -> 305 us).  p
// through shared memory measured slower (487 us), as did blocks of 64 columns
// at 128 channels (893 -> 1,005 us for the step).
//
// Measured: 8,192 causal tokens, 16 heads of 128 on 8, bf16: 0.81-0.90 ms for
// both, the call repeated.  32 images of 197-785 tokens, 6 heads of 64, with a
// bias of 32 buckets: 97 us for dq and 78 for dk and dv in fp16 (one launch at a
// time); a bias adds 53 us to the 119 of the whole backward pass in bf16, and 54
// to the 132 in fp16.  With a look-up through the buckets, one chain of shuffles
// and a lane a bucket dq and dk with dv took 14 and 11 us more.
//
// delta takes out as the forward pass rounded it: its error, that of a mean of
// rounded values, is not above that of the ds rounded beside it, and an fp32 out
// would cost the forward pass twice its writes.
#include <algorithm>

#include "packed_tc.cuh"

namespace mn {
namespace pk {

struct BwdParams {
  mn_packed_args a;
  int group, ntok;
  int span, reach;   // bias: distances held, offset of distance 0
  int ranked;        // key tiles in descending order of the queries that see them
  float* delta;      // [kv_heads][tq * group]
  float* part;       // [kv_heads][slots][buckets * group] sums of ds by bucket
  unsigned* norms;   // fp16: [nseq][kv_heads][2] bits of the a bound of the largest squared norm of a row of dout, of v
  int* err;
};

// p and ds of fp16 inputs.  As they stand they would leave its range: ds
// passes 65,504 under the upstream gradients of a large loss scale and has
// steps of 2^-24 under small ones, and a weight below 2^-14 loses bits (one of
// 16,384 equal keys).  So dv takes 2^14 p, and dq and dk take 2^s ds, with one
// s for all rows of a sequence and key head; the powers are taken off the fp32
// sums.  delta is the mean of a row's dp by its p, so |ds| <= p (1 - p) times the
// span of the dp, half of max|dout| max|v|; that product goes to 2^15, which
// leaves a factor of four for the statistics of very large scores.  A ds below
// 2^-39 of it loses bits.  bf16 has the range of fp32.
constexpr int kPowerP = 14;
template <typename ET>
constexpr bool kPowers = std::is_same<ET, __half>::value;
__device__ __forceinline__ int power_of(const unsigned* norms) {  // s: max|dout| max|v| 2^s <= 2^15, by the bounds of both
  const unsigned x = norms[0], y = norms[1];
  if (x == 0 || y == 0) return 0;
  const int e = (int)(x >> 23) + (int)(y >> 23) - 252;  // (max|dout| max|v|)^2 < 2^e
  return min(max(15 - ((e + 1) >> 1), -40), 40);
}
__device__ __forceinline__ float pow2(int n) { return __int_as_float((127 + n) << 23); }

// The norms: a block takes 256 rows of (token, head of the group) of dout, or
// 256 keys of v, of one sequence and key head; a maximum depends on no order.
// A vector's eight channels of the largest sum stand for all of its eights:
// a bound within two bits, and no shuffles (15 us with them).
// Rows of no sequence and unused keys are not looked at, and rows with an
// infinity or a NaN do not count (their results show it in any case).
// 32 images of 197-785 tokens, 6 heads of 64: 10 us (24 MB from a cold cache),
// and the training step with a bias 232 -> 236 us.
__host__ __device__ constexpr int norm_tokens(int group) { return 256 / group; }
constexpr int kNormKeys = 256;
__global__ void __launch_bounds__(256) norms_kernel(const __grid_constant__ BwdParams p) {
  __shared__ uint32_t found_at[8];
  __shared__ float most[8];
  const mn_packed_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.group;
  const int hk = blockIdx.x % a.kv_heads, slot = blockIdx.x / a.kv_heads;
  const bool keys = blockIdx.y != 0;
  if (warp == 0)
    put_found(found_at, keys ? seq_of_slot<true>(a, kNormKeys, slot) : seq_of_slot<false>(a, norm_tokens(G), slot));
  __syncthreads();
  const Found f = get_found(found_at);
  if (f.seq >= a.nseq || f.local < 0) return;
  const int t0 = f.local * (keys ? kNormKeys : norm_tokens(G));
  const int n = keys ? min(kNormKeys, f.s.nk - t0) : min(norm_tokens(G), f.s.nq - t0) * G;  // vectors of the block
  const int width = a.head_dim / 8;
  int lanes = 1;  // a vector's lanes, eight channels each
  while (lanes < width) lanes *= 2;
  const int sub = lane % lanes, step = 8 * (32 / lanes);  // vectors of the block at a time
  float m = 0.f;
  for (int i0 = warp * (32 / lanes) + lane / lanes; i0 < n; i0 += 8 * step) {
    uint4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * step;
      const __half* row = keys ? static_cast<const __half*>(a.v) + (int64_t)(f.s.k0 + t0 + i) * a.v_st + hk * a.v_sh
                               : static_cast<const __half*>(a.dout) + (int64_t)(f.s.q0 + t0 + i / G) * a.do_st + (hk * G + i % G) * a.do_sh;
      v[u] = i < n && sub < width ? *reinterpret_cast<const uint4*>(row + sub * 8) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const __half* e = reinterpret_cast<const __half*>(&v[u]);
      float x = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) x = fmaf(to_f32(e[c]), to_f32(e[c]), x);
      if (x < INFINITY) m = fmaxf(m, x);
    }
  }
  m *= width;  // at least the largest of the vectors' sums
  m = warp_max(m);
  if (lane == 0) most[warp] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) m = fmaxf(m, most[w]);
    if (m > 0.f) atomicMax(p.norms + ((int64_t)f.seq * a.kv_heads + hk) * 2 + (keys ? 1 : 0), __float_as_uint(m));
  }
}

// Bias tables of a CTA: the bucket of each distance held, and the values of
// each head in log2 units.  Up to 64 channels (FLAT) a value per distance, with
// `pad` more on both sides, so that a warp whose block touches the distances
// held reads a value per score and needs no clamp; at 128 channels there is
// room for a value per bucket only.  The compute warps fill them while the first
// tiles are on their way.
struct BiasSmem {
  float* val;    // [group][len]
  uint8_t* idx;  // [span]
  int len;
};
template <bool FLAT>
__host__ __device__ constexpr int bias_len(int buckets, int group, int span, int pad) {
  // a head's values begin 32 / group banks after the last one's: the lanes of a position read different banks
  return FLAT ? span + 2 * pad + ((32 / group - span - 2 * pad) & 31) : buckets;
}
template <bool FLAT>
__host__ __device__ constexpr uint32_t bias_bytes(int buckets, int group, int span, int pad) {
  return bias_len<FLAT>(buckets, group, span, pad) * group * 4 + (span + 15) / 16 * 16;
}
template <bool FLAT>
__device__ __forceinline__ BiasSmem bias_at(uint8_t* at, int buckets, int group, int span, int pad) {
  BiasSmem s;
  s.val = reinterpret_cast<float*>(at);
  s.len = bias_len<FLAT>(buckets, group, span, pad);
  s.idx = at + s.len * group * 4;
  return s;
}
template <bool FLAT, int THREADS>  // by the compute threads, the first ones of the CTA
__device__ __forceinline__ void fill_bias(const BwdParams& p, const Borders& bo, int hk, const BiasSmem& s, int pad) {
  for (int i = threadIdx.x; i < p.span; i += THREADS) s.idx[i] = (uint8_t)bucket_of(bo, i - p.reach);
  if (FLAT) asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
  for (int g = 0; g < p.group; ++g)
    for (int i = threadIdx.x; i < s.len; i += THREADS)
      s.val[g * s.len + i] = table_value(p.a, FLAT ? s.idx[min(max(i - pad, 0), p.span - 1)] : i, hk * p.group + g);
}

template <typename ET>
__device__ __forceinline__ void put32(uint32_t taddr, const float* v) {
  uint32_t w[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) w[e] = pack2<ET>(v[2 * e], v[2 * e + 1]);
  tc::tmem_st16_nowait(taddr, w);
}
// left operand in tensor memory: the columns of each of a row's threads packed
// over the first half of their own, so that it overwrites only what that thread
// has read; the column of K step kk (16 columns of scores)
template <int CW>
__device__ __forceinline__ uint32_t left_cols(int kk) { return (uint32_t)(kk * 16 / CW * CW + kk * 16 % CW / 2); }

// ----------------------------------------------------------------------- dq
template <int DT, int NB, bool BIAS>
struct Dq {
  static constexpr int W = NB == 64 || BIAS ? 2 : 4;  // threads to a row; the sums by bucket take shared memory a warp
  static constexpr int CW = NB / W, kThreads = 32 * (4 * W + 2), kPerSM = NB == 64 ? 2 : 1;
  static constexpr int HV = DT / 64;
  static constexpr uint32_t kTile = HV * kHalfBytes, kKVHalf = NB * 128, kKV = HV * kKVHalf;
  static constexpr int KS = DT == 64 || !BIAS ? 3 : 2, VS = DT == 64 || !BIAS ? 2 : 1;
  static constexpr uint32_t oQ = 0, oDO = kTile, oK = 2 * kTile, oV = oK + KS * kKV, oBars = oV + VS * kKV;
  static constexpr int bQ = 0, bKF = 1, bKE = bKF + KS, bVF = bKE + KS, bVE = bVF + VS, bS = bVE + VS, bDP = bS + 2, bDS = bDP + 1,
                       bDone = bDS + 1, bDrain = bDone + 1, kNumBars = bDrain + 1;
  static constexpr uint32_t oMisc = oBars + ((kNumBars * 8 + 15) / 16) * 16;
  static constexpr uint32_t oDelta = oMisc + 32;             // [2][128] partial deltas
  // bias: per warp the sums by (head, bucket) and by (chain of keys, head, distance of a block); the bias tables
  static constexpr bool kFlat = DT == 64;
  static constexpr int kChains = DT == 64 ? 4 : 2, kChain = CW / kChains, kPad = 64;
  static_assert(!kFlat || kPad >= CW + 32, "distances of a warp's block past the ones held");
  static constexpr uint32_t oHist = oDelta + 2 * 128 * 4;
  static constexpr int diags(int group) { return kChain + 32 / group + 1; }  // distances of a warp's rows to a chain's keys
  static constexpr uint32_t warp_floats(int buckets, int group) {  // a multiple of 4
    return (buckets * group + kChains * group * diags(group) + group + 3) / 4 * 4;
  }
  static constexpr uint32_t bytes(int buckets, int group, int span) {
    return oHist + (BIAS ? 4 * W * warp_floats(buckets, group) * 4 + bias_bytes<kFlat>(buckets, group, span, kPad) : 0) + 1024;
  }
  static constexpr uint32_t cS = 0, cDP = 2 * NB, cDQ = 3 * NB, kCols = NB == 64 ? 256 : 512;
  static_assert(cDQ + DT <= kCols, "tensor memory");
};

template <typename ET, int DT, int NB, bool BIAS>
__global__ void __launch_bounds__(Dq<DT, NB, BIAS>::kThreads, Dq<DT, NB, BIAS>::kPerSM)
    dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
              const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
              const __grid_constant__ BwdParams p, const __grid_constant__ Borders bo) {
  using C = Dq<DT, NB, BIAS>;
  constexpr int HV = C::HV, KS = C::KS, VS = C::VS, W = C::W, CW = C::CW;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + C::oBars);
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(base + C::oMisc);
  const mn_packed_args& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = p.group;
  const int hk = blockIdx.x % a.kv_heads, slot_id = blockIdx.x / a.kv_heads;
  float* hist = reinterpret_cast<float*>(base + C::oHist);
  const int per_warp = BIAS ? C::warp_floats(a.buckets, G) : 0;
  BiasSmem bs;
  if (BIAS) bs = bias_at<C::kFlat>(base + C::oHist + 4 * W * per_warp * 4, a.buckets, G, p.span, C::kPad);

  if (warp == 0) tc::tmem_alloc(const_cast<uint32_t*>(misc), C::kCols);
  if (warp == 1) {
    put_found(misc + 1, seq_of_slot<false>(a, p.ntok, slot_id));
  }
  if (warp == 2 && lane == 0) {
    for (int i = 0; i < C::kNumBars; ++i) tc::mbar_init(bars + i, i == C::bDS ? 4 * W : 1);
    tc::fence_mbar_init();
  }
  if (warp == 3 && lane == 0) {
    tma::prefetch_map(&tm_q);
    tma::prefetch_map(&tm_do);
    tma::prefetch_map(&tm_k);
    tma::prefetch_map(&tm_v);
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = misc[0];
  const Found found = get_found(misc + 1);
  const Seq& s = found.s;
  const int tiles = (s.nq + p.ntok - 1) / p.ntok, local = found.local;
  const bool present = local >= 0 && local < tiles;
  const int t0 = present ? (a.causal ? tiles - 1 - local : local) * p.ntok : 0;
  const int shift = s.nk - s.nq;
  const int last = min(s.nq, t0 + p.ntok) - 1;
  const int keys = a.causal ? min(s.nk, last + shift + 1) : s.nk;
  const int n = present && keys > 0 ? (keys + NB - 1) / NB : 0;
  constexpr int ab_bf16 = std::is_same<ET, __nv_bfloat16>::value ? 1 : 0;
  bool ok = true;

  if (warp == 4 * W + 1) {
    // ---------------------------------------------------------------- loads
    if (lane == 0 && n > 0) {
      tma::expect_tx(bars + C::bQ, 2u * HV * 128u * (uint32_t)(G * p.ntok));
      for (int h = 0; h < HV; ++h) {
        tma::load_4d(tc::smem_u32(base + C::oQ + h * kHalfBytes), &tm_q, h * 64, 0, hk, s.q0 + t0, bars + C::bQ);
        tma::load_4d(tc::smem_u32(base + C::oDO + h * kHalfBytes), &tm_do, h * 64, 0, hk, s.q0 + t0, bars + C::bQ);
      }
      int nk = 0, nv = 0;
      for (int j = 0; j < n && ok; ++j) {
        const int ks = j % KS, vs = j % VS;
        if (j >= KS && !(ok = wait(bars + C::bKE + ks, (j / KS - 1) & 1, p.err))) break;
        tma::expect_tx(bars + C::bKF + ks, C::kKV);
        for (int h = 0; h < HV; ++h)
          load_3d(tc::smem_u32(base + C::oK + ks * C::kKV + h * C::kKVHalf), &tm_k, h * 64, hk, s.k0 + j * NB, bars + C::bKF + ks);
        nk = j + 1;
        if (j >= VS && !(ok = wait(bars + C::bVE + vs, (j / VS - 1) & 1, p.err))) break;
        tma::expect_tx(bars + C::bVF + vs, C::kKV);
        for (int h = 0; h < HV; ++h)
          load_3d(tc::smem_u32(base + C::oV + vs * C::kKV + h * C::kKVHalf), &tm_v, h * 64, hk, s.k0 + j * NB, bars + C::bVF + vs);
        nv = j + 1;
      }
      if (!ok && p.err) atomicOr(p.err, MN_STATUS_TC_TIMEOUT);
      // every copy issued has landed before the CTA may release its shared memory
      wait(bars + C::bQ, 0, nullptr);
      for (int j = max(0, nk - KS); j < nk; ++j) wait(bars + C::bKF + j % KS, (j / KS) & 1, nullptr);
      for (int j = max(0, nv - VS); j < nv; ++j) wait(bars + C::bVF + j % VS, (j / VS) & 1, nullptr);
    }
    __syncwarp();
  } else if (warp == 4 * W) {
    // ----------------------------------------------------------------- MMAs
    // S runs one block ahead of dP: at ds(j), dP(j + 1), dQ += ds(j) K(j) and
    // S(j + 2) are issued while the compute warps turn S(j + 1) into p
    constexpr uint32_t idesc_q = tc::idesc_f16(ab_bf16, 1, 128, DT);
    auto cols_of = [&](int j) { return min(NB, (s.nk - j * NB + 31) & ~31); };
    // D = A B^T over the channels, both operands 128-byte rows in shared memory
    auto scores = [&](uint32_t d, const uint8_t* x, const uint8_t* y, int cols, uint64_t* bar) {
      if (elect_one()) {
        tc::fence_after_sync();
        const uint64_t dx = tc::sw128_desc(tc::smem_u32(x), 16), dy = tc::sw128_desc(tc::smem_u32(y), 16);
        const uint32_t idesc = tc::idesc_f16(ab_bf16, 0, 128, cols);
#pragma unroll
        for (int kk = 0; kk < DT / 16; ++kk) {
          tc::mma_f16_ss(d, dx + (kk >> 2) * (kHalfBytes >> 4) + 2 * (kk & 3), dy + (kk >> 2) * (C::kKVHalf >> 4) + 2 * (kk & 3), idesc,
                         kk > 0 ? 1u : 0u);
        }
        tc::mma_commit(bar);
      }
      __syncwarp();
    };
    auto issue_s = [&](int j) -> bool {
      const int ks = j % KS;
      if (!wait(bars + C::bKF + ks, (j / KS) & 1, p.err)) return false;
      uint8_t* k = base + C::oK + ks * C::kKV;
      const int cols = cols_of(j);
      // rows behind the last key are an operand of ds K
      if (s.nk - j * NB < cols) zero_rows(k, s.nk - j * NB, cols, HV, C::kKVHalf);
      scores(tmem + C::cS + (j & 1) * NB, base + C::oQ, k, cols, bars + C::bS + (j & 1));
      return true;
    };
    auto issue_dp = [&](int j) -> bool {
      const int vs = j % VS;
      if (!wait(bars + C::bVF + vs, (j / VS) & 1, p.err)) return false;
      uint8_t* v = base + C::oV + vs * C::kKV;
      const int cols = cols_of(j);
      if (s.nk - j * NB < cols) zero_rows(v, s.nk - j * NB, cols, HV, C::kKVHalf);  // 0 (dP - delta) must not meet a NaN
      scores(tmem + C::cDP, base + C::oDO, v, cols, bars + C::bDP);
      return true;
    };
    if (n > 0) {
      ok = wait(bars + C::bQ, 0, p.err) && issue_s(0) && issue_dp(0);
      if (ok && n > 1) ok = issue_s(1);
      for (int j = 0; j < n && ok; ++j) {
        if (!(ok = wait(bars + C::bDS, j & 1, p.err))) break;
        if (j + 1 < n && !(ok = issue_dp(j + 1))) break;
        if (elect_one()) {
          tc::fence_after_sync();
          const int cols = cols_of(j);
          const uint64_t dk = tc::sw128_desc(tc::smem_u32(base + C::oK + (j % KS) * C::kKV), C::kKVHalf);
#pragma unroll
          for (int kk = 0; kk < NB / 16; ++kk)
            if (kk * 16 < cols)
              tc::mma_f16_ts(tmem + C::cDQ, tmem + C::cS + (j & 1) * NB + left_cols<CW>(kk), dk + 128 * kk, idesc_q,
                             (j > 0 || kk > 0) ? 1u : 0u);
          tc::mma_commit(bars + C::bKE + j % KS);
          if (j == n - 1) tc::mma_commit(bars + C::bDone);
        }
        __syncwarp();
        if (j + 2 < n) ok = issue_s(j + 2);
      }
      if (!ok && lane == 0 && p.err) atomicOr(p.err, MN_STATUS_TC_TIMEOUT);
      if (elect_one()) {
        tc::mma_commit(bars + C::bDrain);
        wait(bars + C::bDrain, 0, nullptr);
      }
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------- compute
    if (BIAS) {
      fill_bias<C::kFlat, 128 * W>(p, bo, hk, bs, C::kPad);
      for (int i = tid; i < 4 * W * per_warp; i += 128 * W) hist[i] = 0.f;
      asm volatile("bar.sync 1, %0;" ::"n"(128 * W) : "memory");
    }
    const int w = warp >> 2, r = (warp & 3) * 32 + lane;  // part of the columns, row
    const uint32_t lane_sel = (uint32_t)((warp & 3) * 32) << 16;
    const int my = t0 + r / G, g = r % G;
    const bool mine = present && r < G * p.ntok && my < s.nq;
    const int pos = my + shift;
    const int klim = a.causal && mine ? min(s.nk, pos + 1) : s.nk;
    const int kmin = __reduce_min_sync(MN_FULL_MASK, klim);
    const int pmin = __reduce_min_sync(MN_FULL_MASK, mine ? pos : 0x7fffffff);
    const int pmax = __reduce_max_sync(MN_FULL_MASK, mine ? pos : -0x7fffffff);
    const int64_t row = (int64_t)(s.q0 + my) * G + g, rows = (int64_t)a.tq * G;
    int power = 0;  // fp16: p enters as 2^power p, so that ds comes out as 2^power ds
    if (kPowers<ET>) power = n > 0 ? power_of(p.norms + ((int64_t)found.seq * a.kv_heads + hk) * 2) : 0;
    const float lift = (float)power, off = pow2(-power);
    // delta = dout . out, the channels in 8s in turn to the row's threads
    float* dl = reinterpret_cast<float*>(base + C::oDelta);
    {
      float acc = 0.f;
      if (mine) {
        const ET* x = static_cast<const ET*>(a.dout) + (int64_t)(s.q0 + my) * a.do_st + (hk * G + g) * a.do_sh;
        const ET* y = static_cast<const ET*>(a.out) + ((int64_t)(s.q0 + my) * a.heads + hk * G + g) * a.head_dim;
        for (int c = w; c < a.head_dim / 8; c += W) {
          const uint4 xv = *reinterpret_cast<const uint4*>(x + c * 8), yv = *reinterpret_cast<const uint4*>(y + c * 8);
          const ET* xe = reinterpret_cast<const ET*>(&xv);
          const ET* ye = reinterpret_cast<const ET*>(&yv);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc = fmaf(to_f32(xe[e]), to_f32(ye[e]), acc);
        }
      }
      auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(128 * W) : "memory"); };
      if (W == 4) {  // room for two partial sums a row
        if (w >= 2) dl[(w - 2) * 128 + r] = acc;
        sync();
        if (w < 2) acc += dl[w * 128 + r];
        sync();
      }
      if (w < 2) dl[w * 128 + r] = acc;
      sync();
    }
    const float delta = dl[r] + dl[128 + r];
    if (mine && w == 0) p.delta[hk * rows + row] = delta;
    const float nlse = mine ? -a.lse[hk * rows + row] : -INFINITY;
    const bool big = __any_sync(MN_FULL_MASK, is_big(nlse));  // scores rounded before lse is taken off, as in the forward
    const float sl2 = a.scale * kLog2e;
    const float* val = BIAS ? bs.val + (mine ? g : 0) * bs.len : nullptr;
    const float val_lo = BIAS ? val[C::kFlat ? 0 : bs.idx[0]] : 0.f, val_hi = BIAS ? val[C::kFlat ? bs.len - 1 : bs.idx[p.span - 1]] : 0.f;
    // bias: the warp's sums by (head, bucket), its block's by (chain, head, distance), and each head's first distance
    float* my_hist = hist + warp * per_warp;
    float* diag = my_hist + a.buckets * G;
    const int dist = BIAS ? C::diags(G) : 0, above = (31 - lane) / G;  // lanes of the same head above this one
    int* first = reinterpret_cast<int*>(diag + C::kChains * G * dist);
    float far_lo = 0.f, far_hi = 0.f;
    for (int j = 0; j < n && ok; ++j) {
      const int k0 = j * NB + w * CW;  // this thread's first key
      const int chunks = max(0, min(CW / 32, (min(NB, (s.nk - j * NB + 31) & ~31) - w * CW) >> 5));
      const uint32_t t_s = tmem + C::cS + (j & 1) * NB + w * CW + lane_sel, t_dp = tmem + C::cDP + w * CW + lane_sel;
      if (!(ok = wait(bars + C::bS + (j & 1), (j >> 1) & 1, p.err))) break;
      tc::fence_after_sync();
      float x[CW];
#pragma unroll
      for (int u = 0; u < CW / 32; ++u)
        if (u < chunks) tc::tmem_ld32_nowait(t_s + u * 32, x + u * 32);
      tc::tmem_ld_wait<CW>(x);
      const bool masked = kmin < k0 + CW;
      int kind = 0;  // bias: 1 all below the reach, 2 all above, 3 mixed
      float add = big ? 0.f : kPowers<ET> ? nlse + lift : nlse;
      if (BIAS) {
        kind = k0 + CW - 1 - pmin <= -p.reach ? 1 : k0 - pmax >= p.span - 1 - p.reach ? 2 : 3;
        if (kind == 1) add += val_lo;
        if (kind == 2) add += val_hi;
      }
      if (BIAS && kind == 3) {
        const int at = k0 - (mine ? pos : pmin) + p.reach;
        const float* flat = val + at + C::kPad;
#pragma unroll
        for (int e = 0; e < CW; ++e)
          if (e / 32 < chunks)
            x[e] = fmaf(x[e], sl2, (C::kFlat ? flat[e] : val[bs.idx[min(max(at + e, 0), p.span - 1)]]) + add);
      } else {
        const float2 f2 = make_float2(sl2, sl2), a2 = make_float2(add, add);
#pragma unroll
        for (int e = 0; e < CW / 2; ++e) {
          const float2 y = ffma2(make_float2(x[2 * e], x[2 * e + 1]), f2, a2);
          x[2 * e] = y.x;
          x[2 * e + 1] = y.y;
        }
      }
      if (__builtin_expect(big, 0)) {
#pragma unroll
        for (int e = 0; e < CW; ++e) x[e] = kPowers<ET> ? (x[e] + nlse) + lift : x[e] + nlse;
      }
      if (__builtin_expect(masked, 0)) {  // hidden keys get exactly 0
#pragma unroll
        for (int e = 0; e < CW; ++e)
          if (k0 + e >= klim) x[e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < CW; ++e) x[e] = ex2(x[e]);
      if (!(ok = wait(bars + C::bDP, j & 1, p.err))) break;
      if (tid == 0) tma::arrive(bars + C::bVE + j % VS);  // dP has read V (a commit would cost the MMA warp 200 cycles)
      tc::fence_after_sync();
      const float2 nd = make_float2(-delta, -delta);
#pragma unroll
      for (int u = 0; u < CW / 32; ++u) {
        if (u >= chunks) break;
        float d[32];
        tc::tmem_ld32_nowait(t_dp + u * 32, d);
        tc::tmem_ld_wait<32>(d);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 v = fmul2(make_float2(x[u * 32 + 2 * e], x[u * 32 + 2 * e + 1]), fadd2(make_float2(d[2 * e], d[2 * e + 1]), nd));
          x[u * 32 + 2 * e] = v.x;
          x[u * 32 + 2 * e + 1] = v.y;
        }
        put32<ET>(t_s + u * 16, x + u * 32);
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tma::arrive(bars + C::bDS);
      if (BIAS) {
        // Sums of ds by bucket; hidden keys have ds = 0, rows of no query and
        // chunks that do not exist are left out.
        if (kind == 3) {
          // Rows of one head are G lanes apart and one position on, so a
          // distance's sum moves up G lanes a key: a shuffle and an addition
          // a key for the whole warp, and the uppermost lane of each head has
          // the sum of the next distance (the lower lanes hold the last ones).
          // The keys are cut into chains, whose shuffles run side by side.
          constexpr int NC = C::kChains, L = C::kChain;
          float acc[NC];
#pragma unroll
          for (int e = 0; e < L; ++e)
#pragma unroll
            for (int q = 0; q < NC; ++q) {
              const float own = mine && (q * L + e) / 32 < chunks ? x[q * L + e] : 0.f;
              const float below = e ? __shfl_up_sync(MN_FULL_MASK, acc[q], G) : 0.f;
              acc[q] = (lane < G ? 0.f : below) + own;
              if (lane >= 32 - G) diag[(q * G + g) * dist + e] = acc[q];
            }
#pragma unroll
          for (int q = 0; q < NC; ++q) diag[(q * G + g) * dist + L - 1 + above] = acc[q];
          if (above == 0) first[g] = k0 - pos;
          __syncwarp();
          // Sums by bucket over the (head, distance) pairs in order, two a lane and turn:
          // a bucket's distances are contiguous, so each (head, bucket) is one
          // run of pairs, and the lane where it ends adds its sum.
          const int held = CW + 31 / G, all = G * held;  // a head's distances: CW keys, 31 / G + 1 rows
          for (int i0 = 0; i0 < all; i0 += 64) {
            float v[2];
            int to[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int i = i0 + 2 * lane + h, gg = i / held, t = i - gg * held;
              v[h] = 0.f;
              to[h] = -1;
              if (i < all) {
#pragma unroll
                for (int q = 0; q < NC; ++q)
                  if (t >= q * L && t < q * L + L + 31 / G) v[h] += diag[(q * G + gg) * dist + t - q * L];
                to[h] = gg * a.buckets + bs.idx[min(max(first[gg] + t + p.reach, 0), p.span - 1)];
              }
            }
            const int before = __shfl_up_sync(MN_FULL_MASK, to[1], 1), after = __shfl_down_sync(MN_FULL_MASK, to[0], 1);
            // a run goes on through a lane whose two pairs are of it
            const bool on = lane > 0 && to[0] == to[1] && before == to[0];
            const unsigned starts = ~__ballot_sync(MN_FULL_MASK, on);
            const int start = 31 - __clz(starts & (0xffffffffu >> (31 - lane)));  // the lane where the run at this lane's end began
            float run = v[1] + (to[0] == to[1] ? v[0] : 0.f);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const float t = __shfl_up_sync(MN_FULL_MASK, run, o);
              if (lane - o >= start) run += t;
            }
            const float left = __shfl_up_sync(MN_FULL_MASK, run, 1);
            if (to[0] != to[1]) my_hist[to[0]] += v[0] + (lane > 0 && before == to[0] ? left : 0.f);
            __syncwarp();
            if (to[1] >= 0 && (lane == 31 || after != to[1])) my_hist[to[1]] += run;
            __syncwarp();
          }
        } else if (mine) {
          float2 acc = make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < CW / 2; ++e)
            if (e / 16 < chunks) acc = fadd2(acc, make_float2(x[2 * e], x[2 * e + 1]));
          if (kind == 1) far_lo += acc.x + acc.y;
          else far_hi += acc.x + acc.y;
        }
      }
    }
    if (!ok && lane == 0 && p.err) atomicOr(p.err, MN_STATUS_TC_TIMEOUT);
    if (ok && n > 0) {
      ok = wait(bars + C::bDone, 0, p.err);
      tc::fence_after_sync();
    }
    if (ok) {
      ET* dst = static_cast<ET*>(a.dq) + ((int64_t)(s.q0 + my) * a.heads + hk * G + g) * a.head_dim;
#pragma unroll
      for (int u = w; u < DT / 32; u += W) {
        const int c0 = u * 32;
        float o[32];
        if (n > 0) {
          tc::tmem_ld32(tmem + C::cDQ + c0 + lane_sel, o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (mine) store32<ET>(dst, c0, a.head_dim, o, kPowers<ET> ? a.scale * off : a.scale);
        __syncwarp();
      }
    }
    if (BIAS) {
      __syncwarp();
      diag[lane] = far_lo;  // at least 64 floats: chains x (chain + 1) of them
      diag[32 + lane] = far_hi;
      __syncwarp();
      if (lane < min(G, 32)) {  // the head of this lane: its rows are G lanes apart
        float lo = 0.f, hi = 0.f;
        for (int l = lane; l < 32; l += G) {
          lo += diag[l];
          hi += diag[32 + l];
        }
        my_hist[g * a.buckets + bs.idx[0]] += lo;
        my_hist[g * a.buckets + bs.idx[p.span - 1]] += hi;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(128 * W) : "memory");
      const int per = a.buckets * G;
      const int64_t slots = gridDim.x / a.kv_heads;
      for (int i = tid; i < per; i += 128 * W) {  // in the order of dbias_kernel: [bucket][head]
        const int at = i % G * a.buckets + i / G;
        float acc = 0.f;
        for (int ww = 0; ww < 4 * W; ++ww) acc += hist[ww * per_warp + at];
        p.part[(hk * slots + slot_id) * per + i] = kPowers<ET> ? acc * off : acc;
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, C::kCols);
  }
}

// dtable[u, hk * G + g]: the tiles' sums in order, one block per entry
__global__ void __launch_bounds__(128) dbias_kernel(int heads, int group, int buckets, int slots, const float* __restrict__ part,
                                                    void* __restrict__ out, int dtype) {
  __shared__ float scratch[32];
  const int i = blockIdx.x, hk = blockIdx.y, per = buckets * group;
  float x = 0.f;
  for (int t = threadIdx.x; t < slots; t += 128) x += part[((int64_t)hk * slots + t) * per + i];
  x = block_sum(x, scratch);
  if (threadIdx.x == 0) store_any(out, dtype, (i / group) * heads + hk * group + i % group, x);
}

// ------------------------------------------------------------------- dk, dv
template <int DT, int NB, bool BIAS>
struct Dkv {
  static constexpr int W = NB / 32, CW = 32, kThreads = 32 * (4 * W + 2), kPerSM = NB == 64 ? 2 : 1;
  static constexpr int HV = DT / 64;
  static constexpr uint32_t kTile = HV * kHalfBytes, kQHalf = NB * 128, kQ = HV * kQHalf;
  // Stages of Q and of dout (with lse and delta).  S(i + 1) is issued as soon
  // as S(i) has been read, so its Q has to be there a tile early: three stages,
  // but for the bias tables' room at 128 channels.
  static constexpr int QS = DT == 128 && BIAS ? 2 : 3, OS = 2;
  static constexpr uint32_t oK = 0, oV = kTile, oRing = 2 * kTile, oDO = oRing + QS * kQ, oRows = oDO + OS * kQ;  // [OS][2][NB] floats
  static constexpr uint32_t oBars = oRows + OS * NB * 8;
  // barriers: K and V landed; Q, dout (and its rows) landed; tile i % 3 done; S ready, read; dP ready; p and ds ready
  static constexpr int bKV = 0, bF = 1, bO = bF + QS, bE = bO + OS, bS = bE + 3, bSR = bS + 1, bDP = bSR + 1, bDS = bDP + 1,
                       bDone = bDS + 1, bDrain = bDone + 1, kNumBars = bDrain + 1;
  static constexpr uint32_t oMisc = oBars + ((kNumBars * 8 + 15) / 16) * 16;
  static constexpr bool kFlat = DT == 64;
  static constexpr int pad(int group) { return 128 + NB / group + 2; }  // distances of a tile pair past the ones held
  // of a column, [NB] each: its token, and the place of its head's first value; FLAT: that place less the token instead
  // of the token
  static constexpr uint32_t oCol = oMisc + 48;
  static constexpr uint32_t oTab = oCol + NB * 8;
  static constexpr uint32_t bytes(int buckets, int group, int span) {
    return (BIAS ? oTab + bias_bytes<kFlat>(buckets, group, span, pad(group)) : oCol);
  }
  static constexpr uint32_t cS = 0, cDP = NB, cDV = cDP + NB, cDK = cDV + DT, kCols = NB == 64 ? 256 : 512;
  static_assert(cDK + DT <= kCols, "tensor memory");
};

template <typename ET, int DT, int NB, bool BIAS>
__global__ void __launch_bounds__(Dkv<DT, NB, BIAS>::kThreads, Dkv<DT, NB, BIAS>::kPerSM)
    dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
               const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
               const __grid_constant__ BwdParams p, const __grid_constant__ Borders bo) {
  using C = Dkv<DT, NB, BIAS>;
  constexpr int HV = C::HV, QS = C::QS, OS = C::OS, W = C::W, CW = C::CW;
  // Swizzled tiles begin on 1,024 bytes.  The declaration asks for it: at 128
  // channels the tiles fill shared memory to the last KB, without room to align
  // the start by hand.
  extern __shared__ __align__(1024) uint8_t base[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + C::oBars);
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(base + C::oMisc);
  volatile uint8_t* big = base + C::oMisc + 32;  // [OS] a row's lse is big: scores rounded before it is taken off
  int *col = reinterpret_cast<int*>(base + C::oCol), *col_val = col + NB;
  const mn_packed_args& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = p.group;
  const int hk = blockIdx.x % a.kv_heads, slot_id = blockIdx.x / a.kv_heads;
  BiasSmem bs;
  if (BIAS) bs = bias_at<C::kFlat>(base + C::oTab, a.buckets, G, p.span, C::pad(G));

  if (warp == 0) tc::tmem_alloc(const_cast<uint32_t*>(misc), C::kCols);
  if (warp == 1) {
    put_found(misc + 1, p.ranked ? ranked_slot<true>(a, 128, slot_id) : seq_of_slot<true>(a, 128, slot_id));
  }
  if (warp == 2 && lane == 0) {
    for (int i = 0; i < C::kNumBars; ++i)
      tc::mbar_init(bars + i, i >= C::bO && i < C::bE ? 2 : i == C::bSR || i == C::bDS ? 4 * W : 1);
    tc::fence_mbar_init();
  }
  if (warp == 3 && lane == 0) {
    tma::prefetch_map(&tm_q);
    tma::prefetch_map(&tm_do);
    tma::prefetch_map(&tm_k);
    tma::prefetch_map(&tm_v);
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = misc[0];
  const Found found = get_found(misc + 1);
  const Seq& s = found.s;
  const int local = found.local, k0 = local * 128;
  const bool present = local >= 0 && k0 < s.slot;
  const int shift = s.nk - s.nq;
  // query tiles that see a key of this tile: [i0, i0 + n)
  const int i0 = a.causal ? max(0, k0 - shift) / p.ntok : 0;
  const int n = present && k0 < s.nk ? max(0, (s.nq + p.ntok - 1) / p.ntok - i0) : 0;
  constexpr int ab_bf16 = std::is_same<ET, __nv_bfloat16>::value ? 1 : 0;
  // bias of a whole tile pair: 1 all distances below the reach, 2 all above, 3 mixed
  auto kind_of = [&](int t0) {
    return k0 + 127 - (t0 + shift) <= -p.reach ? 1 : k0 - (t0 + p.ntok - 1 + shift) >= p.span - 1 - p.reach ? 2 : 3;
  };
  // fp16: 2^kPowerP p, and with dp and delta times 2^(power - kPowerP) 2^power ds
  int power = 0;
  if (kPowers<ET>) power = n > 0 ? power_of(p.norms + ((int64_t)found.seq * a.kv_heads + hk) * 2) : 0;
  const float lift = kPowers<ET> ? (float)kPowerP : 0.f, dp_by = kPowers<ET> ? pow2(power - kPowerP) : 1.f;
  bool ok = true;

  if (warp == 4 * W + 1) {
    // ---------------------------------------------------------------- loads
    if (n > 0) {
      if (lane == 0) {
        tma::expect_tx(bars + C::bKV, 2 * C::kTile);
        for (int h = 0; h < HV; ++h) {
          load_3d(tc::smem_u32(base + C::oK + h * kHalfBytes), &tm_k, h * 64, hk, s.k0 + k0, bars + C::bKV);
          load_3d(tc::smem_u32(base + C::oV + h * kHalfBytes), &tm_v, h * 64, hk, s.k0 + k0, bars + C::bKV);
        }
      }
      int q_done = 0, done = 0;
      const int64_t rows = (int64_t)a.tq * G;
      for (int i = 0; i < n && ok; ++i) {
        const int st = i % OS, t0 = (i0 + i) * p.ntok;
        const uint32_t bytes = (uint32_t)(HV * 128 * G * p.ntok);
        // tile i - 2 done: its dout stage is free, and with three stages of Q (whose
        // last tile's end was waited for a turn ago) Q need not wait for it
        auto before = [&] { return i < 2 || wait(bars + C::bE + (i - 2) % 3, ((i - 2) / 3) & 1, p.err); };
        if (QS == 2 && !(ok = before())) break;
        if (lane == 0) {
          tma::expect_tx(bars + C::bF + i % QS, bytes);
          for (int h = 0; h < HV; ++h)
            tma::load_4d(tc::smem_u32(base + C::oRing + (i % QS) * C::kQ + h * C::kQHalf), &tm_q, h * 64, 0, hk, s.q0 + t0,
                         bars + C::bF + i % QS);
        }
        q_done = i + 1;
        if (QS == 3 && !(ok = before())) break;
        if (lane == 0) {
          tma::expect_tx(bars + C::bO + st, bytes);
          for (int h = 0; h < HV; ++h)
            tma::load_4d(tc::smem_u32(base + C::oDO + st * C::kQ + h * C::kQHalf), &tm_do, h * 64, 0, hk, s.q0 + t0,
                         bars + C::bO + st);
        }
        if (BIAS && i == 0) {  // the bias tables are there
          __syncwarp();
          asm volatile("bar.sync 2, %0;" ::"n"(128 * W + 32) : "memory");
        }
        // -lse (with the bias where it is the same for the whole tile) and
        // -delta of the rows; rows of no query give p = 0
        float* x = reinterpret_cast<float*>(base + C::oRows) + st * 2 * NB;
        const int valid = min(p.ntok, s.nq - t0) * G;
        const int64_t first = hk * rows + (int64_t)(s.q0 + t0) * G;
        const int kind = BIAS ? kind_of(t0) : 0;
        const int lo = !BIAS || C::kFlat ? 0 : bs.idx[0], hi = !BIAS ? 0 : C::kFlat ? bs.len - 1 : bs.idx[p.span - 1];
        float l[NB / 32];
        bool any_big = false;
#pragma unroll
        for (int e = 0; e < NB / 32; ++e) {
          const int r = e * 32 + lane;
          l[e] = r < valid ? -a.lse[first + r] : -INFINITY;
          any_big |= is_big(l[e]);
          x[NB + r] = r < valid ? -p.delta[first + r] * dp_by : 0.f;
        }
        any_big = __any_sync(MN_FULL_MASK, any_big);
        if (lane == 0) big[st] = any_big;
#pragma unroll
        for (int e = 0; e < NB / 32; ++e) {
          const int r = e * 32 + lane;
          if (BIAS && kind != 3 && !any_big && r < valid) l[e] += bs.val[col_val[r] + (kind == 1 ? lo : hi)];
          if (kPowers<ET> && !any_big) l[e] += lift;
          x[r] = l[e];
        }
        __syncwarp();
        if (lane == 0) tma::arrive(bars + C::bO + st);
        done = i + 1;
      }
      if (lane == 0) {
        if (!ok && p.err) atomicOr(p.err, MN_STATUS_TC_TIMEOUT);
        // every copy issued has landed before the CTA may release its shared memory
        wait(bars + C::bKV, 0, nullptr);
        for (int i = max(0, q_done - QS); i < q_done; ++i) wait(bars + C::bF + i % QS, (i / QS) & 1, nullptr);
        for (int i = max(0, done - OS); i < done; ++i) wait(bars + C::bO + i % OS, (i / OS) & 1, nullptr);
      }
    }
    __syncwarp();
  } else if (warp == 4 * W) {
    // ----------------------------------------------------------------- MMAs
    // p(i) and ds(i) both go over dP(i), whose values the compute warps have in
    // registers by then, so S's columns are free from the moment S(i) has been
    // read: S(i + 1) is computed under the exponentials of tile i, and
    // dV += p(i) dout, dK += ds(i) Q and dP(i + 1) under those of tile i + 1.
    constexpr uint32_t idesc_s = tc::idesc_f16(ab_bf16, 0, 128, NB), idesc_g = tc::idesc_f16(ab_bf16, 1, 128, DT);
    auto q_at = [&](int i) { return base + C::oRing + (i % QS) * C::kQ; };
    auto do_at = [&](int i) { return base + C::oDO + (i % OS) * C::kQ; };
    auto scores = [&](uint32_t d, const uint8_t* x, const uint8_t* y, uint64_t* bar) {
      if (elect_one()) {
        tc::fence_after_sync();
        const uint64_t dx = tc::sw128_desc(tc::smem_u32(x), 16), dy = tc::sw128_desc(tc::smem_u32(y), 16);
#pragma unroll
        for (int kk = 0; kk < DT / 16; ++kk) {
          tc::mma_f16_ss(d, dx + (kk >> 2) * (kHalfBytes >> 4) + 2 * (kk & 3), dy + (kk >> 2) * (C::kQHalf >> 4) + 2 * (kk & 3), idesc_s,
                         kk > 0 ? 1u : 0u);
        }
        tc::mma_commit(bar);
      }
      __syncwarp();
    };
    auto issue_s = [&](int i) -> bool {
      if (!wait(bars + C::bF + i % QS, (i / QS) & 1, p.err)) return false;
      const int valid = min(p.ntok, s.nq - (i0 + i) * p.ntok) * G;
      if (valid < NB) zero_rows(q_at(i), valid, NB, HV, C::kQHalf);  // rows of no query are an operand of dK ...
      scores(tmem + C::cS, base + C::oK, q_at(i), bars + C::bS);
      return true;
    };
    auto issue_dp = [&](int i) -> bool {
      if (!wait(bars + C::bO + i % OS, (i / OS) & 1, p.err)) return false;
      const int valid = min(p.ntok, s.nq - (i0 + i) * p.ntok) * G;
      if (valid < NB) zero_rows(do_at(i), valid, NB, HV, C::kQHalf);  // ... and of dV
      scores(tmem + C::cDP, base + C::oV, do_at(i), bars + C::bDP);
      return true;
    };
    auto grads = [&](uint32_t d, uint32_t left, const uint8_t* x, bool more) {  // D += left x
      const uint64_t dx = tc::sw128_desc(tc::smem_u32(x), C::kQHalf);
#pragma unroll
      for (int kk = 0; kk < NB / 16; ++kk)
        tc::mma_f16_ts(d, left + left_cols<CW>(kk), dx + 128 * kk, idesc_g, (more || kk > 0) ? 1u : 0u);
    };
    if (n > 0) {
      ok = wait(bars + C::bKV, 0, p.err);
      ok = ok && issue_s(0) && issue_dp(0);
      for (int i = 0; i < n && ok; ++i) {
        if (i + 1 < n && !(ok = wait(bars + C::bSR, i & 1, p.err) && issue_s(i + 1))) break;
        if (!(ok = wait(bars + C::bDS, i & 1, p.err))) break;
        if (elect_one()) {
          tc::fence_after_sync();
          grads(tmem + C::cDV, tmem + C::cDP, do_at(i), i > 0);
          grads(tmem + C::cDK, tmem + C::cDP + CW / 2, q_at(i), i > 0);
          tc::mma_commit(bars + C::bE + i % 3);
          if (i == n - 1) tc::mma_commit(bars + C::bDone);
        }
        __syncwarp();
        if (i + 1 < n) ok = issue_dp(i + 1);
      }
      if (!ok && lane == 0 && p.err) atomicOr(p.err, MN_STATUS_TC_TIMEOUT);
      if (elect_one()) {
        tc::mma_commit(bars + C::bDrain);
        wait(bars + C::bDrain, 0, nullptr);
      }
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------- compute
    if (BIAS && n > 0) {
      fill_bias<C::kFlat, 128 * W>(p, bo, hk, bs, C::pad(G));
      if (tid < NB) {
        col_val[tid] = tid % G * bs.len;
        col[tid] = C::kFlat ? col_val[tid] - tid / G : tid / G;
      }
      asm volatile("bar.sync 2, %0;" ::"n"(128 * W + 32) : "memory");  // with the load warp
    }
    const int w = warp >> 2, r = (warp & 3) * 32 + lane;  // part of the columns, key row
    const uint32_t lane_sel = (uint32_t)((warp & 3) * 32) << 16;
    const int key = k0 + r;
    const float sl2 = a.scale * kLog2e;
    for (int i = 0; i < n && ok; ++i) {
      const int st = i % OS, t0 = (i0 + i) * p.ntok;
      const uint32_t t_s = tmem + C::cS + w * CW + lane_sel, t_dp = tmem + C::cDP + w * CW + lane_sel;
      const float* nl = reinterpret_cast<const float*>(base + C::oRows) + st * 2 * NB + w * CW;
      // columns from here on see this key; the warp's last key sees the latest start
      const int c0 = a.causal ? (key - shift - t0) * G - w * CW : 0;
      const bool masked = a.causal && (k0 + ((warp & 3) * 32 + 31) - shift - t0) * G > w * CW;
      if (!(ok = wait(bars + C::bO + st, (i / OS) & 1, p.err))) break;  // lse and delta are there
      if (!(ok = wait(bars + C::bS, i & 1, p.err))) break;
      tc::fence_after_sync();
      float x[CW];
      tc::tmem_ld32_nowait(t_s, x);
      tc::tmem_ld_wait<CW>(x);
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tma::arrive(bars + C::bSR);
      const bool apart = big[st] != 0;
      const int at = key - t0 - shift + p.reach;  // place of token 0's distance among those held
      const float* flat = bs.val + at + C::pad(G);
      auto bias = [&](int c, int cv) {  // of a column, in a tile pair that touches the distances held
        return C::kFlat ? flat[c] : bs.val[cv + bs.idx[min(max(at - c, 0), p.span - 1)]];
      };
      auto bias_any = [&](int c, int cv) {  // in any tile pair
        return C::kFlat ? bs.val[cv + min(max(at + C::pad(G) + c - cv, 0), bs.len - 1)] : bias(c, cv);
      };
      if (__builtin_expect(apart, 0)) {
#pragma unroll
        for (int e = 0; e < CW; ++e) {
          const float b = BIAS ? bias_any(col[w * CW + e], col_val[w * CW + e]) : 0.f;
          x[e] = __fmaf_rn(x[e], sl2, b) + nl[e];
          if (kPowers<ET>) x[e] += lift;
        }
      } else if (BIAS && kind_of(t0) == 3) {
#pragma unroll
        for (int e = 0; e < CW / 4; ++e) {
          const float4 l = reinterpret_cast<const float4*>(nl)[e];
          const int4 c = reinterpret_cast<const int4*>(col + w * CW)[e];
          const int4 cv = C::kFlat ? c : reinterpret_cast<const int4*>(col_val + w * CW)[e];
          x[4 * e] = fmaf(x[4 * e], sl2, l.x + bias(c.x, cv.x));
          x[4 * e + 1] = fmaf(x[4 * e + 1], sl2, l.y + bias(c.y, cv.y));
          x[4 * e + 2] = fmaf(x[4 * e + 2], sl2, l.z + bias(c.z, cv.z));
          x[4 * e + 3] = fmaf(x[4 * e + 3], sl2, l.w + bias(c.w, cv.w));
        }
      } else {
        const float2 f2 = make_float2(sl2, sl2);
#pragma unroll
        for (int e = 0; e < CW / 4; ++e) {
          const float4 l = reinterpret_cast<const float4*>(nl)[e];
          const float2 y0 = ffma2(make_float2(x[4 * e], x[4 * e + 1]), f2, make_float2(l.x, l.y));
          const float2 y1 = ffma2(make_float2(x[4 * e + 2], x[4 * e + 3]), f2, make_float2(l.z, l.w));
          x[4 * e] = y0.x; x[4 * e + 1] = y0.y; x[4 * e + 2] = y1.x; x[4 * e + 3] = y1.y;
        }
      }
      if (__builtin_expect(masked, 0)) {
#pragma unroll
        for (int e = 0; e < CW; ++e)
          if (e < c0) x[e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < CW; ++e) x[e] = ex2(x[e]);  // hidden keys and columns of no query: exactly 0
      if (!(ok = wait(bars + C::bDP, i & 1, p.err))) break;
      tc::fence_after_sync();
      float d[CW];
      tc::tmem_ld32_nowait(t_dp, d);
      tc::tmem_ld_wait<CW>(d);
#pragma unroll
      for (int e = 0; e < CW / 4; ++e) {
        const float4 nd = reinterpret_cast<const float4*>(nl + NB)[e];
        const float2 d0 = make_float2(d[4 * e], d[4 * e + 1]), d1 = make_float2(d[4 * e + 2], d[4 * e + 3]);
        const float2 n0 = make_float2(nd.x, nd.y), n1 = make_float2(nd.z, nd.w), by = make_float2(dp_by, dp_by);
        const float2 y0 = fmul2(make_float2(x[4 * e], x[4 * e + 1]), kPowers<ET> ? ffma2(d0, by, n0) : fadd2(d0, n0));
        const float2 y1 = fmul2(make_float2(x[4 * e + 2], x[4 * e + 3]), kPowers<ET> ? ffma2(d1, by, n1) : fadd2(d1, n1));
        d[4 * e] = y0.x; d[4 * e + 1] = y0.y; d[4 * e + 2] = y1.x; d[4 * e + 3] = y1.y;
      }
      // p over the first half of this thread's columns, ds over the second
      put32<ET>(t_dp, x);
      put32<ET>(t_dp + CW / 2, d);
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tma::arrive(bars + C::bDS);
    }
    if (!ok && lane == 0 && p.err) atomicOr(p.err, MN_STATUS_TC_TIMEOUT);
    if (ok && n > 0) {
      ok = wait(bars + C::bDone, 0, p.err);
      tc::fence_after_sync();
    }
    if (ok) {
      const bool mine = present && key < s.slot;
#pragma unroll
      for (int q = w; q < DT / 16; q += W) {  // chunks of dV, then of dK
        const bool is_v = q < DT / 32;
        const int c0 = (is_v ? q : q - DT / 32) * 32;
        float o[32];
        if (n > 0) tc::tmem_ld32(tmem + (is_v ? C::cDV : C::cDK) + c0 + lane_sel, o);
        if (n == 0 || key >= s.nk) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (mine)
          store32<ET>(static_cast<ET*>(is_v ? a.dv : a.dk) + ((int64_t)(s.k0 + key) * a.kv_heads + hk) * a.head_dim, c0, a.head_dim,
                      o, is_v ? pow2(kPowers<ET> ? -kPowerP : 0) : kPowers<ET> ? a.scale * pow2(-power) : a.scale);
        __syncwarp();
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, C::kCols);
  }
}

// ------------------------------------------------------------------- host
struct BwdSizes {
  int ntok, ntok_k;  // tokens to a tile of the query side, to a block of the key side
  int64_t q_slots, k_slots;
  size_t delta_bytes, norm_bytes, bytes;
};
// Up to 64 channels: blocks of 64 columns and two CTAs to an SM, so that one's
// start and end run under the other's products; not where a token's heads
// would fill such a block badly.
static bool small_blocks(const mn_packed_args* a) { return a->head_dim <= 64 && a->heads / a->kv_heads <= 32; }
static BwdSizes sizes_of(const mn_packed_args* a) {
  BwdSizes z;
  const int g = a->heads / a->kv_heads;
  z.ntok = 128 / g;
  z.ntok_k = small_blocks(a) ? 64 / g : z.ntok;
  z.q_slots = tile_slots(a->tq, a->nseq, z.ntok);
  z.k_slots = tile_slots(a->tk, a->nseq, 128);
  z.delta_bytes = ((size_t)a->tq * a->heads * 4 + 255) / 256 * 256;
  z.norm_bytes = a->dtype == MN_F16 ? ((size_t)a->nseq * a->kv_heads * 8 + 255) / 256 * 256 : 0;
  z.bytes = z.delta_bytes + z.norm_bytes + (a->bias_table ? (size_t)z.q_slots * a->heads * a->buckets * 4 : 0);
  return z;
}

template <typename ET, int DT, int NB, bool BIAS>
static bool launch_bwd(const mn_packed_args* a, const Borders& bo, const BwdSizes& z, void* ws, int* err, cudaStream_t st) {
  constexpr bool bf16 = std::is_same<ET, __nv_bfloat16>::value;
  BwdParams p;
  p.a = *a;
  p.group = a->heads / a->kv_heads;
  p.ntok = z.ntok;
  p.span = p.reach = 0;
  p.ranked = a->nseq > 1 && a->nseq <= kRanked && (z.k_slots - 1) * a->kv_heads > sm_count();  // more than a wave
  if (BIAS) {
    const int last = bo.n ? bo.at[bo.n - 1] : 1;
    p.reach = last;
    p.span = (bo.two_sided ? 2 : 1) * last + 1;
  }
  p.delta = static_cast<float*>(ws);
  p.norms = reinterpret_cast<unsigned*>(static_cast<char*>(ws) + z.delta_bytes);
  p.part = reinterpret_cast<float*>(static_cast<char*>(ws) + z.delta_bytes + z.norm_bytes);
  p.err = err;
  CUtensorMap mq, mdo, mk, mv, nq, ndo, nk, nv;  // m: the query-side kernel's, n: the key-side kernel's
  const void *k = a->tk ? a->k : a->q, *v = a->tk ? a->v : a->q;
  const int tk = std::max(a->tk, 1);
  if (!bind_context() || !map_q(&mq, bf16, a->q, a->q_st, a->q_sh, a->tq, a->heads, a->kv_heads, a->head_dim, z.ntok) ||
      !map_q(&mdo, bf16, a->dout, a->do_st, a->do_sh, a->tq, a->heads, a->kv_heads, a->head_dim, z.ntok) ||
      !map_k(&mk, bf16, k, a->k_st, a->k_sh, tk, a->kv_heads, a->head_dim, NB) ||
      !map_k(&mv, bf16, v, a->v_st, a->v_sh, tk, a->kv_heads, a->head_dim, NB) ||
      !map_q(&nq, bf16, a->q, a->q_st, a->q_sh, a->tq, a->heads, a->kv_heads, a->head_dim, z.ntok_k) ||
      !map_q(&ndo, bf16, a->dout, a->do_st, a->do_sh, a->tq, a->heads, a->kv_heads, a->head_dim, z.ntok_k) ||
      !map_k(&nk, bf16, k, a->k_st, a->k_sh, tk, a->kv_heads, a->head_dim, 128) ||
      !map_k(&nv, bf16, v, a->v_st, a->v_sh, tk, a->kv_heads, a->head_dim, 128))
    return false;
  auto kq = dq_kernel<ET, DT, NB, BIAS>;
  auto kkv = dkv_kernel<ET, DT, NB, BIAS>;
  const size_t sq = Dq<DT, NB, BIAS>::bytes(a->buckets, p.group, p.span), skv = Dkv<DT, NB, BIAS>::bytes(a->buckets, p.group, p.span);
  if (!ensure_smem(kq, sq) || !ensure_smem(kkv, skv)) return false;
  if constexpr (kPowers<ET>) {
    const int64_t qs = tile_slots(a->tq, a->nseq, norm_tokens(p.group)), ks = tile_slots(a->tk, a->nseq, kNormKeys);
    if (cudaMemsetAsync(p.norms, 0, z.norm_bytes, st) != cudaSuccess) return false;
    norms_kernel<<<dim3((unsigned)(std::max(qs, ks) * a->kv_heads), 2), 256, 0, st>>>(p);
  }
  kq<<<(unsigned)(z.q_slots * a->kv_heads), Dq<DT, NB, BIAS>::kThreads, sq, st>>>(mq, mdo, mk, mv, p, bo);
  BwdParams pk = p;
  pk.ntok = z.ntok_k;
  if (a->tk > 0) kkv<<<(unsigned)(z.k_slots * a->kv_heads), Dkv<DT, NB, BIAS>::kThreads, skv, st>>>(nq, ndo, nk, nv, pk, bo);
  if (BIAS)
    dbias_kernel<<<dim3(a->buckets * p.group, a->kv_heads), 128, 0, st>>>(a->heads, p.group, a->buckets, (int)z.q_slots, p.part,
                                                                         a->dbias, a->bias_dtype);
  return true;
}

template <typename ET, int DT>
static bool launch_bwd_d(const mn_packed_args* a, const Borders& bo, const BwdSizes& z, void* ws, int* err, cudaStream_t st) {
  if constexpr (DT == 64) {
    if (small_blocks(a))
      return a->bias_table ? launch_bwd<ET, DT, 64, true>(a, bo, z, ws, err, st) : launch_bwd<ET, DT, 64, false>(a, bo, z, ws, err, st);
    return launch_bwd<ET, DT, 128, false>(a, bo, z, ws, err, st);  // a bias comes with at most 16 grouped heads
  } else {
    return a->bias_table ? launch_bwd<ET, DT, 128, true>(a, bo, z, ws, err, st) : launch_bwd<ET, DT, 128, false>(a, bo, z, ws, err, st);
  }
}

}  // namespace pk
}  // namespace mn

using namespace mn;

extern "C" size_t mn_packed_attention_backward_workspace_bytes(const mn_packed_args* a) {
  Borders bo;
  if (pk::check(a, &bo, true) != MN_OK || a->tq == 0) return 0;
  return pk::sizes_of(a).bytes;
}

extern "C" int mn_packed_attention_backward(const mn_packed_args* a, void* workspace, size_t workspace_bytes, int* status,
                                            void* stream) {
  Borders bo;
  const int rc = pk::check(a, &bo, true);
  if (rc != MN_OK) return rc;
  if (a->tq == 0) return MN_ERR_ARG;  // no query: the gradients are 0, nothing to launch
  const pk::BwdSizes z = pk::sizes_of(a);
  if (!workspace || !pk::aligned({workspace}) || workspace_bytes < z.bytes) return MN_ERR_WORKSPACE;
  cudaGetLastError();
  auto st = static_cast<cudaStream_t>(stream);
  bool done;
  if (a->dtype == MN_F16)
    done = a->head_dim <= 64 ? pk::launch_bwd_d<__half, 64>(a, bo, z, workspace, status, st)
                             : pk::launch_bwd_d<__half, 128>(a, bo, z, workspace, status, st);
  else
    done = a->head_dim <= 64 ? pk::launch_bwd_d<__nv_bfloat16, 64>(a, bo, z, workspace, status, st)
                             : pk::launch_bwd_d<__nv_bfloat16, 128>(a, bo, z, workspace, status, st);
  if (!done) return MN_ERR_UNSUPPORTED;
  return cudaGetLastError() == cudaSuccess ? MN_OK : MN_ERR_LAUNCH;
}
