// Attention over packed sequences (mn_packed_attention), on the tensor cores.
//
//   x = scale Q K^T + bias,  out = softmax(x) V  within each sequence
//
// A tile is 128 rows of (token, head of the group), token-major: the heads
// that share a key head sit in one tile, so grouped heads read their keys and
// values once and one token's form is a tile of its heads.  Per block of keys:
//
//   * a load warp brings K and V (a ring of tiles) by TMA;
//   * an MMA warp issues S = Q K^T into tensor memory and, once the softmax
//     warps have written the probabilities over it as 16-bit values, O += P V
//     with P read from tensor memory;
//   * four softmax warps a tile, one row a thread, keep the row's running
//     maximum and sum.  O is rescaled in place only when a row's maximum has
//     grown by more than 2^8 since its last scale, so rarely.
//
// The softmax warps bound the kernel: an exponential with its scaling, sum and
// conversion takes a scheduler about 9 cycles with two warps on it, 8 of them
// the special-function unit (a polynomial on the FMA pipe takes as long: a
// packed FMA of two values issues in two cycles), so 1,180 cycles for 128 rows
// x 128 keys, against 8 D = 1,024 cycles of products at 128 channels.
//
// Up to 64 channels one CTA works on one tile and two CTAs share an SM; blocks
// of 64 keys, three S buffers, so that the softmax warps run back to back.
// Up to 128 channels one CTA works on two tiles that share K and V (a single
// tile would ask the L2 for 64 bytes a cycle and SM); tensor memory then holds
// one S a tile, and the tiles take turns: one's products run under the
// other's softmax.  Blocks of 128 keys: with two S buffers of 64 keys instead
// the products of 64 columns became the bound (16,384 causal tokens, 16 heads
// of 128, the same call repeated: 1.13 ms against 0.99-1.08 ms).
//
// Measured among calls on other inputs: 16,384 causal tokens, 16 heads of 128
// on 4 key heads, bf16: 1.09-1.11 ms, 990-1,010 TFLOP/s; 128 images of 393-785
// tokens, 6 heads of 64, fp16: 0.185-0.19 ms; 64 tokens against caches of 700 to
// 8,192, 32 heads on 8 of 128: 0.24-0.256 ms, 5.0-5.3 TB/s of the cache in use
// (0.228 ms, 5.6 TB/s, repeated on one input).
//
// With few rows and many keys (SPLIT) the keys are divided over grid.y, and
// within a CTA of two tile slots the blocks alternate between the slots; the
// parts are joined by a second kernel in a fixed order.
#include <algorithm>

#include "packed_tc.cuh"

namespace mn {
namespace pk {

constexpr float kRescaleLog2 = 8.0f;  // growth of a row's maximum before O is rescaled

template <int DT, bool BIAS>
struct Fwd {
  static constexpr int NQ = DT == 64 ? 1 : 2;     // tile slots of a CTA
  static constexpr int KB = DT == 64 ? 64 : 128;  // keys of a block
  static constexpr int NS = DT == 64 ? 3 : 1;     // S buffers of a slot
  static constexpr int kHalves = DT / 64;
  static constexpr int kStages = DT == 64 ? 10 : (BIAS ? 4 : 5);  // ring: K and V tiles of the blocks in turn
  static_assert(kStages >= 2 * NQ * NS, "S runs NS blocks of a slot ahead");
  // Four softmax warps a slot, the MMA and the load warp.  A softmax thread
  // holds a row's scores; with 128 of them it takes registers from a third
  // group of four warps, two of them idle.  The shares stay within what the
  // CTA was launched with.
  static constexpr bool kExchange = KB == 128;
  static constexpr int kThreads = kExchange ? 128 * (NQ + 1) : 32 * (4 * NQ + 2);
  static constexpr int kLaunchRegs = kExchange ? 168 : 0, kMore = 208, kLess = 80;
  static_assert(!kExchange || NQ * kMore + kLess <= (NQ + 1) * kLaunchRegs, "register exchange");
  static constexpr uint32_t kTile = kHalves * kHalfBytes, kKVHalf = KB * 128, kKV = kHalves * kKVHalf;
  static constexpr uint32_t kQ = 0, kRing = NQ * kTile, kBars = kRing + kStages * kKV;
  // barriers: Q landed; ring stages full, empty; per slot and S buffer S
  // ready, P ready (by 64 keys), the last P V done; drain
  static constexpr int kParts = KB / 64;
  static constexpr int bQ = 0, bFull = 1, bEmpty = bFull + kStages, bS = bEmpty + kStages, bP = bS + NQ * NS,
                       bPV = bP + NQ * NS * kParts, bDrain = bPV + NQ * NS, kNumBars = bDrain + 1;
  static constexpr uint32_t kMisc = kBars + ((kNumBars * 8 + 15) / 16) * 16;  // TMEM base, sequence
  static constexpr uint32_t kLut = kMisc + 32;
  // Bias: a value per distance and head.  Up to 64 channels with a margin on
  // both sides, so that a warp whose block touches the distances held needs no
  // clamp (forward over 32 images with a bias of 32 buckets: 60 -> 56 us); at 128
  // channels there is no room for it.
  static constexpr int margin(int group) { return DT == 64 ? KB + 32 / group + 1 : 0; }
  static constexpr uint32_t bytes(int group, int span) { return kLut + (BIAS ? group * (span + 2 * margin(group)) * 4 : 0) + 1024; }
  // TMEM columns: the slots' S buffers, then their O
  static constexpr uint32_t kCols = DT == 64 ? 256 : 512, cO = NQ * NS * KB;
  static_assert(cO + NQ * DT <= kCols, "tensor memory");
};

struct FwdParams {
  mn_packed_args a;
  int group, ntok;          // heads to a key head, tokens to a tile
  int span, reach;          // bias: distances held, offset of distance 0
  int splits;               // grid.y
  int ranked;               // tiles in descending order of their keys
  float* part_o;            // [part][kv_heads][tq * group][head_dim]
  float* part_lse;          // [part][kv_heads][tq * group]
  int* err;
};

template <typename ET, int DT, bool BIAS, bool SPLIT>
__global__ void __launch_bounds__(Fwd<DT, BIAS>::kThreads, DT == 64 ? 2 : 1)
    forward_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ FwdParams p,
                   const __grid_constant__ Borders bo) {
  using F = Fwd<DT, BIAS>;
  constexpr int NQ = F::NQ, NS = F::NS, ST = F::kStages, HV = F::kHalves, kKeys = F::KB;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + F::kBars);
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(base + F::kMisc);
  float* lut = reinterpret_cast<float*>(base + F::kLut);
  const mn_packed_args& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hk = blockIdx.x % a.kv_heads, slot_id = blockIdx.x / a.kv_heads;
  const int tile_tokens = SPLIT ? p.ntok : NQ * p.ntok;  // SPLIT: both slots work on one tile
  const int G = p.group;
  const int margin = BIAS ? F::margin(G) : 0, row_len = p.span + 2 * margin;

  if (warp == 0) tc::tmem_alloc(const_cast<uint32_t*>(misc), F::kCols);
  if (warp == 1) {
    put_found(misc + 1, SPLIT && p.ranked ? ranked_slot<false>(a, tile_tokens, slot_id) : seq_of_slot<false>(a, tile_tokens, slot_id));
    if (blockIdx.x == 0 && blockIdx.y == 0 && p.err &&
        bad_lengths(a.cu_q, a.cu_k, a.len_k, a.nseq, a.tq, a.tk, lane, 32))
      atomicOr(p.err, MN_STATUS_BAD_LENGTHS);
  }
  if (warp == 2 && lane == 0) {
    for (int i = 0; i < F::kNumBars; ++i)
      tc::mbar_init(bars + i, i >= F::bP && i < F::bPV ? 4 : 1);  // the softmax warps' arrivals
    tc::fence_mbar_init();
  }
  if (warp == 3 && lane == 0) {
    tma::prefetch_map(&tm_q);
    tma::prefetch_map(&tm_k);
    tma::prefetch_map(&tm_v);
  }
  if (BIAS)
    for (int i = tid; i < G * row_len; i += F::kThreads) {
      const int g = i / row_len, r = i % row_len - margin - p.reach;
      lut[i] = table_value(a, bucket_of(bo, r), hk * G + g);
    }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = misc[0];
  const Found found = get_found(misc + 1);
  const Seq& s = found.s;
  const int tiles = (s.nq + tile_tokens - 1) / tile_tokens, local = found.local;
  const bool present = local >= 0 && local < tiles;
  // the last tiles see the most keys under a causal mask: they go first
  const int t0 = present ? (a.causal ? tiles - 1 - local : local) * tile_tokens : 0;
  const int shift = s.nk - s.nq;  // position of query 0

  // key blocks of slot i: [0, end[i]) in whole, [j0, j1) of this split
  int end[NQ], tok[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    tok[i] = SPLIT ? t0 : t0 + i * p.ntok;
    const int last = min(s.nq, tok[i] + p.ntok) - 1;  // last token of the tile
    const int keys = a.causal ? min(s.nk, last + shift + 1) : s.nk;
    end[i] = present && last >= tok[i] && keys > 0 ? (keys + kKeys - 1) / kKeys : 0;
  }
  const int nblk = max(end[0], end[NQ - 1]);
  const int j0 = SPLIT ? (int)((int64_t)nblk * blockIdx.y / p.splits) : 0;
  const int j1 = SPLIT ? (int)((int64_t)nblk * (blockIdx.y + 1) / p.splits) : nblk;
  // slot i takes block j?  its first block, and the one after j
  auto takes = [&](int i, int j) { return SPLIT ? (NQ == 1 || ((j - j0) & 1) == i) : j < end[i]; };
  auto first_of = [&](int i) { return SPLIT ? j0 + (NQ == 1 ? 0 : i) : j0; };
  constexpr int kStep = SPLIT ? NQ : 1;
  auto end_of = [&](int i) { return SPLIT ? j1 : end[i]; };
  auto last_user = [&](int j) {  // the highest slot that takes block j
    return SPLIT ? (NQ == 1 ? 0 : (j - j0) & 1) : (NQ > 1 && j < end[NQ - 1] ? NQ - 1 : 0);
  };
  constexpr int ab_bf16 = std::is_same<ET, __nv_bfloat16>::value ? 1 : 0;
  constexpr bool kCommitV = DT == 64 || SPLIT;  // a V tile is freed by P V's own commit
  bool ok = true;

  if (warp >= 4 * NQ) {
    if (F::kExchange) regs_give<F::kLess>();
    if (warp == 4 * NQ + 1) {
      // ---------------------------------------------------------------- loads
      if (lane == 0 && j1 > j0) {
        int nq_tiles = 0;
        for (int i = 0; i < (SPLIT ? 1 : NQ); ++i) nq_tiles += end[i] > 0 || i == 0;
        tma::expect_tx(bars + F::bQ, (uint32_t)nq_tiles * HV * 128u * (uint32_t)(G * p.ntok));
        for (int i = 0; i < nq_tiles; ++i)
          for (int h = 0; h < HV; ++h)
            tma::load_4d(tc::smem_u32(base + F::kQ + i * F::kTile + h * kHalfBytes), &tm_q, h * 64, 0, hk, s.q0 + tok[i],
                         bars + F::bQ);
        int n = 0;  // tiles loaded: K(j0), V(j0), K(j0 + 1), ...
        for (; n < 2 * (j1 - j0) && ok; ++n) {
          const int st = n % ST;
          if (n >= ST && !(ok = wait(bars + F::bEmpty + st, (n / ST - 1) & 1, p.err))) break;
          tma::expect_tx(bars + F::bFull + st, F::kKV);
          for (int h = 0; h < HV; ++h)
            load_3d(tc::smem_u32(base + F::kRing + st * F::kKV + h * F::kKVHalf), (n & 1) ? &tm_v : &tm_k, h * 64, hk,
                    s.k0 + (j0 + n / 2) * kKeys, bars + F::bFull + st);
        }
        if (!ok && p.err) atomicOr(p.err, MN_STATUS_TC_TIMEOUT);
        // every copy issued has landed before the CTA may release its shared memory
        wait(bars + F::bQ, 0, nullptr);
        for (int m = max(0, n - ST); m < n; ++m) wait(bars + F::bFull + m % ST, (m / ST) & 1, nullptr);
      }
      __syncwarp();
    } else if (warp == 4 * NQ) {
      // ----------------------------------------------------------------- MMAs
      // S(c + NS) goes into the buffer of P(c) right behind P V(c): the products
      // of a CTA run in the order of issue, so P(c) has been read by then
      constexpr uint32_t idesc_o = tc::idesc_f16(ab_bf16, 1, 128, DT);
      int done[NQ];  // blocks of the slot so far
#pragma unroll
      for (int i = 0; i < NQ; ++i) done[i] = 0;
      auto cols_of = [&](int j) { return min(kKeys, (s.nk - j * kKeys + 31) & ~31); };  // keys of block j, in 32s
      auto s_cols = [&](int i, int c) { return tmem + (uint32_t)(i * NS + c % NS) * kKeys; };
      auto issue_s = [&](int i, int j, int c) -> bool {  // c: the slot's count of block j
        const int n = 2 * (j - j0);
        if (!wait(bars + F::bFull + n % ST, (n / ST) & 1, p.err)) return false;
        const uint64_t dq = tc::sw128_desc(tc::smem_u32(base + F::kQ + (SPLIT ? 0 : i) * F::kTile), 16);
        const uint64_t dk = tc::sw128_desc(tc::smem_u32(base + F::kRing + (n % ST) * F::kKV), 16);
        const uint32_t idesc_s = tc::idesc_f16(ab_bf16, 0, 128, cols_of(j)), d = s_cols(i, c);
        if (elect_one()) {
          tc::fence_after_sync();
#pragma unroll
          for (int kk = 0; kk < DT / 16; ++kk)
            tc::mma_f16_ss(d, dq + (kk >> 2) * (kHalfBytes >> 4) + 2 * (kk & 3), dk + (kk >> 2) * (F::kKVHalf >> 4) + 2 * (kk & 3),
                           idesc_s, kk > 0 ? 1u : 0u);
          tc::mma_commit(bars + F::bS + i * NS + c % NS);
        }
        __syncwarp();
        return true;
      };
      auto issue_pv = [&](int i, int j, int c) -> bool {
        const int n = 2 * (j - j0) + 1, cols = cols_of(j);
        if (!wait(bars + F::bFull + n % ST, (n / ST) & 1, p.err)) return false;
        uint8_t* v = base + F::kRing + (n % ST) * F::kKV;
        if (s.nk - j * kKeys < cols && (SPLIT || i == 0 || j >= end[0])) zero_rows(v, s.nk - j * kKeys, cols, HV, F::kKVHalf);
        const uint64_t dv = tc::sw128_desc(tc::smem_u32(v), F::kKVHalf);
        const uint32_t t_o = tmem + F::cO + i * DT, t_p = s_cols(i, c);
#pragma unroll
        for (int part = 0; part < F::kParts; ++part) {  // 64 keys while the softmax works on the next
          if (!wait(bars + F::bP + (i * NS + c % NS) * F::kParts + part, (c / NS) & 1, p.err)) return false;
          if (elect_one()) {
            tc::fence_after_sync();
#pragma unroll
            for (int kk = part * 4; kk < part * 4 + 4; ++kk)
              if (kk * 16 < cols) tc::mma_f16_ts(t_o, t_p + kk * 8, dv + 128 * kk, idesc_o, (c > 0 || kk > 0) ? 1u : 0u);
            // a commit takes its thread some 200 cycles: where the products bound the
            // kernel only the one that no S behind it replaces
            if (kCommitV && part == F::kParts - 1 && i == last_user(j)) tc::mma_commit(bars + F::bEmpty + n % ST);
            if (part == F::kParts - 1 && j + NS * kStep >= end_of(i)) tc::mma_commit(bars + F::bPV + i * NS + c % NS);
          }
          __syncwarp();
        }
        return true;
      };
      if (j1 > j0) {
        ok = wait(bars + F::bQ, 0, p.err);
#pragma unroll
        for (int c = 0; c < NS; ++c)
#pragma unroll
          for (int i = 0; i < NQ; ++i)
            if (ok && first_of(i) + c * kStep < end_of(i)) ok = issue_s(i, first_of(i) + c * kStep, c);
        for (int j = j0; j < j1 && ok; ++j) {
#pragma unroll
          for (int i = 0; i < NQ; ++i) {
            if (!ok || !takes(i, j)) continue;
            const int c = done[i]++;
            ok = issue_pv(i, j, c);
            if (ok && j + NS * kStep < end_of(i)) ok = issue_s(i, j + NS * kStep, c + NS);
          }
        }
        if (!ok && lane == 0 && p.err) atomicOr(p.err, MN_STATUS_TC_TIMEOUT);
        if (elect_one()) {  // every MMA issued has completed before the CTA may release its memory
          tc::mma_commit(bars + F::bDrain);
          wait(bars + F::bDrain, 0, nullptr);
        }
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------- softmax
    if (F::kExchange) regs_take<F::kMore>();
    const int i = warp >> 2, wq = warp & 3;
    const int r = wq * 32 + lane;
    const uint32_t lane_sel = (uint32_t)(wq * 32) << 16;
    const uint32_t t_o = tmem + F::cO + i * DT + lane_sel;
    const float sl2 = a.scale * kLog2e;  // scores enter the softmax in log2 units
    const int my = tok[i] + r / G, g = r % G;
    const bool mine = present && r < G * p.ntok && my < s.nq;  // a row of the sequence
    const int pos = my + shift;
    const int klim = a.causal && mine ? min(s.nk, pos + 1) : s.nk;  // keys this row sees
    const bool live = __any_sync(MN_FULL_MASK, mine);
    const int kmin = __reduce_min_sync(MN_FULL_MASK, klim), kmax = __reduce_max_sync(MN_FULL_MASK, mine ? klim : 0);
    const int pmin = __reduce_min_sync(MN_FULL_MASK, mine ? pos : 0x7fffffff);
    const int pmax = __reduce_max_sync(MN_FULL_MASK, mine ? pos : -0x7fffffff);
    const float* row_lut = lut + (BIAS ? (mine ? g : 0) * row_len : 0);
    float m_run = -INFINITY, l_run = 0.f;
    int c = 0;
    const int total = first_of(i) < end_of(i) ? (end_of(i) - first_of(i) + kStep - 1) / kStep : 0;
    // P V of the slot's block b has completed: S(b + NS) is behind it, or its own commit
    auto pv_done = [&](int b) {
      return b + NS < total ? wait(bars + F::bS + i * NS + b % NS, (b / NS + 1) & 1, p.err)
                            : wait(bars + F::bPV + i * NS + b % NS, 0, p.err);
    };
    for (int j = first_of(i); j < end_of(i) && ok; j += kStep, ++c) {
      const int buf = c % NS;
      const uint32_t t_s = tmem + (uint32_t)(i * NS + buf) * kKeys + lane_sel;
      if (!(ok = wait(bars + F::bS + i * NS + buf, (c / NS) & 1, p.err))) break;
      // S(j) is there: K(j) has been read, and V of the block whose P V came before S(j)
      if (wq == 0 && lane == 0) {
        const int jp = j - NS * kStep;
        if (i == last_user(j)) tma::arrive(bars + F::bEmpty + (2 * (j - j0)) % ST);
        if (!kCommitV && c >= NS && i == last_user(jp)) tma::arrive(bars + F::bEmpty + (2 * (jp - j0) + 1) % ST);
      }
      tc::fence_after_sync();
      const int k0 = j * kKeys;
      const int nch = (min(kKeys, s.nk - k0) + 31) >> 5;          // chunks of 32 columns that S and P hold
      const bool fast = nch == kKeys / 32 && kmin >= k0 + kKeys;  // the warp's rows see the whole block
      float f = sl2, add = 0.f;                                   // x enters the softmax as f x + add
      float x[kKeys], mx = -INFINITY;
      if (__builtin_expect(fast, 1)) {
        if (live) {
          tc::tmem_ld32_nowait(t_s, x);
          tc::tmem_ld32_nowait(t_s + 32, x + 32);
          tc::tmem_ld_wait<64>(x);
          if constexpr (kKeys == 128) {
            tc::tmem_ld32_nowait(t_s + 64, x + 64);
            tc::tmem_ld32_nowait(t_s + 96, x + 96);
            if (!BIAS) mx = max32(x + 32, max32(x, mx));
            tc::tmem_ld_wait<64>(x + 64);
          }
        }
      } else if (live) {
        const int wch = min(nch, max(0, (kmax - k0 + 31) >> 5));  // chunks that some row of the warp sees
#pragma unroll
        for (int u = 0; u < kKeys / 32; ++u)
          if (u < wch) tc::tmem_ld32_nowait(t_s + u * 32, x + u * 32);
        tc::tmem_ld_wait<kKeys>(x);
      }
      if (live) {
        if (BIAS) {
          const int lo = k0 - pmax, hi = k0 + kKeys - 1 - pmin;  // distances of the warp's rows
          if (hi <= -p.reach) {
            add = row_lut[0];
          } else if (lo >= p.span - 1 - p.reach) {
            add = row_lut[row_len - 1];
          } else {
            const int at = k0 - (mine ? pos : pmin) + p.reach + margin;
#pragma unroll
            for (int e = 0; e < kKeys; ++e) x[e] = fmaf(x[e], sl2, row_lut[DT == 64 ? at + e : min(max(at + e, 0), p.span - 1)]);
            f = 1.f;
          }
        }
        if (__builtin_expect(!fast, 0)) {  // hidden keys get exactly 0
#pragma unroll
          for (int e = 0; e < kKeys; ++e)
            if (k0 + e >= klim) x[e] = -INFINITY;
        }
        if (kKeys == 64 || BIAS || !fast) mx = max32(x + 32, max32(x, mx));
        if constexpr (kKeys == 128) mx = max32(x + 96, max32(x + 64, mx));
        const float m_new = fmaxf(m_run, fmaf(mx, f, add));
        const bool up = m_new - m_run > kRescaleLog2;  // the first keys of a row included
        const bool big = mine && is_big(m_new);
        if (__builtin_expect(__any_sync(MN_FULL_MASK, (c > 0 && up) || big), 0)) {
          // rescale the running output rows, at rest once P V of the block before has completed
          if (c > 0 && __any_sync(MN_FULL_MASK, up)) {
            if (!(ok = pv_done(c - 1))) break;
            tc::fence_after_sync();
            const float corr = up ? ex2(m_run - m_new) : 1.f;
            l_run *= corr;
            float o[32];
#pragma unroll
            for (int u = 0; u < DT / 32; ++u) {
              tc::tmem_ld32(t_o + u * 32, o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] *= corr;
              tc::tmem_st32(t_o + u * 32, o);
            }
          }
          if (__any_sync(MN_FULL_MASK, big)) {
#pragma unroll
            for (int e = 0; e < kKeys; ++e) x[e] = fmaf(x[e], f, add);
            f = 1.f;
            add = 0.f;
          }
        }
        if (up) m_run = m_new;
      }
      const float nm1 = add - (m_run == -INFINITY ? 0.f : m_run);
      const float2 nm = make_float2(nm1, nm1), f2 = make_float2(f, f);
      float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int part = 0; part < F::kParts; ++part) {
        if (live) {
#pragma unroll
          for (int u = part * 2; u < part * 2 + 2; ++u) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 y = ffma2(make_float2(x[u * 32 + 2 * e], x[u * 32 + 2 * e + 1]), f2, nm);
              const float2 q = make_float2(ex2(y.x), ex2(y.y));
              sum2[e & 1] = fadd2(sum2[e & 1], q);
              pk[e] = pack2<ET>(q.x, q.y);
            }
            tc::tmem_st16_nowait(t_s + u * 16, pk);
          }
          tc::tmem_wait_st();
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tma::arrive(bars + F::bP + (i * NS + buf) * F::kParts + part);
      }
      const float2 ss = fadd2(sum2[0], sum2[1]);
      l_run += ss.x + ss.y;
    }
    if (!ok && lane == 0 && p.err) atomicOr(p.err, MN_STATUS_TC_TIMEOUT);
    if (ok && c > 0) {
      ok = pv_done(c - 1);
      tc::fence_after_sync();
    }
    if (ok && live) {
      const float inv = l_run == 0.f ? 0.f : 1.f / l_run;  // NaN stays
      const int64_t row = (int64_t)(s.q0 + my) * G + g;     // packed row of the key head
      const int part = SPLIT ? blockIdx.y * NQ + i : 0;
      const int64_t rows = (int64_t)a.tq * G;
#pragma unroll
      for (int u = 0; u < DT / 32; ++u) {
        float o[32];
        if (c > 0) {
          tc::tmem_ld32(t_o + u * 32, o);  // the whole warp takes part
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (mine && SPLIT && c > 0) {
          float4* dst = reinterpret_cast<float4*>(p.part_o + ((part * a.kv_heads + hk) * rows + row) * a.head_dim + u * 32);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (u * 32 + 4 * e < a.head_dim)
              dst[e] = make_float4(o[4 * e] * inv, o[4 * e + 1] * inv, o[4 * e + 2] * inv, o[4 * e + 3] * inv);
        }
        if (mine && !SPLIT)
          store32<ET>(static_cast<ET*>(a.out) + ((int64_t)(s.q0 + my) * a.heads + hk * G + g) * a.head_dim, u * 32, a.head_dim,
                      o, inv);
        __syncwarp();
      }
      if (mine) {
        if (SPLIT)
          p.part_lse[(part * a.kv_heads + hk) * rows + row] = l_run == 0.f ? -INFINITY : m_run + log2f(l_run);
        else if (a.lse)
          a.lse[hk * rows + row] = l_run == 0.f ? INFINITY : m_run + log2f(l_run);
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, F::kCols);
  }
}

// out = sum over the parts of 2^(lse_i - max) out_i over the sum of those
// weights; one block a row.  Its warps take the parts in turn and their sums
// are added in order.
constexpr int kJoinWarps = 8;
template <typename ET>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ mn_packed_args a, int parts,
                                                               const float* __restrict__ part_o,
                                                               const float* __restrict__ part_lse) {
  __shared__ float4 sums[kJoinWarps][32];
  __shared__ float totals[kJoinWarps];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5, G = a.heads / a.kv_heads;
  const int64_t rows = (int64_t)a.tq * G, all = rows * a.kv_heads, at = blockIdx.x;
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 32) m = fmaxf(m, part_lse[i * all + at]);
  m = warp_max(m);
  const int c = lane * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float total = 0.f;
#pragma unroll 4
  for (int i = w; i < parts; i += nw) {
    const float lse = part_lse[i * all + at];
    // a part without keys has no weight and wrote no output; NaN stays
    const float f = lse == -INFINITY ? 0.f : m == -INFINITY ? 1.f : ex2(lse - m);
    total += f;
    if (c < a.head_dim && f != 0.f) {
      const float4 o = *reinterpret_cast<const float4*>(part_o + (i * all + at) * a.head_dim + c);
      acc.x += f * o.x; acc.y += f * o.y; acc.z += f * o.z; acc.w += f * o.w;
    }
  }
  if (nw > 1) {
    sums[w][lane] = acc;
    if (lane == 0) totals[w] = total;
    __syncthreads();
    if (w > 0) return;
    for (int i = 1; i < nw; ++i) {
      const float4 o = sums[i][lane];
      acc.x += o.x; acc.y += o.y; acc.z += o.z; acc.w += o.w;
      total += totals[i];
    }
  }
  const int hk = (int)(at / rows);
  const int64_t row = at % rows, t = row / G, g = row % G;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (c < a.head_dim)
    *reinterpret_cast<uint2*>(static_cast<ET*>(a.out) + (t * a.heads + hk * G + g) * a.head_dim + c) =
        make_uint2(pack2<ET>(acc.x * inv, acc.y * inv), pack2<ET>(acc.z * inv, acc.w * inv));
  if (a.lse && lane == 0) a.lse[at] = total == 0.f ? INFINITY : m + log2f(total);
}

int check(const mn_packed_args* a, Borders* bo, bool backward) {
  if (!a || a->nseq < 1 || a->tq < 0 || a->tk < 0 || a->heads < 1 || a->kv_heads < 1) return MN_ERR_ARG;
  if (a->heads % a->kv_heads || a->head_dim < 1 || !(a->scale > 0.f) || !(a->scale <= 0x1p127f)) return MN_ERR_ARG;
  if (!a->cu_q || !a->cu_k || (a->tq > 0 && (!a->q || !a->out)) || (a->tk > 0 && (!a->k || !a->v))) return MN_ERR_ARG;
  if (backward && a->tq > 0 && (!a->dout || !a->lse || !a->dq)) return MN_ERR_ARG;
  if (backward && a->tk > 0 && (!a->dk || !a->dv)) return MN_ERR_ARG;
  if (a->dtype != MN_F16 && a->dtype != MN_BF16) return MN_ERR_UNSUPPORTED;
  const int g = a->heads / a->kv_heads;
  if (a->head_dim > 128 || a->head_dim % 8 || g > 128 || a->kv_heads > 65535) return MN_ERR_UNSUPPORTED;
  if ((int64_t)a->tq * g >= (1 << 30) || (int64_t)a->tk * g >= (1 << 30)) return MN_ERR_UNSUPPORTED;
  // grids of a block a row and head, and of the tiles of either side, at most
  if ((int64_t)a->tq * a->heads > 0x7fffffff) return MN_ERR_UNSUPPORTED;
  if (std::max(tile_slots(a->tq, a->nseq, 128 / g), tile_slots(a->tk, a->nseq, 128)) * a->kv_heads > 0x7fffffff)
    return MN_ERR_UNSUPPORTED;
  if (!rows_ok(a->q, a->q_st, a->q_sh, a->tq, a->heads, g) || !rows_ok(a->k, a->k_st, a->k_sh, a->tk, a->kv_heads, 1) ||
      !rows_ok(a->v, a->v_st, a->v_sh, a->tk, a->kv_heads, 1) ||
      (backward && !rows_ok(a->dout, a->do_st, a->do_sh, a->tq, a->heads, g)))
    return MN_ERR_UNSUPPORTED;
  if (!aligned({a->out}) || (backward && !aligned({a->dq, a->dk, a->dv}))) return MN_ERR_UNSUPPORTED;
  bo->n = 0;
  if (a->bias_table) {
    if (a->bias_dtype < 0 || a->bias_dtype > 2 || (backward && !a->dbias)) return MN_ERR_ARG;
    if (!make_borders(bo, a->buckets, a->two_sided, a->num_borders, a->borders)) return MN_ERR_ARG;
    const int last = bo->n ? bo->at[bo->n - 1] : 1;
    if (g > 16 || a->buckets > 48 || ((a->two_sided ? 2 : 1) * (int64_t)last + 1) * g > 8192) return MN_ERR_UNSUPPORTED;
  }
  return MN_OK;
}

// How the call is divided: 0 parts means whole rows.
struct Plan {
  int ntok, parts, splits, ranked;
};
static Plan plan_of(const mn_packed_args* a) {
  const int g = a->heads / a->kv_heads, slots = a->head_dim <= 64 ? 1 : 2;
  Plan pl{128 / g, 0, 1, 0};
  // Tiles that have rows, at most; a call that leaves the card part empty, or
  // whose tiles are mostly empty rows, and whose sequences are long on average
  // is divided over the keys.
  const int64_t tiles = ((int64_t)a->tq / pl.ntok + a->nseq) * a->kv_heads;
  const int64_t ctas = (int64_t)sm_count() * (slots == 1 ? 2 : 1);
  const int64_t blocks = a->tk / a->nseq / 128;
  if (blocks >= 4 && (tiles <= ctas || (int64_t)a->tq * g <= (int64_t)a->nseq * 64)) {
    // the division whose waves of CTAs end first; a CTA's start and end take
    // it about as long as four blocks of 128 keys, joining the parts as six
    double best = 0;
    for (int64_t n = 1; n <= 64 && (n == 1 || n * 2 * slots <= blocks); ++n) {
      const double cost = (double)((tiles * n + ctas - 1) / ctas) * ((double)blocks / n + 4) + (n * slots > 1 ? 6 : 0);
      if (n == 1 || cost < best) {
        best = cost;
        pl.splits = (int)n;
      }
    }
    if (pl.splits * slots > 1) pl.parts = pl.splits * slots;
    pl.ranked = a->nseq > 1 && a->nseq <= kRanked && tiles * pl.splits > ctas;  // more than a wave
  }
  return pl;
}
static size_t part_bytes(const mn_packed_args* a, const Plan& pl) {
  return (size_t)pl.parts * a->tq * a->heads * (a->head_dim + 1) * 4;
}

template <typename ET, int DT, bool BIAS, bool SPLIT>
static bool launch(const mn_packed_args* a, const Borders& bo, const Plan& pl, void* ws, int* err, cudaStream_t st) {
  using F = Fwd<DT, BIAS>;
  constexpr bool bf16 = std::is_same<ET, __nv_bfloat16>::value;
  CUtensorMap mq, mk, mv;
  if (!bind_context()) return false;
  if (!map_q(&mq, bf16, a->q, a->q_st, a->q_sh, a->tq, a->heads, a->kv_heads, a->head_dim, pl.ntok)) return false;
  if (!map_k(&mk, bf16, a->tk ? a->k : a->q, a->k_st, a->k_sh, std::max(a->tk, 1), a->kv_heads, a->head_dim, F::KB)) return false;
  if (!map_k(&mv, bf16, a->tk ? a->v : a->q, a->v_st, a->v_sh, std::max(a->tk, 1), a->kv_heads, a->head_dim, F::KB)) return false;
  FwdParams p;
  p.a = *a;
  p.group = a->heads / a->kv_heads;
  p.ntok = pl.ntok;
  p.splits = pl.splits;
  p.ranked = pl.ranked;
  p.span = p.reach = 0;
  if (BIAS) {
    const int last = bo.n ? bo.at[bo.n - 1] : 1;
    p.reach = last;
    p.span = (bo.two_sided ? 2 : 1) * last + 1;
  }
  p.part_o = static_cast<float*>(ws);
  p.part_lse = p.part_o + (size_t)pl.parts * a->tq * a->heads * a->head_dim;
  p.err = err;
  const size_t smem = F::bytes(p.group, p.span);
  auto kern = forward_kernel<ET, DT, BIAS, SPLIT>;
  if (!ensure_smem(kern, smem) || !launch_regs(kern, F::kLaunchRegs)) return false;
  const int64_t slots = tile_slots(a->tq, a->nseq, SPLIT ? pl.ntok : F::NQ * pl.ntok) * a->kv_heads;
  kern<<<dim3((unsigned)slots, pl.splits), F::kThreads, smem, st>>>(mq, mk, mv, p, bo);
  if (SPLIT) {
    const int64_t rows = (int64_t)a->tq * a->heads;
    join_kernel<ET><<<(unsigned)rows, 32 * std::min(kJoinWarps, (pl.parts + 3) / 4), 0, st>>>(*a, pl.parts, p.part_o, p.part_lse);
  }
  return true;
}

template <typename ET, int DT>
static bool launch_d(const mn_packed_args* a, const Borders& bo, const Plan& pl, void* ws, int* err, cudaStream_t st) {
  if (a->bias_table)
    return pl.parts ? launch<ET, DT, true, true>(a, bo, pl, ws, err, st) : launch<ET, DT, true, false>(a, bo, pl, ws, err, st);
  return pl.parts ? launch<ET, DT, false, true>(a, bo, pl, ws, err, st) : launch<ET, DT, false, false>(a, bo, pl, ws, err, st);
}

}  // namespace pk
}  // namespace mn

using namespace mn;

extern "C" size_t mn_packed_attention_workspace_bytes(const mn_packed_args* a) {
  Borders bo;
  if (pk::check(a, &bo, false) != MN_OK || a->tq == 0) return 0;
  const pk::Plan pl = pk::plan_of(a);
  return pl.parts ? pk::part_bytes(a, pl) : 0;
}

extern "C" int mn_packed_attention(const mn_packed_args* a, void* workspace, size_t workspace_bytes, int* status, void* stream) {
  Borders bo;
  const int rc = pk::check(a, &bo, false);
  if (rc != MN_OK) return rc;
  if (a->tq == 0) return MN_OK;
  const pk::Plan pl = pk::plan_of(a);
  if (pl.parts && (!workspace || !pk::aligned({workspace}) || workspace_bytes < pk::part_bytes(a, pl))) return MN_ERR_WORKSPACE;
  cudaGetLastError();
  auto st = static_cast<cudaStream_t>(stream);
  bool done;
  if (a->dtype == MN_F16)
    done = a->head_dim <= 64 ? pk::launch_d<__half, 64>(a, bo, pl, workspace, status, st)
                             : pk::launch_d<__half, 128>(a, bo, pl, workspace, status, st);
  else
    done = a->head_dim <= 64 ? pk::launch_d<__nv_bfloat16, 64>(a, bo, pl, workspace, status, st)
                             : pk::launch_d<__nv_bfloat16, 128>(a, bo, pl, workspace, status, st);
  if (!done) return MN_ERR_UNSUPPORTED;
  return cudaGetLastError() == cudaSuccess ? MN_OK : MN_ERR_LAUNCH;
}
