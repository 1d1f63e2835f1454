// What the kernels of the packed attention share: the sequences' offsets and
// the bucket of a distance.
#pragma once

#include "common.cuh"

namespace mn {

constexpr int kMaxBorders = 127;

// Ascending distances at which the next bucket begins (passed by value).
struct Borders {
  int n;
  int two_sided;
  int side;  // buckets to a side
  int at[(kMaxBorders + 7) / 8 * 8];  // behind the last one: beyond every distance
};

// Bucket of r = key position - query position: the number of borders at or
// below the distance; keys ahead take the second side.
__device__ __forceinline__ int bucket_of(const Borders& b, int r) {
  const int n = b.two_sided ? abs(r) : max(-r, 0);
  int u = 0;
  for (int i = 0; i < b.n; i += 8)  // eight reads on their way at a time
#pragma unroll
    for (int e = 0; e < 8; ++e) u += b.at[i + e] <= n ? 1 : 0;
  return u + (b.two_sided && r > 0 ? b.side : 0);
}

// First and last relative position of bucket u (empty where borders coincide):
// one side's bucket k is the run of distances [at[k - 1], at[k]).
__device__ __forceinline__ int2 bucket_range(const Borders& b, int u) {
  const bool ahead = u >= b.side;
  const int k = ahead ? u - b.side : u;
  const int near = k == 0 ? 0 : b.at[k - 1], far = k < b.n ? b.at[k] - 1 : 0x3fffffff;
  if (ahead) return make_int2(max(near, 1), far);
  return make_int2(-far, k == 0 && !b.two_sided ? 0x3fffffff : -near);  // one-sided: all that is ahead as well
}

// false when the arguments describe no valid buckets
inline bool make_borders(Borders* b, int buckets, int two_sided, int num_borders, const int32_t* at) {
  b->two_sided = two_sided ? 1 : 0;
  b->side = two_sided ? buckets / 2 : buckets;
  b->n = num_borders;
  if (buckets < 1 || (two_sided && buckets % 2) || num_borders != b->side - 1 || num_borders > kMaxBorders ||
      (num_borders > 0 && !at))
    return false;
  for (int i = 0; i < num_borders; ++i) {
    if (at[i] < 1 || (i > 0 && at[i] < at[i - 1])) return false;
    b->at[i] = at[i];
  }
  for (int i = num_borders; i < (kMaxBorders + 7) / 8 * 8; ++i) b->at[i] = 0x7fffffff;
  return true;
}

// One sequence: query rows [q0, q0 + nq), key rows [k0, k0 + nk) of a slot of
// `slot` rows.  Offsets are clamped to the tensors, so that whatever they hold
// no access leaves them.
struct Seq {
  int q0, nq, k0, nk, slot;
};

// Data condition of the offsets, looked at by one thread block.
__device__ __forceinline__ bool bad_lengths(const int32_t* cu_q, const int32_t* cu_k, const int32_t* len_k, int n, int tq,
                                            int tk, int first, int step) {
  bool bad = false;
  for (int b = first; b < n; b += step) {
    const int q0 = cu_q[b], q1 = cu_q[b + 1], k0 = cu_k[b], k1 = cu_k[b + 1];
    bad |= q0 < 0 || q1 < q0 || q1 > tq || k0 < 0 || k1 < k0 || k1 > tk || (b == 0 && (q0 != 0 || k0 != 0));
    if (len_k) bad |= len_k[b] < 0 || len_k[b] > k1 - k0;
  }
  return bad;
}

}  // namespace mn
