// The largest of n numbers, found by one workgroup: the k-th largest by counting digits from the highest down, and then one walk that hands out
// the places of those above it, and of the first ones that equal it, in their order.
#pragma once
#include "qfa_paged_work.h"

namespace qfa {

// An order-preserving 32-bit key of a float: 1 at least for every number, NaN among them below all others (-0 is 0); 0 is left for what
// does not take part, TOP_ALWAYS lies above all of them
constexpr unsigned TOP_ALWAYS = 0xffffffffu;
__device__ __forceinline__ unsigned top_key(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.0f);
  const unsigned k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return x != x ? 1u : k;
}

// T threads; digits of BITS bits, of which a thread counts BINS / T
template <int T, int BITS> struct TopSearch {
  static constexpr int BINS = 1 << BITS, PER = BINS / T, WAVES = T / 64;
  static_assert(BINS % T == 0, "every thread owns some of the digit's values");
  unsigned count[BINS];
  unsigned sums[2][WAVES];   // per wave, of two steps in turn
  unsigned found[2];

  // The k-th largest key, and how many of those that equal it are among the k largest.  1 <= k <= n; key(i): of place i, any number of times
  template <typename Key> __device__ __forceinline__ void threshold(int n, unsigned k, Key key, unsigned &at, unsigned &equal) {
    const int tid = threadIdx.x, wave = tid / 64;
    unsigned prefix = 0, mask = 0;
    for (int shift = 32 - BITS;; shift = max(0, shift - BITS)) {
      const unsigned digits = (~mask) >> shift;   // of this step, at their place
#pragma unroll
      for (int e = 0; e < PER; ++e) count[tid + T * e] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += T) {
        const unsigned u = key(i);
        if ((u & mask) == prefix) atomicAdd(&count[(u >> shift) & digits], 1u);
      }
      __syncthreads();
      // from the largest digit down; a thread's digits lie side by side
      unsigned mine = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) mine += count[BINS - 1 - (tid * PER + e)];
      const unsigned sum = wave_scan(mine);
      if (tid % 64 == 63) sums[0][wave] = sum;
      __syncthreads();
      unsigned before = sum - mine;
      for (int w = 0; w < wave; ++w) before += sums[0][w];
      if (before < k && k <= before + mine) {   // (of one thread)
        int e = 0;
        for (unsigned c; k > before + (c = count[BINS - 1 - (tid * PER + e)]); ++e) before += c;
        found[0] = (unsigned)(BINS - 1 - (tid * PER + e));
        found[1] = k - before;
      }
      __syncthreads();
      prefix |= found[0] << shift;
      k = found[1];
      mask |= digits << shift;
      if (shift == 0) break;
    }
    at = prefix;
    equal = k;
  }

  // take(place among the taken ones, i) for the keys above `at` and the first `equal` ones of those that equal it.  Returns how many were taken
  template <typename Key, typename Take> __device__ __forceinline__ unsigned walk(int n, unsigned at, unsigned equal, Key key, Take take) {
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    unsigned above = 0, same = 0;   // before this step
    int step = 0;
    for (int i0 = 0; i0 < n; i0 += T, step ^= 1) {
      const int i = i0 + tid;
      const unsigned u = i < n ? key(i) : 0u;
      const bool gt = u > at, eq = (u == at) & (i < n);
      const uint64_t all_gt = __builtin_amdgcn_ballot_w64(gt), all_eq = __builtin_amdgcn_ballot_w64(eq);
      if (lane == 0) sums[step][wave] = (unsigned)__builtin_popcountll(all_gt) << 16 | (unsigned)__builtin_popcountll(all_eq);   // (T < 2^16)
      __syncthreads();   // (the next step writes the other half: none is overwritten before all have read it)
      unsigned before = 0, total = 0;
      for (int w = 0; w < WAVES; ++w) {
        const unsigned c = sums[step][w];
        before += w < wave ? c : 0u;
        total += c;
      }
      const uint64_t lower = (1ull << lane) - 1;
      const unsigned my_gt = above + (before >> 16) + (unsigned)__builtin_popcountll(all_gt & lower);
      const unsigned my_eq = same + (before & 0xffffu) + (unsigned)__builtin_popcountll(all_eq & lower);
      if (gt | (eq & (my_eq < equal))) take(my_gt + min(my_eq, equal), i);
      above += total >> 16;
      same += total & 0xffffu;
    }
    return above + min(same, equal);
  }
};

}  // namespace qfa
