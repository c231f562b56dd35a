// The largest of n numbers, found by one workgroup: the k-th largest first, then the places of those above it, and of the first ones that
// equal it, in their order.
//
// Up to 16384 numbers are brought to LDS once, and their first digit is counted on the way; more are read anew for every walk, eight at a time.
// Digits are counted in LDS: the first one holds the exponent and the first bits of the mantissa, behind it few numbers are left, and the
// search ends as soon as all that begin alike are wanted.  8 x 5120 numbers and a list of them: 10.7 us; 512 x 3000:
// 13.4; scores and selection of 2 x 5 x 333 times 219 numbers, by a wave each: 15.6.
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

// A wave by itself, 256 numbers at most, in registers: bit by bit from the top, how many keys are at least the candidate is a comparison and a
// population count for each 64 of them, and the search ends as soon as there are just k
struct TopFew {
  template <typename Number, typename Key, typename Take>
  __device__ __forceinline__ unsigned run(int n, unsigned k, Number number, Key key_of, Take take) {
    const int lane = threadIdx.x % 64;
    float x[4];
    unsigned u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = number(min(64 * e + lane, n - 1));
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = 64 * e + lane < n ? key_of(64 * e + lane, x[e]) : 0u;
    auto count = [&](unsigned from) __attribute__((always_inline)) -> unsigned {
      unsigned c = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) c += (unsigned)__builtin_popcountll(__builtin_amdgcn_ballot_w64(u[e] >= from));
      return c;
    };
    unsigned at = 0, equal = 0;   // taken: keys above at, and so many that equal it
    bool exact = false;
    for (unsigned bit = 0x80000000u; bit != 0 && !exact; bit >>= 1) {
      const unsigned c = count(at | bit);
      if (c >= k) at |= bit;
      exact = c == k;
    }
    if (exact) at -= 1;
    else if (at != 0) equal = at == ~0u ? k : k - count(at + 1);
    unsigned gt = 0, eq = 0;
    const uint64_t lower = (1ull << lane) - 1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool same = (u[e] == at) & (at != 0);
      const uint64_t all_gt = __builtin_amdgcn_ballot_w64(u[e] > at), all_eq = __builtin_amdgcn_ballot_w64(same);
      const unsigned my_gt = gt + (unsigned)__builtin_popcountll(all_gt & lower), my_eq = eq + (unsigned)__builtin_popcountll(all_eq & lower);
      if ((u[e] > at) | (same & (my_eq < equal))) take(my_gt + min(my_eq, equal), 64 * e + lane, x[e]);
      gt += (unsigned)__builtin_popcountll(all_gt);
      eq += (unsigned)__builtin_popcountll(all_eq);
    }
    return gt + min(eq, equal);
  }
};

// T threads, N numbers at most (0: any number of them, which stay where they are); digits of BITS bits, of which a thread counts BINS / T.  A wave's numbers lie
// side by side, 64 of them a step
template <int T, int N, int BITS> struct TopHeld {
  static constexpr int BINS = 1 << BITS, PER = BINS / T, WAVES = T / 64, AT_ONCE = N > 0 ? 4 : 8;
  static_assert(BINS % T == 0, "every thread owns some of the digit's values");
  float held[N > 0 ? N : 1];
  unsigned count[BINS];
  unsigned sums[3][WAVES];
  unsigned found[3];

  // number(i) of places i = 0 .. n - 1, n <= N, its key(i, x); take(place among the taken ones, i, x) for the k largest of those whose key is not 0 (of
  // equal ones the first), in order.  Returns how many there are.  1 <= k; n >= 1
  template <typename Number, typename Key, typename Take>
  __device__ __forceinline__ unsigned run(int n, unsigned k, Number number, Key key_of, Take take) {
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
#pragma unroll
    for (int e = 0; e < PER; ++e) count[tid + T * e] = 0;
    __syncthreads();
#pragma unroll 8
    for (int i = tid; i < n; i += T) {
      const float x = number(i);
      if constexpr (N > 0) held[i] = x;
      atomicAdd(&count[key_of(i, x) >> (32 - BITS)], 1u);
    }
    auto again = [&](int i) __attribute__((always_inline)) -> float {
      if constexpr (N > 0) return held[i];
      else return number(i);
    };
    const int steps = (n + T - 1) / T, i0 = 64 * steps * wave + lane, i1 = min(n, 64 * steps * (wave + 1));
    // ---- taken: keys above at, and so many that equal it
    unsigned at, equal = 0, need = min(k, (unsigned)n), from = 0;   // the need-th largest of those that begin as `from` does, down to bit `shift`
    for (int shift = 32 - BITS;;) {
      __syncthreads();
      // from the largest digit down; a thread's digits lie side by side
      unsigned mine = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) mine += count[BINS - 1 - (tid * PER + e)];
      const unsigned sum = wave_scan(mine);
      unsigned before = sum - mine;
      if constexpr (WAVES > 1) {
        if (lane == 63) sums[0][wave] = sum;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) before += w < wave ? sums[0][w] : 0u;
      }
      if (before < need && need <= before + mine) {   // (of one thread)
        for (int e = 0; e < PER; ++e) {
          const int digit = BINS - 1 - (tid * PER + e);
          const unsigned c = count[digit];
          if (need > before && need <= before + c) {
            found[0] = (unsigned)digit;
            found[1] = need - before;
            found[2] = c;
          }
          before += c;
        }
      }
      __syncthreads();
      from |= found[0] << shift;
      need = found[1];
      if (found[2] == need || shift == 0) {
        // all that begin like this (but what does not take part), or of those that are this
        at = from == 0 ? 0 : shift == 0 ? from : from - 1;
        equal = from == 0 || shift != 0 ? 0 : need;
        break;
      }
      const int before_shift = shift;
      shift = max(0, shift - BITS);
      const unsigned digits = (1u << (before_shift - shift)) - 1;
#pragma unroll
      for (int e = 0; e < PER; ++e) count[tid + T * e] = 0;
      __syncthreads();
#pragma unroll AT_ONCE
      for (int i = i0; i < i1; i += 64) {
        const unsigned u = key_of(i, again(i));
        if ((u >> before_shift) == (from >> before_shift)) atomicAdd(&count[(u >> shift) & digits], 1u);
      }
    }
    // ---- their places
    unsigned mine_gt = 0, mine_eq = 0;   // (each its own count: there may be more than 2^16 of both)
#pragma unroll AT_ONCE
    for (int i = i0; i < i1; i += 64) {
      const unsigned u = key_of(i, again(i));
      mine_gt += u > at ? 1u : 0u;
      mine_eq += ((u == at) & (at != 0)) ? 1u : 0u;
    }
    const unsigned wave_gt = __builtin_amdgcn_readlane((int)wave_scan(mine_gt), 63), wave_eq = __builtin_amdgcn_readlane((int)wave_scan(mine_eq), 63);
    unsigned gt = 0, eq = 0, total_gt = wave_gt, total_eq = wave_eq;
    if constexpr (WAVES > 1) {
      if (lane == 0) {
        sums[1][wave] = wave_gt;
        sums[2][wave] = wave_eq;
      }
      __syncthreads();
      total_gt = total_eq = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const unsigned g = sums[1][w], e = sums[2][w];
        gt += w < wave ? g : 0u;
        eq += w < wave ? e : 0u;
        total_gt += g;
        total_eq += e;
      }
    }
    const uint64_t lower = (1ull << lane) - 1;
    for (int first = i0 - lane; first < i1; first += 64 * AT_ONCE) {   // (some steps at once, of all lanes: one by one each would wait for its numbers)
      float x[AT_ONCE];
      unsigned u[AT_ONCE];
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) x[e] = again(min(first + 64 * e + lane, n - 1));
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) u[e] = first + 64 * e + lane < i1 ? key_of(first + 64 * e + lane, x[e]) : 0u;
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {
        const bool same = (u[e] == at) & (at != 0);
        const uint64_t all_gt = __builtin_amdgcn_ballot_w64(u[e] > at), all_eq = __builtin_amdgcn_ballot_w64(same);
        const unsigned my_gt = gt + (unsigned)__builtin_popcountll(all_gt & lower), my_eq = eq + (unsigned)__builtin_popcountll(all_eq & lower);
        if ((u[e] > at) | (same & (my_eq < equal))) take(my_gt + min(my_eq, equal), first + 64 * e + lane, x[e]);
        gt += (unsigned)__builtin_popcountll(all_gt);
        eq += (unsigned)__builtin_popcountll(all_eq);
      }
    }
    return total_gt + min(total_eq, equal);
  }
};

}  // namespace qfa
