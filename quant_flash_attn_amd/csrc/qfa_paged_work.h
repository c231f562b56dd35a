// How the keys of a batch of sequences of any lengths are dealt to a fixed number of workgroups.
//
// The lengths are on the device and the host does not wait for them (a captured graph is replayed while they grow), so the
// division is made here, by every workgroup for itself.  All tiles of keys that the call has to look at are numbered through:
// sequence by sequence, in it head by head, in it block of rows by block of rows, in it key tile by key tile.  Workgroup w
// takes the tiles [w * each, (w + 1) * each): every one the same number, whatever the lengths.  Where that cuts an item (one
// sequence, head and block of rows), the pieces' unnormalised results go to the workgroups' slots and a second kernel joins them.
//
// Rows of a sequence are its queries times the query heads that share a key head: row = query * G + head % G.
#pragma once
#include "qfa_device.h"
#include "qfa_host.h"

namespace qfa {

// One launch: the sequences' own keys, from `prefix` on (SHARED false), or the prefix that all of them share, once for the rows
// of all (SHARED true: one problem whose rows are the sequences' rows one after the other).
struct PagedWork {
  const int32_t *starts, *counts;   // counts: nullable
  int B, Hk, G, N, causal;
  int prefix, capacity;             // keys; what the page table has room for
  int grid, least;                  // workgroups; the fewest tiles that one of them takes
  float *slots, *slots_ml;          // [2 * grid][block rows][D] and (m in log2 units, l): of a piece that does not begin its item, one that does
  float *whole, *whole_ml;          // nullable: items in one piece, [problem, head, row] (null: they are normalised and stored)
};

template <bool SHARED, int BR, int TK> struct PagedDeal {
  const PagedWork &a;
  int rows, blocks, problems;       // rows and blocks of rows of a problem
  unsigned total, each;
  __device__ __forceinline__ int tokens(int p) const { return a.counts ? max(0, min(a.counts[p], a.N)) : a.N; }
  // the keys of a block of rows end here
  __device__ __forceinline__ int end(int p, int rb) const {
    if (SHARED) return min(a.prefix, a.capacity);
    const int n = tokens(p), first = rb * BR / a.G;
    if (first >= n) return 0;
    const int64_t last = a.causal ? min(((rb + 1) * BR - 1) / a.G, n - 1) : n - 1;
    return (int)max((int64_t)0, min((int64_t)a.starts[p] + last + 1, (int64_t)a.capacity));
  }
  __device__ __forceinline__ int begin() const { return SHARED ? 0 : a.prefix; }
  __device__ __forceinline__ unsigned tiles(int p, int rb) const {
    const int e = end(p, rb), b = begin();
    return e > b ? (unsigned)((e + TK - 1) / TK - b / TK) : 0u;
  }
  __device__ __forceinline__ unsigned tiles_of_problem(int p) const {   // of one head
    if (SHARED || !a.causal) return (unsigned)blocks * tiles(p, 0) - (SHARED ? 0u : missing(p));
    unsigned s = 0;
    for (int rb = 0; rb < blocks; ++rb) s += tiles(p, rb);
    return s;
  }
  // not causal: all blocks see the same keys, but for those behind the last token
  __device__ __forceinline__ unsigned missing(int p) const {
    const int n = tokens(p), with = (n * a.G + BR - 1) / BR;
    return (unsigned)(blocks - with) * tiles(p, 0);
  }
  // (every wave adds up for itself: 64 problems at a time, nothing to wait for but their lengths)
  __device__ __forceinline__ unsigned below(int p, unsigned x) const { return p < problems ? x : 0u; }
  __device__ __forceinline__ PagedDeal(const PagedWork &a_) : a(a_) {
    rows = (SHARED ? a.B : 1) * a.N * a.G;
    blocks = (rows + BR - 1) / BR;
    problems = SHARED ? 1 : a.B;
    unsigned sum = 0;
    for (int p = threadIdx.x % 64; p < problems; p += 64) sum += tiles_of_problem(p);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    total = __builtin_amdgcn_readfirstlane((int)(sum * (unsigned)a.Hk));
    each = max((unsigned)a.least, (total + a.grid - 1) / a.grid);
  }
  // Number of the first tile of an item
  __device__ __forceinline__ unsigned first_tile(int p, int h, int rb) const {
    unsigned sum = 0;
    for (int i = threadIdx.x % 64; i < p; i += 64) sum += tiles_of_problem(i);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    sum = sum * (unsigned)a.Hk + (unsigned)h * tiles_of_problem(p);
    for (int i = 0; i < rb; ++i) sum += tiles(p, i);
    return __builtin_amdgcn_readfirstlane((int)sum);
  }
  // The item that tile x < total belongs to, and which of its tiles it is
  struct Item { int p, h, rb; unsigned at; };
  __device__ __forceinline__ Item find(unsigned x) const {
    const int lane = threadIdx.x % 64;
    unsigned before = 0;
    Item it = {0, 0, 0, 0u};
    for (int base = 0; base < problems; base += 64) {
      const unsigned mine = base + lane < problems ? tiles_of_problem(base + lane) * (unsigned)a.Hk : 0u;
      unsigned sum = mine;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const unsigned y = __shfl_up(sum, off, 64);
        if (lane >= off) sum += y;
      }
      const uint64_t past = __builtin_amdgcn_ballot_w64(before + sum > x);
      if (past != 0) {
        const int l = __builtin_ctzll(past);
        it.p = base + l;
        it.at = x - before - __builtin_amdgcn_readlane((int)(sum - mine), l);
        break;
      }
      before += __builtin_amdgcn_readlane((int)sum, 63);
    }
    const unsigned per_head = __builtin_amdgcn_readfirstlane((int)tiles_of_problem(it.p));
    it.h = (int)(it.at / per_head);
    it.at -= (unsigned)it.h * per_head;
    for (unsigned t; it.rb < blocks - 1 && it.at >= (t = tiles(it.p, it.rb)); ++it.rb) it.at -= t;
    it.p = __builtin_amdgcn_readfirstlane(it.p);
    it.h = __builtin_amdgcn_readfirstlane(it.h);
    it.rb = __builtin_amdgcn_readfirstlane(it.rb);
    it.at = __builtin_amdgcn_readfirstlane((int)it.at);
    return it;
  }
  // the next item that has tiles (there is one)
  __device__ __forceinline__ void next(Item &it) const {
    it.at = 0;
    do {
      if (++it.rb == blocks) {
        it.rb = 0;
        if (++it.h == a.Hk) {
          it.h = 0;
          ++it.p;
        }
      }
    } while (tiles(it.p, it.rb) == 0);
  }
  // Row r of problem p: its sequence, query and query head (of key head h)
  struct Row { int b, i, qh; };
  __device__ __forceinline__ Row row(int p, int h, int r) const {
    const int per = a.N * a.G, b = SHARED ? r / per : p, in = SHARED ? r - b * per : r;
    const int i = in / a.G;
    return {b, i, h * a.G + in - i * a.G};
  }
  // The last key that a row sees (-1 and below: none)
  __device__ __forceinline__ int last_key(const Row &r) const {
    const int n = tokens(r.b);
    if (r.i >= n) return -1;
    const int64_t k = (int64_t)a.starts[r.b] + (a.causal ? r.i : n - 1);
    return (int)max((int64_t)-1, min(k, (int64_t)(SHARED ? a.prefix : a.capacity) - 1));
  }
};

}  // namespace qfa
