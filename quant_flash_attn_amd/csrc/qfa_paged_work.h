// How the keys of a batch of sequences of any lengths are dealt to a fixed number of workgroups.
//
// The lengths are on the device and the host does not wait for them (a captured graph is replayed while they grow), so the
// division is made here, by every workgroup for itself.  All work of the call is numbered through in units: sequence by sequence,
// in it head by head, in it block of rows by block of rows -- an item --, and of an item first a few units for its start and end,
// then one for every tile of its keys.  Workgroup w takes the units [w * each, (w + 1) * each): every one the same number, whatever
// the lengths.  Where that cuts an item, the pieces' unnormalised results go to the workgroups' slots and a second kernel joins them.
// (Without the units for an item's start, a workgroup that gets many short sequences takes several times as long as the others: a
// start costs the time of about twelve tiles of 32 keys, or four of 64 expanded ones: 8 in place of 12 1 to 4 % more, 6 in place of 4
// between 3 % less and 3 % more.)
//
// Every load that another one waits for costs about a microsecond at a workgroup's start, and so do a few thousand bytes of code
// that no cache holds yet: the lengths of 64 sequences are loaded once, a sequence in each lane, and read out of the lanes from
// there on; where an item begins is left in memory for the kernel that joins the pieces.
//
// Nothing here branches on what differs between lanes (& in place of &&, values before their selection): where the branches of some
// lanes join again the compiler has saved registers of all lanes before it turned the others back on, a thread's own index among
// them, in kernels that have none to spare.
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
  int grid;                         // workgroups (0: this launch is not made)
  int br, tk;                       // rows of a block, keys of a tile: powers of two
  int extra;                        // units of an item beside its tiles, and the fewest units that a workgroup takes
  unsigned *first;                  // [items] the unit of an item's first tile, [items] that one's units per workgroup (own keys)
  float *slots, *slots_ml;          // [2 * grid][br][D] and (m in log2 units, l): of a piece that does not begin its item, one that does
  float *whole, *whole_ml;          // nullable: items in one piece, [problem, head, row] (null: they are normalised and stored)
};

// A sequence's position of its first new token, and how many it brings
struct PagedSeq { int start, tokens; };

// inclusive sum over the wave's lanes (the last one has all of it)
__device__ __forceinline__ unsigned wave_scan(unsigned x) {
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true);   // row_shr 1, 2, 4, 8
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true);
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true);
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true);
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);  // the row before's last lane, to rows 1 and 3
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);  // the lower half's last lane, to the upper half
  return x;
}

// ONE: a problem has a single block of rows
template <bool SHARED, bool ONE> struct PagedDeal {
  static constexpr bool ONE_PROBLEM = SHARED, LIST = false;
  static __device__ __forceinline__ unsigned workgroup() { return blockIdx.x; }
  const PagedWork &a;
  const int BR, TK;                 // work.br and work.tk, constants in the kernels that are made for them
  int rows, blocks, problems;       // rows and blocks of rows of a problem
  unsigned total, each;             // units of the call, of a workgroup
  int held;                         // the 64 sequences from here on are in the lanes
  PagedSeq lanes;
  __device__ __forceinline__ PagedSeq load(int p) const {
    const int i = min(p, a.B - 1), n = a.counts ? max(0, min(a.counts[i], a.N)) : a.N;
    return {a.starts[i], n};
  }
  // sequence p, uniform over the wave
  __device__ __forceinline__ PagedSeq seq(int p) {
    if (SHARED) return {0, 0};
    if ((p & ~63) != held) {
      held = p & ~63;
      lanes = load(held + threadIdx.x % 64);
    }
    return {__builtin_amdgcn_readlane(lanes.start, p & 63), __builtin_amdgcn_readlane(lanes.tokens, p & 63)};
  }
  // the keys of a block of rows end here
  __device__ __forceinline__ int end(const PagedSeq &s, int rb) const {
    if (SHARED) return min(a.prefix, a.capacity);
    int last = s.tokens - 1;
    const bool none = last < (ONE ? 0 : rb * BR / a.G);
    if (!ONE && a.causal) last = min(((rb + 1) * BR - 1) / a.G, last);
    const int e = (int)max((int64_t)0, min((int64_t)s.start + last + 1, (int64_t)a.capacity));
    return none ? 0 : e;
  }
  __device__ __forceinline__ int begin() const { return SHARED ? 0 : a.prefix; }
  __device__ __forceinline__ unsigned tiles(const PagedSeq &s, int rb) const {
    const int e = end(s, rb), b = begin();
    const unsigned n = (unsigned)((int)(((unsigned)e + TK - 1) / TK) - b / TK);
    return e > b ? n : 0u;
  }
  __device__ __forceinline__ unsigned units(const PagedSeq &s, int rb) const {
    const unsigned n = tiles(s, rb);
    return n ? n + (unsigned)a.extra : 0u;
  }
  __device__ __forceinline__ unsigned units_of_head(const PagedSeq &s) const {
    if (ONE) return units(s, 0);
    if (SHARED) return (unsigned)blocks * units(s, 0);
    if (!a.causal) return (unsigned)((s.tokens * a.G + BR - 1) / BR) * units(s, 0);   // (all blocks with a token see the same keys)
    unsigned sum = 0;
    for (int rb = 0; rb < blocks; ++rb) sum += units(s, rb);
    return sum;
  }
  __device__ __forceinline__ void divide() { each = max((unsigned)a.extra, (total + a.grid - 1) / a.grid); }
  __device__ __forceinline__ PagedDeal(const PagedWork &a_, int br, int tk) : a(a_), BR(br), TK(tk) {
    rows = (SHARED ? a.B : 1) * a.N * a.G;
    blocks = ONE ? 1 : (rows + BR - 1) / BR;
    problems = SHARED ? 1 : a.B;
    held = 0;
    if (SHARED) {
      total = units_of_head({0, 0}) * (unsigned)a.Hk;
      divide();
    }
  }
  // An item, its sequence, which of its `tiles` tiles is the next, and the unit of its first one
  struct Item { int p, h, rb; unsigned at, tiles, first; PagedSeq s; };
  // Divides the work and finds unit blockIdx.x * each.  False: there is no such unit.  (x moves on to an item's first tile.)
  __device__ __forceinline__ bool find(unsigned &x, Item &it) {
    unsigned in = 0;   // which unit of the problem
    it.p = 0;
    it.s = {0, 0};
    if (SHARED) {
      x = blockIdx.x * each;
      if (x >= total) return false;
      in = x;
    } else {
      const int lane = threadIdx.x % 64;
      lanes = load(lane);
      // (of a sequence that there is)
      const auto units_of = [&](const PagedSeq &s, int p) __attribute__((always_inline)) -> unsigned {
        const unsigned u = units_of_head(s) * (unsigned)a.Hk;
        return p < problems ? u : 0u;
      };
      unsigned mine = units_of(lanes, lane), sum = wave_scan(mine);
      total = (unsigned)__builtin_amdgcn_readlane((int)sum, 63);
      for (int base = 64; base < problems; base += 64) {
        const unsigned u = units_of(load(base + lane), base + lane);
        total += (unsigned)__builtin_amdgcn_readlane((int)wave_scan(u), 63);
      }
      divide();
      x = blockIdx.x * each;
      if (x >= total) return false;
      unsigned before = 0;
      for (;;) {
        const uint64_t past = __builtin_amdgcn_ballot_w64(before + sum > x);
        if (past != 0) {
          const int l = __builtin_ctzll(past);
          it.p = held + l;
          in = x - before - (unsigned)__builtin_amdgcn_readlane((int)(sum - mine), l);
          break;
        }
        before += (unsigned)__builtin_amdgcn_readlane((int)sum, 63);   // (x < total: a later sequence has it)
        held += 64;
        lanes = load(held + lane);
        mine = units_of(lanes, held + lane);
        sum = wave_scan(mine);
      }
      it.s = seq(it.p);
    }
    const unsigned per_head = __builtin_amdgcn_readfirstlane((int)units_of_head(it.s));
    it.h = __builtin_amdgcn_readfirstlane((int)(in / per_head));
    in -= (unsigned)it.h * per_head;
    it.rb = 0;
    if (!ONE) {
      if (SHARED || !a.causal) {
        it.rb = (int)(in / units(it.s, 0));
        in -= (unsigned)it.rb * units(it.s, 0);
      } else {
        for (unsigned t; it.rb < blocks - 1 && in >= (t = units(it.s, it.rb)); ++it.rb) in -= t;
      }
      it.rb = __builtin_amdgcn_readfirstlane(it.rb);
    }
    in = __builtin_amdgcn_readfirstlane((int)in);
    it.tiles = __builtin_amdgcn_readfirstlane((int)tiles(it.s, it.rb));
    it.first = x - in + (unsigned)a.extra;
    if (in < (unsigned)a.extra) x = it.first;
    it.at = x - it.first;
    return x < total;
  }
  // the next item that has tiles, behind unit x where the last one ended; false: that is not this workgroup's
  __device__ __forceinline__ bool next(unsigned &x, unsigned x_end, Item &it) {
    x += (unsigned)a.extra;
    if (x >= x_end) return false;
    it.first = x;
    it.at = 0;
    do {   // (x_end is at most the last item's end: there is one)
      if (ONE || ++it.rb == blocks) {
        it.rb = 0;
        if (++it.h == a.Hk) {
          it.h = 0;
          it.s = seq(++it.p);
        }
      }
      it.tiles = __builtin_amdgcn_readfirstlane((int)tiles(it.s, it.rb));
    } while (it.tiles == 0);
    return true;
  }
  __device__ __forceinline__ int item_index(int p, int h, int rb) const { return (p * a.Hk + h) * blocks + rb; }
  // Row r of problem p: its sequence, query and query head (of key head h)
  struct Row { int b, i, qh; };
  __device__ __forceinline__ Row row(int p, int h, int r) const {
    const int per = a.N * a.G, b = SHARED ? r / per : p, in = SHARED ? r - b * per : r;
    const int i = a.N == 1 ? 0 : in / a.G;
    return {b, i, h * a.G + in - i * a.G};
  }
  // The last key that a row sees (-1 and below: none).  s: its sequence
  __device__ __forceinline__ int last_key(const Row &r, const PagedSeq &s) const {
    const int64_t k = (int64_t)s.start + (a.causal ? r.i : s.tokens - 1);
    return (int)max((int64_t)-1, min(k, (int64_t)(SHARED ? a.prefix : a.capacity) - 1));
  }
};

// Lists of blocks: a problem is a token, its rows the query heads that share a key head, and its keys the blocks of its list, which are as many
// for all tokens.  So every item has the same number of units, the host divides them, and nothing has to be noted for the kernel that joins
// the pieces.
struct PagedListDeal {
  static constexpr bool ONE_PROBLEM = false, LIST = true;
  const PagedWork &a;
  const int BR;
  int rows, blocks;
  unsigned total, each, per_item;
  typedef PagedDeal<false, false> Keys;
  typedef Keys::Row Row;
  struct Item { int p, h, rb; unsigned at, tiles, first; PagedSeq s; };
  unsigned item_tiles;
  __device__ __forceinline__ PagedListDeal(const PagedWork &a_, int br, int) : a(a_), BR(br) {
    rows = a.G;
    blocks = (rows + BR - 1) / BR;
  }
  // tiles of an item, units of a workgroup: before anything else is asked
  __device__ __forceinline__ void lists(unsigned tiles, unsigned units) {
    item_tiles = tiles;
    per_item = tiles + (unsigned)a.extra;
    each = units;
    total = (unsigned)(a.B * a.N * a.Hk * blocks) * per_item;
  }
  __device__ __forceinline__ PagedSeq seq(int p) const {
    const int b = p / a.N, n = a.counts ? max(0, min(a.counts[b], a.N)) : a.N;
    return {__builtin_amdgcn_readfirstlane(a.starts[b]), __builtin_amdgcn_readfirstlane(n)};
  }
  // Consecutive workgroups go round the 8 XCDs.  Where a sequence has several tokens, whose lists share blocks, each XCD takes an eighth of the work side by
  // side: the tokens of a key head then find each other's keys in one L2 (2 x 333 tokens, 8 key heads, 2048 keys each, with paged_rows_kernel: 352 us without, 302 with it)
  __device__ __forceinline__ unsigned workgroup() const {
    const unsigned n = gridDim.x, xcd = blockIdx.x % 8, at = blockIdx.x / 8;
    return a.N == 1 ? blockIdx.x : xcd * (n / 8) + min(xcd, n % 8) + at;
  }
  // The item of that number: blocks of rows of a token, tokens of a head, heads, sequences
  __device__ __forceinline__ void item(unsigned n, Item &it) const {
    const unsigned token = n / (unsigned)blocks, bh = token / (unsigned)a.N, b = bh / (unsigned)a.Hk;
    it.rb = (int)(n - token * (unsigned)blocks);
    it.h = (int)(bh - b * (unsigned)a.Hk);
    it.p = (int)(b * (unsigned)a.N + token - bh * (unsigned)a.N);
    it.tiles = item_tiles;
    it.first = n * per_item + (unsigned)a.extra;
    it.at = 0;
    it.s = seq(it.p);
  }
  __device__ __forceinline__ bool find(unsigned &x, Item &it) const {
    x = workgroup() * each;
    if (x >= total) return false;
    item(x / per_item, it);
    x = max(x, it.first);
    it.at = x - it.first;
    return x < total;
  }
  __device__ __forceinline__ bool next(unsigned &x, unsigned x_end, Item &it) const {
    x += (unsigned)a.extra;
    if (x >= x_end) return false;
    item(x / per_item, it);
    return true;
  }
  __device__ __forceinline__ int begin() const { return 0; }
  __device__ __forceinline__ Row row(int p, int h, int r) const {
    const int b = p / a.N;
    return {b, p - b * a.N, h * a.G + r};
  }
  __device__ __forceinline__ int last_key(const Row &r, const PagedSeq &s) const {
    const int64_t k = (int64_t)s.start + r.i;
    return r.i >= s.tokens ? -1 : (int)max((int64_t)-1, min(k, (int64_t)a.capacity - 1));
  }
};

}  // namespace qfa
