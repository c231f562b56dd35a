// Which blocks (pages) of a long cache a token's attention reads: those whose keys may have the largest scores.
//
// Bounds of a page and key head: low_d = min, high_d = max over its rows of k^_d = scale * (code - zero point); the two rows are quantized
// like tokens, with zero points of 16 bits for rows of one sign (quant_row).  No key of the page has a larger product with a query q than
// sum_d max(q_d low_d, q_d high_d), but for that rounding and the query's.  (Zero points of 8 bits, as tokens have them, cut such rows at their span: of
// zero-mean keys 44 % of the largest elements of 64 rows and 76 % of those of 128.  Bounds that come with them are served as they are.)  With the query's own whole numbers e = code - zero point, e+ = max(e, 0), e- = max(-e, 0):
//     score = scale_q * (scale_high * sum e+ (c_high - z_high) - scale_low * sum e- (c_low - z_low)),
// and of the query heads that share a key head the largest.  The sums are whole numbers below 2^27, exact on INT8 MFMA; what is left is
// in 64 bits (the products with 24-bit scales are exact there) and rounded to 32 once, so that the order of blocks is the same wherever
// it is computed.  e+ and e- reach 255: the operands are e+ - 128 and e- - 128, and 128 times the bounds' own sums (a product with ones)
// come on top.
//
// Scores, then for every token and key head the `keep` best (qfa_topk.h), in one launch or two.
//
// Waits bound all of it, not the 2 (D + 6) bytes of a block: page number, bounds, the digits of a selection come one behind the other.  One token of 64 sequences
// of 5 to 512 blocks, 8 key heads of 4 x 128, 34 MB: 18.5 us (2 TB/s), vector pipe 10 % busy; 333 tokens of 2 sequences of 219 blocks, 5 key heads of 4 x 64:
// 15.6; one token of 2048 blocks: 5.9 and 8.4 for the selection.  Not faster: eight waves that take all blocks at once (22.8; with 128 registers each 32), bounds
// brought in the order in which they lie and turned in LDS (17.6; 256 elements run out of registers).
#include <cfloat>

#include "qfa_host.h"
#include "qfa_quant_row.h"
#include "qfa_skv_common.h"
#include "qfa_topk.h"

namespace qfa {

// ---------------------------------------------------------------------------------------------------------------- bounds
// A wave takes a page and key head: D/16 lanes hold a row, each its minima and maxima of 16 elements, which meet at the end.  A launch with its waits: one token of
// 64 sequences, 8 key heads of 128, 16 rows a page 4.2 us, one token, 64 rows 5.2; of whole prompts, 131072 tokens in pages of 64, 31.6 us (4.5 TB/s), 4 x 8192 tokens in pages of 16 18
template <typename S, int D, typename Z> __global__ __launch_bounds__(256) void page_bounds_kernel(PagedSelectArgs a, int pages_each) {
  constexpr int LPR = D / 16, RPW = 64 / LPR;
  const int lane = threadIdx.x % 64, sub = lane % LPR, rg = lane / LPR;
  const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);   // (uniform over the wave, as all that follows from it)
  const int64_t bt = index_div(item, a.Hk), h = item - bt * a.Hk, b = index_div(bt, pages_each), t = bt - b * pages_each;
  if (b >= a.B) return;
  const int64_t n = a.counts ? max(0, min((int64_t)a.counts[b], a.N)) : a.N, start = a.starts[b], end = start + n;
  const int64_t j = (max((int64_t)0, start) >> a.page_log2) + t, first = j << a.page_log2;
  if (n == 0 || first >= end || j >= a.width) return;
  const int64_t id = a.page_table[b * a.stb + j * a.stw];
  if (id < 0 || id >= a.pages) return;
  const int rows = (int)min(end - first, (int64_t)1 << a.page_log2);
  const int64_t at = (id * a.Hk + h) << a.page_log2;
  const int8_t *codes = a.cache.k_codes + at * D + 16 * sub, *zero = a.cache.k_zero + at;
  const S *scale = static_cast<const S *>(a.cache.k_scale) + at;
  float low[16], high[16];   // high: negated, so that both are minima
#pragma unroll
  for (int e = 0; e < 16; ++e) low[e] = high[e] = INFINITY;
#pragma unroll 2
  for (int r0 = 0; r0 < rows; r0 += RPW) {
    const int r = min(r0 + rg, rows - 1);   // (a row twice changes nothing)
    const u32x4 w = *reinterpret_cast<const u32x4 *>(codes + (int64_t)r * D);
    const float s = (float)scale[r];
    const int z = zero[r];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float x = (float)((int)(signed char)(w[e / 4] >> (8 * (e % 4))) - z) * s;
      low[e] = fminf(low[e], x);
      high[e] = fminf(high[e], -x);
    }
  }
  // groups of lanes in turn go on with the low row and the high one
  const bool up = rg & 1;
  float v[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float other = __shfl_xor(up ? low[e] : high[e], LPR, 64);
    v[e] = fminf(up ? high[e] : low[e], other);
  }
#pragma unroll
  for (int off = 2 * LPR; off < 64; off <<= 1)
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = fminf(v[e], __shfl_xor(v[e], off, 64));
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = up ? -v[e] : v[e];
  const QuantRow<16> q = quant_row<LPR, false, 16, sizeof(Z) == 2>(v, true);
  if (rg < 2) {
    const int64_t to = 2 * (id * a.Hk + h) + rg;
    *reinterpret_cast<u32x4 *>(a.codes + to * D + 16 * sub) = u32x4{q.codes[0], q.codes[1], q.codes[2], q.codes[3]};
    if (sub == 0) {
      a.scale[to] = q.scale;
      static_cast<Z *>(a.zero)[to] = (Z)(int)q.zp;
    }
  }
}

template <typename S, typename Z> static int launch_bounds_sz(const PagedSelectArgs &a, hipStream_t st) {
  const int64_t page = (int64_t)1 << a.page_log2, each = (a.N + page - 2) / page + 1, waves = a.B * each * a.Hk;   // pages that N tokens may touch
  if (waves > 0x7fffffffLL) return set_error(QFA_EUNSUPPORTED, "paged_bounds: too many pages for one launch");
  const dim3 grid((unsigned)((waves + 3) / 4)), block(256);
  if (a.D == 64) page_bounds_kernel<S, 64, Z><<<grid, block, 0, st>>>(a, (int)each);
  else if (a.D == 128) page_bounds_kernel<S, 128, Z><<<grid, block, 0, st>>>(a, (int)each);
  else page_bounds_kernel<S, 256, Z><<<grid, block, 0, st>>>(a, (int)each);
  return check_launch("qfa_paged_bounds");
}
template <typename S> static int launch_bounds_s(const PagedSelectArgs &a, hipStream_t st) {
  return a.zero_bits == 16 ? launch_bounds_sz<S, int16_t>(a, st) : launch_bounds_sz<S, int8_t>(a, st);
}
int launch_paged_bounds(const PagedSelectArgs &a, hipStream_t st) {
  if (a.scale_dtype == QFA_F32) return launch_bounds_s<float>(a, st);
  if (a.scale_dtype == QFA_F16) return launch_bounds_s<_Float16>(a, st);
  return launch_bounds_s<__bf16>(a, st);
}

// The list of one token, by T threads (tid: which of them): the blocks with the `keep` largest scores, number(i) of block i
template <int T, typename Top, typename Number>
__device__ __forceinline__ void select_blocks(Top &top, const PagedSelectArgs &x, int64_t item, int64_t pos, int tid, Number number) {
  const int blocks = pos < 0 ? 0 : (int)min((pos >> x.page_log2) + 1, x.width);   // (a token past the table's end sees all of it)
  const int keep = (int)x.keep, first = (int)x.first, last = blocks - 1 - (int)x.last;
  int32_t *to = x.blocks + item * keep;
  unsigned taken = 0;
  if (blocks > 0)
    taken = top.run(blocks, (unsigned)keep, number,
                    [&](int i, float s) __attribute__((always_inline)) -> unsigned {
                      return s == -INFINITY ? 0u : ((i < first) | (i > last)) ? TOP_ALWAYS : top_key(s);
                    },
                    [&](unsigned place, int i, float) __attribute__((always_inline)) { to[place] = i; });
  for (int i = (int)taken + tid; i < keep; i += T) to[i] = -1;
}

// ---------------------------------------------------------------------------------------------------------------- scores
struct SelectKernelArgs {
  PagedSelectArgs x;
  int G, tokens_each, token_tiles, row_blocks;   // tokens of a workgroup (its 16 rows hold whole groups of heads; larger groups take several blocks of rows)
  int steps, chunks;                             // of 16 blocks of each wave; workgroups that share a token's blocks
  bool round;                                    // all heads and tokens of a chunk run on one XCD
};

// The position of token n of sequence b: below 0 where it brings none
__device__ __forceinline__ int64_t token_position(const PagedSelectArgs &x, int64_t b, int64_t n) {
  const int64_t brings = x.counts ? max(0, min((int64_t)x.counts[b], x.N)) : x.N;
  return n < brings ? (int64_t)x.starts[b] + n : -1;
}

// The zero points of a block's two rows as they lie there, and the one of the low row or the high one
__device__ __forceinline__ unsigned load_zeros(const PagedSelectArgs &x, int64_t row) {
  if (x.zero_bits == 16) return *reinterpret_cast<const unsigned *>(static_cast<const int16_t *>(x.zero) + row);
  return *reinterpret_cast<const unsigned short *>(static_cast<const int8_t *>(x.zero) + row);
}
__device__ __forceinline__ int zero_of(const PagedSelectArgs &x, unsigned zeros, bool high) {
  return (int)__builtin_amdgcn_sbfe((int)zeros, high ? (unsigned)x.zero_bits : 0u, (unsigned)x.zero_bits);
}

// What a workgroup works on
struct SelectPlace {
  int chunk, tile, n0, tokens;
  int64_t b, h, start, brings;
  bool live;
  __device__ __forceinline__ SelectPlace(const SelectKernelArgs &p) {
    const PagedSelectArgs &x = p.x;
    // consecutive workgroups go round the 8 XCDs: all heads and tokens of a chunk to one of them, whose L2 then has the scales and zero points of its
    // pages once (8 bytes and 2 for each head, of lines of 128)
    const unsigned inner = (unsigned)(x.Hk * p.token_tiles), xcd = p.round ? blockIdx.x % 8 : 0, place = p.round ? blockIdx.x / 8 : blockIdx.x;
    const unsigned outer = p.round ? place / inner * 8 + xcd : place / inner, in = place % inner;
    live = outer < (unsigned)(x.B * p.chunks);
    // (sequences before chunks: not every sequence has blocks in the later chunks)
    chunk = (int)(outer / (unsigned)x.B);
    tile = (int)(in % (unsigned)p.token_tiles);
    h = in / (unsigned)p.token_tiles;
    b = live ? outer - (unsigned)chunk * (unsigned)x.B : 0;
    n0 = tile * p.tokens_each;
    tokens = min(p.tokens_each, (int)x.N - n0);
    start = x.starts[b];
    brings = x.counts ? max((int64_t)0, min((int64_t)x.counts[b], x.N)) : x.N;
  }
  // the position of token t of the tile (-1: it sees nothing), and its last block
  __device__ __forceinline__ int64_t position(int t) const {
    const int64_t pos = start + n0 + t;
    return t >= 0 && t < tokens && n0 + t < brings && pos >= 0 ? pos : -1;
  }
  __device__ __forceinline__ int64_t last_block(const PagedSelectArgs &x, int t) const { return position(t) >> x.page_log2; }
  __device__ __forceinline__ int64_t item(const PagedSelectArgs &x, int t) const { return (b * x.Hk + h) * x.N + n0 + t; }
  // ... and that any of them sees
  __device__ __forceinline__ int64_t last_block(const PagedSelectArgs &x) const { return last_block(x, (int)min((int64_t)tokens, brings - n0) - 1); }
};

// 16 rows of a tile of tokens, quantized and split: a thread holds 8 elements of PASSES rows
template <int D> struct SplitRows {
  static constexpr int LPT = D / 8, TPP = 256 / LPT, PASSES = (16 + TPP - 1) / TPP;
  struct Lds {
    unsigned char codes[2][16 * D];   // e+ - 128, e- - 128
    float scale[16];
    int sums[2][16];                  // of e+ and e-
  };
  float v[PASSES][8];
  __device__ __forceinline__ void load(const SelectKernelArgs &p, const SelectPlace &at, int rb, int nrows) {
    const PagedSelectArgs &x = p.x;
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int row = ps * TPP + threadIdx.x / LPT, sub = threadIdx.x % LPT, r = 16 * rb + min(row, nrows - 1), i = r / p.G;
      const int64_t off = at.b * x.sq[0] + (at.h * p.G + r - i * p.G) * x.sq[1] + (at.n0 + i) * x.sq[2] + sub * 8;
      if (x.q_dtype == QFA_F32) Load8<float>::run(static_cast<const float *>(x.q) + off, v[ps]);
      else if (x.q_dtype == QFA_BF16) Load8<__bf16>::run(static_cast<const __bf16 *>(x.q) + off, v[ps]);
      else Load8<_Float16>::run(static_cast<const _Float16 *>(x.q) + off, v[ps]);
    }
  }
  __device__ __forceinline__ void split(Lds &lds, int nrows) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int row = ps * TPP + threadIdx.x / LPT, sub = threadIdx.x % LPT;
      if (ps * TPP + wave * (64 / LPT) >= nrows) break;   // (uniform over the wave; the rows behind hold anything, and nobody looks at their scores)
      const QuantRow<8> q = quant_row<LPT, false, 8>(v[ps], true);
      const int z = (int)q.zp;
      unsigned plus[2] = {0, 0}, minus[2] = {0, 0};
      int sp = 0, sm = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int w = (int)(signed char)(q.codes[e / 4] >> (8 * (e % 4))) - z, up = max(w, 0), down = max(-w, 0);
        plus[e / 4] |= (unsigned)((up ^ 0x80) & 0xff) << (8 * (e % 4));
        minus[e / 4] |= (unsigned)((down ^ 0x80) & 0xff) << (8 * (e % 4));
        sp += up;
        sm += down;
      }
      sp = group_sum<LPT>(sp);
      sm = group_sum<LPT>(sm);
      if (row < 16) {
        *reinterpret_cast<u32x2 *>(&lds.codes[0][row * D + sub * 8]) = u32x2{plus[0], plus[1]};
        *reinterpret_cast<u32x2 *>(&lds.codes[1][row * D + sub * 8]) = u32x2{minus[0], minus[1]};
        if (sub == 0) {
          lds.scale[row] = q.scale;
          lds.sums[0][row] = sp;
          lds.sums[1][row] = sm;
        }
      }
    }
  }
};
__device__ __forceinline__ i32x4 select_mfma(i32x4 a, i32x4 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
// a row's score on a block: dot products of e+ - 128 with the high row and of e- - 128 with the low one, the rows' own sums
__device__ __forceinline__ float block_score(int dot_high, int dot_low, int own_high, int own_low, int zh, int zl, double sh, double sl, int sum_plus, int sum_minus,
                                             double sq) {
  const int ih = dot_high + 128 * own_high - zh * sum_plus, il = dot_low + 128 * own_low - zl * sum_minus;
  return fmaxf(-FLT_MAX, (float)((sh * (double)ih - sl * (double)il) * sq));   // (what is not a number counts as the least)
}

// Up to four rows (a token's heads, mostly): they stand four times among the 16 rows of a product, so that every group of lanes has the products of all
// rows with all of four tiles of 16 blocks, and goes on with one of them: a lane has one block.  A wave takes 64 blocks at a time.
// WHOLE: a workgroup has all blocks of its tokens, keeps their scores, and selects.
constexpr int SELECT_WHOLE_FEW = 1024, SELECT_WHOLE = 256;   // blocks at most
template <int D, bool WHOLE> __global__ __launch_bounds__(256, 2) void block_scores_few_kernel(SelectKernelArgs p) {
  constexpr int KM = D / 64;
  __shared__ float held[WHOLE ? 4 : 1][WHOLE ? SELECT_WHOLE_FEW : 1];
  __shared__ __attribute__((aligned(16))) typename SplitRows<D>::Lds lds;
  const PagedSelectArgs &x = p.x;
  const int tid = threadIdx.x, lane = tid % 64, c16 = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const SelectPlace at(p);
  if (!at.live) return;
  const int64_t begin = (int64_t)at.chunk * 256 * p.steps, end = min(x.width, begin + 256 * p.steps);
  auto page_of = [&](int64_t j) __attribute__((always_inline)) -> int {
    const int page = x.page_table[at.b * x.stb + min(j, x.width - 1) * x.stw];
    return j < x.width && page >= 0 && page < x.pages ? page : -1;
  };
  int page = page_of(begin + 64 * wave + lane);
  SplitRows<D> rows;
  const int nrows = at.tokens * p.G;
  rows.load(p, at, 0, nrows);
  const int64_t seen = min(end, at.last_block(x) + 1);
  float *to = x.scores + ((at.b * x.Hk + at.h) * x.N + at.n0) * x.width;
  if (begin >= seen) {
    if (x.all_scores)
      for (int64_t i = begin + tid; i < end; i += 256)
        for (int t = 0; t < at.tokens; ++t) to[t * x.width + i] = -INFINITY;
    if (WHOLE)
      for (int64_t i = tid; i < at.tokens * x.keep; i += 256) x.blocks[at.item(x, 0) * x.keep + i] = -1;
    return;
  }
  i32x4 qf[2][KM];
  const i32x4 ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
  for (int step = 0; step < p.steps; ++step) {
    const int64_t j0 = begin + 256 * step + 64 * wave, j = j0 + lane;
    const bool work = j0 < seen;   // (uniform over the wave)
    i32x4 k[4][2][KM];
    f32x2 sk = {0.f, 0.f};
    unsigned zk = 0;
    if (work) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int64_t row = 2 * ((int64_t)max(__shfl(page, 16 * t + c16, 64), 0) * x.Hk + at.h);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int m = 0; m < KM; ++m) k[t][s][m] = *reinterpret_cast<const i32x4 *>(x.codes + (row + s) * D + 64 * m + 16 * g);
      }
      const int64_t row = 2 * ((int64_t)max(page, 0) * x.Hk + at.h);
      sk = *reinterpret_cast<const f32x2 *>(x.scale + row);
      zk = load_zeros(x, row);
    }
    const bool there = page >= 0;
    if (step + 1 < p.steps) page = page_of(j + 256);
    if (step == 0) {
      rows.split(lds, nrows);
      __syncthreads();
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int m = 0; m < KM; ++m) qf[s][m] = *reinterpret_cast<const i32x4 *>(&lds.codes[s][c16 % 4 * D + 64 * m + 16 * g]);
    }
    if (work) {
      i32x4 dot[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};   // of e- with the low row, e+ with the high one
      int own[2] = {0, 0};
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          i32x4 d = {0, 0, 0, 0}, o = {0, 0, 0, 0};
#pragma unroll
          for (int m = 0; m < KM; ++m) {
            d = select_mfma(qf[1 - s][m], k[t][s][m], d);
            o = select_mfma(ones, k[t][s][m], o);
          }
#pragma unroll
          for (int v = 0; v < 4; ++v) dot[s][v] = g == t ? d[v] : dot[s][v];
          own[s] = g == t ? o[0] : own[s];
        }
      const int zl = zero_of(x, zk, false), zh = zero_of(x, zk, true);
      float y[4];
#pragma unroll
      for (int v = 0; v < 4; ++v)
        y[v] = block_score(dot[1][v], dot[0][v], own[1], own[0], zh, zl, sk[1], sk[0], lds.sums[0][v], lds.sums[1][v], lds.scale[v]);
      for (int t = 0; t < at.tokens; ++t) {   // (rows in order: tokens, and in them the heads)
        float best = -FLT_MAX;
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (v / p.G == t) best = fmaxf(best, y[v]);
        const float score = there && j <= at.last_block(x, t) ? best : -INFINITY;
        if (WHOLE && j < end) held[t][j] = score;
        if ((!WHOLE || x.all_scores) && j < end) to[t * x.width + j] = score;
      }
    } else if (x.all_scores && j < end) {
      for (int t = 0; t < at.tokens; ++t) to[t * x.width + j] = -INFINITY;
    }
  }
  if constexpr (WHOLE) {
    __shared__ TopHeld<256, SELECT_WHOLE_FEW, 8> top;
    __syncthreads();
    for (int t = 0; t < at.tokens; ++t) {
      if (t > 0) __syncthreads();   // the token before is done with
      select_blocks<256>(top, x, at.item(x, t), at.position(t), tid, [&](int i) __attribute__((always_inline)) { return held[t][i]; });
    }
  }
}

// A workgroup = 4 waves = some tokens of a sequence and key head, and a chunk of its blocks, 16 of them at a time in a wave: queries are the rows
// of the product, blocks its columns.  The pages of up to four steps are one load, a step's bounds are requested a step ahead, and the
// first ones before the queries are quantized.
constexpr int SELECT_STEPS = 4;
template <int D, bool WHOLE> __global__ __launch_bounds__(256, D == 256 ? 2 : 3) void block_scores_kernel(SelectKernelArgs p) {
  constexpr int KM = D / 64;
  __shared__ float held[WHOLE ? 16 : 1][WHOLE ? SELECT_WHOLE : 1];
  __shared__ __attribute__((aligned(16))) typename SplitRows<D>::Lds lds;
  __shared__ float out[4][16][17];       // per wave: rows, blocks
  const PagedSelectArgs &x = p.x;
  const int tid = threadIdx.x, lane = tid % 64, c16 = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const SelectPlace at(p);
  if (!at.live) return;
  const int64_t b = at.b, h = at.h;
  const int tokens = at.tokens;
  const int64_t begin = (int64_t)at.chunk * 64 * p.steps, end = min(x.width, begin + 64 * p.steps);
  // lane (g, c16): the page of its wave's block c16 of step g
  const int64_t j_mine = begin + 64 * g + 16 * wave + c16;
  const int page_mine = x.page_table[b * x.stb + min(j_mine, x.width - 1) * x.stw];
  const int64_t seen = min(end, at.last_block(x) + 1);
  float *to = x.scores + ((b * x.Hk + h) * x.N + at.n0) * x.width;
  if (begin >= seen) {
    if (x.all_scores)
      for (int64_t i = begin + tid; i < end; i += 256)
        for (int t = 0; t < tokens; ++t) to[t * x.width + i] = -INFINITY;
    if (WHOLE)
      for (int64_t i = tid; i < tokens * x.keep; i += 256) x.blocks[at.item(x, 0) * x.keep + i] = -1;
    return;
  }
  struct Bounds {
    i32x4 k[2][KM];
    f32x2 s;
    unsigned z;
    bool there;
  };
  auto load = [&](Bounds &k, int step) __attribute__((always_inline)) {
    const int page = __shfl(page_mine, 16 * step + c16, 64);
    k.there = begin + 64 * step + 16 * wave + c16 < x.width && page >= 0 && page < x.pages;
    const int64_t at = 2 * ((k.there ? page : 0) * x.Hk + h);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int m = 0; m < KM; ++m) k.k[s][m] = *reinterpret_cast<const i32x4 *>(x.codes + (at + s) * D + 64 * m + 16 * g);
    k.s = *reinterpret_cast<const f32x2 *>(x.scale + at);
    k.z = load_zeros(x, at);
  };
  const i32x4 ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
  const bool folds = p.G <= 16 && (p.G & (p.G - 1)) == 0;   // the rows of a token lie in one lane, or in lanes a power of two apart
  for (int rb = 0; rb < p.row_blocks; ++rb) {
    const int nrows = min(16, (p.row_blocks > 1 ? p.G - 16 * rb : tokens * p.G));
    SplitRows<D> rows;
    rows.load(p, at, rb, nrows);
    Bounds next;
    load(next, 0);
    if (rb > 0) __syncthreads();   // the rows before are done with
    rows.split(lds, nrows);
    __syncthreads();
    i32x4 qf[2][KM];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int m = 0; m < KM; ++m) qf[s][m] = *reinterpret_cast<const i32x4 *>(&lds.codes[s][c16 * D + 64 * m + 16 * g]);
    double sq[4];
    int sum[2][4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      sq[v] = (double)lds.scale[4 * g + v];
      sum[0][v] = lds.sums[0][4 * g + v];
      sum[1][v] = lds.sums[1][4 * g + v];
    }
    for (int step = 0; step < p.steps; ++step) {
      const int64_t j0 = begin + 64 * step + 16 * wave, j = j0 + c16;
      if (j0 >= seen) break;   // (uniform over the wave; no barrier follows inside)
      const Bounds k = next;
      if (step + 1 < p.steps) load(next, step + 1);
      i32x4 dot[2], own[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        dot[s] = own[s] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < KM; ++m) {   // e+ with the high row, e- with the low one
          dot[s] = select_mfma(qf[1 - s][m], k.k[s][m], dot[s]);
          own[s] = select_mfma(ones, k.k[s][m], own[s]);
        }
      }
      const int zl = zero_of(x, k.z, false), zh = zero_of(x, k.z, true);
      const double sl = k.s[0], sh = k.s[1];
      float y[4];   // rows 4 g + v on block c16
#pragma unroll
      for (int v = 0; v < 4; ++v) y[v] = block_score(dot[1][v], dot[0][v], own[1][v], own[0][v], zh, zl, sh, sl, sum[0][v], sum[1][v], sq[v]);
      // ---- of a token's heads the largest
      auto store = [&](int t, float best) __attribute__((always_inline)) {
        if (t >= tokens || j >= end) return;
        if (rb > 0) best = fmaxf(best, WHOLE ? held[t][j] : to[t * x.width + j]);   // (this lane wrote it)
        const float score = k.there && j <= at.last_block(x, t) ? best : -INFINITY;
        if (WHOLE) held[t][j] = score;
        if (!WHOLE || x.all_scores) to[t * x.width + j] = score;
      };
      if (folds) {
        if (p.G == 1) {
#pragma unroll
          for (int v = 0; v < 4; ++v) store(4 * g + v, y[v]);
        } else if (p.G == 2) {
          store(2 * g, fmaxf(y[0], y[1]));
          store(2 * g + 1, fmaxf(y[2], y[3]));
        } else {
          float best = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
          if (p.G >= 8) best = fmaxf(best, __shfl_xor(best, 16, 64));
          if (p.G == 16) best = fmaxf(best, __shfl_xor(best, 32, 64));
          if ((4 * g & (p.G - 1)) == 0) store(4 * g / p.G, best);
        }
      } else {
#pragma unroll
        for (int v = 0; v < 4; ++v) out[wave][4 * g + v][c16] = y[v];
        __builtin_amdgcn_wave_barrier();   // (the wave reads what it wrote itself)
        const int rows = p.row_blocks > 1 ? nrows : p.G, outs = p.row_blocks > 1 ? 1 : tokens;
        for (int t = g; t < outs; t += 4) {
          float best = -FLT_MAX;
          for (int r = 0; r < rows; ++r) best = fmaxf(best, out[wave][t * p.G + r][c16]);
          store(t, best);
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
  if (x.all_scores)   // blocks behind the last one that is seen, of waves that have left the loop above
    for (int64_t i = (seen + 15) / 16 * 16 + tid; i < end; i += 256)
      for (int t = 0; t < tokens; ++t) to[t * x.width + i] = -INFINITY;
  if constexpr (WHOLE) {   // a wave for each token
    __syncthreads();
    TopFew top;
    for (int t = wave; t < tokens; t += 4)
      select_blocks<64>(top, x, at.item(x, t), at.position(t), lane, [&](int i) __attribute__((always_inline)) { return held[t][i]; });
  }
}

// ------------------------------------------------------------------------------------------------------------- the best
// Top: TopFew or TopHeld, of T threads
template <typename Top, int T> __global__ __launch_bounds__(T) void block_select_kernel(PagedSelectArgs x) {
  __shared__ Top top;
  const int64_t item = blockIdx.x, bh = index_div(item, x.N), n = item - bh * x.N, b = index_div(bh, x.Hk);
  const float *scores = x.scores + item * x.width;
  select_blocks<T>(top, x, item, token_position(x, b, n), threadIdx.x, [&](int i) __attribute__((always_inline)) { return scores[i]; });
}
template <typename Top, int T> static void launch_top(const PagedSelectArgs &x, hipStream_t st) {
  block_select_kernel<Top, T><<<dim3((unsigned)(x.B * x.Hk * x.N)), dim3(T), 0, st>>>(x);
}

template <int D> static void launch_scores(const SelectKernelArgs &p, bool few, bool whole, dim3 grid, hipStream_t st) {
  const dim3 block(256);
  if (few && whole) block_scores_few_kernel<D, true><<<grid, block, 0, st>>>(p);
  else if (few) block_scores_few_kernel<D, false><<<grid, block, 0, st>>>(p);
  else if (whole) block_scores_kernel<D, true><<<grid, block, 0, st>>>(p);
  else block_scores_kernel<D, false><<<grid, block, 0, st>>>(p);
}
int launch_paged_select(const PagedSelectArgs &x, hipStream_t st) {
  SelectKernelArgs p;
  p.x = x;
  p.G = (int)(x.H / x.Hk);
  p.tokens_each = p.G >= 16 ? 1 : (int)min((int64_t)(16 / p.G), x.N);
  p.token_tiles = (int)((x.N + p.tokens_each - 1) / p.tokens_each);
  p.row_blocks = (p.G + 15) / 16;
  const int64_t groups = x.B * x.Hk * p.token_tiles;
  const bool few = p.row_blocks == 1 && p.tokens_each * p.G <= 4;
  const int step = few ? 256 : 64;   // blocks of a workgroup's step
  p.steps = 1;
  // Scores and selection in one launch where a workgroup can hold all blocks of its tokens, and has one step of them or enough others beside it.  Four query
  // heads of 128 elements, us with two launches and with one: 256 blocks of 1, 8 and 32 sequences with 8 key heads 9.5, 9.7, 10.2 and 8.8, 8.9, 9.1;
  // 1000 blocks of 1, 8, 32 and 64 12.9, 14.2, 25.5, 37.7 and 19.9, 20.5, 24.6, 35.  What decides is the table's width, for the host does not know the lengths: 32 sequences of 256
  // blocks under a table of 2048, 16384 and 32768 pages 13.0, 19.7 and 29.4
  const bool whole = x.width <= SELECT_WHOLE || (few && x.width <= SELECT_WHOLE_FEW && groups >= 256);
  if (whole) p.steps = (int)((x.width + step - 1) / step);   // (SELECT_STEPS at most)
  while (!whole && p.steps < SELECT_STEPS && groups * ((x.width + 2 * step * p.steps - 1) / (2 * step * p.steps)) >= 512) p.steps *= 2;
  p.chunks = (int)((x.width + step * p.steps - 1) / (step * p.steps));
  const int64_t outer = x.B * p.chunks;
  p.round = xcd_whole_heads(outer);
  const int64_t outer_grid = p.round ? (outer + 7) / 8 * 8 : outer, grid_size = outer_grid * x.Hk * p.token_tiles;
  const double most = (double)outer_grid * (double)x.Hk * (double)p.token_tiles, items = (double)x.B * (double)x.Hk * (double)x.N;
  if (most > 2147483647.0 || items > 2147483647.0) return set_error(QFA_EUNSUPPORTED, "paged_select: too many tokens and blocks for one launch");
  const dim3 grid((unsigned)grid_size);
  if (x.D == 64) launch_scores<64>(p, few, whole, grid, st);
  else if (x.D == 128) launch_scores<128>(p, few, whole, grid, st);
  else launch_scores<256>(p, few, whole, grid, st);
  if (int e = check_launch("qfa_paged_select (scores)")) return e;
  if (whole) return 0;
  // one wave for a few blocks (3330 x 219: 5.8 us, with a wave and counters in LDS 7.5, with four 9.3), more for many
  if (x.width <= 256) launch_top<TopFew, 64>(x, st);
  else if (x.width <= 1024) launch_top<TopHeld<256, 1024, 8>, 256>(x, st);
  else if (x.width <= 16384) launch_top<TopHeld<1024, 16384, 11>, 1024>(x, st);
  else launch_top<TopHeld<1024, 0, 11>, 1024>(x, st);
  return check_launch("qfa_paged_select");
}

}  // namespace qfa
