// Which blocks (pages) of a long cache a token's attention reads: those whose keys may have the largest scores.
//
// Bounds of a page and key head: low_d = min, high_d = max over its rows of k^_d = scale * (code - zero point); the two rows are quantized
// like tokens.  No key of the page has a larger product with a query q than  sum_d max(q_d low_d, q_d high_d), but for that rounding and the
// query's.  With the query's own whole numbers e = code - zero point, e+ = max(e, 0), e- = max(-e, 0):
//     score = scale_q * (scale_high * sum e+ (c_high - z_high) - scale_low * sum e- (c_low - z_low)),
// and of the query heads that share a key head the largest.  The sums are whole numbers below 2^24, exact on INT8 MFMA; what is left is
// in 64 bits (the products of 24-bit numbers are exact there) and rounded to 32 once, so that the order of blocks is the same wherever
// it is computed.  e+ and e- reach 255: the operands are e+ - 128 and e- - 128, and 128 times the bounds' own sums (a product with ones)
// come on top.
//
// Two launches: scores, then for every token and key head the `keep` best (qfa_topk.h).
#include <cfloat>

#include "qfa_host.h"
#include "qfa_quant_row.h"
#include "qfa_skv_common.h"
#include "qfa_topk.h"

namespace qfa {

// ---------------------------------------------------------------------------------------------------------------- bounds
// A wave takes a page and key head: D/16 lanes hold a row, each its minima and maxima of 16 elements, which meet at the end
template <typename S, int D> __global__ __launch_bounds__(256) void page_bounds_kernel(PagedSelectArgs a, int pages_each) {
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
  float low[16], high[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    low[e] = INFINITY;
    high[e] = -INFINITY;
  }
#pragma unroll 4
  for (int r0 = 0; r0 < rows; r0 += RPW) {
    const int r = min(r0 + rg, rows - 1);   // (a row twice changes nothing)
    const u32x4 w = *reinterpret_cast<const u32x4 *>(codes + (int64_t)r * D);
    const float s = (float)scale[r];
    const int z = zero[r];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float x = (float)((int)(signed char)(w[e / 4] >> (8 * (e % 4))) - z) * s;
      low[e] = fminf(low[e], x);
      high[e] = fmaxf(high[e], x);
    }
  }
#pragma unroll
  for (int off = LPR; off < 64; off <<= 1)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      low[e] = fminf(low[e], __shfl_xor(low[e], off, 64));
      high[e] = fmaxf(high[e], __shfl_xor(high[e], off, 64));
    }
  const QuantRow<16> ql = quant_row<LPR, false, 16>(low, true), qh = quant_row<LPR, false, 16>(high, true);
  if (rg < 2) {   // the first lanes store the low row, the next ones the high one
    const int64_t to = 2 * (id * a.Hk + h) + rg;
    *reinterpret_cast<u32x4 *>(a.codes + to * D + 16 * sub) =
        rg ? u32x4{qh.codes[0], qh.codes[1], qh.codes[2], qh.codes[3]} : u32x4{ql.codes[0], ql.codes[1], ql.codes[2], ql.codes[3]};
    if (sub == 0) {
      a.scale[to] = rg ? qh.scale : ql.scale;
      a.zero[to] = (int8_t)(int)(rg ? qh.zp : ql.zp);
    }
  }
}

template <typename S> static int launch_bounds_s(const PagedSelectArgs &a, hipStream_t st) {
  const int64_t page = (int64_t)1 << a.page_log2, each = (a.N + page - 2) / page + 1, waves = a.B * each * a.Hk;   // pages that N tokens may touch
  if (waves > 0x7fffffffLL) return set_error(QFA_EUNSUPPORTED, "paged_bounds: too many pages for one launch");
  const dim3 grid((unsigned)((waves + 3) / 4)), block(256);
  if (a.D == 64) page_bounds_kernel<S, 64><<<grid, block, 0, st>>>(a, (int)each);
  else if (a.D == 128) page_bounds_kernel<S, 128><<<grid, block, 0, st>>>(a, (int)each);
  else page_bounds_kernel<S, 256><<<grid, block, 0, st>>>(a, (int)each);
  return check_launch("qfa_paged_bounds");
}
int launch_paged_bounds(const PagedSelectArgs &a, hipStream_t st) {
  if (a.scale_dtype == QFA_F32) return launch_bounds_s<float>(a, st);
  if (a.scale_dtype == QFA_F16) return launch_bounds_s<_Float16>(a, st);
  return launch_bounds_s<__bf16>(a, st);
}

// ---------------------------------------------------------------------------------------------------------------- scores
struct SelectKernelArgs {
  PagedSelectArgs x;
  int G, tokens_each, token_tiles, row_blocks;   // tokens of a workgroup (its 16 rows hold whole groups of heads; larger groups take several blocks of rows)
  int steps, chunks;                             // of 16 blocks of each wave; workgroups that share a token's blocks
};

// The position of token n of sequence b: below 0 where it brings none
__device__ __forceinline__ int64_t token_position(const PagedSelectArgs &x, int64_t b, int64_t n) {
  const int64_t brings = x.counts ? max(0, min((int64_t)x.counts[b], x.N)) : x.N;
  return n < brings ? (int64_t)x.starts[b] + n : -1;
}

// A workgroup = 4 waves = some tokens of a sequence and key head, and a chunk of its blocks, 16 of them at a time in a wave: queries are the rows
// of the product, blocks its columns
template <int D> __global__ __launch_bounds__(256) void block_scores_kernel(SelectKernelArgs p) {
  constexpr int KM = D / 64, LPT = D / 8, TPP = 256 / LPT, PASSES = (16 + TPP - 1) / TPP;
  __shared__ __attribute__((aligned(16))) unsigned char codes[2][16 * D];   // e+ - 128, e- - 128
  __shared__ float scale[16];
  __shared__ int sums[2][16];            // of e+ and e-
  __shared__ float out[4][16][17];       // per wave: rows, blocks
  const PagedSelectArgs &x = p.x;
  const int tid = threadIdx.x, lane = tid % 64, c16 = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  unsigned id = blockIdx.x;
  const int chunk = (int)(id % (unsigned)p.chunks);
  id /= (unsigned)p.chunks;
  const int tile = (int)(id % (unsigned)p.token_tiles);
  id /= (unsigned)p.token_tiles;
  const int64_t h = id % (unsigned)x.Hk, b = id / (unsigned)x.Hk;
  const int n0 = tile * p.tokens_each, tokens = min(p.tokens_each, (int)x.N - n0);
  // the last block that any of the tokens sees
  int64_t last = -1;
  for (int i = 0; i < tokens; ++i) last = max(last, token_position(x, b, n0 + i));
  const int64_t begin = (int64_t)chunk * 64 * p.steps, end = min(x.width, begin + 64 * p.steps), seen = min(end, (last >> x.page_log2) + 1);
  float *to = x.scores + ((b * x.Hk + h) * x.N + n0) * x.width;
  if (last < 0 || begin >= seen) {
    if (x.all_scores)
      for (int64_t i = begin + tid; i < end; i += 256)
        for (int t = 0; t < tokens; ++t) to[t * x.width + i] = -INFINITY;
    return;
  }
  const i32x4 ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
  for (int rb = 0; rb < p.row_blocks; ++rb) {
    const int nrows = min(16, (p.row_blocks > 1 ? p.G - 16 * rb : tokens * p.G));
    if (rb > 0) __syncthreads();   // the rows before are done with
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int row = ps * TPP + tid / LPT, sub = tid % LPT, r = 16 * rb + min(row, nrows - 1), i = r / p.G;
      const int64_t off = b * x.sq[0] + (h * p.G + r - i * p.G) * x.sq[1] + (n0 + i) * x.sq[2] + sub * 8;
      float v[8];
      if (x.q_dtype == QFA_F32) Load8<float>::run(static_cast<const float *>(x.q) + off, v);
      else if (x.q_dtype == QFA_BF16) Load8<__bf16>::run(static_cast<const __bf16 *>(x.q) + off, v);
      else Load8<_Float16>::run(static_cast<const _Float16 *>(x.q) + off, v);
      const QuantRow<8> q = quant_row<LPT, false, 8>(v, true);
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
        *reinterpret_cast<u32x2 *>(&codes[0][row * D + sub * 8]) = u32x2{plus[0], plus[1]};
        *reinterpret_cast<u32x2 *>(&codes[1][row * D + sub * 8]) = u32x2{minus[0], minus[1]};
        if (sub == 0) {
          scale[row] = q.scale;
          sums[0][row] = sp;
          sums[1][row] = sm;
        }
      }
    }
    __syncthreads();
    i32x4 qf[2][KM];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int m = 0; m < KM; ++m) qf[s][m] = *reinterpret_cast<const i32x4 *>(&codes[s][c16 * D + 64 * m + 16 * g]);
    float sq[4];
    int sum[2][4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      sq[v] = scale[4 * g + v];
      sum[0][v] = sums[0][4 * g + v];
      sum[1][v] = sums[1][4 * g + v];
    }
    for (int step = 0; step < p.steps; ++step) {
      const int64_t j0 = begin + 64 * step + 16 * wave, j = j0 + c16;
      if (j0 >= seen) break;   // (uniform over the wave; no barrier follows inside)
      const int64_t page = x.page_table[b * x.stb + min(j, x.width - 1) * x.stw];
      const bool there = j < x.width && page >= 0 && page < x.pages;
      const int64_t at = 2 * ((there ? page : 0) * x.Hk + h);
      i32x4 k[2][KM];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int m = 0; m < KM; ++m) k[s][m] = *reinterpret_cast<const i32x4 *>(x.codes + (at + s) * D + 64 * m + 16 * g);
      const f32x2 sk = *reinterpret_cast<const f32x2 *>(x.scale + at);
      const unsigned zk = *reinterpret_cast<const unsigned short *>(x.zero + at);
      i32x4 dot[2], own[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        dot[s] = own[s] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < KM; ++m) {   // e+ with the high row, e- with the low one
          dot[s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(qf[1 - s][m], k[s][m], dot[s], 0, 0, 0);
          own[s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(ones, k[s][m], own[s], 0, 0, 0);
        }
      }
      const int zl = (int)(signed char)zk, zh = (int)(signed char)(zk >> 8);
      const double sl = sk[0], sh = sk[1];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int ih = dot[1][v] + 128 * own[1][v] - zh * sum[0][v], il = dot[0][v] + 128 * own[0][v] - zl * sum[1][v];
        const double u = (sh * (double)ih - sl * (double)il) * (double)sq[v];
        out[wave][4 * g + v][c16] = (float)u;
      }
      // ---- of a token's heads the largest
      __builtin_amdgcn_wave_barrier();   // (the wave reads what it wrote itself)
      const int outs = p.row_blocks > 1 ? 16 : tokens * 16;
      for (int o = lane; o < outs; o += 64) {
        const int t = o / 16, c = o % 16;
        const int64_t jc = j0 + c;
        float best = -FLT_MAX;   // (what is not a number counts as the least)
        const int rows = p.row_blocks > 1 ? nrows : p.G;
        for (int r = 0; r < rows; ++r) best = fmaxf(best, out[wave][t * p.G + r][c]);
        if (jc >= end) continue;
        const int64_t pos = token_position(x, b, n0 + t), id_c = x.page_table[b * x.stb + jc * x.stw];
        const bool candidate = pos >= 0 && jc <= pos >> x.page_log2 && id_c >= 0 && id_c < x.pages;
        if (rb > 0) best = fmaxf(best, to[t * x.width + jc]);   // (this lane wrote it)
        to[t * x.width + jc] = candidate ? best : -INFINITY;
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  if (x.all_scores)   // blocks behind the last one that is seen, of waves that have left the loop above
    for (int64_t i = (seen + 15) / 16 * 16 + tid; i < end; i += 256)
      for (int t = 0; t < tokens; ++t) to[t * x.width + i] = -INFINITY;
}

// ------------------------------------------------------------------------------------------------------------- the best
constexpr int SELECT_THREADS = 256;
__global__ __launch_bounds__(SELECT_THREADS) void block_select_kernel(PagedSelectArgs x) {
  __shared__ TopSearch<SELECT_THREADS, 8> top;
  const int64_t item = blockIdx.x, bh = index_div(item, x.N), n = item - bh * x.N, b = index_div(bh, x.Hk);
  const int64_t pos = token_position(x, b, n);
  const int mine = pos < 0 ? -1 : (int)min(pos >> x.page_log2, x.width - 1), blocks = mine + 1, keep = (int)x.keep;
  const float *scores = x.scores + item * x.width;
  int32_t *to = x.blocks + item * keep;
  const int64_t own = pos >> x.page_log2;   // (past the table's width: the last blocks are counted from there)
  unsigned taken = 0;
  if (blocks > 0) {
    auto key = [&](int i) __attribute__((always_inline)) -> unsigned {
      const float s = scores[i];
      const bool always = (i < x.first) | (i > own - x.last);
      return s == -INFINITY ? 0u : always ? TOP_ALWAYS : top_key(s);
    };
    unsigned at, equal;
    top.threshold(blocks, (unsigned)min(keep, blocks), key, at, equal);
    taken = top.walk(blocks, at, at == 0u ? 0u : equal, key, [&](unsigned place, int i) __attribute__((always_inline)) { to[place] = i; });
  }
  for (int i = (int)taken + (int)threadIdx.x; i < keep; i += SELECT_THREADS) to[i] = -1;
}

int launch_paged_select(const PagedSelectArgs &x, hipStream_t st) {
  SelectKernelArgs p;
  p.x = x;
  p.G = (int)(x.H / x.Hk);
  p.tokens_each = p.G >= 16 ? 1 : (int)min((int64_t)(16 / p.G), x.N);
  p.token_tiles = (int)((x.N + p.tokens_each - 1) / p.tokens_each);
  p.row_blocks = (p.G + 15) / 16;
  const int64_t groups = x.B * x.Hk * p.token_tiles;
  p.steps = 1;
  while (p.steps < 8 && groups * ((x.width + 128 * p.steps - 1) / (128 * p.steps)) >= 1024) p.steps *= 2;
  p.chunks = (int)((x.width + 64 * p.steps - 1) / (64 * p.steps));
  const double most = (double)groups * p.chunks, items = (double)x.B * (double)x.Hk * (double)x.N;
  if (most > 2147483647.0 || items > 2147483647.0) return set_error(QFA_EUNSUPPORTED, "paged_select: too many tokens and blocks for one launch");
  const dim3 grid((unsigned)(groups * p.chunks)), block(256);
  if (x.D == 64) block_scores_kernel<64><<<grid, block, 0, st>>>(p);
  else if (x.D == 128) block_scores_kernel<128><<<grid, block, 0, st>>>(p);
  else block_scores_kernel<256><<<grid, block, 0, st>>>(p);
  if (int e = check_launch("qfa_paged_select (scores)")) return e;
  block_select_kernel<<<dim3((unsigned)(x.B * x.Hk * x.N)), dim3(SELECT_THREADS), 0, st>>>(x);
  return check_launch("qfa_paged_select");
}

}  // namespace qfa
