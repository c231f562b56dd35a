// Attention of up to 16 rows on the pages of an INT8 cache: the kernel, and the sum of the pieces that its workgroups leave.
// What it computes and why so: qfa_paged_attn.hip, where sequences read all their keys; qfa_paged_list.hip, where every token has a
// list of blocks.  Both are compiled with -ffp-contract=off (see qfa_quant_row.h).
#pragma once
#include "qfa_host.h"
#include "qfa_merge.h"
#include "qfa_paged_attn.h"
#include "qfa_quant_row.h"
#include "qfa_skv_common.h"

namespace qfa {

constexpr int PAGED_ROWS = 16;
constexpr int PAGED_WGS = 256 * 2;   // two on a CU

__device__ __forceinline__ i32x4 paged_mfma_i8(i32x4 a, i32x4 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

// the binary16 number of a small whole number; 1152 less than two of them; what two numbers have beside their binary16 parts, as such parts
__device__ __forceinline__ unsigned half_of(int x) { return (unsigned)__builtin_bit_cast(unsigned short, (_Float16)(short)x); }
__device__ __forceinline__ unsigned without_offset(unsigned two) {
  const f16x2 x = __builtin_bit_cast(f16x2, two), offset = {(_Float16)1152.f, (_Float16)1152.f};
  return __builtin_bit_cast(unsigned, x - offset);
}
__device__ __forceinline__ unsigned rest_h2(float x, float y, unsigned parts) {
  const f16x2 p = __builtin_bit_cast(f16x2, parts);
  return pack_h2(x - (float)p[0], y - (float)p[1]);
}

// Deal: how the work is dealt -- PagedDeal, every sequence's keys from a place on, or PagedListDeal, those of listed blocks.
// FINE: p' in two binary16 parts, 22 bits, and codes without an offset, for queries in fp32 on lists: one part is 2^-11 off, and the offset takes 10 bits of the sums
template <typename S, int D, typename Deal, bool STREAM, bool FINE = false> __global__ __launch_bounds__(256, 2) void paged_rows_kernel(PagedAttnKernelArgs a) {
  constexpr bool SHARED = Deal::ONE_PROBLEM, LIST = Deal::LIST;
  constexpr int KM = D / 64;    // 64-wide k-steps of the score product
  constexpr int DB = D / 16;    // 16-row blocks of O^T
  constexpr int VB = D / 16;    // bytes of a V row per lane
  constexpr int VD = VB / 4;    // ... in dwords
  constexpr int HINT = STREAM ? LOAD_ONCE : 0;
  constexpr int LPT = D / 8, TPP = 256 / LPT;   // quantizer: lanes per token, tokens per pass
  // LDS: query codes and constants, per-wave token constants; the merge of the four waves overlays them
  constexpr int OFF_ST = 16 * D, OFF_TC = OFF_ST + 3 * 16 * 4, MERGE = 4 * 16 * (D + 2) * 4;
  constexpr int TC = 512 + 128;   // per wave: [64] x (scale, zero point operand), exponents of the 32 values' scales
  constexpr int TOTAL = MERGE > OFF_TC + 4 * TC ? MERGE : OFF_TC + 4 * TC;
  __shared__ __attribute__((aligned(16))) unsigned char smem[TOTAL];

  Deal deal(a.work, PAGED_ROWS, SKV_TILE);
  if constexpr (LIST) deal.lists(a.list_tiles, a.list_each);
  unsigned x;
  typename Deal::Item item;
  if (!deal.find(x, item)) return;
  const unsigned x_end = min((deal.workgroup() + 1) * deal.each, deal.total);
  if (x >= x_end) return;
  const int tid = threadIdx.x, lane = tid % 64, q16 = lane % 16, G = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);

  struct Tile {
    i32x4 k[2][KM];
    unsigned v[8][VD];
    unsigned sc, zp;   // scale (its bits) and zero point: lanes 0-31 of key lane, lanes 32-63 of value lane - 32
    int ok;            // bit per half: its page exists
    int key[LIST ? 2 : 1];   // of a list: the position of each half's first key
  };
  const int k_off = q16 * D + 16 * G, v_off = 4 * G * D + VB * q16;
  const S *sc_base = reinterpret_cast<const S *>(lane < 32 ? a.ks : a.vs);
  const int8_t *zp_base = lane < 32 ? a.kz : a.vz;
  const int page_halves_log2 = a.page_log2 - 4;
  const i32x4 ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
  unsigned *tc = reinterpret_cast<unsigned *>(smem + OFF_TC + wave * TC);

  for (;;) {
    const int ntiles = (int)min(item.tiles - item.at, x_end - x);
    const int t0 = deal.begin() / SKV_TILE + (int)item.at;
    int my_tiles = ntiles > wave ? (ntiles - wave + 3) / 4 : 0;
    const int32_t *list = nullptr;
    int last_of_list = -1;   // the last key that the item's token sees
    if constexpr (LIST) {
      list = a.blocks + ((int64_t)deal.row(item.p, item.h, 0).b * a.work.Hk + item.h) * a.work.N * a.keep + (int64_t)deal.row(item.p, item.h, 0).i * a.keep;
      last_of_list = deal.last_key(deal.row(item.p, item.h, 0), item.s);
    }
    const int seq = SHARED ? 0 : LIST ? deal.row(item.p, item.h, 0).b : item.p;   // whose pages
    const int nrows = min(PAGED_ROWS, deal.rows - PAGED_ROWS * item.rb);

    // pages of this wave's tiles: lane 2 i + half of tile i of 32 (a place past the last one is read as the last one, and counts for nothing:
    // no branch that some lanes take, see qfa_paged_work.h)
    auto pages_from = [&](int i0, int &pos) __attribute__((always_inline)) -> int {
      const int i = i0 + lane / 2, half = 2 * (t0 + wave + 4 * i) + lane % 2;
      int at = half >> page_halves_log2;
      if constexpr (LIST) {
        const int block = list[min(at, a.keep - 1)];
        const bool listed = (at < a.keep) & (block >= 0) & (block < a.width);
        at = listed ? block : a.width;
        pos = listed ? (block << a.page_log2) + ((half & ((1 << page_halves_log2) - 1)) << 4) : 0;
      }
      const int id = a.page_table[seq * a.stb + min(at, a.width - 1) * a.stw];
      const bool there = (i < my_tiles) & (at < a.width) & (id >= 0) & (id < a.pages);
      return there ? id : -1;
    };
    int pos = 0, pos_next = 0;   // of a list: where the halves' keys begin
    int pg = pages_from(0, pos), pg_next = my_tiles > 32 ? pages_from(32, pos_next) : -1;
    if constexpr (LIST) {   // nothing is done for what stands behind a short list's blocks
      const uint64_t there = __builtin_amdgcn_ballot_w64((pg >= 0) & (pos <= last_of_list));
      if (my_tiles <= 32) my_tiles = there != 0 ? (63 - __builtin_clzll(there)) / 2 + 1 : 0;
    }
    // (every load is issued whether the tile exists or not -- a missing one has an empty descriptor and fetches nothing)
    int64_t first[2];   // first row of each half among all rows
    auto load_keys = [&](Tile &t, int i) __attribute__((always_inline)) {
      if (i > 0 && i % 32 == 0) {
        pg = pg_next;
        pos = pos_next;
        pg_next = i + 32 < my_tiles ? pages_from(i + 32, pos_next) : -1;
      }
      const int tile = t0 + wave + 4 * i;
      t.ok = 0;
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        const int id = __builtin_amdgcn_readlane(pg, 2 * (i % 32) + rb);
        bool ok = id >= 0;
        if constexpr (LIST) {
          t.key[rb] = __builtin_amdgcn_readlane(pos, 2 * (i % 32) + rb);
          ok = ok & (t.key[rb] <= last_of_list);
        }
        t.ok |= ok ? 1 << rb : 0;
        first[rb] = (((int64_t)(ok ? id : 0) * a.work.Hk + item.h) << a.page_log2) + (((2 * tile + rb) & ((1 << page_halves_log2) - 1)) << 4);
        const rsrc_t rk = make_rsrc(a.kc + first[rb] * D, ok ? 16 * D : 0);
#pragma unroll
        for (int m = 0; m < KM; ++m)
          t.k[rb][m] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off, 64 * m, HINT));
      }
      const int64_t at = (lane % 32 < 16 ? first[0] : first[1]) + lane % 16;
      if constexpr (sizeof(S) == 4) t.sc = __builtin_bit_cast(unsigned, sc_base[at]);
      else t.sc = __builtin_bit_cast(unsigned short, sc_base[at]);
      t.zp = (unsigned)(unsigned char)zp_base[at];
    };
    auto load_values = [&](Tile &t) __attribute__((always_inline)) {
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        const rsrc_t rv = make_rsrc(a.vc + first[rb] * D, t.ok >> rb & 1 ? 16 * D : 0);
#pragma unroll
        for (int e = 4 * rb; e < 4 * rb + 4; ++e) {
          const int soff = (e % 4) * D;
          if constexpr (VD == 4) {
            const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, v_off, soff, HINT));
#pragma unroll
            for (int y = 0; y < 4; ++y) t.v[e][y] = w[y];
          } else if constexpr (VD == 2) {
            const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rv, v_off, soff, HINT));
            t.v[e][0] = w[0];
            t.v[e][1] = w[1];
          } else {
            t.v[e][0] = (unsigned)__builtin_amdgcn_raw_buffer_load_b32(rv, v_off, soff, HINT);
          }
        }
      }
    };
    auto load = [&](Tile &t, int i) __attribute__((always_inline)) {
      load_keys(t, i);
      load_values(t);
    };

    // the block's queries are requested beside the pages, and quantized while the first keys are on their way
    constexpr int PASSES = (16 + TPP - 1) / TPP;
    float qv[PASSES][8];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int tok = p * TPP + tid / LPT, sub = tid % LPT;
      const auto r = deal.row(item.p, item.h, PAGED_ROWS * item.rb + min(tok, nrows - 1));
      const int64_t off = r.b * a.sqb + r.qh * a.sqh + r.i * a.sqn + sub * 8;
      if (a.q_dtype == QFA_F32) Load8<float>::run(static_cast<const float *>(a.q) + off, qv[p]);
      else if (a.q_dtype == QFA_BF16) Load8<__bf16>::run(static_cast<const __bf16 *>(a.q) + off, qv[p]);
      else Load8<_Float16>::run(static_cast<const _Float16 *>(a.q) + off, qv[p]);
    }
    // last key of this lane's row; a row that is not there, or brings no token, goes along with the others and is not looked at
    // (Without a branch that some lanes take, see qfa_paged_work.h.)
    const int lo = deal.begin();
    int lim = last_of_list;   // (of a list: all rows are the same token's)
    if constexpr (!LIST) {
      const int block_end = deal.end(item.s, item.rb) - 1;
      const auto r = deal.row(item.p, item.h, PAGED_ROWS * item.rb + min(q16, nrows - 1));
      const PagedSeq s = SHARED ? deal.load(r.b) : item.s;
      const int key = deal.last_key(r, s);
      const bool seen = (q16 < nrows) & (r.i < s.tokens);
      lim = seen ? key : block_end;
    }

    Tile ta;
    load(ta, 0);

    // ---- the block's queries, quantized: codes to LDS, a = scale * sm_scale * log2(e), zero point and c = sum - D * zp
    float *st_a = reinterpret_cast<float *>(smem + OFF_ST);
    int *st_z = reinterpret_cast<int *>(smem + OFF_ST + 64), *st_c = reinterpret_cast<int *>(smem + OFF_ST + 128);
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int tok = p * TPP + tid / LPT, sub = tid % LPT;
      const QuantRow<8> row = quant_row<LPT, false, 8>(qv[p], true);
      if (tok < 16) {
        *reinterpret_cast<u32x2 *>(smem + tok * D + sub * 8) = u32x2{row.codes[0], row.codes[1]};
        if (sub == 0) {
          const float f = row.scale * a.sm_scale_log2;
          st_a[tok] = f < 0x1p-126f ? 0x1p-126f : f;   // (not zero: the mask's -inf is multiplied by it)
          st_z[tok] = (int)row.zp;
          st_c[tok] = row.sum - D * (int)row.zp;
        }
      }
    }
    __syncthreads();
    i32x4 qf[KM];
#pragma unroll
    for (int m = 0; m < KM; ++m) qf[m] = *reinterpret_cast<const i32x4 *>(smem + q16 * D + 64 * m + 16 * G);
    const float a_i = st_a[q16];
    const int zq = st_z[q16], c_i = st_c[q16];
    int first_lim = lim;
    if constexpr (!LIST) {
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) first_lim = min(first_lim, __shfl_xor(first_lim, off, 64));
    }
    first_lim = __builtin_amdgcn_readfirstlane(first_lim);

    f32x4 oacc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) oacc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ref = NO_KEY, l_run = 0.f, w_run = 0.f;   // p = 2^(a_i * u - ref)

    // next: called once the tile's keys are done with
    auto tile = [&](Tile &t, int i, auto next) __attribute__((always_inline)) {
      const int there = t.ok, t_key[2] = {t.key[0], t.key[LIST ? 1 : 0]};   // (next may load into t)
      const int key0 = (t0 + wave + 4 * i) * SKV_TILE;
      // token constants: K (scale, zp as an integer), V (scale, the binary16 number 1152 + zp)
      {
        u32x2 w;
        w[0] = __builtin_bit_cast(unsigned, scale_to_f32<S>(t.sc));
        w[1] = lane < 32 ? (unsigned)(int)(signed char)t.zp : FINE ? half_of((int)(signed char)t.zp) : (0x6400u | (t.zp ^ 0x80u));
        *reinterpret_cast<u32x2 *>(tc + 2 * lane) = w;
      }
      // ---- scores of keys 16rb + 4G + v
      f32x4 f[2];
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        i32x4 s = {0, 0, 0, 0}, rk = {0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < KM; ++m) {
          s = paged_mfma_i8(t.k[rb][m], qf[m], s);
          rk = paged_mfma_i8(t.k[rb][m], ones, rk);
        }
        const u32x4 c0 = *reinterpret_cast<const u32x4 *>(tc + 2 * (16 * rb + 4 * G)),
                    c1 = *reinterpret_cast<const u32x4 *>(tc + 2 * (16 * rb + 4 * G) + 4);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const unsigned scw = v < 2 ? c0[2 * v] : c1[2 * v - 4], zw = v < 2 ? c0[2 * v + 1] : c1[2 * v - 3];
          const int dot = s[v] - __mul24(zq, rk[v]) - __mul24((int)zw, c_i);
          f[rb][v] = (float)dot * __builtin_bit_cast(float, scw);
        }
      }
      next();
      if constexpr (LIST) {
        if (t_key[0] > first_lim - 15 || t_key[1] > first_lim - 15 || there != 3) {
#pragma unroll
          for (int rb = 0; rb < 2; ++rb)
#pragma unroll
            for (int v = 0; v < 4; ++v)
              if (4 * G + v > first_lim - t_key[rb] || !(there >> rb & 1)) f[rb][v] = -INFINITY;
        }
      } else if (key0 + SKV_TILE - 1 > first_lim || key0 < lo || there != 3) {
        const int last = lim - key0 - 4 * G, first = lo - key0 - 4 * G;   // (this lane's keys are key0 + 4 G + 16 rb + v)
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            if (16 * rb + v > last || 16 * rb + v < first || !(there >> rb & 1)) f[rb][v] = -INFINITY;
      }
      // ---- p and its row sum, p' = p * scale_j and the largest of them
      float ps[8], mx = 0.f, l_new = 0.f;
      unsigned zz[4];   // the binary16 numbers 1152 + zero point
      u32x4 cv[4];      // keys 16(x/2) + 4G + 2(x%2) + {0, 1}: scale, 1152 + zero point, and again
#pragma unroll
      for (int y = 0; y < 4; ++y) cv[y] = *reinterpret_cast<const u32x4 *>(tc + 2 * (32 + 16 * (y / 2) + 4 * G + 2 * (y % 2)));
      auto probs = [&]() __attribute__((always_inline)) {
        mx = 0.f;
        l_new = l_run;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const unsigned s0 = cv[y][0], z0 = cv[y][1], s1 = cv[y][2], z1 = cv[y][3];   // (a bit cast of a vector's element takes element 0)
          zz[y] = z0 | (z1 << 16);
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(a_i, f[y / 2][2 * (y % 2)], -ref));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(a_i, f[y / 2][2 * (y % 2) + 1], -ref));
          l_new += p0 + p1;
          ps[2 * y] = mul_zero_wins(p0, __builtin_bit_cast(float, s0));   // (what is hidden may hold any scale)
          ps[2 * y + 1] = mul_zero_wins(p1, __builtin_bit_cast(float, s1));
          mx = fmaxf(mx, fmaxf(fabsf(ps[2 * y]), fabsf(ps[2 * y + 1])));
        }
      };
      // a new reference, common to the four lanes of a row: log2 of the tile's largest p' (and p itself within fp32), but for the
      // scale's mantissa
      auto move = [&]() __attribute__((always_inline)) -> float {
        float *tl = reinterpret_cast<float *>(tc + 128);
        if (lane >= 32) tl[lane - 32] = __builtin_floorf(__builtin_amdgcn_logf(fabsf((*reinterpret_cast<const f32x2 *>(tc + 2 * lane))[0])));
        float t_max = -INFINITY, u = -INFINITY;
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
          const f32x4 ls = *reinterpret_cast<const f32x4 *>(tl + 16 * rb + 4 * G);
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            t_max = fmaxf(t_max, !(f[rb][v] > -INFINITY) ? -INFINITY : __builtin_fmaf(a_i, f[rb][v], ls[v]));
            u = fmaxf(u, f[rb][v]);
          }
        }
        t_max = fmaxf(t_max - PAGED_P_REF, __builtin_fmaf(a_i, u, -100.0f));
        t_max = fmaxf(t_max, __shfl_xor(t_max, 16, 64));
        t_max = fmaxf(t_max, __shfl_xor(t_max, 32, 64));
        t_max = fmaxf(t_max, ref);
        const float alpha = __builtin_amdgcn_exp2f(ref - t_max);
        ref = t_max;
        return alpha;
      };
      if (i == 0) move();   // (nothing summed yet)
      probs();
      if (i != 0 && __builtin_amdgcn_ballot_w64(mx > PAGED_P_MAX || !(l_new <= 0x1p100f)) != 0) {
        const float alpha = move();
        l_run *= alpha;
        w_run *= alpha;
#pragma unroll
        for (int j = 0; j < DB; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) oacc[j][v] *= alpha;
        probs();
      }
      l_run = l_new;
      // ---- p' as binary16, offset term
      u32x4 pf, pl;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const unsigned pp = pack_h2(ps[2 * y], ps[2 * y + 1]);
        pf[y] = pp;
        w_run = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pp), __builtin_bit_cast(f16x2, zz[y]), w_run, false);
        if constexpr (FINE) {
          const unsigned rest = rest_h2(ps[2 * y], ps[2 * y + 1], pp);   // (a bit cast of a vector's element takes element 0)
          pl[y] = rest;
          w_run = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, rest), __builtin_bit_cast(f16x2, zz[y]), w_run, false);
        }
      }
      // ---- O^T += (1152 + codes)^T . P'^T
#pragma unroll
      for (int j = 0; j < DB; ++j) {
        u32x4 vf;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          constexpr unsigned pick = 0x0c040c00u;
          vf[e] = __builtin_amdgcn_perm(t.v[2 * e + 1][j / 4], t.v[2 * e][j / 4], pick + (unsigned)(j % 4) * 0x00010001u) ^ 0x64806480u;
          if constexpr (FINE) vf[e] = without_offset(vf[e]);
        }
        oacc[j] = mfma_h16(vf, pf, oacc[j]);
        if constexpr (FINE) oacc[j] = mfma_h16(vf, pl, oacc[j]);
      }
    };
    // Rows of 256 elements: two tiles in registers would leave room for one workgroup on a CU (1 to 12 % slower); a tile's keys and values
    // are requested anew as soon as they are done with
    if constexpr (D == 256) {
      for (int i = 0; i < my_tiles; ++i) {
        tile(ta, i, [&]() __attribute__((always_inline)) { load_keys(ta, i + 1); });
        load_values(ta);
      }
    } else {
      Tile tb;
      for (int i = 0; i < my_tiles; i += 2) {
        load(tb, i + 1);
        tile(ta, i, []() {});
        load(ta, i + 2);
        if (i + 1 < my_tiles) tile(tb, i + 1, []() {});
      }
    }

    // ---- merge of the four waves, through LDS: [wave][row][D] and (m, l) behind
    float l_tot = l_run + __shfl_xor(l_run, 16, 64), w_tot = w_run + __shfl_xor(w_run, 16, 64);
    l_tot += __shfl_xor(l_tot, 32, 64);
    w_tot += __shfl_xor(w_tot, 32, 64);
    __syncthreads();   // query codes and token constants are done with
    float *mg = reinterpret_cast<float *>(smem), *ml = mg + 4 * 16 * D;
    if (q16 < nrows) {
      float *dst = mg + (wave * 16 + q16) * D;
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int j = 0; j < DB; j += 4) {
          f32x4 y;
#pragma unroll
          for (int z = 0; z < 4; ++z) y[z] = oacc[j + z][v] - w_tot;
          *reinterpret_cast<f32x4 *>(dst + VB * (4 * G + v) + j) = y;
        }
      if (G == 0) {
        ml[2 * (wave * 16 + q16)] = ref;
        ml[2 * (wave * 16 + q16) + 1] = l_tot;
      }
    }
    __syncthreads();
    const bool whole = item.at == 0 && ntiles == (int)item.tiles;
    if constexpr (!SHARED && !LIST) {
      if (item.at == 0 && tid == 0) {   // where the pieces are, for those who join them
        a.work.first[2 * deal.item_index(item.p, item.h, item.rb)] = item.first;
        a.work.first[2 * deal.item_index(item.p, item.h, item.rb) + 1] = deal.each;
      }
    }
    const int64_t slot = ((int64_t)deal.workgroup() * 2 + (item.at == 0 ? 1 : 0)) * PAGED_ROWS;
    for (int y = tid; y < nrows * (D / 4); y += 256) {
      const int q = y / (D / 4), d = 4 * (y % (D / 4)), r = PAGED_ROWS * item.rb + q;
      float m = NO_KEY, l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[2 * (16 * w + q)]);
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float s = __builtin_amdgcn_exp2f(ml[2 * (16 * w + q)] - m);
        l += ml[2 * (16 * w + q) + 1] * s;
        const f32x4 z = *reinterpret_cast<const f32x4 *>(mg + (16 * w + q) * D + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += z[e] * s;
      }
      if (whole && !a.work.whole) {
        const auto row = deal.row(item.p, item.h, r);
        const bool none = row.i >= item.s.tokens || l == 0.f;   // (not of a shared prefix)
        const float inv = none ? 0.f : 1.0f / l;
        const f32x4 out = none ? f32x4{0.f, 0.f, 0.f, 0.f} : f32x4{acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
        const int64_t off = (((int64_t)row.b * a.work.Hk * a.work.G + row.qh) * a.work.N + row.i) * D;
        store4(static_cast<char *>(a.o) + off * (a.q_dtype == QFA_F32 ? 4 : 2), a.q_dtype, d, out);
      } else {
        const int64_t to = whole ? ((int64_t)item.p * a.work.Hk + item.h) * deal.rows + r : slot + q;
        float *po = whole ? a.work.whole : a.work.slots, *pml = whole ? a.work.whole_ml : a.work.slots_ml;
        *reinterpret_cast<f32x4 *>(po + to * D + d) = acc;
        if (d == 0) *reinterpret_cast<f32x2 *>(pml + 2 * to) = f32x2{m, l};
      }
    }
    x += (unsigned)ntiles;
    if (x >= x_end || !deal.next(x, x_end, item)) return;
    __syncthreads();   // the merge is read
  }
}

// Where a row's pieces are
struct PagedPieces {
  unsigned w0 = 1, w1 = 0;       // workgroups that have one (none)
  int64_t whole = -1;            // row among the items in one piece
  int in_block = 0;
  __device__ __forceinline__ PagedPieces(unsigned first, unsigned each, unsigned n, int64_t whole_row, int in_block_) {
    if (n == 0) return;
    w0 = first / each;
    w1 = (first + n - 1) / each;
    in_block = in_block_;
    if (w0 == w1) whole = whole_row;
  }
};
struct PagedSum { float m, l; f32x4 acc; };
// Adds a row's pieces, or those of R rows that lie `step` apart in their blocks.  Four are loaded at a time (past the last piece: once more
// that one, which then counts for nothing); one by one, each would wait for its own loads
template <int D, int R> __device__ __forceinline__ void paged_add(const PagedWork &work, const PagedPieces &at, int d, int group, int groups, PagedSum (&x)[R],
                                                                  int step) {
  constexpr int AT_ONCE = 4 / R;
  const float *po = at.whole >= 0 ? work.whole : work.slots, *pml = at.whole >= 0 ? work.whole_ml : work.slots_ml;
  for (unsigned w = at.w0 + group; w <= at.w1; w += AT_ONCE * groups) {
    f32x2 ml[R][AT_ONCE];
    f32x4 y[R][AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const unsigned wj = min(w + j * groups, at.w1);
      const int64_t i = at.whole >= 0 ? at.whole : ((int64_t)wj * 2 + (wj == at.w0 ? 1 : 0)) * work.br + at.in_block;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        ml[r][j] = *reinterpret_cast<const f32x2 *>(pml + 2 * (i + r * step));
        y[r][j] = *reinterpret_cast<const f32x4 *>(po + (i + r * step) * D + d);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float m_new = x[r].m;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const float l = ml[r][j][1];
        if ((w + j * groups > at.w1) | (l == 0.f)) ml[r][j] = f32x2{NO_KEY, 0.f};   // (a piece that saw no key: its sums are zero)
        m_new = fmaxf(m_new, ml[r][j][0]);
      }
      const float s0 = __builtin_amdgcn_exp2f(x[r].m - m_new);
      x[r].m = m_new;
      x[r].l *= s0;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[r].acc[e] *= s0;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const float l = ml[r][j][1], s1 = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[r][j][0] - m_new);
        x[r].l += l * s1;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[r].acc[e] += mul_zero_wins(s1, y[r][j][e]);
      }
    }
  }
}

}  // namespace qfa
