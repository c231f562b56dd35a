// Attention of the queries at the end of every sequence of a batch on the pages of an INT8 cache:
//     O = softmax(sm_scale * Q^ K^^T) V^,   X^ = scale * (codes - zero_point) per token,
// with the arithmetic of the kernel for a cache in one piece (qfa_cache.hip): queries quantized per token here, Q K^T on INT8
// MFMA with the exact zero-point term, V as its exact codes in binary16, softmax statistics and sums in fp32.
//
// Bound by reading the cache once (2 D + 6 bytes per key and key head): 64 sequences of 65 to 8192 keys, 8 key heads of 128, 550 MB in
// 99 us (5.6 TB/s); of short work the start, where lengths, page numbers and keys are three loads that wait for each other (4 us), and
// the kernel that joins the pieces (5 us): 16 heads of 16384 keys 22 us.  A workgroup = 4 waves = 16 rows (queries times the
// query heads that share a key head) of one sequence and key head, and a piece of its keys (qfa_paged_work.h); 32-key tiles are
// dealt to the waves, each with its own online softmax.  A tile lives in registers, double-buffered (but for 256 elements) as there.  A page holds 16
// keys or a multiple, so the two halves of a tile lie in one page each: their pages' numbers are fetched 32 tiles ahead, one
// lane per half, and read out of the lanes as scalars, so that no load of keys waits for the page table.
//
// What the mask hides may hold anything (pages that were never written): its scores are replaced, its probability is zero and
// zero wins over whatever its scale holds.
#include "qfa_host.h"
#include "qfa_merge.h"
#include "qfa_paged_attn.h"
#include "qfa_quant_row.h"
#include "qfa_skv_common.h"

namespace qfa {

constexpr int PAGED_ROWS = 16;
constexpr int PAGED_WGS = 256 * 2;   // two on a CU

__device__ __forceinline__ i32x4 paged_mfma_i8(i32x4 a, i32x4 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

template <typename S, int D, bool SHARED, bool ONE, bool STREAM> __global__ __launch_bounds__(256, 2) void paged_rows_kernel(PagedAttnKernelArgs a) {
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

  typedef PagedDeal<SHARED, ONE> Deal;
  Deal deal(a.work, PAGED_ROWS, SKV_TILE);
  unsigned x;
  typename Deal::Item item;
  if (!deal.find(x, item)) return;
  const unsigned x_end = min((blockIdx.x + 1) * deal.each, deal.total);
  if (x >= x_end) return;
  const int tid = threadIdx.x, lane = tid % 64, q16 = lane % 16, G = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);

  struct Tile {
    i32x4 k[2][KM];
    unsigned v[8][VD];
    unsigned sc, zp;   // scale (its bits) and zero point: lanes 0-31 of key lane, lanes 32-63 of value lane - 32
    int ok;            // bit per half: its page exists
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
    const int my_tiles = ntiles > wave ? (ntiles - wave + 3) / 4 : 0;
    const int seq = SHARED ? 0 : item.p;   // whose pages
    const int nrows = min(PAGED_ROWS, deal.rows - PAGED_ROWS * item.rb);

    // pages of this wave's tiles: lane 2 i + half of tile i of 32 (a place past the last one is read as the last one, and counts for nothing:
    // no branch that some lanes take, see qfa_paged_work.h)
    auto pages_from = [&](int i0) __attribute__((always_inline)) -> int {
      const int i = i0 + lane / 2, half = 2 * (t0 + wave + 4 * i) + lane % 2, at = half >> page_halves_log2;
      const int id = a.page_table[seq * a.stb + min(at, a.width - 1) * a.stw];
      const bool there = (i < my_tiles) & (at < a.width) & (id >= 0) & (id < a.pages);
      return there ? id : -1;
    };
    int pg = pages_from(0), pg_next = my_tiles > 32 ? pages_from(32) : -1;
    // (every load is issued whether the tile exists or not -- a missing one has an empty descriptor and fetches nothing)
    int64_t first[2];   // first row of each half among all rows
    auto load_keys = [&](Tile &t, int i) __attribute__((always_inline)) {
      if (i > 0 && i % 32 == 0) {
        pg = pg_next;
        pg_next = i + 32 < my_tiles ? pages_from(i + 32) : -1;
      }
      const int tile = t0 + wave + 4 * i;
      t.ok = 0;
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        const int id = __builtin_amdgcn_readlane(pg, 2 * (i % 32) + rb);
        const bool ok = id >= 0;
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
    const int block_end = deal.end(item.s, item.rb) - 1, lo = deal.begin();
    int lim;
    {
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
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) first_lim = min(first_lim, __shfl_xor(first_lim, off, 64));
    first_lim = __builtin_amdgcn_readfirstlane(first_lim);

    f32x4 oacc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) oacc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ref = NO_KEY, l_run = 0.f, w_run = 0.f;   // p = 2^(a_i * u - ref)

    // next: called once the tile's keys are done with
    auto tile = [&](Tile &t, int i, auto next) __attribute__((always_inline)) {
      const int there = t.ok;
      const int key0 = (t0 + wave + 4 * i) * SKV_TILE;
      // token constants: K (scale, zp as an integer), V (scale, the binary16 number 1152 + zp)
      {
        u32x2 w;
        w[0] = __builtin_bit_cast(unsigned, scale_to_f32<S>(t.sc));
        w[1] = lane < 32 ? (unsigned)(int)(signed char)t.zp : (0x6400u | (t.zp ^ 0x80u));
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
      if (key0 + SKV_TILE - 1 > first_lim || key0 < lo || there != 3) {
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
      u32x4 pf;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const unsigned pp = pack_h2(ps[2 * y], ps[2 * y + 1]);
        pf[y] = pp;
        w_run = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pp), __builtin_bit_cast(f16x2, zz[y]), w_run, false);
      }
      // ---- O^T += (1152 + codes)^T . P'^T
#pragma unroll
      for (int j = 0; j < DB; ++j) {
        u32x4 vf;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          constexpr unsigned pick = 0x0c040c00u;
          vf[e] = __builtin_amdgcn_perm(t.v[2 * e + 1][j / 4], t.v[2 * e][j / 4], pick + (unsigned)(j % 4) * 0x00010001u) ^ 0x64806480u;
        }
        oacc[j] = mfma_h16(vf, pf, oacc[j]);
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
    if (!SHARED && item.at == 0 && tid == 0) {   // where the pieces are, for those who join them
      a.work.first[2 * deal.item_index(item.p, item.h, item.rb)] = item.first;
      a.work.first[2 * deal.item_index(item.p, item.h, item.rb) + 1] = deal.each;
    }
    const int64_t slot = ((int64_t)blockIdx.x * 2 + (item.at == 0 ? 1 : 0)) * PAGED_ROWS;
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

// O from the pieces of its rows: a workgroup joins up to 16 rows of one sequence and key head, D/4 lanes of four columns each; with
// fewer rows than 1024/D the pieces of a row are dealt to several groups of lanes, which meet in LDS.  Rows that lie in one piece
// have been stored already (no shared prefix); rows that see no key become zeros.
struct PagedMergeArgs {
  PagedWork own, shared;   // shared.grid 0: none
  void *o;
  int o_dtype, chunks, chunk_rows;   // chunks of rows of a sequence and key head, a power of two that divides a block
};
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

template <int D> __global__ __launch_bounds__(256) void paged_merge_kernel(PagedMergeArgs a) {
  constexpr int CL = D / 4, SLOTS = 256 / CL;
  __shared__ float red[SLOTS][D + 4];
  const int tid = threadIdx.x, d = 4 * (tid % CL), slot = tid / CL;
  const PagedDeal<false, false> own(a.own, a.own.br, a.own.tk);
  const int bh = (int)(blockIdx.x / (unsigned)a.chunks), chunk = (int)(blockIdx.x % (unsigned)a.chunks), b = bh / a.own.Hk, h = bh % a.own.Hk;
  const int r0 = chunk * a.chunk_rows, n = min(a.chunk_rows, own.rows - r0), rb = r0 / own.BR;
  const unsigned *note = a.own.first + 2 * own.item_index(b, h, rb), first = note[0], each = max(note[1], 1u);   // (nobody's, without tiles)
  const PagedSeq seq = own.load(b);
  const PagedPieces mine(first, each, own.tiles(seq, rb), (int64_t)bh * own.rows + r0, r0 % own.BR);
  if (!a.own.whole && mine.whole >= 0) return;   // stored
  auto store = [&](int r, const PagedSum &x) __attribute__((always_inline)) {
    const int i = r / a.own.G;
    const float inv = i >= seq.tokens || x.l == 0.f ? 0.f : 1.0f / x.l;
    const int64_t off = (((int64_t)b * a.own.Hk * a.own.G + h * a.own.G + r % a.own.G) * a.own.N + i) * D;
    store4(static_cast<char *>(a.o) + off * (a.o_dtype == QFA_F32 ? 4 : 2), a.o_dtype, d,
           f32x4{mul_zero_wins(x.acc[0], inv), mul_zero_wins(x.acc[1], inv), mul_zero_wins(x.acc[2], inv), mul_zero_wins(x.acc[3], inv)});
  };
  if (n > SLOTS && a.shared.grid == 0) {   // two rows at a time
    for (int k = slot; k < n; k += 2 * SLOTS) {
      PagedSum x[2] = {{NO_KEY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}}, {NO_KEY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}}};
      PagedPieces p = mine;
      p.in_block += k;
      paged_add<D, 2>(a.own, p, d, 0, 1, x, k + SLOTS < n ? SLOTS : 0);
      store(r0 + k, x[0]);
      if (k + SLOTS < n) store(r0 + k + SLOTS, x[1]);
    }
    return;
  }
  const int groups = n >= SLOTS ? 1 : SLOTS / n;   // of pieces
  for (int first = 0; first < n; first += SLOTS) {
    const int k = groups == 1 ? first + slot : slot % n, group = groups == 1 ? 0 : slot / n;   // row of the chunk
    const bool live = k < n && group < groups;
    const int r = r0 + min(k, n - 1), i = r / a.own.G;
    PagedSum x[1] = {{NO_KEY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}}};
    if (live && i < seq.tokens) {
      PagedPieces p = mine;
      p.in_block += r - r0;
      if (p.whole >= 0) p.whole += r - r0;
      paged_add<D, 1>(a.own, p, d, group, groups, x, 0);
      if (a.shared.grid > 0) {
        const PagedDeal<true, false> all(a.shared, a.shared.br, a.shared.tk);
        const int rs = b * own.rows + r, item = h * all.blocks + rs / all.BR;
        const unsigned u = all.units({0, 0}, 0);
        const PagedPieces q((unsigned)item * u + (unsigned)a.shared.extra, all.each, all.tiles({0, 0}, 0), (int64_t)h * all.rows + rs, rs % all.BR);
        paged_add<D, 1>(a.shared, q, d, group, groups, x, 0);
      }
    }
    if (groups > 1) {
      *reinterpret_cast<f32x4 *>(&red[slot][d]) = x[0].acc;
      if (tid % CL == 0) {
        red[slot][D] = x[0].m;
        red[slot][D + 1] = x[0].l;
      }
      __syncthreads();
      if (slot >= n) return;
      x[0] = {NO_KEY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}};
      for (int g = 0; g < groups; ++g) x[0].m = fmaxf(x[0].m, red[g * n + slot][D]);
      for (int g = 0; g < groups; ++g) {
        const float s = __builtin_amdgcn_exp2f(red[g * n + slot][D] - x[0].m);
        x[0].l += red[g * n + slot][D + 1] * s;
        const f32x4 y = *reinterpret_cast<const f32x4 *>(&red[g * n + slot][d]);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[0].acc[e] += y[e] * s;
      }
    } else if (!live) {
      return;
    }
    store(r, x[0]);
  }
}

// Rows of a block, in a launch over `problems` (sequences times key heads) of that many rows: 16, or the tiles' 64 or 128 beyond.
// Two blocks of 16 read the keys twice but need no other launch and leave no wave without rows; 20 rows of 256 elements, 3000 keys
// of 8 sequences: 39 us against 47 on tiles; 32 rows, 8192 keys of one sequence, 128 elements: 23 against 29, of 64 sequences with
// 64 elements 167 against 193, but with 128 elements, where the keys no longer stay in the last cache, 313 against 250.
// (48 rows on three blocks: 68 us against 59.)
static int block_rows(int64_t rows, int D, int64_t problems) {
  if (rows <= PAGED_ROWS || (rows <= 2 * PAGED_ROWS && (D != 128 || problems <= 128))) return PAGED_ROWS;
  return rows <= 64 ? 64 : 128;
}
static int tile_keys(int br) { return br == PAGED_ROWS ? SKV_TILE : PAGED_TILE; }
static int item_units(int br) { return br == PAGED_ROWS ? 12 : 4; }   // beside its tiles, see qfa_paged_work.h
static int work_grid(int br, int D) { return br == PAGED_ROWS ? PAGED_WGS : paged_tile_grid(D); }
// bytes of a launch's slots, and of its whole items
static int64_t slots_bytes(int br, int D) { return 2LL * work_grid(br, D) * br * (D + 2) * 4; }
static int64_t whole_bytes(int64_t rows, int D) { return (rows * (D + 2) * 4 + 15) / 16 * 16; }
static int64_t first_bytes(int64_t problems, int64_t rows, int br) { return (8 * problems * ((rows + br - 1) / br) + 15) / 16 * 16; }
static int64_t quantized_bytes(int64_t rows, int D) { return (rows * D + 4 * rows + rows + 15) / 16 * 16; }
int64_t paged_attn_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t prefix) {
  const int64_t rows = N * (H / Hk);
  const int own = block_rows(rows, D, B * Hk), shared = prefix > 0 ? block_rows(B * rows, D, Hk) : 0;
  int64_t bytes = slots_bytes(own, D) + first_bytes(B * Hk, rows, own);
  if (prefix > 0) bytes += slots_bytes(shared, D) + 2 * whole_bytes(B * H * N, D);
  if (own > PAGED_ROWS || shared > PAGED_ROWS) bytes += quantized_bytes(B * H * N, D);   // (blocks of 16 quantize their own)
  return bytes;
}

// Units of work (qfa_paged_work.h) that a launch of the call has at most, if every sequence fills its `keys` keys
double paged_attn_most_units(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t prefix, int64_t keys) {
  const auto most = [&](int64_t problems, int64_t rows, int64_t n) {
    const int br = block_rows(rows, D, problems);
    return (double)problems * (double)((rows + br - 1) / br) * ((double)n / tile_keys(br) + 2 + item_units(br));
  };
  const double own = most(B * Hk, N * (H / Hk), keys), shared = prefix > 0 ? most(Hk, B * N * (H / Hk), prefix) : 0.0;
  return own > shared ? own : shared;
}

// How long a pass over `keys` keys takes for problems * rows rows beside its start, in us: every block of rows reads them again, at the
// rate (TB/s, of a chip that is full) that its kernel has in its caches
static double pass_us(int64_t problems, int64_t rows, int64_t keys, int D) {
  const int br = block_rows(rows, D, problems);
  const double rate = br == PAGED_ROWS ? 11.0 : br == 64 ? (D == 128 ? 5.5 : 3.75) : (D == 128 ? 3.4 : 2.5);
  return (double)problems * (double)((rows + br - 1) / br) * (double)keys * 2 * D / (rate * 1e6);
}
// Whether a prefix gets a pass of its own.  That one has its start, its queries quantized and results of all rows written and joined
// again against it: where it saves less, every sequence reads the prefix from its own pages.  Of 240 calls timed both ways (4 to 64
// sequences, 1 to 300 rows, prefixes of 400, 2000 and 8000 keys, D 64, 128 and 256) 34 get one: 31 of them take 0.33 to 1.0 of the time
// without and three, of 256 elements, 1.09 to 1.29; of the others 201 take 1.01 to 2.4 of the time with it, five 0.78 to 0.95.
int64_t paged_attn_shared_prefix(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t prefix) {
  const int64_t rows = N * (H / Hk);
  const double start = block_rows(B * rows, D, Hk) == PAGED_ROWS ? 6.0 + D / 64 : 13.0 + 3.5 * (D / 64);
  const double joined = (double)(B * H * N) * (D + 2) * 16 / 4.5e6;   // written twice, read twice
  return B > 1 && pass_us(B * Hk, rows, prefix, D) > pass_us(Hk, B * rows, prefix, D) + start + joined ? prefix : 0;
}

template <typename S, int D, bool SHARED> static int launch_rows(const PagedAttnKernelArgs &a, bool one, bool stream, hipStream_t st) {
  const dim3 grid((unsigned)a.work.grid), block(256);
  if (!one) paged_rows_kernel<S, D, SHARED, false, false><<<grid, block, 0, st>>>(a);
  else if (!SHARED && stream) paged_rows_kernel<S, D, false, true, true><<<grid, block, 0, st>>>(a);
  else paged_rows_kernel<S, D, SHARED, true, false><<<grid, block, 0, st>>>(a);
  return check_launch(SHARED ? "qfa_attn_paged (prefix)" : "qfa_attn_paged");
}
template <typename S, int D> static int launch_rows(const PagedAttnKernelArgs &a, bool shared, bool one, bool stream, hipStream_t st) {
  return shared ? launch_rows<S, D, true>(a, one, stream, st) : launch_rows<S, D, false>(a, one, stream, st);
}
template <int D> static int launch_d(const PagedAttnArgs &x, hipStream_t st) {
  PagedAttnKernelArgs a = {};
  a.q = x.q; a.kc = x.cache.k_codes; a.ks = x.cache.k_scale; a.kz = x.cache.k_zero;
  a.vc = x.cache.v_codes; a.vs = x.cache.v_scale; a.vz = x.cache.v_zero; a.o = x.o; a.page_table = x.page_table;
  a.pages = x.pages; a.stb = x.stb; a.stw = x.stw; a.sqb = x.sq[0]; a.sqh = x.sq[1]; a.sqn = x.sq[2];
  a.width = (int)x.width; a.page_log2 = x.page_log2; a.q_dtype = x.q_dtype;
  a.sm_scale_log2 = x.sm_scale * kLog2e;
  const int G = (int)(x.H / x.Hk);
  const int64_t rows = x.B * x.H * x.N, problem[2] = {x.N * G, x.B * x.N * G};
  PagedWork w[2];
  float *mem = static_cast<float *>(x.workspace);
  for (int i = 0; i < 2; ++i) {
    const int br = block_rows(problem[i], D, (i == 0 ? x.B : 1) * x.Hk), grid = x.prefix > 0 || i == 0 ? work_grid(br, D) : 0;
    w[i] = {x.starts, x.counts, (int)x.B, (int)x.Hk, G, (int)x.N, x.causal, (int)x.prefix, (int)(x.width << x.page_log2), grid, br,
            tile_keys(br), item_units(br), nullptr, nullptr, nullptr, nullptr, nullptr};
    if (grid == 0) continue;
    if (i == 0) {
      w[i].first = reinterpret_cast<unsigned *>(mem);
      mem += first_bytes(x.B * x.Hk, problem[0], br) / 4;
    }
    w[i].slots = mem;
    w[i].slots_ml = mem + 2LL * grid * br * D;
    mem += slots_bytes(br, D) / 4;
    if (x.prefix > 0) {
      w[i].whole = mem;
      w[i].whole_ml = mem + rows * D;
      mem += whole_bytes(rows, D) / 4;
    }
  }
  if (w[0].br > PAGED_ROWS || (w[1].grid > 0 && w[1].br > PAGED_ROWS)) {   // many rows: quantized once, every piece of keys needs them
    int8_t *codes = reinterpret_cast<int8_t *>(mem), *zero = codes + rows * (D + 4);
    float *scale = reinterpret_cast<float *>(codes + rows * D);
    // (one token each: a sequence's heads as tokens of one head, which fill the quantizer's workgroups)
    const bool one = x.N == 1;
    if (int e = launch_quant(x.q, x.q_dtype, codes, scale, nullptr, 0, zero, nullptr, x.B, one ? 1 : x.H, one ? x.H : x.N, D, x.sq[0], one ? x.sq[2] : x.sq[1],
                             one ? x.sq[1] : x.sq[2], x.H * x.N * D, one ? D : x.N * D, D, st))
      return e;
    a.q_codes = codes; a.q_scale = scale; a.q_zero = zero;
  }
  // Non-temporal loads (LOAD_ONCE) where the keys and values that a call may reach outgrow the last-level cache (256 MiB) for good.  One token
  // of 64 sequences, 8 key heads of 64, 128 and 256 elements, us with plain loads and with these: 128 MiB 29.1, 27.4, 28.4 and 28.8, 28.1,
  // 28.3; 256 MiB 49.2, 46.3, 47.4 and 49.7, 48.1, 47.7; 320 MiB 65.4, 61.5, 62.1 and 60.8, 58.1, 57.1; 512 MiB 105, 99, 100 and 93, 88, 87.
  // The lengths are not known here: short sequences under a table of 4 GiB are read with these too, 16 to 128 MiB of them in the same time
  // and 256 in 49.0 us in place of 46.7.  Two blocks of rows, which read every key twice, keep plain loads (20 rows, 512 MiB, 64, 128 and 256
  // elements: 200, 176 and 191 us; with these 180, 182 and 181).
  const bool stream = (double)(x.pages < x.B * x.width ? x.pages : x.B * x.width) * (double)(x.Hk << x.page_log2) * 2 * D >= 320.0 * (1 << 20);
  for (int i = 1; i >= 0; --i) {
    if (w[i].grid == 0) continue;
    a.work = w[i];
    int e;
    if (w[i].br > PAGED_ROWS) e = launch_paged_tile(a, i == 1, D, x.scale_dtype, w[i].br / 32, st);
    else if (x.scale_dtype == QFA_F32) e = launch_rows<float, D>(a, i == 1, problem[i] <= PAGED_ROWS, stream, st);
    else if (x.scale_dtype == QFA_F16) e = launch_rows<_Float16, D>(a, i == 1, problem[i] <= PAGED_ROWS, stream, st);
    else e = launch_rows<__bf16, D>(a, i == 1, problem[i] <= PAGED_ROWS, stream, st);
    if (e) return e;
  }
  // rows per workgroup: few, whose pieces many lanes share, while that leaves no more than 1024 workgroups (2048 rows one by one: 9.4 us
  // against 6.4 two by two, with a prefix 12.9 against 10.5; in 512 workgroups 5.7 and 11.4)
  int chunk_rows = 1;
  while (chunk_rows < 16 && x.B * x.Hk * ((problem[0] + chunk_rows - 1) / chunk_rows) > 1024) chunk_rows *= 2;
  const int chunks = (int)((problem[0] + chunk_rows - 1) / chunk_rows);
  const PagedMergeArgs m = {w[0], w[1], x.o, x.q_dtype, chunks, chunk_rows};
  paged_merge_kernel<D><<<dim3((unsigned)(x.B * x.Hk * chunks)), dim3(256), 0, st>>>(m);
  return check_launch("qfa_attn_paged (merge)");
}
int launch_paged_attn(const PagedAttnArgs &x, hipStream_t st) {
  if (x.D == 64) return launch_d<64>(x, st);
  if (x.D == 128) return launch_d<128>(x, st);
  return launch_d<256>(x, st);
}

}  // namespace qfa
