// Attention on a paged INT8 cache for many rows at once: a piece of a prompt, or the queries of all sequences that share a prefix.
// The same arithmetic as qfa_paged_attn.hip; there 16 rows read a key's codes, here 64 or 128 share them.
//
// The four waves together turn a tile of 64 keys and of their values into binary16 integers code - zero_point (exact) in LDS, in
// the layout of the shared-KV kernels (qfa_skv_tile.h): rows come out of it for the score product, columns (transposing reads) for
// the P.V product, and nothing has to be corrected afterwards.  The queries are integers of that kind too, so a score is the same
// exact integer as on INT8 MFMA (255 * 255 * 256 < 2^24): that product would take half the matrix cycles, but its zero-point terms
// cost four vector instructions more for every score, and the vector pipe is what bounds this kernel.
//
// A wave takes 32 rows.  Four waves side by side (128 rows) take both blocks of 32 keys of a tile, two (64 rows) share them with the
// other two and meet in LDS at the end.  The next tile's codes are on their way in registers while a tile is worked on; pieces of
// the keys are dealt as qfa_paged_work.h says.
#include <type_traits>

#include "qfa_host.h"
#include "qfa_merge.h"
#include "qfa_paged_attn.h"
#include "qfa_quant_row.h"
#include "qfa_skv_tile.h"

namespace qfa {

template <int D, int QW> struct PagedTileGeom {
  static constexpr int TK = PAGED_TILE, BR = 32 * QW, KW = 4 / QW, NB = TK / 32 / KW;   // NB: blocks of 32 keys per wave and tile
  static constexpr int CPR = D / 16, SLAB = TK * 32 + 128;
  static constexpr int SIDE = CPR * SLAB;               // one side's expanded tile
  static constexpr int CONST_K = 2 * SIDE, CONST_V = CONST_K + TK * 4, CONST_L = CONST_V + TK * 4;   // scales of both, log2 of V's
  static constexpr int BUF = CONST_L + TK * 4;
  static constexpr int QROW = 2 * D + 16;               // a query row on its way into operands
  static constexpr int MERGE = (D / 2 + 2) * 256;       // partial result of a wave
  static_assert(BR * QROW <= 2 * BUF && (KW - 1) * QW * MERGE <= 2 * BUF, "what overlays the tiles");
};

// A thread's share of one side of a tile: N chunks of 16 codes with their rows' zero points
template <int D> struct PagedChunks {
  static constexpr int CPR = D / 16, RPW = 64 / CPR, N = PAGED_TILE * CPR / 256, STEP = 4 * RPW;
  static_assert(RPW <= 16 && 16 % RPW == 0, "a wave's rows of a chunk lie in one page");
  u32x4 w[N];
  unsigned z[N];
};

template <int D, int QW, bool SHARED> __global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_tile_kernel(PagedAttnKernelArgs a, int scale_dtype) {
  typedef PagedTileGeom<D, QW> GM;
  typedef PagedChunks<D> Chunks;
  constexpr int TK = GM::TK, NB = GM::NB, KW = GM::KW, BR = GM::BR, DB = D / 32, KD = D / 16, SLAB = GM::SLAB;
  constexpr int LPT = D / 8, TPP = 256 / LPT;   // quantizer: lanes per row, rows per pass
  __shared__ __attribute__((aligned(256))) unsigned char smem[2 * GM::BUF];
  __shared__ float row_a[BR];

  typedef PagedDeal<SHARED, false> Deal;
  Deal deal(a.work, BR, TK);
  unsigned x;
  typename Deal::Item item;
  if (!deal.find(x, item)) return;
  const unsigned x_end = min((blockIdx.x + 1) * deal.each, deal.total);
  if (x >= x_end) return;
  const int tid = threadIdx.x, lane = tid % 64, lr = lane % 32, g = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int kw = wave / QW;
  const SkvTileReads<SLAB> rd(lane);
  const int page_quarters_log2 = a.page_log2 - 4;   // 16 keys each

  // a thread's chunks: 4 columns of chunks by 4 rows per 16 lanes, as SkvTileStage has them
  // (made again where it is needed, from a lane that is opaque there: kept over the tiles it would cost registers that are not there)
  constexpr int CH = GM::CPR / 4;
  const int quarter_mask = (1 << page_quarters_log2) - 1;
  auto opaque = [](int y) __attribute__((always_inline)) -> int {
    asm volatile("" : "+v"(y));
    return y;
  };
  auto chunk_row = [&](int l) __attribute__((always_inline)) -> int { return wave * Chunks::RPW + l / 4 % 4 + 4 * (l / 16 / CH); };
  auto chunk_col = [&](int l) __attribute__((always_inline)) -> int { return l % 4 + 4 * (l / 16 % CH); };

  for (;;) {
    const int nt = (int)min(item.tiles - item.at, x_end - x);
    const int t0 = deal.begin() / TK + (int)item.at;
    const int seq = SHARED ? 0 : item.p, nrows = min(BR, deal.rows - BR * item.rb);
    const int slot = (wave + item.h) % QW;   // (turned by the head: waves without rows should not all sit on the same SIMD)
    const bool active = 32 * slot < nrows;

    // pages of 16 tiles: lane 4 t + quarter
    auto pages_from = [&](int first) __attribute__((always_inline)) -> int {
      const int l = opaque(lane), t = first + l / 4, quarter = 4 * (t0 + t) + l % 4, at = quarter >> page_quarters_log2;
      int id = -1;
      if (t < nt && at < a.width) id = a.page_table[seq * a.stb + at * a.stw];
      return id >= 0 && id < a.pages ? id : -1;
    };
    int pg = pages_from(0);
    Chunks ck, cv;
    unsigned sc;       // wave 0: scales of the keys, wave 1: of the values
    unsigned ok_next;  // quarters of the tile on its way whose pages are there
    // request tile t (of a page that is not there: of some other; its keys are hidden)
    auto issue = [&](int t) __attribute__((always_inline)) {
      if (t > 0 && t % 16 == 0) pg = pages_from(t);
      ok_next = (unsigned)(__builtin_amdgcn_ballot_w64(pg >= 0) >> (4 * (t % 16))) & 15u;
      const int tile = t0 + t, l = opaque(lane), in = chunk_row(l) % 16, off = in * D + 16 * chunk_col(l);
#pragma unroll
      for (int i = 0; i < Chunks::N; ++i) {
        // (chunk i lies STEP rows further: the same row of its 16, another quarter)
        static_assert(Chunks::STEP % 16 == 0, "a thread's chunks differ in the quarter");
        const int quarter = (wave * Chunks::RPW + Chunks::STEP * i) / 16;
        const int id = __builtin_amdgcn_readlane(pg, 4 * (t % 16) + quarter);
        const int64_t at = (((int64_t)max(id, 0) * a.work.Hk + item.h) << a.page_log2) + (((4 * tile + quarter) & quarter_mask) << 4);
        const rsrc_t rk = make_rsrc(a.kc + at * D, 16 * D), rv = make_rsrc(a.vc + at * D, 16 * D);
        ck.w[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, off, 0, 0));
        cv.w[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, off, 0, 0));
        ck.z[i] = (unsigned char)__builtin_amdgcn_raw_buffer_load_b8(make_rsrc(a.kz + at, 16), in, 0, 0);
        cv.z[i] = (unsigned char)__builtin_amdgcn_raw_buffer_load_b8(make_rsrc(a.vz + at, 16), in, 0, 0);
      }
      if (wave < 2) {
        const int id = __shfl(pg, 4 * (t % 16) + l / 16, 64);
        const int64_t at = (((int64_t)max(id, 0) * a.work.Hk + item.h) << a.page_log2) + (((4 * tile + l / 16) & quarter_mask) << 4) + l % 16;
        const void *p = wave == 0 ? a.ks : a.vs;
        asm("" : "+s"(p));
        sc = scale_dtype == QFA_F32 ? static_cast<const unsigned *>(p)[at] : static_cast<const unsigned short *>(p)[at];
      }
    };
    auto expand = [&](unsigned char *side, const Chunks &c, int chunk_lds) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < Chunks::N; ++i) {
        const unsigned nz = 0xe400u | (c.z[i] ^ 0x80u), nz2 = nz | nz << 16;   // -(1152 + zero_point), twice
        const f16x2 neg = __builtin_bit_cast(f16x2, nz2);
        u32x4 e[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const u32x4 m = expand_codes(c.w[i][2 * k], c.w[i][2 * k + 1]);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const unsigned my = m[y];
            e[k][y] = __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, my) + neg);
          }
        }
        *reinterpret_cast<u32x4 *>(side + chunk_lds + i * (Chunks::STEP * 32)) = e[0];
        *reinterpret_cast<u32x4 *>(side + (chunk_lds ^ 16) + i * (Chunks::STEP * 32)) = e[1];
      }
    };
    auto commit = [&](unsigned char *buf) __attribute__((always_inline)) {
      const int l = opaque(lane), chunk_lds = skv_tile_off<SLAB>(chunk_row(l), chunk_col(l), 0);
      expand(buf, ck, chunk_lds);
      expand(buf + GM::SIDE, cv, chunk_lds);
      if (wave < 2) {
        const float f = scale_dtype == QFA_F32 ? __builtin_bit_cast(float, sc) : scale_dtype == QFA_F16 ? lo_to_f32<_Float16>(sc) : lo_to_f32<__bf16>(sc);
        *reinterpret_cast<float *>(buf + (wave == 0 ? GM::CONST_K : GM::CONST_V) + l * 4) = f;
        if (wave == 1) *reinterpret_cast<float *>(buf + GM::CONST_L + l * 4) = __builtin_floorf(__builtin_amdgcn_logf(fabsf(f)));
      }
    };

    // ---- the block's queries: quantized, code - zero point as binary16 rows in LDS, a = scale * sm_scale * log2(e).  Four passes'
    // rows are requested together
    const int tid_q = opaque(tid), sub = tid_q % LPT;
    constexpr int PASSES = BR / TPP, TOGETHER = PASSES < 4 ? PASSES : 4;
    // last key of this lane's row; a row that is not there, or brings no token, goes along with the others and is not looked at
    const int block_end = deal.end(item.s, item.rb) - 1, lo = deal.begin();
    int lim = block_end;
    const int row_q = 32 * slot + tid_q % 32;
    if (row_q < nrows) {
      const auto r = deal.row(item.p, item.h, BR * item.rb + row_q);
      const PagedSeq s = SHARED ? deal.load(r.b) : item.s;
      if (r.i < s.tokens) lim = deal.last_key(r, s);
    }
    for (int p0 = 0; p0 < PASSES && p0 * TPP < nrows; p0 += TOGETHER) {
      float v[TOGETHER][8];
#pragma unroll
      for (int p = 0; p < TOGETHER; ++p) {
        const auto r = deal.row(item.p, item.h, BR * item.rb + min((p0 + p) * TPP + tid_q / LPT, nrows - 1));
        const int64_t off = r.b * a.sqb + r.qh * a.sqh + r.i * a.sqn + sub * 8;
        if (a.q_dtype == QFA_F32) Load8<float>::run(static_cast<const float *>(a.q) + off, v[p]);
        else if (a.q_dtype == QFA_BF16) Load8<__bf16>::run(static_cast<const __bf16 *>(a.q) + off, v[p]);
        else Load8<_Float16>::run(static_cast<const _Float16 *>(a.q) + off, v[p]);
      }
      if (p0 == 0) issue(0);   // (behind the first rows, which the pages do not wait for)
#pragma unroll
      for (int p = 0; p < TOGETHER; ++p) {
        const int q = (p0 + p) * TPP + tid_q / LPT;
        const QuantRow<8> row = quant_row<LPT, false, 8>(v[p], true);
        const u32x4 m = expand_codes(row.codes[0], row.codes[1]);
        const _Float16 neg = (_Float16)(-1152.0f - row.zp);
        const f16x2 neg2 = {neg, neg};
        u32x4 e;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const unsigned my = m[y];
          e[y] = __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, my) + neg2);
        }
        *reinterpret_cast<u32x4 *>(smem + q * GM::QROW + sub * 16) = e;
        if (sub == 0) {
          const float f = row.scale * a.sm_scale_log2;
          row_a[q] = f < 0x1p-126f ? 0x1p-126f : f;   // (not zero: the mask's -inf is multiplied by it)
        }
      }
    }
    __syncthreads();
    u32x4 qf[KD];
    float a_i = 0.f;
    if (active) {   // (rows past the last hold what is there: their columns of the products are nobody's)
#pragma unroll
      for (int m = 0; m < KD; ++m) qf[m] = *reinterpret_cast<const u32x4 *>(smem + (32 * slot + lr) * GM::QROW + 32 * m + 16 * g);
      a_i = 32 * slot + lr < nrows ? row_a[32 * slot + lr] : 0x1p-126f;
      if (32 * slot + lr >= nrows) {
#pragma unroll
        for (int m = 0; m < KD; ++m) qf[m] = u32x4{0u, 0u, 0u, 0u};
      }
    }
    int first_lim = lim;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) first_lim = min(first_lim, __shfl_xor(first_lim, off, 64));
    first_lim = __builtin_amdgcn_readfirstlane(first_lim);
    __syncthreads();   // the queries are read
    commit(smem);
    unsigned ok = ok_next;
    if (nt > 1) issue(1);
    __syncthreads();

    f32x16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[db][v] = 0.f;
    float ref = NO_KEY, l_run = 0.f;   // p = 2^(a_i * u - ref)
    bool begun = false;

    // rows kr .. kr + 31 of the tile in buf, whose first key is key0: scores in s
    auto scores = [&](const unsigned char *buf, int kr, f32x16 &s) __attribute__((always_inline)) {
      constexpr int AHEAD = KD < 8 ? KD : 8;   // fragments requested together (their registers are free until the probabilities)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[v] = 0.f;
#pragma unroll
      for (int m0 = 0; m0 < KD; m0 += AHEAD) {
        u32x4 kf[AHEAD];
#pragma unroll
        for (int m = 0; m < AHEAD; ++m) kf[m] = rd.rows(buf + kr * 32, m0 + m);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int m = 0; m < AHEAD; ++m) s = mfma_h(kf[m], qf[m0 + m], s);
      }
    };
    auto block = [&](const unsigned char *buf, int kr, int key0, unsigned okb, f32x16 &s, auto masked_tag) __attribute__((always_inline)) {
      constexpr bool MASKED = decltype(masked_tag)::value;
      const int at0 = key0 + kr + 4 * g, last = lim - at0, first = lo - at0;   // (this lane's keys are at0 + 8 aa + v)
#pragma unroll
      for (int aa = 0; aa < 4; ++aa) {
        const f32x4 sk = *reinterpret_cast<const f32x4 *>(buf + GM::CONST_K + (kr + 8 * aa + 4 * g) * 4);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          s[4 * aa + v] *= sk[v];
          if (MASKED && (8 * aa + v > last || 8 * aa + v < first || !(okb >> (kr / 16 + aa / 2) & 1))) s[4 * aa + v] = -INFINITY;
        }
      }
      float sum, mx;
      u32x4 pf[2];
      auto probs = [&]() __attribute__((always_inline)) {
        sum = 0.f;
        mx = 0.f;
        const unsigned char *at = buf + GM::CONST_V + opaque(kr + 4 * g) * 4;   // (opaque: read again for each use, not kept)
#pragma unroll
        for (int aa = 0; aa < 4; ++aa) {
          const f32x4 sv = *reinterpret_cast<const f32x4 *>(at + 32 * aa);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(a_i, s[4 * aa + 2 * y], -ref)),
                        p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(a_i, s[4 * aa + 2 * y + 1], -ref));
            sum += p0 + p1;
            // (what is hidden may hold any scale)
            const float x0 = MASKED ? mul_zero_wins(p0, sv[2 * y]) : p0 * sv[2 * y], x1 = MASKED ? mul_zero_wins(p1, sv[2 * y + 1]) : p1 * sv[2 * y + 1];
            mx = __builtin_fmaxf(mx, __builtin_fmaxf(fabsf(x0), fabsf(x1)));
            pf[aa / 2][2 * (aa % 2) + y] = pack_h2(x0, x1);
          }
        }
      };
      // a new reference, common to the two lanes of a row: see PAGED_P_REF
      auto move = [&]() __attribute__((always_inline)) -> float {
        float t = -INFINITY, u = -INFINITY;
#pragma unroll
        for (int aa = 0; aa < 4; ++aa) {
          const f32x4 ls = *reinterpret_cast<const f32x4 *>(buf + GM::CONST_L + (kr + 8 * aa + 4 * g) * 4);
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float y = s[4 * aa + v];
            t = fmaxf(t, MASKED && !(y > -INFINITY) ? -INFINITY : __builtin_fmaf(a_i, y, ls[v]));
            u = fmaxf(u, y);
          }
        }
        t = fmaxf(max_across_halves(fmaxf(t - PAGED_P_REF, __builtin_fmaf(a_i, u, -100.0f))), ref);
        const float alpha = __builtin_amdgcn_exp2f(ref - t);
        ref = t;
        return alpha;
      };
      if (!begun) {
        move();
        begun = true;
      }
      probs();
      if (__builtin_amdgcn_ballot_w64(mx > PAGED_P_MAX || !(l_run + sum <= 0x1p100f)) != 0) {
        const float alpha = move();
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[db][v] *= alpha;
        probs();
      }
      l_run += sum;
      __builtin_amdgcn_sched_barrier(0);
      // (columns are requested two products ahead, and not earlier: their registers are needed by then)
      const unsigned char *p = buf + GM::SIDE + kr * 32;
      u32x4 vf[2][2] = {{rd.cols(p, 0, 0), rd.cols(p, 0, 1)}, {}};
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        if (db + 1 < DB) {
          vf[(db + 1) % 2][0] = rd.cols(p, db + 1, 0);
          vf[(db + 1) % 2][1] = rd.cols(p, db + 1, 1);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) acc[db] = mfma_h(vf[db % 2][hh], pf[hh], acc[db]);
      }
    };

    int cur = 0;
    for (int t = 0; t < nt; ++t) {
      const unsigned char *buf = smem + cur * GM::BUF;
      const int key0 = (t0 + t) * TK;
      if (active) {
        const bool masked = key0 + TK - 1 > first_lim || key0 < lo || ok != 15u;
#pragma unroll 1
        for (int nb = 0; nb < NB; ++nb) {
          const int kr = 32 * (NB * kw + nb);
          f32x16 s;
          scores(buf, kr, s);
          __builtin_amdgcn_sched_barrier(0);
          if (masked) block(buf, kr, key0, ok, s, std::true_type{});
          else block(buf, kr, key0, ok, s, std::false_type{});
        }
      }
      cur ^= 1;
      if (t + 1 < nt) {
        commit(smem + cur * GM::BUF);
        ok = ok_next;
        if (t + 2 < nt) issue(t + 2);
      }
      __syncthreads();
    }

    if (!SHARED && item.at == 0 && tid == 0) {   // where the pieces are, for those who join them
      a.work.first[2 * deal.item_index(item.p, item.h, item.rb)] = item.first;
      a.work.first[2 * deal.item_index(item.p, item.h, item.rb) + 1] = deal.each;
    }
    // ---- the wave's (or the two waves') result
    float l = l_run + swap32_f(l_run);
    float *mine = reinterpret_cast<float *>(smem) + slot * (GM::MERGE / 4) + lane;
    if (KW > 1) {
      if (kw > 0 && active) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int v = 0; v < 16; ++v) mine[(16 * db + v) * 64] = acc[db][v];
        mine[16 * DB * 64] = ref;
        mine[(16 * DB + 1) * 64] = l;
      }
      __syncthreads();
    }
    const int r = 32 * slot + opaque(lr);
    if (active && kw == 0) {
      if (KW > 1) {
        const float m2 = mine[16 * DB * 64], m_all = fmaxf(ref, m2), s0 = __builtin_amdgcn_exp2f(ref - m_all), s1 = __builtin_amdgcn_exp2f(m2 - m_all);
        l = l * s0 + mine[(16 * DB + 1) * 64] * s1;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[db][v] = acc[db][v] * s0 + mine[(16 * db + v) * 64] * s1;
        ref = m_all;
      }
      const bool whole = item.at == 0 && nt == (int)item.tiles;
      if (r < nrows) {
        const int rg = BR * item.rb + r;
        const auto row = deal.row(item.p, item.h, rg);
        if (whole && !a.work.whole) {
          const bool none = row.i >= item.s.tokens || l == 0.f;   // (not of a shared prefix)
          const float inv = none ? 0.f : 1.0f / l;
          const int64_t off = (((int64_t)row.b * a.work.Hk * a.work.G + row.qh) * a.work.N + row.i) * D;
          char *o = static_cast<char *>(a.o) + off * (a.q_dtype == QFA_F32 ? 4 : 2);
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int aa = 0; aa < 4; ++aa) {
              f32x4 y;
#pragma unroll
              for (int v = 0; v < 4; ++v) y[v] = none ? 0.f : acc[db][4 * aa + v] * inv;
              store4(o, a.q_dtype, 32 * db + 8 * aa + 4 * g, y);
            }
        } else {
          const int64_t to = whole ? ((int64_t)item.p * a.work.Hk + item.h) * deal.rows + rg : ((int64_t)blockIdx.x * 2 + (item.at == 0 ? 1 : 0)) * BR + r;
          float *po = (whole ? a.work.whole : a.work.slots) + to * D, *pml = whole ? a.work.whole_ml : a.work.slots_ml;
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int aa = 0; aa < 4; ++aa)
              *reinterpret_cast<f32x4 *>(po + 32 * db + 8 * aa + 4 * g) = f32x4{acc[db][4 * aa], acc[db][4 * aa + 1], acc[db][4 * aa + 2], acc[db][4 * aa + 3]};
          if (g == 0) *reinterpret_cast<f32x2 *>(pml + 2 * to) = f32x2{ref, l};
        }
      }
    }
    x += (unsigned)nt;
    if (x >= x_end || !deal.next(x, x_end, item)) return;
    __syncthreads();   // what is in LDS is read
  }
}

template <int D, int QW> static void launch_t(const PagedAttnKernelArgs &a, bool shared, int scale_dtype, hipStream_t st) {
  if (shared) paged_tile_kernel<D, QW, true><<<dim3((unsigned)a.work.grid), dim3(256), 0, st>>>(a, scale_dtype);
  else paged_tile_kernel<D, QW, false><<<dim3((unsigned)a.work.grid), dim3(256), 0, st>>>(a, scale_dtype);
}
template <int D> static void launch_q(const PagedAttnKernelArgs &a, bool shared, int scale_dtype, int qw, hipStream_t st) {
  if (qw == 2) launch_t<D, 2>(a, shared, scale_dtype, st);
  else launch_t<D, 4>(a, shared, scale_dtype, st);
}
int launch_paged_tile(const PagedAttnKernelArgs &a, bool shared, int D, int scale_dtype, int qw, hipStream_t st) {
  if (D == 64) launch_q<64>(a, shared, scale_dtype, qw, st);
  else if (D == 128) launch_q<128>(a, shared, scale_dtype, qw, st);
  else launch_q<256>(a, shared, scale_dtype, qw, st);
  return check_launch(shared ? "qfa_attn_paged (prefix, tiles)" : "qfa_attn_paged (tiles)");
}

}  // namespace qfa
