// Attention on a paged INT8 cache for many rows at once: a piece of a prompt, or the queries of all sequences that share a prefix.
// The same arithmetic as qfa_paged_attn.hip; there 16 rows read a key's codes, here 64 or 128 share them.
// 2 x 32 heads, 333 rows on 6500 keys of 128: 146 us (480 TFLOP/s); 256 rows of each of 8 heads on 16384 keys 47 us, of which start and
// end are 10.  Of the former the vector pipe is busy for 48 %, the matrix pipe for 22 %, LDS for 30 %, and the waves wait for 36 % of their
// cycles: two waves on a SIMD, each of them a chain of scores, probabilities and products, fill none of the three.  The expansion of the
// codes is about 120 of a wave's 315 vector instructions of a tile, the keys' half of it.
//
// The four waves together turn a tile of 64 keys and of their values into binary16 integers code - zero_point (exact) in LDS, in
// the layout of the shared-KV kernels (qfa_skv_tile.h): rows come out of it for the score product, columns (transposing reads) for
// the P.V product, and nothing has to be corrected afterwards.  The queries are integers of that kind too, so a score is the same
// exact integer as on INT8 MFMA (255 * 255 * 256 < 2^24): that product would take half the matrix cycles and leave the keys unexpanded,
// but its zero-point terms, formed for every score, cost four vector instructions each.  (The dense forward, qfa_fwd.hip, takes them in a
// correction product; that has not been tried here.)
//
// A wave takes 32 rows.  Four waves side by side (128 rows) take both blocks of 32 keys of a tile, two (64 rows) share them with the
// other two and meet in LDS at the end.  The next tile's codes are on their way in registers while a tile is worked on; pieces of
// the keys are dealt as qfa_paged_work.h says.
#include "qfa_host.h"
#include "qfa_merge.h"
#include "qfa_paged_attn.h"
#include "qfa_skv_tile.h"

namespace qfa {

template <int D, int QW> struct PagedTileGeom {
  static constexpr int TK = PAGED_TILE, BR = 32 * QW, KW = 4 / QW, NB = TK / 32 / KW;   // NB: blocks of 32 keys per wave and tile
  static constexpr int CPR = D / 16, SLAB = TK * 32 + 128;
  static constexpr int SIDE = CPR * SLAB;               // one side's expanded tile
  static constexpr int CONST_K = 2 * SIDE, CONST_V = CONST_K + TK * 4, CONST_L = CONST_V + TK * 4;   // scales of both, log2 of V's
  static constexpr int CONST_X = CONST_L + TK * 4, BUF = CONST_X + TK * 4;
  static constexpr int MERGE = (D / 2 + 2) * 256;       // partial result of a wave
  static_assert((KW - 1) * QW * MERGE <= 2 * BUF, "what overlays the tiles");
};

// A thread's share of one side of a tile: N chunks of 16 codes with their rows' zero points
template <int D> struct PagedChunks {
  static constexpr int CPR = D / 16, RPW = 64 / CPR, N = PAGED_TILE * CPR / 256, STEP = 4 * RPW;
  static_assert(RPW <= 16 && 16 % RPW == 0, "a wave's rows of a chunk lie in one page");
  u32x4 w[N];
  unsigned z[N];
};

typedef const __attribute__((address_space(1))) unsigned char *GlobalBytes;
typedef const __attribute__((address_space(1))) u32x4 *GlobalWords;

template <int D, int QW, bool SHARED> __global__ __launch_bounds__(256, D == 256 ? 1 : D == 64 ? 3 : 2) void paged_tile_kernel(PagedAttnKernelArgs a_, int scale_dtype) {
  typedef PagedTileGeom<D, QW> GM;
  typedef PagedChunks<D> Chunks;
  constexpr int TK = GM::TK, NB = GM::NB, KW = GM::KW, BR = GM::BR, DB = D / 32, KD = D / 16, SLAB = GM::SLAB;
  __shared__ __attribute__((aligned(256))) unsigned char smem[2 * GM::BUF];

  const PagedAttnKernelArgs &a = a_;
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
  constexpr int CH = GM::CPR / 4;
  const unsigned quarter_mask = (1u << page_quarters_log2) - 1;
  auto opaque = [](auto y) __attribute__((always_inline)) {
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

    // pages of 16 tiles (lane 4 t + quarter): requested, and made into their first rows among all pages' rows (counted in 32 bits, see
    // qfa_paged_api.cpp) where that is needed.  A page that is not there: some other one's rows, hidden
    int pg;
    unsigned first_row = 0;
    uint64_t pages_ok = 0;
    auto request_pages = [&](int t) __attribute__((always_inline)) {
      const int l = opaque(lane);
      pg = a.page_table[seq * a.stb + min((4 * (t0 + t) + l) >> page_quarters_log2, a.width - 1) * a.stw];
    };
    auto take_pages = [&](int t) __attribute__((always_inline)) {
      const int l = opaque(lane), quarter = 4 * (t0 + t) + l;
      const bool ok = (4 * t + l < 4 * nt) & (quarter >> page_quarters_log2 < a.width) & (pg >= 0) & (pg < a.pages);
      pages_ok = __builtin_amdgcn_ballot_w64(ok);
      first_row = (((unsigned)(ok ? pg : 0) * (unsigned)a.work.Hk + (unsigned)item.h) << a.page_log2) + (((unsigned)quarter & quarter_mask) << 4);
    };
    Chunks ck, cv;
    unsigned sc;       // even waves: scales of the keys, odd ones: of the values (each of a pair writes the same)
    unsigned ok_next;  // quarters of the tile on its way whose pages are there
    // request tile t
    auto issue = [&](int t) __attribute__((always_inline)) {
      if (t % 16 == 0) {
        if (t > 0) request_pages(t);
        take_pages(t);
      }
      ok_next = (unsigned)(pages_ok >> (4 * (t % 16))) & 15u;
      const int l = opaque(lane);
      const unsigned scale_row = (unsigned)__shfl((int)first_row, 4 * (t % 16) + l / 16, 64) + l % 16;
      const unsigned in = (unsigned)chunk_row(lane) % 16, off = in * D + 16 * (unsigned)chunk_col(lane);
#pragma unroll
      for (int i = 0; i < Chunks::N; ++i) {
        // (chunk i lies STEP rows further: the same row of its 16, another quarter)
        static_assert(Chunks::STEP % 16 == 0, "a thread's chunks differ in the quarter");
        const int quarter = (wave * Chunks::RPW + Chunks::STEP * i) / 16;
        const unsigned at = (unsigned)__builtin_amdgcn_readlane((int)first_row, 4 * (t % 16) + quarter);
        GlobalBytes k = (GlobalBytes)(a.kc + (uint64_t)at * D), v = (GlobalBytes)(a.vc + (uint64_t)at * D), zk = (GlobalBytes)(a.kz + at),
                    zv = (GlobalBytes)(a.vz + at);
        asm("" : "+s"(k), "+s"(v), "+s"(zk), "+s"(zv));   // (scalar bases: else the lanes' 64-bit addresses are kept)
        ck.w[i] = *(GlobalWords)(k + off);
        cv.w[i] = *(GlobalWords)(v + off);
        ck.z[i] = zk[in];
        cv.z[i] = zv[in];
      }
      const void *p = wave % 2 == 0 ? a.ks : a.vs;
      sc = scale_dtype == QFA_F32 ? static_cast<const unsigned *>(p)[scale_row] : static_cast<const unsigned short *>(p)[scale_row];
    };
    request_pages(0);
    // one chunk of the tile on its way, as binary16 integers code - zero point, into buf (i: the keys' chunks, then the values')
    auto commit_chunk = [&](unsigned char *buf, int lds, int i) __attribute__((always_inline)) {
      const Chunks &c = i < Chunks::N ? ck : cv;
      const int n = i % Chunks::N;
      // (What was loaded is looked at here and not before: the compiler moves what both callers begin with, and with it the wait for the
      // loads, in front of the tile.)
      const unsigned zero = opaque(c.z[n]), nz = 0xe400u | (zero ^ 0x80u), nz2 = nz | nz << 16;   // -(1152 + zero_point), twice
      const f16x2 neg = __builtin_bit_cast(f16x2, nz2);
      unsigned char *side = buf + (i < Chunks::N ? 0 : GM::SIDE) + n * (Chunks::STEP * 32);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const unsigned w0 = opaque(c.w[n][2 * k]), w1 = opaque(c.w[n][2 * k + 1]);
        const u32x4 m = expand_codes(w0, w1);
        u32x4 e;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const unsigned my = m[y];
          e[y] = __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, my) + neg);
        }
        *reinterpret_cast<u32x4 *>(side + (k == 0 ? lds : lds ^ 16)) = e;
      }
    };
    auto commit_scales = [&](unsigned char *buf) __attribute__((always_inline)) {
      const int l = opaque(lane);
      const unsigned raw = opaque(sc);
      const float f = scale_dtype == QFA_F32 ? __builtin_bit_cast(float, raw) : scale_dtype == QFA_F16 ? lo_to_f32<_Float16>(raw) : lo_to_f32<__bf16>(raw);
      *reinterpret_cast<float *>(buf + (wave % 2 == 0 ? GM::CONST_K : GM::CONST_V) + l * 4) = f;
      // (log2 of the keys' scales goes where nobody reads it)
      *reinterpret_cast<float *>(buf + (wave % 2 == 0 ? GM::CONST_X : GM::CONST_L) + l * 4) = __builtin_floorf(__builtin_amdgcn_logf(fabsf(f)));
    };
    auto commit = [&](unsigned char *buf) __attribute__((always_inline)) {
      const int lds = skv_tile_off<SLAB>(chunk_row(lane), chunk_col(lane), 0);
#pragma unroll
      for (int i = 0; i < 2 * Chunks::N; ++i) commit_chunk(buf, lds, i);
      commit_scales(buf);
    };

    // ---- this lane's row: half of its codes, as binary16 integers code - zero point (k-step m, k-group g holds columns
    // 16m + 8g + {0..7}), and a = scale * sm_scale * log2(e).  Rows past the last are zeros.
    const int row_q = 32 * slot + opaque(lr), block_end = deal.end(item.s, item.rb) - 1, lo = deal.begin();
    int lim;   // last key of the row; one that is not there, or brings no token, goes along with the others and is not looked at
    u32x2 qc[KD];
    const bool have = row_q < nrows;
    const auto r_q = deal.row(item.p, item.h, BR * item.rb + min(row_q, nrows - 1));
    const int64_t at_q = ((int64_t)r_q.b * a.work.Hk * a.work.G + r_q.qh) * a.work.N + r_q.i;
    const int8_t *codes = a.q_codes + at_q * D + 8 * g;
#pragma unroll
    for (int m = 0; m < KD; ++m) qc[m] = *reinterpret_cast<const u32x2 *>(codes + 16 * m);
    const float scale_q = a.q_scale[at_q];
    const int8_t zero_q = a.q_zero[at_q];
    PagedSeq seq_q = item.s;
    if (SHARED) seq_q = {a.work.starts[r_q.b], a.work.counts ? a.work.counts[r_q.b] : a.work.N};
    __builtin_amdgcn_sched_barrier(0);
    issue(0);   // (waits for the pages alone, which were requested first)
    __builtin_amdgcn_sched_barrier(0);
    float a_i;
    {
      const float f = scale_q * a.sm_scale_log2;
      if (SHARED) seq_q.tokens = max(0, min(seq_q.tokens, a.work.N));
      const int key = deal.last_key(r_q, seq_q);   // (no branches: see qfa_paged_work.h)
      const bool seen = have & (r_q.i < seq_q.tokens), small = !have | (f < 0x1p-126f);
      a_i = small ? 0x1p-126f : f;   // (not zero: the mask's -inf is multiplied by it)
      lim = seen ? key : block_end;
    }
    u32x4 qf[KD];
    {
      const _Float16 neg = (_Float16)(-1152.0f - (float)zero_q);
      const f16x2 neg2 = {neg, neg};
#pragma unroll
      for (int m = 0; m < KD; ++m) {
        const unsigned w0 = qc[m][0], w1 = qc[m][1];
        const u32x4 e = expand_codes(w0, w1);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const unsigned ey = e[y];
          qf[m][y] = have ? __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, ey) + neg2) : 0u;
        }
      }
    }
    int first_lim = lim;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) first_lim = min(first_lim, __shfl_xor(first_lim, off, 64));
    first_lim = __builtin_amdgcn_readfirstlane(first_lim);
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
    // ---- Rows kr .. kr + 31 of the tile in buf, and their scores in code units in four steps
    constexpr int KS = KD / 4;   // k-steps of a step, and of the fragments requested together
    auto request = [&](const unsigned char *buf, int kr, int step, u32x4 (&kf)[KS]) __attribute__((always_inline)) {
#pragma unroll
      for (int m = 0; m < KS; ++m) kf[m] = rd.rows(buf + kr * 32, step * KS + m);
    };
    auto scores = [&](f32x16 &s, int step, const u32x4 (&kf)[KS]) __attribute__((always_inline)) {
      if (step == 0) {
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = 0.f;
      }
#pragma unroll
      for (int m = 0; m < KS; ++m) s = mfma_h(kf[m], qf[step * KS + m], s);
    };
    // What keys 8 aa + 4 g + {0..3} of rows kr .. have at `at`: their scales, their values' scales or those's log2
    auto constants = [&](const unsigned char *buf, int at, int kr, int aa) __attribute__((always_inline)) -> f32x4 {
      return *reinterpret_cast<const f32x4 *>(buf + at + 16 * g + kr * 4 + 32 * aa);
    };
    // The scores times the keys' scales; hidden keys become -inf.  (A branch of its own around the mask and nothing else: with a masked
    // and an unmasked copy of the whole tile the compiler keeps the accumulators twice; and one for the whole block: it moves what stands
    // between several of them behind the last one.)
    auto scale = [&](const unsigned char *buf, int kr, int key0, unsigned okb, bool masked, f32x16 &s) __attribute__((always_inline)) {
#pragma unroll
      for (int aa = 0; aa < 4; ++aa) {
        const f32x4 c = constants(buf, GM::CONST_K, kr, aa);
#pragma unroll
        for (int v = 0; v < 4; ++v) s[4 * aa + v] *= c[v];
      }
      if (masked) {
        const int at0 = key0 + kr + opaque(4 * g), last = lim - at0, first = lo - at0;
#pragma unroll
        for (int aa = 0; aa < 4; ++aa) {
          const bool page = okb >> (kr / 16 + aa / 2) & 1;
#pragma unroll
          for (int v = 0; v < 4; ++v)
            if (8 * aa + v > last || 8 * aa + v < first || !page) s[4 * aa + v] = -INFINITY;
        }
      }
    };
    // p' = p * scale as binary16, the sum of p, the largest p' as bits (of a negative scale: larger than any limit)
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    struct Probs { u32x4 f[2]; float sum; u16x2 top; };
    auto probs = [&](const f32x4 &sv, const f32x16 &s, Probs &r, int aa) __attribute__((always_inline)) {
      if (aa == 0) {
        r.sum = 0.f;
        r.top = u16x2{0, 0};
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(a_i, s[4 * aa + 2 * y], -ref)),
                    p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(a_i, s[4 * aa + 2 * y + 1], -ref));
        r.sum += p0 + p1;
        const float x0 = mul_zero_wins(p0, sv[2 * y]), x1 = mul_zero_wins(p1, sv[2 * y + 1]);   // (what is hidden may hold any scale)
        const unsigned w = pack_h2(x0, x1);
        r.top = __builtin_elementwise_max(r.top, __builtin_bit_cast(u16x2, w));
        r.f[aa / 2][2 * (aa % 2) + y] = w;
      }
    };
    // A new reference, common to the two lanes of a row (see PAGED_P_REF): the factor for what has been summed up
    auto move = [&](const unsigned char *buf, int kr, const f32x16 &s) __attribute__((always_inline)) -> float {
      float t = -INFINITY, u = -INFINITY;
#pragma unroll
      for (int aa = 0; aa < 4; ++aa) {
        const f32x4 ls = constants(buf, GM::CONST_L, kr, aa);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float y = s[4 * aa + v];
          t = fmaxf(t, !(y > -INFINITY) ? -INFINITY : __builtin_fmaf(a_i, y, ls[v]));
          u = fmaxf(u, y);
        }
      }
      t = fmaxf(max_across_halves(fmaxf(t - PAGED_P_REF, __builtin_fmaf(a_i, u, -100.0f))), ref);
      const float alpha = __builtin_amdgcn_exp2f(ref - t);
      ref = t;
      return alpha;
    };
    // The reference moves where some p' (or the sum) has become too large, and at the first keys; what was made of it is made again
    auto check = [&](const unsigned char *buf, int kr, const f32x16 &s, Probs &r) __attribute__((always_inline)) {
      if (__builtin_amdgcn_ballot_w64(max((unsigned)r.top[0], (unsigned)r.top[1]) > PAGED_P_MAX_BITS || !(l_run + r.sum <= 0x1p100f)) != 0) {
        const float alpha = move(buf, kr, s);
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[db][v] *= alpha;
#pragma unroll
        for (int aa = 0; aa < 4; ++aa) probs(constants(buf, GM::CONST_V, kr, aa), s, r, aa);
      }
      l_run += r.sum;
    };
    // A tile.  The matrix products of one block of keys run beside the probabilities of the other one, the last ones beside what
    // makes the next tile out of codes: four steps each, written down in the order in which they are to be issued.  (Left alone, the
    // compiler puts every kind in a row of its own, a load, a wait and a product at a time, and two waves per SIMD do not fill that.)
    auto fence = []() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };
    auto tile = [&](const unsigned char *buf, unsigned char *nbuf, int key0, unsigned okb, bool masked) __attribute__((always_inline)) {
      const int kr = 32 * NB * kw;
      f32x16 s0, s1;
      Probs r0, r1;
      // fragments on their way: rows of the keys four steps ahead of their products, columns of the values two
      u32x4 kf[4][KS], vf[DB][2];
      __builtin_amdgcn_s_setprio(1);   // (the other wave of the SIMD may be making a tile out of codes: 2%)
      auto columns = [&](int row, int db) __attribute__((always_inline)) {
        const unsigned char *p = buf + GM::SIDE + row * 32;
        vf[db][0] = rd.cols(p, db, 0);
        vf[db][1] = rd.cols(p, db, 1);
      };
      auto product = [&](const Probs &r, int db) __attribute__((always_inline)) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) acc[db] = mfma_h(vf[db][hh], r.f[hh], acc[db]);
      };
      constexpr int PER = DB > 4 ? DB / 4 : 1, EVERY = DB < 4 ? 4 / DB : 1;   // column blocks of a step, steps of a column block
      auto step_columns = [&](int row, int j) __attribute__((always_inline)) {
        if (j % EVERY == 0)
#pragma unroll
          for (int x = 0; x < PER; ++x) columns(row, j / EVERY * PER + x);
      };
      // all products with r, `step` in four parts beside them; next_row: whose columns come after these (-1: none)
      auto products = [&](const Probs &r, int row, int next_row, auto step) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j % EVERY == 0) {
#pragma unroll
            for (int x = 0; x < PER; ++x) product(r, j / EVERY * PER + x);
          }
          if (j < 2) step_columns(row, j + 2);
          else if (next_row >= 0) step_columns(next_row, j - 2);
          step(j);
          fence();
        }
      };
      f32x4 c[2];   // the values' scales
#pragma unroll
      for (int i = 0; i < 4; ++i) request(buf, kr, i, kf[i]);
      fence();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        scores(s0, i, kf[i]);
        if (NB == 2) request(buf, kr + 32, i, kf[i]);
      }
      scale(buf, kr, key0, okb, masked, s0);
      c[0] = constants(buf, GM::CONST_V, kr, 0);
      fence();
#pragma unroll
      for (int aa = 0; aa < 4; ++aa) {
        if (aa < 3) c[(aa + 1) % 2] = constants(buf, GM::CONST_V, kr, aa + 1);
        if (NB == 2) scores(s1, aa, kf[aa]);
        if (aa >= 2) step_columns(kr, aa - 2);
        probs(c[aa % 2], s0, r0, aa);
        fence();
      }
      check(buf, kr, s0, r0);
      if (NB == 2) {
        scale(buf, kr + 32, key0, okb, masked, s1);
        c[0] = constants(buf, GM::CONST_V, kr + 32, 0);
      }
      fence();
      if (NB == 2) {
        products(r0, kr, kr + 32, [&](int aa) __attribute__((always_inline)) {
          if (aa < 3) c[(aa + 1) % 2] = constants(buf, GM::CONST_V, kr + 32, aa + 1);
          probs(c[aa % 2], s1, r1, aa);
        });
        check(buf, kr + 32, s1, r1);
        fence();
      }
      __builtin_amdgcn_s_setprio(0);
      const int lds = skv_tile_off<SLAB>(chunk_row(lane), chunk_col(lane), 0);
      products(NB == 2 ? r1 : r0, NB == 2 ? kr + 32 : kr, -1, [&](int j) __attribute__((always_inline)) {
        // (past the last tile: once more what is there)
        constexpr int N2 = 2 * Chunks::N;
#pragma unroll
        for (int i = j * N2 / 4; i < (j + 1) * N2 / 4; ++i) commit_chunk(nbuf, lds, i);
        if (j == 0) commit_scales(nbuf);
      });
    };

    int cur = 0;
    for (int t = 0; t < nt; ++t) {
      const unsigned char *buf = smem + cur * GM::BUF;
      const int key0 = (t0 + t) * TK;
      cur ^= 1;
      unsigned char *nbuf = smem + cur * GM::BUF;
      if (active) tile(buf, nbuf, key0, ok, key0 + TK - 1 > first_lim || key0 < lo || ok != 15u);
      else commit(nbuf);
      if (t + 1 < nt) {
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
