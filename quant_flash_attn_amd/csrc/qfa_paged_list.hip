// Attention of every token on a list of blocks (pages) of its sequence, those that a cheap score has selected (qfa_paged_select.hip):
//     O = softmax(sm_scale * Q^ K^^T) V^   over the keys of the listed blocks at or before the token,
// with the arithmetic of attention on all keys (qfa_paged_attn.hip), and its kernel, or one for few rows.  Probabilities times scales are binary16 numbers for
// queries of 16 bits, 2^-11 off relative to a sum of p |v|: a second part of them, which queries in fp32 get (FINE), takes 26 % longer for 2 x 333 tokens.  A token and key head are an item: the query heads that
// share the key head are its rows, the list's blocks one behind the other its keys.  A half of a tile lies in one block, so what the mask
// asks is where each half's keys begin; the list is read beside the page numbers, 32 tiles ahead.
//
// Lists of one token each are bound by reading the cache, 64 sequences, 8 key heads of 4 x 128, 1024 keys of each, 134 MB in 29 us (4.6 TB/s), or by a start and a
// few tiles that wait for each other: 8 x 5 tokens, 4 key heads of 4 x 256, 640 keys 15.3 us.
#include "qfa_paged_block.h"

namespace qfa {

constexpr int LIST_WGS = 256 * 2;   // two on a CU
constexpr int LIST_EXTRA = 12;      // units of an item beside its tiles, as there

// Up to four rows.  Of the sixteen columns of a product they would be four real ones and twelve copies, for whose scores the vector pipe
// works as long as for real ones.  So the columns are the four rows four times over, and of a tile of 64 keys every copy takes 16 and
// is a softmax of its own: the score products add up in one accumulator, each 16 keys' with the queries of their copy and zeros elsewhere,
// and a lane has four scores of 64 keys in place of eight of 32.  The probabilities enter the P.V product likewise.  The copies meet at the end,
// as the waves do: two, so that an item costs little beside its tiles.  A value's bytes, offset by 128, are binary16 numbers of 2^-24 each as they stand.
// 2 x 333 tokens, 8 key heads of 4 x 128, 2048 keys each, us: 165 against 291 of paged_rows_kernel (calls in a row 140 against 244, of one block of 64 keys each 28 against 64); 64 x 1 token,
// 1024 keys: 29.1 against 29.5.  With one wave to an item 161 and 30.4, with four 190 and 29.7.  Every step against the one before it, where it was taken: values 8 bytes a lane in
// the products' order 179, through LDS 198, 16 bytes a lane 171 (two workgroups less on a CU 197), and that with an offset of 128 in place of 1152, an instruction less for two
// values, 168.  Keys and values come from L2 (99 %): 2.9 GB, 17 TB/s.  The way from the L1 cache to registers is busy for 76 % of the time, its tags for 52 %, the
// vector pipe for 60 %, the matrix pipe for 24 %: a tile takes 240 vector instructions, 96 of them the values' conversion.
constexpr int FEW_ROWS = 4, FEW_TILE = 64, FEW_WAVES = 2;
template <typename S, int D, bool FINE> __global__ __launch_bounds__(64 * FEW_WAVES, D == 256 ? 2 : 3) void paged_list_few_kernel(PagedAttnKernelArgs a) {
  constexpr int KM = D / 64;
  // A lane holds 16 bytes of a value: D / 16 lanes of 16 have a row, so that the 16 rows of the products' first operand are PARTS times the elements,
  // each part of keys of its own: those of copies part * 4 / PARTS and on.  What a part's rows sum up for the other copies is not looked at
  constexpr int PARTS = 256 / D, VE = 16 / PARTS, VH = D == 256 ? 2 : 1;   // loads of a tile, products
  constexpr int LPT = D / 8;
  constexpr int OFF_ONES = (FEW_ROWS + 1) * D, OFF_ST = OFF_ONES + 16, OFF_TC = OFF_ST + 3 * 16;   // (query codes; D bytes of zeros; ones)
  constexpr int TC = 512 + 512 + 256;   // [64] x (scale, zero point operand) of keys, of values, exponents of the values' scales
  constexpr int OFF_K = OFF_TC + TC, EACH = OFF_K + FEW_TILE * D;   // a tile's keys; the copies' sums
  __shared__ __attribute__((aligned(16))) unsigned char all[FEW_WAVES * EACH];

  PagedListDeal deal(a.work, PAGED_ROWS, FEW_TILE);
  deal.lists(a.list_tiles, a.list_each);
  PagedListDeal::Item item;
  deal.item(deal.workgroup(), item);
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), q16 = lane % 16, G = lane / 16;
  const int copy = q16 / 4, row_of = q16 % 4;   // this lane's column: copy * 4 + row; its keys of a tile: 16 copy + 4 G + v
  const auto token = deal.row(item.p, item.h, 0);
  const int tiles = ((int)item.tiles - wave + FEW_WAVES - 1) / FEW_WAVES, last = deal.last_key(token, item.s), nrows = deal.rows;   // (4 rows at most)

  unsigned char *smem = all + wave * EACH;
  struct Tile {
    u32x4 v[VE];
    unsigned ks, kz, vs, vz;   // scale (its bits) and zero point of key lane and value lane
    int ok, key[4];            // bit per 16 keys: their page exists; the position of the first of them
  };
  const int part = q16 / (16 / PARTS), v_off = 4 * G * D + 16 * (q16 % (16 / PARTS));
  // Keys are loaded into LDS as they lie, 16 bytes a lane, and read from there in the fragments' order: loaded in that order,
  // neighbouring lanes' bytes are of different rows, and each lane is an access of its own to the L1 cache.  Within a row the 16-byte
  // parts are exchanged by its number, for the banks.
  constexpr int CHUNKS = D / 16, PER_LINE = CHUNKS < 8 ? 8 / CHUNKS : 1, TURNS = CHUNKS < 8 ? CHUNKS : 8;   // (rows in 128 bytes)
  auto k_at = [](int row, int part) __attribute__((always_inline)) -> int { return row * D + 16 * (part ^ (row / PER_LINE % TURNS)); };
  unsigned char *kl = smem + OFF_K;
  int k_off[4];   // (KM of them)
#pragma unroll
  for (int m = 0; m < KM; ++m) k_off[m] = k_at(m * (1024 / D) + lane / CHUNKS, lane % CHUNKS) - 1024 * m;
  const int page_parts_log2 = a.page_log2 - 4;
  unsigned *tc = reinterpret_cast<unsigned *>(smem + OFF_TC);
  const int32_t *list = a.blocks + (((int64_t)token.b * a.work.Hk + item.h) * a.work.N + token.i) * a.keep;

  // pages of 16 tiles: lane 4 i + part of tile i, and where the part's keys begin
  auto pages_from = [&](int i0, int &pos) __attribute__((always_inline)) -> int {
    const int i = i0 + lane / 4, part = 4 * (FEW_WAVES * i + wave) + lane % 4, place = part >> page_parts_log2;
    const int block = list[min(place, a.keep - 1)];
    const bool listed = (place < a.keep) & (block >= 0) & (block < a.width);
    const int id = a.page_table[token.b * a.stb + (listed ? block : a.width - 1) * a.stw];
    pos = listed ? (block << a.page_log2) + ((part & ((1 << page_parts_log2) - 1)) << 4) : 0;
    const bool there = (i < tiles) & listed & (id >= 0) & (id < a.pages) & (pos <= last);
    return there ? id : -1;
  };
  int pos = 0, pos_next = 0;
  int pg = pages_from(0, pos), pg_next = tiles > 16 ? pages_from(16, pos_next) : -1;
  unsigned first[4];   // first row of each 16 keys among all rows (fewer than 2^32)
  auto load_keys = [&](Tile &t, int i) __attribute__((always_inline)) {
    if (i > 0 && i % 16 == 0) {
      pg = pg_next;
      pos = pos_next;
      pg_next = i + 16 < tiles ? pages_from(i + 16, pos_next) : -1;
    }
    t.ok = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int id = __builtin_amdgcn_readlane(pg, 4 * (i % 16) + g);
      t.key[g] = __builtin_amdgcn_readlane(pos, 4 * (i % 16) + g);
      const bool ok = id >= 0;
      t.ok |= ok ? 1 << g : 0;
      first[g] = (((unsigned)(ok ? id : 0) * (unsigned)a.work.Hk + (unsigned)item.h) << a.page_log2) + ((unsigned)t.key[g] & ((1u << a.page_log2) - 1));
    }
    const unsigned f0 = first[0], f1 = first[1], f2 = first[2], f3 = first[3];
    const unsigned at = (G < 2 ? (G == 0 ? f0 : f1) : (G == 2 ? f2 : f3)) + (unsigned)q16;
    const S *ks = static_cast<const S *>(a.ks) + at, *vs = static_cast<const S *>(a.vs) + at;
    if constexpr (sizeof(S) == 4) {
      t.ks = __builtin_bit_cast(unsigned, *ks);
      t.vs = __builtin_bit_cast(unsigned, *vs);
    } else {
      t.ks = __builtin_bit_cast(unsigned short, *ks);
      t.vs = __builtin_bit_cast(unsigned short, *vs);
    }
    t.kz = (unsigned)(unsigned char)a.kz[at];
    t.vz = (unsigned)(unsigned char)a.vz[at];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const rsrc_t rk = make_rsrc(a.kc + (int64_t)first[g] * D, t.ok >> g & 1 ? 16 * D : 0);
#pragma unroll
      for (int m = 0; m < KM; ++m) __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lptr_t)(kl + 16 * D * g + 1024 * m), 16, k_off[m], 1024 * m, 0, 0);
    }
  };
  auto load_values = [&](Tile &t) __attribute__((always_inline)) {   // (of a page that is not there those of another; they count for nothing)
    const unsigned f0 = first[0], f1 = first[1], f2 = first[2], f3 = first[3];
#pragma unroll
    for (int y = 0; y < VE / 4; ++y) {
      unsigned at;
      if constexpr (PARTS == 1) at = first[y];
      else if constexpr (PARTS == 2) at = y == 0 ? (part == 0 ? f0 : f2) : (part == 0 ? f1 : f3);
      else at = part < 2 ? (part == 0 ? f0 : f1) : (part == 2 ? f2 : f3);
      const int8_t *from = a.vc + (int64_t)at * D + v_off;
#pragma unroll
      for (int e = 0; e < 4; ++e) t.v[4 * y + e] = *reinterpret_cast<const u32x4 *>(from + e * D);
    }
  };

  // the queries are requested beside the pages, and quantized while the first keys are on their way
  constexpr int PASSES = D == 256 ? 2 : 1;
  float qv[PASSES][8];
#pragma unroll
  for (int ps = 0; ps < PASSES; ++ps) {
    const auto r = deal.row(item.p, item.h, min(ps * (64 / LPT) + lane / LPT, nrows - 1));
    const int64_t off = r.b * a.sqb + r.qh * a.sqh + r.i * a.sqn + lane % LPT * 8;
    if (a.q_dtype == QFA_F32) Load8<float>::run(static_cast<const float *>(a.q) + off, qv[ps]);
    else if (a.q_dtype == QFA_BF16) Load8<__bf16>::run(static_cast<const __bf16 *>(a.q) + off, qv[ps]);
    else Load8<_Float16>::run(static_cast<const _Float16 *>(a.q) + off, qv[ps]);
  }
  Tile ta;
  load_keys(ta, 0);
  asm volatile("" ::: "memory");
  load_values(ta);
  float *st_a = reinterpret_cast<float *>(smem + OFF_ST);
  int *st_z = reinterpret_cast<int *>(smem + OFF_ST + 16), *st_c = reinterpret_cast<int *>(smem + OFF_ST + 32);
  if (lane <= D / 16)   // (the zeros, and the ones behind them)
    *reinterpret_cast<i32x4 *>(smem + FEW_ROWS * D + 16 * lane) = lane < D / 16 ? i32x4{0, 0, 0, 0} : i32x4{0x01010101, 0x01010101, 0x01010101, 0x01010101};
#pragma unroll
  for (int ps = 0; ps < PASSES; ++ps) {
    const QuantRow<8> row = quant_row<LPT, false, 8>(qv[ps], true);
    const int r = ps * (64 / LPT) + lane / LPT;
    if (r < FEW_ROWS) {
      *reinterpret_cast<u32x2 *>(smem + r * D + lane % LPT * 8) = u32x2{row.codes[0], row.codes[1]};
      if (lane % LPT == 0) {
        const float f = row.scale * a.sm_scale_log2;
        st_a[r] = f < 0x1p-126f ? 0x1p-126f : f;   // (not zero: the mask's -inf is multiplied by it)
        st_z[r] = (int)row.zp;
        st_c[r] = row.sum - D * (int)row.zp;
      }
    }
  }
  __syncthreads();
  // where the queries of each copy stand, zeros elsewhere; ones likewise
  int q_at[4], one_at[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    q_at[g] = (copy == g ? row_of : FEW_ROWS) * D + 16 * G;
    one_at[g] = copy == g ? OFF_ONES : FEW_ROWS * D;
  }
  const float a_i = st_a[row_of];
  const int zq = st_z[row_of], c_i = st_c[row_of];

  f32x4 oacc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) oacc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float ref = NO_KEY, l_run = 0.f, w_run = 0.f;   // p = 2^(a_i * u - ref)

  auto tile = [&](Tile &t, int i) __attribute__((always_inline)) {
    {
      u32x2 w;
      w[0] = __builtin_bit_cast(unsigned, scale_to_f32<S>(t.ks));
      w[1] = (unsigned)(int)(signed char)t.kz;
      *reinterpret_cast<u32x2 *>(tc + 2 * lane) = w;
      w[0] = __builtin_bit_cast(unsigned, scale_to_f32<S>(t.vs));
      w[1] = FINE ? half_of((int)(signed char)t.vz) : half_of((int)(t.vz ^ 0x80u));   // the binary16 number of the zero point (or of 128 + it)
      *reinterpret_cast<u32x2 *>(tc + 128 + 2 * lane) = w;
    }
    const int mine = 16 * copy + 4 * G;   // this lane's first key
    // The keys are in LDS once no more than the loads of values behind them are on their way.  (The compiler moves no access
    // of memory across a statement like this, or the one behind the products; a register that it spilled would be counted too.  The build looks at all of it.)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(VE) : "memory");
    i32x4 s = {0, 0, 0, 0}, rk = {0, 0, 0, 0};
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const i32x4 ones = *reinterpret_cast<const i32x4 *>(smem + one_at[g]);
#pragma unroll
      for (int m = 0; m < KM; ++m) {
        const i32x4 kf = *reinterpret_cast<const i32x4 *>(kl + 16 * D * g + k_at(q16, 4 * m + G));
        s = paged_mfma_i8(kf, *reinterpret_cast<const i32x4 *>(smem + q_at[g] + 64 * m), s);
        rk = paged_mfma_i8(kf, ones, rk);
      }
    }
    const u32x4 cv[2] = {*reinterpret_cast<const u32x4 *>(tc + 128 + 2 * mine), *reinterpret_cast<const u32x4 *>(tc + 128 + 2 * mine + 4)};
    f32x4 f;
    {
      const u32x4 c0 = *reinterpret_cast<const u32x4 *>(tc + 2 * mine), c1 = *reinterpret_cast<const u32x4 *>(tc + 2 * mine + 4);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const unsigned scw = v < 2 ? c0[2 * v] : c1[2 * v - 4], zw = v < 2 ? c0[2 * v + 1] : c1[2 * v - 3];
        const int dot = s[v] - __mul24(zq, rk[v]) - __mul24((int)zw, c_i);
        f[v] = (float)dot * __builtin_bit_cast(float, scw);
      }
    }
    const int k0 = t.key[0], k1 = t.key[1], k2 = t.key[2], k3 = t.key[3];
    if (max(max(k0, k1), max(k2, k3)) > last - 15 || t.ok != 15) {
      const int begin = copy < 2 ? (copy == 0 ? k0 : k1) : (copy == 2 ? k2 : k3);
      const int seen = t.ok >> copy & 1 ? last - begin - 4 * G : -1;   // (v up to it)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (v > seen) f[v] = -INFINITY;
    }
    // the next tile's keys go where the products have read: not before all of their reads have returned
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    load_keys(t, i + 1);
    // ---- p and its row sum, p' = p * scale_j and the largest of them
    float ps[4], mx = 0.f, l_new = 0.f;
    auto probs = [&]() __attribute__((always_inline)) {
      mx = 0.f;
      l_new = l_run;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const unsigned s0 = cv[y][0], s1 = cv[y][2];   // (a bit cast of a vector's element takes element 0)
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(a_i, f[2 * y], -ref));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(a_i, f[2 * y + 1], -ref));
        l_new += p0 + p1;
        ps[2 * y] = mul_zero_wins(p0, __builtin_bit_cast(float, s0));   // (what is hidden may hold any scale)
        ps[2 * y + 1] = mul_zero_wins(p1, __builtin_bit_cast(float, s1));
        mx = fmaxf(mx, fmaxf(fabsf(ps[2 * y]), fabsf(ps[2 * y + 1])));
      }
    };
    // a new reference, common to the four lanes of a column (as in paged_rows_kernel)
    auto move = [&]() __attribute__((always_inline)) -> float {
      float *tl = reinterpret_cast<float *>(tc + 256);
      tl[lane] = __builtin_floorf(__builtin_amdgcn_logf(fabsf((*reinterpret_cast<const f32x2 *>(tc + 128 + 2 * lane))[0])));
      const f32x4 ls = *reinterpret_cast<const f32x4 *>(tl + mine);
      float t_max = -INFINITY, u = -INFINITY;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        t_max = fmaxf(t_max, !(f[v] > -INFINITY) ? -INFINITY : __builtin_fmaf(a_i, f[v], ls[v]));
        u = fmaxf(u, f[v]);
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
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) oacc[j][v] *= alpha;
      probs();
    }
    l_run = l_new;
    // ---- p' as binary16, offset term
    u32x4 pf[VH], pl[VH];
#pragma unroll
    for (int h = 0; h < VH; ++h) pf[h] = pl[h] = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const unsigned pp = pack_h2(ps[2 * y], ps[2 * y + 1]), zz = cv[y][1] | (cv[y][3] << 16);
      w_run = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pp), __builtin_bit_cast(f16x2, zz), w_run, false);
      unsigned rest = 0;
      if constexpr (FINE) {
        rest = rest_h2(ps[2 * y], ps[2 * y + 1], pp);
        w_run = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, rest), __builtin_bit_cast(f16x2, zz), w_run, false);
      }
      if constexpr (PARTS == 4) {
        pf[0][y] = pp;
        pl[0][y] = rest;
      } else {
#pragma unroll
        for (int g = 0; g < 2 * VH; ++g) {
          pf[g / 2][2 * (g % 2) + y] = copy % (2 * VH) == g ? pp : 0u;
          pl[g / 2][2 * (g % 2) + y] = copy % (2 * VH) == g ? rest : 0u;
        }
      }
    }
    // ---- O^T += (128 + codes)^T . P'^T, the former as the binary16 numbers 2^-24 (128 + code), which are their bytes (FINE: codes^T . P'^T)
#pragma unroll
    for (int e = 0; e < VE && !FINE; ++e)
#pragma unroll
      for (int y = 0; y < 4; ++y) t.v[e][y] ^= 0x80808080u;
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int h = 0; h < VH; ++h) {
        u32x4 vf = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < (PARTS == 4 ? 2 : 4); ++e) {
          constexpr unsigned pick = 0x0c040c00u;
          const unsigned lo = t.v[8 * h + 2 * e][j / 4], hi = t.v[8 * h + 2 * e + 1][j / 4];
          vf[e] = __builtin_amdgcn_perm(hi, lo, pick + (unsigned)(j % 4) * 0x00010001u);
          if constexpr (FINE) vf[e] = without_offset(vf[e] ^ 0x64806480u);
        }
        oacc[j] = mfma_h16(vf, pf[h], oacc[j]);
        if constexpr (FINE) oacc[j] = mfma_h16(vf, pl[h], oacc[j]);
      }
    asm volatile("" ::: "memory");
    load_values(t);
  };
  for (int i = 0; i < tiles; ++i) tile(ta, i);

  // ---- merge of the copies, through LDS: [column][D] where the keys were, (m, l) where the tokens' constants were
  float l_tot = l_run + __shfl_xor(l_run, 16, 64), w_tot = w_run + __shfl_xor(w_run, 16, 64);
  l_tot += __shfl_xor(l_tot, 32, 64);
  w_tot += __shfl_xor(w_tot, 32, 64);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing is on its way into LDS
  __syncthreads();
  float *mg = reinterpret_cast<float *>(smem + OFF_K), *ml = reinterpret_cast<float *>(tc);
  {
    float *dst = mg + q16 * D;
    if (4 * G / (16 / PARTS) == copy * PARTS / 4) {   // (this lane's four rows are one part's)
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          f32x4 y;
#pragma unroll
          for (int z = 0; z < 4; ++z) y[z] = __builtin_fmaf(oacc[j + z][v], FINE ? 1.0f : 0x1p24f, -w_tot);
          *reinterpret_cast<f32x4 *>(dst + 16 * ((4 * G + v) % (16 / PARTS)) + j) = y;
        }
    }
    if (G == 0) {
      ml[2 * q16] = ref;
      ml[2 * q16 + 1] = l_tot;
    }
  }
  __syncthreads();
  for (int y = threadIdx.x; y < nrows * (D / 4); y += 64 * FEW_WAVES) {
    const int q = y / (D / 4), d = 4 * (y % (D / 4));
    const float *from = reinterpret_cast<const float *>(all) + (OFF_K / 4 + q * D + d), *ml = reinterpret_cast<const float *>(all) + (OFF_TC / 4 + 2 * q);
    constexpr int STEP = EACH / 4;
    float m = NO_KEY, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4 * FEW_WAVES; ++w) m = fmaxf(m, ml[w / 4 * STEP + 8 * (w % 4)]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4 * FEW_WAVES; ++w) {
      const float sc = __builtin_amdgcn_exp2f(ml[w / 4 * STEP + 8 * (w % 4)] - m);
      l += ml[w / 4 * STEP + 8 * (w % 4) + 1] * sc;
      const f32x4 z = *reinterpret_cast<const f32x4 *>(from + w / 4 * STEP + 4 * D * (w % 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += z[e] * sc;
    }
    const auto row = deal.row(item.p, item.h, q);
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const f32x4 o = l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : f32x4{acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    const int64_t off = (((int64_t)row.b * a.work.Hk * a.work.G + row.qh) * a.work.N + row.i) * D;
    store4(static_cast<char *>(a.o) + off * (a.q_dtype == QFA_F32 ? 4 : 2), a.q_dtype, d, o);
  }
}

// O of the items that several workgroups share
struct PagedListMergeArgs {
  PagedWork work;
  void *o;
  int o_dtype;
  unsigned tiles, each;
};
template <int D> __global__ __launch_bounds__(256) void paged_list_merge_kernel(PagedListMergeArgs a) {
  constexpr int CL = D / 4, SLOTS = 256 / CL;
  __shared__ float red[SLOTS][D + 4];
  const int tid = threadIdx.x, d = 4 * (tid % CL), slot = tid / CL;
  PagedListDeal deal(a.work, PAGED_ROWS, SKV_TILE);
  deal.lists(a.tiles, a.each);
  PagedListDeal::Item it;
  deal.item(blockIdx.x, it);
  const PagedPieces mine(it.first, deal.each, it.tiles, 0, 0);
  if (mine.whole >= 0) return;   // stored
  const int r0 = PAGED_ROWS * it.rb, n = min(PAGED_ROWS, deal.rows - r0);
  auto store = [&](int r, const PagedSum &x) __attribute__((always_inline)) {
    const auto row = deal.row(it.p, it.h, r0 + r);
    const float inv = row.i >= it.s.tokens || x.l == 0.f ? 0.f : 1.0f / x.l;
    const int64_t off = (((int64_t)row.b * a.work.Hk * a.work.G + row.qh) * a.work.N + row.i) * D;
    store4(static_cast<char *>(a.o) + off * (a.o_dtype == QFA_F32 ? 4 : 2), a.o_dtype, d,
           f32x4{mul_zero_wins(x.acc[0], inv), mul_zero_wins(x.acc[1], inv), mul_zero_wins(x.acc[2], inv), mul_zero_wins(x.acc[3], inv)});
  };
  const int groups = n >= SLOTS ? 1 : SLOTS / n;   // of pieces
  for (int first = 0; first < n; first += SLOTS) {
    const int k = groups == 1 ? first + slot : slot % n, group = groups == 1 ? 0 : slot / n;
    const bool live = k < n && group < groups;
    PagedSum x[1] = {{NO_KEY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}}};
    if (live) {
      PagedPieces p = mine;
      p.in_block += k;
      paged_add<D, 1>(a.work, p, d, group, groups, x, 0);
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
    store(k, x[0]);
  }
}

// How the items are divided: each to a workgroup of its own, or, where few items with long lists leave CUs idle, all units evenly to two workgroups on
// every CU.  The kernel that joins the pieces costs 5.5 us, as much as about 32 tiles of a workgroup (20 of 256 elements).  Items of T
// tiles, us whole and cut:  64 elements 8 items T 32: 10.5, 11.7, T 48: 13.2, 11.6; 192 items T 64: 16.6, 19.6, T 256: 49, 43.8;  128: 8 items T 32: 12.4, 12.0,
// 64 items T 32: 12.7, 12.6, T 64: 19.8, 16.1, 192 items T 128: 36.3, 39.8;  256: 8 items T 16: 11.9, 13.6, T 32: 16.4, 13.8, 64 items T 32: 18.1, 15.6,
// 192 items T 256: 142, 151.
// (A list's places are counted, not what stands in them: the kernel for few rows walks all of them, the other one ends at the last block that the token sees.  2 x 333 tokens from
// position 0, us: 46.5 with lists of the 6 blocks that there are, 136 with 26 places of -1 behind them.)
// The kernel for up to four rows is as fast or faster from 512 items on (1024 of 256 elements), and for few keys: items x keys, us of
// paged_rows_kernel (whole or cut) and of it:  64 elements 8 x 128: 6.5, 6.2, 8 x 512: 7.9, 8.4, 256 x 512: 8.0, 8.6, 512 x 512: 11.7, 11.0,
// 1024 x 64: 10.6, 6.2, 1024 x 4096: 106, 104;  128: 8 x 256: 7.8, 7.2, 8 x 1024: 12.4, 14.3, 128 x 4096: 29.7, 43.6, 512 x 256: 11.4, 10.0,
// 512 x 4096: 99.4, 100.6, 1024 x 64: 14.6, 8.4;  256: 8 x 128: 8.6, 9.3, 512 x 512: 26.6, 29.1, 512 x 2048: 97, 102, 1024 x 64: 19.2, 14.3,
// 1024 x 2048: 189, 190, 2664 (333 tokens of one sequence) x 2048: 200, 152.
struct PagedListPlan {
  unsigned tiles, each;
  int grid;
  bool cut, few;
};
static PagedListPlan list_plan(int64_t items, int64_t keep, int page_log2, int64_t G, int D) {
  PagedListPlan p;
  p.few = G <= FEW_ROWS && (items >= (D == 256 ? 1024 : 512) || (D < 256 && keep << page_log2 <= 256));
  if (p.few) {
    p.tiles = (unsigned)(((keep << page_log2) + FEW_TILE - 1) / FEW_TILE);
    p.each = 0;
    p.grid = (int)items;
    p.cut = false;
    return p;
  }
  p.tiles = (unsigned)(((keep << page_log2) + SKV_TILE - 1) / SKV_TILE);
  const int64_t unit = p.tiles + LIST_EXTRA, total = items * unit, full = D == 256 ? 192 : 256;   // items that keep the chip busy
  p.cut = items < full && (int64_t)p.tiles * (full - items) > (D == 256 ? 20 : 32) * full;
  p.each = (unsigned)(p.cut ? max((int64_t)LIST_EXTRA, (total + LIST_WGS - 1) / LIST_WGS) : unit);
  p.grid = (int)((total + p.each - 1) / p.each);
  return p;
}
static int64_t list_items(int64_t B, int64_t N, int64_t Hk, int64_t G) { return B * N * Hk * ((G + PAGED_ROWS - 1) / PAGED_ROWS); }
int64_t paged_list_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t keep, int page_log2) {
  const PagedListPlan p = list_plan(list_items(B, N, Hk, H / Hk), keep, page_log2, H / Hk, D);
  return p.cut ? 2LL * p.grid * PAGED_ROWS * (D + 2) * 4 : 0;
}
double paged_list_units(int64_t B, int64_t H, int64_t Hk, int64_t N, int64_t keep, int page_log2) {
  return (double)list_items(B, N, Hk, H / Hk) * ((double)keep * (1 << page_log2) / SKV_TILE + 1 + LIST_EXTRA);
}

template <typename S, int D> static void launch_list(const PagedAttnKernelArgs &a, bool few, dim3 grid, hipStream_t st) {
  const bool fine = a.q_dtype == QFA_F32;
  if (few && fine) paged_list_few_kernel<S, D, true><<<grid, dim3(64 * FEW_WAVES), 0, st>>>(a);
  else if (few) paged_list_few_kernel<S, D, false><<<grid, dim3(64 * FEW_WAVES), 0, st>>>(a);
  else if (fine) paged_rows_kernel<S, D, PagedListDeal, false, true><<<grid, dim3(256), 0, st>>>(a);
  else paged_rows_kernel<S, D, PagedListDeal, false, false><<<grid, dim3(256), 0, st>>>(a);
}
template <int D> static int launch_d(const PagedListArgs &l, hipStream_t st) {
  const PagedAttnArgs &x = l.x;
  const int G = (int)(x.H / x.Hk);
  const int64_t items = list_items(x.B, x.N, x.Hk, G);
  const PagedListPlan p = list_plan(items, l.keep, x.page_log2, G, D);
  PagedAttnKernelArgs a = {};
  a.q = x.q; a.kc = x.cache.k_codes; a.ks = x.cache.k_scale; a.kz = x.cache.k_zero;
  a.vc = x.cache.v_codes; a.vs = x.cache.v_scale; a.vz = x.cache.v_zero; a.o = x.o; a.page_table = x.page_table;
  a.pages = x.pages; a.stb = x.stb; a.stw = x.stw; a.sqb = x.sq[0]; a.sqh = x.sq[1]; a.sqn = x.sq[2];
  a.width = (int)x.width; a.page_log2 = x.page_log2; a.q_dtype = x.q_dtype;
  a.sm_scale_log2 = x.sm_scale * kLog2e;
  a.blocks = l.blocks; a.keep = (int)l.keep; a.list_tiles = p.tiles; a.list_each = p.each;
  float *slots = static_cast<float *>(x.workspace);
  a.work = {x.starts, x.counts, (int)x.B, (int)x.Hk, G, (int)x.N, 1, 0, (int)(x.width << x.page_log2), p.grid, PAGED_ROWS, SKV_TILE, LIST_EXTRA, nullptr,
            slots, p.cut ? slots + 2LL * p.grid * PAGED_ROWS * D : nullptr, nullptr, nullptr};
  const dim3 grid((unsigned)p.grid), block(256);
  if (x.scale_dtype == QFA_F32) launch_list<float, D>(a, p.few, grid, st);
  else if (x.scale_dtype == QFA_F16) launch_list<_Float16, D>(a, p.few, grid, st);
  else launch_list<__bf16, D>(a, p.few, grid, st);
  if (int e = check_launch("qfa_attn_paged_blocks")) return e;
  if (!p.cut) return 0;
  paged_list_merge_kernel<D><<<dim3((unsigned)items), block, 0, st>>>({a.work, x.o, x.q_dtype, p.tiles, p.each});
  return check_launch("qfa_attn_paged_blocks (merge)");
}
int launch_paged_list(const PagedListArgs &x, hipStream_t st) {
  if (x.x.D == 64) return launch_d<64>(x, st);
  if (x.x.D == 128) return launch_d<128>(x, st);
  return launch_d<256>(x, st);
}

}  // namespace qfa
