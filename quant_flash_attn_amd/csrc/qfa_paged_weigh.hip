// The attention weight that every key of a paged INT8 cache gets from the rows of a call:
//     out[b, h, j] = decay * before[b, h, j] + sum over tokens n and the query heads g of key head h of  exp(sm_scale * q^_gn . k^_j - lse_gn),
// with the scores of attention itself (qfa_paged_attn.hip: INT8 products, exact zero-point terms) and its log-sum-exp, so that the sum is the
// one over that softmax's probabilities.
//
// One pass over the keys (D + 3 bytes of each), no exchange between workgroups and no atomics: a wave holds 64 keys, all rows pass by, and a
// key's sum is made in a fixed order.  Rows are the rows of the product and keys its columns, so a key's scale and zero point are one value
// per lane and its sum is three lane exchanges for 64 keys.  Up to 16 rows are quantized in the workgroup and stay in registers while it
// takes several times 256 keys; more are quantized once by a launch in front (up to 32 by every workgroup, where those are few), and pass
// through LDS in panels of 64, the next one on its way while one is worked on.
//
// Few rows are bound by reading the keys: 64 sequences of 65 to 8192 keys, 8 key heads of 4 x 128, 16 keys a page: 64 us, 4.9 TB/s (at the 5 TB/s of a large
// copy 62 us).  128 rows on 4 x 4000 to 8000 keys, 8 key heads of 128: 18.6 us behind 4.2 of the launch in front.  All workgroups run at once and wait, for
// page numbers, keys and one block of rows after the other: the vector pipe, seven instructions a score, is busy for 30 % of the time, the matrix pipe 6 %.
#include "qfa_host.h"
#include "qfa_quant_row.h"
#include "qfa_skv_common.h"

namespace qfa {

struct WeighKernelArgs {
  PagedWeighArgs w;
  int G, steps, chunks, rows;
  float sm_scale_log2;
  const unsigned char *panels;   // many rows: those of every sequence and key head, ready to be copied to LDS
  int panels_each;
  bool here;   // ... made by every workgroup itself
};

template <int D, int PR> struct __attribute__((aligned(16))) WeighPanel {
  static constexpr int CPR = D / 16;
  unsigned char codes[PR * D];   // rows, their chunks of 16 bytes moved by the row: 16 rows at one chunk lie in different banks
  float a[PR], lse[PR];          // scale * sm_scale * log2(e); the log-sum-exp in log2 units (infinite: the row counts for nothing)
  int zero[PR], c[PR], last[PR]; // - zero point; D * zero point - code sum; the last key that the row sees
  static __device__ __forceinline__ int chunk(int row, int c) { return row * D + ((c ^ (row % CPR)) << 4); }
  // the constants of a row, token i's of `tokens`
  __device__ __forceinline__ void constants(int at, bool there, float scale, int z, int sum, float row_lse, int row_last) {
    a[at] = there ? (scale < 0x1p-126f ? 0x1p-126f : scale) : 0.f;
    lse[at] = there ? row_lse * kLog2e : INFINITY;
    zero[at] = -z;
    c[at] = D * z - sum;
    last[at] = row_last;
  }
};

// A sequence's tokens and the last keys that they see
struct WeighSeq {
  int start, tokens, slots, last;   // last: of any row
  __device__ __forceinline__ WeighSeq(const PagedAttnArgs &x, int64_t b) {
    start = x.starts[b];
    tokens = (int)(x.counts ? max((int64_t)0, min((int64_t)x.counts[b], x.N)) : x.N);
    slots = (int)(x.width << x.page_log2);
    last = tokens == 0 ? -1 : (int)max((int64_t)-1, min((int64_t)start + tokens - 1, (int64_t)slots - 1));
  }
  __device__ __forceinline__ int last_of(const PagedAttnArgs &x, int i) const {   // token i's
    return x.causal ? (int)max((int64_t)-1, min((int64_t)start + i, (int64_t)slots - 1)) : last;
  }
};

// 16 rows of a sequence and key head (row = token * G + head), quantized into a panel at r0 % PR: D/8 lanes hold a row.  A row that is not there, or is
// padding, counts for nothing
template <int D> struct WeighRows {
  static constexpr int LPT = D / 8, TPP = 256 / LPT, PASSES = (16 + TPP - 1) / TPP;
  float v[PASSES][8], lse[PASSES];
  __device__ __forceinline__ void load(const WeighKernelArgs &p, int64_t b, int64_t h, int r0) {
    const PagedAttnArgs &x = p.w.x;
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int row = ps * TPP + threadIdx.x / LPT, sub = threadIdx.x % LPT, r = min(r0 + row, p.rows - 1), i = r / p.G;
      const int64_t head = h * p.G + r - i * p.G, off = b * x.sq[0] + head * x.sq[1] + i * x.sq[2] + sub * 8;
      lse[ps] = p.w.lse[(b * x.H + head) * x.N + i];
      if (x.q_dtype == QFA_F32) Load8<float>::run(static_cast<const float *>(x.q) + off, v[ps]);
      else if (x.q_dtype == QFA_BF16) Load8<__bf16>::run(static_cast<const __bf16 *>(x.q) + off, v[ps]);
      else Load8<_Float16>::run(static_cast<const _Float16 *>(x.q) + off, v[ps]);
    }
  }
  template <typename Panel> __device__ __forceinline__ void put(const WeighKernelArgs &p, const WeighSeq &seq, Panel &panel, int r0) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int row = ps * TPP + threadIdx.x / LPT, sub = threadIdx.x % LPT, r = r0 + row;
      if (r0 + ps * TPP + wave * (64 / LPT) >= p.rows) break;   // (uniform over the wave)
      const QuantRow<8> q = quant_row<LPT, false, 8>(v[ps], true);
      if (row < 16 && r < p.rows) {
        const int at = r % (int)(sizeof(panel.a) / 4), i = r / p.G;
        *reinterpret_cast<u32x2 *>(panel.codes + Panel::chunk(at, sub / 2) + 8 * (sub % 2)) = u32x2{q.codes[0], q.codes[1]};
        const bool there = i < seq.tokens;
        if (sub == 0) panel.constants(at, there, q.scale * p.sm_scale_log2, (int)q.zp, q.sum, lse[ps], there ? seq.last_of(p.w.x, i) : seq.last);
      }
    }
    const int r = r0 + threadIdx.x;   // (the codes behind hold anything)
    if (threadIdx.x < 16 && r >= p.rows) panel.constants(r % (int)(sizeof(panel.a) / 4), false, 0.f, 0, 0, 0.f, seq.last);
  }
};

constexpr int WEIGH_PANEL = 64;
// Many rows: the panels of every sequence and key head, 16 rows of one a workgroup
template <int D> __global__ __launch_bounds__(256) void weigh_rows_kernel(WeighKernelArgs p) {
  typedef WeighPanel<D, WEIGH_PANEL> Panel;
  const int per = p.panels_each * (WEIGH_PANEL / 16);
  const int64_t bh = index_div(blockIdx.x, per), b = index_div(bh, p.w.x.Hk), h = bh - b * p.w.x.Hk;
  const int r0 = 16 * (int)(blockIdx.x - bh * per);
  const WeighSeq seq(p.w.x, b);
  WeighRows<D> rows;
  rows.load(p, b, h, r0);
  rows.put(p, seq, reinterpret_cast<Panel *>(const_cast<unsigned char *>(p.panels))[bh * p.panels_each + r0 / WEIGH_PANEL], r0);
}

template <typename S, int D, bool ONE, bool STREAM> __global__ __launch_bounds__(256, D == 256 ? 2 : ONE && !STREAM ? 5 : 4) void paged_weigh_kernel(WeighKernelArgs p) {
  constexpr int KM = D / 64, PR = ONE ? 16 : WEIGH_PANEL;
  typedef WeighPanel<D, PR> Panel;
  // many rows: two panels, each with room for whole copies of 1024 bytes
  constexpr int PIECES = (sizeof(Panel) + 1023) / 1024, BUF = ONE ? sizeof(Panel) : 1024 * PIECES;
  __shared__ __attribute__((aligned(16))) unsigned char smem[ONE ? BUF : 2 * BUF];
  __shared__ __attribute__((aligned(16))) unsigned char held[STREAM ? 256 * D : 16];   // the keys of a step
  const PagedAttnArgs &x = p.w.x;
  const int tid = threadIdx.x, lane = tid % 64, c16 = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  // (sequences before chunks of keys: not every sequence has keys in the later ones)
  const unsigned unit = blockIdx.x / (unsigned)x.Hk;
  const int64_t chunk = unit / (unsigned)x.B, b = unit - (unsigned)chunk * (unsigned)x.B, h = blockIdx.x % (unsigned)x.Hk, bh = b * x.Hk + h;
  const WeighSeq seq(x, b);
  const int slots = seq.slots, last = seq.last;
  const float *before = p.w.before ? p.w.before + bh * slots : nullptr;
  float *out = p.w.out + bh * slots;
  const int begin = (int)chunk * 256 * p.steps;
  if (begin > last) {   // slots behind the last key, all loads at once (step by step these workgroups would keep the others from the CUs for several waits)
    const int end = min(slots, begin + 256 * p.steps);
    if (before == out && p.w.decay == 1.0f) return;
#pragma unroll 4
    for (int i = begin + tid; i < end; i += 256) out[i] = before ? p.w.decay * before[i] : 0.f;
    return;
  }
  const i32x4 ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
  i32x4 qf[KM];
  float a[4], lse[4];
  int zq[4], cq[4], lim[4];
  auto rows_from = [&](const Panel &panel, int r0) __attribute__((always_inline)) {   // 16 rows out of the panel
#pragma unroll
    for (int m = 0; m < KM; ++m) qf[m] = *reinterpret_cast<const i32x4 *>(panel.codes + Panel::chunk(r0 + c16, 4 * m + g));
    const f32x4 av = *reinterpret_cast<const f32x4 *>(panel.a + r0 + 4 * g), lv = *reinterpret_cast<const f32x4 *>(panel.lse + r0 + 4 * g);
    const i32x4 zv = *reinterpret_cast<const i32x4 *>(panel.zero + r0 + 4 * g), cv = *reinterpret_cast<const i32x4 *>(panel.c + r0 + 4 * g),
                kv = *reinterpret_cast<const i32x4 *>(panel.last + r0 + 4 * g);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      a[v] = av[v];
      lse[v] = lv[v];
      zq[v] = zv[v];
      cq[v] = cv[v];
      lim[v] = kv[v];
    }
  };
  // 64 keys of a step: the page of each, a key's constants in its lane, the codes of four tiles of 16
  struct Keys {
    i32x4 k[4][KM];
    float scale;
    int zero, there;   // there: bit per tile, its page exists
  };
  // Keys that are not to stay in the caches (STREAM) are loaded into LDS as they lie, 16 bytes a lane, and read from there in the fragments'
  // order: loaded in that order, two loads of 64 bytes share a line, which would be fetched twice.  Within a row the 16-byte parts are
  // exchanged by its number, for the banks.
  constexpr int PARTS = D / 16, PER_LINE = PARTS < 8 ? 8 / PARTS : 1, TURNS = PARTS < 8 ? PARTS : 8;   // (rows in 128 bytes)
  auto k_at = [](int row, int part) __attribute__((always_inline)) -> int { return row * D + 16 * (part ^ (row / PER_LINE % TURNS)); };
  unsigned char *kl = held + 64 * D * wave;
  int k_off[4];   // (KM of them)
#pragma unroll
  for (int m = 0; m < KM; ++m) k_off[m] = k_at(m * (1024 / D) + lane / PARTS, lane % PARTS) - 1024 * m;
  const S *scales = static_cast<const S *>(x.cache.k_scale);
  auto page_of = [&](int key) __attribute__((always_inline)) -> int {
    const int at = key >> x.page_log2;
    const int page = x.page_table[b * x.stb + min(at, (int)x.width - 1) * x.stw];
    return at < x.width && page >= 0 && page < x.pages && key <= last ? page : -1;
  };
  auto load = [&](Keys &t, int key0, int id) __attribute__((always_inline)) {
    const int64_t row = (((int64_t)max(id, 0) * x.Hk + h) << x.page_log2) + ((key0 + lane) & ((1 << x.page_log2) - 1));
    t.scale = (float)scales[row];
    t.zero = x.cache.k_zero[row];
    t.there = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int id_t = __builtin_amdgcn_readlane(id, 16 * i);   // (-1 behind the last key: of a tile that ends in a sequence the first keys exist)
      t.there |= id_t >= 0 ? 1 << i : 0;
      const int64_t first = (((int64_t)max(id_t, 0) * x.Hk + h) << x.page_log2) + ((key0 + 16 * i) & ((1 << x.page_log2) - 1));
      const rsrc_t rs = make_rsrc(x.cache.k_codes + first * D, id_t >= 0 ? 16 * D : 0);
#pragma unroll
      for (int m = 0; m < KM; ++m)
        if constexpr (STREAM) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lptr_t)(kl + 16 * D * i + 1024 * m), 16, k_off[m], 1024 * m, 0, LOAD_ONCE);
        else t.k[i][m] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, c16 * D + 16 * g, 64 * m, 0));
    }
  };
  int page = page_of(begin + 64 * wave + lane);
  Keys keys;
  const rsrc_t panels = make_rsrc(ONE ? nullptr : p.panels + bh * p.panels_each * (int64_t)sizeof(Panel), ONE ? 0u : (unsigned)(p.panels_each * sizeof(Panel)));
  auto fetch = [&](int panel) __attribute__((always_inline)) {   // (past the last panel's end: zeros)
#pragma unroll
    for (int e = 0; e < (PIECES + 3) / 4; ++e) {
      const int piece = wave + 4 * e;
      if (PIECES % 4 == 0 || piece < PIECES)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(panels, (lptr_t)(smem + (panel & 1) * BUF + 1024 * piece), 16, 16 * lane, panel * (int)sizeof(Panel) + 1024 * piece, 0, 0);
    }
  };
  if constexpr (ONE) {
    WeighRows<D> rows;
    rows.load(p, b, h, 0);
    rows.put(p, seq, *reinterpret_cast<Panel *>(smem), 0);
    __syncthreads();
    rows_from(*reinterpret_cast<const Panel *>(smem), 0);
  } else {
    if (!p.here) fetch(0);
    load(keys, begin + 64 * wave, page);
    if (p.here)
      for (int r0 = 0; r0 < p.rows; r0 += 16) {
        WeighRows<D> rows;
        rows.load(p, b, h, r0);
        rows.put(p, seq, *reinterpret_cast<Panel *>(smem), r0);
      }
  }

  for (int step = 0; step < p.steps; ++step) {
    const int key0 = begin + 256 * step + 64 * wave, key = key0 + lane;
    if (ONE && key0 >= slots) break;   // (many rows: all waves go to the barriers)
    const bool mine = key0 <= last;    // (uniform over the wave)
    const float was = before ? before[min(key, slots - 1)] : 0.f;   // (asked for beside the keys: behind them a step would wait for it alone)
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    if (mine || !ONE) {   // (of one block of rows a wave that is past the last key stays so)
      if constexpr (ONE) {   // (many rows: one step, and its keys are on their way already)
        if constexpr (STREAM) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the keys before are read)
        load(keys, key0, page);
        if (step + 1 < p.steps) page = page_of(key + 256);
        if constexpr (STREAM) {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the keys are in LDS
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int m = 0; m < KM; ++m) keys.k[t][m] = *reinterpret_cast<const i32x4 *>(kl + 16 * D * t + k_at(c16, 4 * m + g));
        }
      }
      i32x4 (&k)[4][KM] = keys.k;
      const int there = keys.there;
      int rk[4], zk[4];
      float sk[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        sk[t] = __shfl(keys.scale, 16 * t + c16, 64);
        zk[t] = __shfl(keys.zero, 16 * t + c16, 64);
        i32x4 r = {0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < KM; ++m) r = __builtin_amdgcn_mfma_i32_16x16x64_i8(ones, k[t][m], r, 0, 0, 0);
        rk[t] = r[0];
      }
      // ---- the weights that 16 rows give
      auto add = [&](int first_row) __attribute__((always_inline)) {
        // (rows are in the order of their tokens: the first one sees the least)
        const bool masked = key0 + 63 > seq.last_of(x, first_row / p.G) || there != 15;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          i32x4 s = {0, 0, 0, 0};
#pragma unroll
          for (int m = 0; m < KM; ++m) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(qf[m], k[t][m], s, 0, 0, 0);
          float w[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int dot = s[v] + __mul24(zq[v], rk[t]) + __mul24(cq[v], zk[t]);
            w[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(a[v], (float)dot * sk[t], -lse[v]));
          }
          if (masked) {
#pragma unroll
            for (int v = 0; v < 4; ++v)
              if (key0 + 16 * t + c16 > lim[v] || !(there >> t & 1)) w[v] = 0.f;
          }
          sum[t] += (w[0] + w[1]) + (w[2] + w[3]);
        }
      };
      if constexpr (ONE) {
        add(0);
      } else {
        for (int i = 0; i < p.panels_each; ++i) {
          dma_wait();
          __syncthreads();   // this panel is there, and nobody looks at the one before any more
          if (i + 1 < p.panels_each) fetch(i + 1);
          if (mine) {
            const Panel &panel = *reinterpret_cast<const Panel *>(smem + (i & 1) * BUF);
            const int n = min(PR, p.rows - PR * i);
            for (int r = 0; r < n; r += 16) {
              rows_from(panel, r);
              add(PR * i + r);
            }
          }
        }
      }
    }
    // ---- of the four groups of lanes, each with its rows' part of four tiles: group t gets tile t
    float y[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float keep = g >= 2 ? sum[2 + t] : sum[t], send = g >= 2 ? sum[t] : sum[2 + t];
      y[t] = keep + __shfl_xor(send, 32, 64);
    }
    const float keep = g & 1 ? y[1] : y[0], send = g & 1 ? y[0] : y[1];
    const float total = keep + __shfl_xor(send, 16, 64);
    if (key < slots) out[key] = before ? __builtin_fmaf(p.w.decay, was, total) : total;
  }
}

// (the panels that the launch in front makes)
static int64_t panel_count(int64_t rows) { return (rows + WEIGH_PANEL - 1) / WEIGH_PANEL; }
int64_t paged_weigh_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int D) {
  const int64_t rows = N * (H / Hk);
  return rows <= 16 ? 0 : B * Hk * panel_count(rows) * (WEIGH_PANEL * (D + 20));
}
template <typename S, int D> static int launch_sd(const PagedWeighArgs &w, hipStream_t st) {
  const PagedAttnArgs &x = w.x;
  static_assert(sizeof(WeighPanel<D, WEIGH_PANEL>) == WEIGH_PANEL * (D + 20), "as the workspace counts them");
  WeighKernelArgs p = {};
  p.w = w;
  p.G = (int)(x.H / x.Hk);
  p.rows = (int)(x.N * p.G);
  p.sm_scale_log2 = x.sm_scale * kLog2e;
  p.panels = static_cast<const unsigned char *>(x.workspace);
  p.panels_each = (int)panel_count(p.rows);
  const int64_t BH = x.B * x.Hk, slots = x.width << x.page_log2;
  const bool one = p.rows <= 16;
  p.steps = 1;
  while (one && p.steps < 4 && BH * ((slots + 512 * p.steps - 1) / (512 * p.steps)) >= 2048) p.steps *= 2;
  p.chunks = (int)((slots + 256 * p.steps - 1) / (256 * p.steps));
  const double quarters = (double)BH * p.panels_each * (WEIGH_PANEL / 16);
  if ((double)BH * p.chunks > 2147483647.0 || quarters > 2147483647.0 || (double)p.panels_each * (WEIGH_PANEL * (D + 20)) > 2147483647.0)
    return set_error(QFA_EUNSUPPORTED, "paged_weights: too many keys or rows for one launch");
  // Up to two blocks of rows are quantized by every workgroup itself where those are few: the launch in front costs more.  8 key heads, keys x sequences, us
  // with the launch and without:  32 rows of 64 elements 512 x 1: 10.3, 6.4, 2048 x 16: 10.8, 9.2, 8192 x 16: 24.4, 31.1;  of 128 512 x 1: 8.7, 6.4, 32768 x 1: 13.3,
  // 12.6, 8192 x 16: 31.4, 37.0;  of 256 512 x 1: 10.9, 9.2, 2048 x 16: 21.0, 23.8;  64 rows of 128 512 x 1: 9.4, 9.4, 8192 x 4: 15.7, 19.0
  p.here = !one && p.rows <= 32 && BH * p.chunks <= (D == 256 ? 512 : 1024);
  if (!one && !p.here) {
    weigh_rows_kernel<D><<<dim3((unsigned)quarters), dim3(256), 0, st>>>(p);
    if (int e = check_launch("qfa_paged_weights (rows)")) return e;
  }
  const dim3 grid((unsigned)(BH * p.chunks)), block(256);
  // Keys that outgrow the last-level cache, with what else is read of it, are not to stay there.  One token, 32 sequences with 8 key heads, keys in MiB, us without
  // and with:  64 elements 128: 32.4, 36.0, 256: 58.0, 63.5, 384: 100.9, 93.3, 1024: 265, 237;  128: 256: 49.8, 55.4, 384: 90.6, 82.0, 1024: 238, 215;  256: 256: 48.7,
  // 54.6, 384: 83.2, 83.3, 1024: 217, 208.  (Non-temporal loads in the fragments' order: 64 sequences of 65 to 8192 keys 83 instead of 72 and, these, 64.)
  // The table's slots are counted, for the host does not know the lengths, and all of them are written: 64 sequences of 65 to 1024 keys 13.0 under their own table of 1024 slots, 17.4
  // under one of 8192 (32 MiB of weights in and out), 53.3 under one of 32768 (128 MiB); of 65 to 8192 keys 64 and, under 32768 slots, 99.5.
  const bool stream = one && (double)BH * (double)slots * D > 320.0 * (1 << 20);
  if (stream) paged_weigh_kernel<S, D, true, true><<<grid, block, 0, st>>>(p);
  else if (one) paged_weigh_kernel<S, D, true, false><<<grid, block, 0, st>>>(p);
  else paged_weigh_kernel<S, D, false, false><<<grid, block, 0, st>>>(p);
  return check_launch("qfa_paged_weights");
}
template <typename S> static int launch_s(const PagedWeighArgs &w, hipStream_t st) {
  if (w.x.D == 64) return launch_sd<S, 64>(w, st);
  if (w.x.D == 128) return launch_sd<S, 128>(w, st);
  return launch_sd<S, 256>(w, st);
}
int launch_paged_weigh(const PagedWeighArgs &w, hipStream_t st) {
  if (w.x.scale_dtype == QFA_F32) return launch_s<float>(w, st);
  if (w.x.scale_dtype == QFA_F16) return launch_s<_Float16>(w, st);
  return launch_s<__bf16>(w, st);
}

}  // namespace qfa
