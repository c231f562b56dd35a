// The attention weight that every key of a paged INT8 cache gets from the rows of a call:
//     out[b, h, j] = decay * before[b, h, j] + sum over tokens n and the query heads g of key head h of  exp(sm_scale * q^_gn . k^_j - lse_gn),
// with the scores of attention itself (qfa_paged_attn.hip: INT8 products, exact zero-point terms) and its log-sum-exp, so that the sum is the
// one over that softmax's probabilities.
//
// One pass over the keys (D + 3 bytes of each), no exchange between workgroups and no atomics: a wave holds 64 keys, all rows pass by, and a
// key's sum is made in a fixed order.  Rows are the rows of the product and keys its columns, so a key's scale and zero point are one value
// per lane and its sum is three lane exchanges for 64 keys.  Up to 16 rows are quantized in the workgroup and stay in registers while it
// takes several times 256 keys; more are quantized once by a launch in front and pass through LDS 64 at a time.
#include "qfa_host.h"
#include "qfa_quant_row.h"
#include "qfa_skv_common.h"

namespace qfa {

struct WeighKernelArgs {
  PagedWeighArgs w;
  int G, steps, chunks, rows;
  float sm_scale_log2;
  const int8_t *q_codes; const float *q_scale; const int8_t *q_zero; const int32_t *q_sum;   // many rows: quantized, dense
};

template <int D, int PR> struct WeighPanel {
  static constexpr int CPR = D / 16;
  unsigned char codes[PR * D];   // rows, their chunks of 16 bytes moved by the row: 16 rows at one chunk lie in different banks
  float a[PR], lse[PR];          // scale * sm_scale * log2(e); the log-sum-exp in log2 units (infinite: the row counts for nothing)
  int zero[PR], c[PR], last[PR]; // zero point; code sum - D * zero point; the last key that the row sees
  static __device__ __forceinline__ int chunk(int row, int c) { return row * D + ((c ^ (row % CPR)) << 4); }
};

template <typename S, int D, bool ONE> __global__ __launch_bounds__(256) void paged_weigh_kernel(WeighKernelArgs p) {
  constexpr int KM = D / 64, PR = ONE ? 16 : 64;
  typedef WeighPanel<D, PR> Panel;
  __shared__ __attribute__((aligned(16))) Panel panel;
  const PagedAttnArgs &x = p.w.x;
  const int tid = threadIdx.x, lane = tid % 64, c16 = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int64_t bh = index_div(blockIdx.x, p.chunks), chunk = blockIdx.x - bh * p.chunks, b = index_div(bh, x.Hk), h = bh - b * x.Hk;
  const int start = x.starts[b], tokens = (int)(x.counts ? max((int64_t)0, min((int64_t)x.counts[b], x.N)) : x.N);
  const int slots = (int)(x.width << x.page_log2);
  // the last key that any row sees
  const int last = tokens == 0 ? -1 : (int)max((int64_t)-1, min((int64_t)start + tokens - 1, (int64_t)slots - 1));
  const float *before = p.w.before ? p.w.before + bh * slots : nullptr;
  float *out = p.w.out + bh * slots;
  const int begin = (int)chunk * 256 * p.steps;
  if (begin > last && before == out && p.w.decay == 1.0f) return;
  auto last_of = [&](int i) __attribute__((always_inline)) -> int {   // token i's
    return x.causal ? (int)max((int64_t)-1, min((int64_t)start + i, (int64_t)slots - 1)) : last;
  };
  const bool work = begin <= last;   // (uniform)
  const i32x4 ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
  i32x4 qf[KM];
  float a[4], lse[4];
  int zq[4], cq[4], lim[4], least = 0;
  auto rows_from = [&](int r0) __attribute__((always_inline)) {   // 16 rows out of the panel
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
    least = min(min(lim[0], lim[1]), min(lim[2], lim[3]));
    least = min(least, __shfl_xor(least, 16, 64));
    least = __builtin_amdgcn_readfirstlane(min(least, __shfl_xor(least, 32, 64)));
  };
  // constants of row r (of the call's sequence and key head), for lane 0 of those that hold it
  auto constants = [&](int at, int r, float scale, int zero, int sum) __attribute__((always_inline)) {
    const int i = min(r, p.rows - 1) / p.G;
    const int64_t row = (b * x.H + h * p.G + min(r, p.rows - 1) - i * p.G) * x.N + i;
    const float f = scale * p.sm_scale_log2;
    const bool there = r < p.rows && i < tokens;
    panel.a[at] = there ? (f < 0x1p-126f ? 0x1p-126f : f) : 0.f;
    panel.lse[at] = there ? p.w.lse[row] * kLog2e : INFINITY;
    panel.zero[at] = zero;
    panel.c[at] = sum - D * zero;
    panel.last[at] = there ? last_of(i) : last;
  };
  if (ONE && work) {
    constexpr int LPT = D / 8, TPP = 256 / LPT, PASSES = (16 + TPP - 1) / TPP;
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int row = ps * TPP + tid / LPT, sub = tid % LPT, r = min(row, p.rows - 1), i = r / p.G;
      const int64_t off = b * x.sq[0] + (h * p.G + r - i * p.G) * x.sq[1] + i * x.sq[2] + sub * 8;
      float v[8];
      if (x.q_dtype == QFA_F32) Load8<float>::run(static_cast<const float *>(x.q) + off, v);
      else if (x.q_dtype == QFA_BF16) Load8<__bf16>::run(static_cast<const __bf16 *>(x.q) + off, v);
      else Load8<_Float16>::run(static_cast<const _Float16 *>(x.q) + off, v);
      const QuantRow<8> q = quant_row<LPT, false, 8>(v, true);
      if (row < 16) {
        *reinterpret_cast<u32x2 *>(panel.codes + Panel::chunk(row, sub / 2) + 8 * (sub % 2)) = u32x2{q.codes[0], q.codes[1]};
        if (sub == 0) constants(row, row, q.scale, (int)q.zp, q.sum);
      }
    }
    __syncthreads();
    rows_from(0);
  }

  const S *scales = static_cast<const S *>(x.cache.k_scale);
  for (int step = 0; step < p.steps; ++step) {
    const int key0 = begin + 256 * step + 64 * wave, key = key0 + lane;
    if (ONE && key0 >= slots) break;   // (many rows: all waves go to the barriers)
    const bool mine = key0 <= last;    // (uniform over the wave)
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    if (mine || (!ONE && work)) {
      // ---- 64 keys: the page of each, a key's constants in its lane, the codes of four tiles of 16
      const int at = key >> x.page_log2;
      const int page = x.page_table[b * x.stb + min(at, (int)x.width - 1) * x.stw];
      const int id = at < x.width && page >= 0 && page < x.pages && key <= last ? page : -1;
      const int64_t row = (((int64_t)max(id, 0) * x.Hk + h) << x.page_log2) + (key & ((1 << x.page_log2) - 1));
      const float scale_mine = (float)scales[row];
      const int zero_mine = x.cache.k_zero[row];
      i32x4 k[4][KM];
      int rk[4], zk[4], there = 0;
      float sk[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int id_t = __builtin_amdgcn_readlane(id, 16 * t);   // (-1 behind the last key: of a tile that ends in a sequence the first keys exist)
        there |= id_t >= 0 ? 1 << t : 0;
        const int64_t first = (((int64_t)max(id_t, 0) * x.Hk + h) << x.page_log2) + ((key0 + 16 * t) & ((1 << x.page_log2) - 1));
        const rsrc_t rs = make_rsrc(x.cache.k_codes + first * D, id_t >= 0 ? 16 * D : 0);
#pragma unroll
        for (int m = 0; m < KM; ++m) k[t][m] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, c16 * D + 16 * g, 64 * m, 0));
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        sk[t] = __shfl(scale_mine, 16 * t + c16, 64);
        zk[t] = __shfl(zero_mine, 16 * t + c16, 64);
        i32x4 r = {0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < KM; ++m) r = __builtin_amdgcn_mfma_i32_16x16x64_i8(ones, k[t][m], r, 0, 0, 0);
        rk[t] = r[0];
      }
      // ---- the weights that 16 rows give
      auto add = [&]() __attribute__((always_inline)) {
        const bool masked = key0 + 63 > least || there != 15;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          i32x4 s = {0, 0, 0, 0};
#pragma unroll
          for (int m = 0; m < KM; ++m) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(qf[m], k[t][m], s, 0, 0, 0);
          float w[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int dot = s[v] - __mul24(zq[v], rk[t]) - __mul24(zk[t], cq[v]);
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
        add();
      } else {
        for (int r0 = 0; r0 < p.rows; r0 += PR) {
          __syncthreads();   // the rows before are done with
          for (int y = tid; y < PR * Panel::CPR; y += 256) {
            const int at_row = y / Panel::CPR, r = min(r0 + at_row, p.rows - 1), i = r / p.G;
            const int64_t from = (b * x.H + h * p.G + r - i * p.G) * x.N + i;
            *reinterpret_cast<u32x4 *>(panel.codes + Panel::chunk(at_row, y % Panel::CPR)) =
                *reinterpret_cast<const u32x4 *>(p.q_codes + from * D + 16 * (y % Panel::CPR));
          }
          if (tid < PR) {
            const int r = min(r0 + tid, p.rows - 1), i = r / p.G;
            const int64_t from = (b * x.H + h * p.G + r - i * p.G) * x.N + i;
            constants(tid, r0 + tid, p.q_scale[from], p.q_zero[from], p.q_sum[from]);
          }
          __syncthreads();
          if (mine) {
            const int n = min(PR, p.rows - r0);
            for (int r = 0; r < n; r += 16) {
              rows_from(r);
              add();
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
    if (key < slots) out[key] = before ? __builtin_fmaf(p.w.decay, before[key], total) : total;
  }
}

// (rows as the launch in front quantizes them)
int64_t paged_weigh_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int D) {
  return N * (H / Hk) <= 16 ? 0 : (B * H * N * (D + 9) + 15) / 16 * 16;
}
template <typename S, int D> static int launch_sd(const PagedWeighArgs &w, hipStream_t st) {
  const PagedAttnArgs &x = w.x;
  WeighKernelArgs p = {};
  p.w = w;
  p.G = (int)(x.H / x.Hk);
  p.rows = (int)(x.N * p.G);
  p.sm_scale_log2 = x.sm_scale * kLog2e;
  const int64_t BH = x.B * x.Hk, slots = x.width << x.page_log2;
  const bool one = p.rows <= 16;
  p.steps = 1;
  while (one && p.steps < 4 && BH * ((slots + 512 * p.steps - 1) / (512 * p.steps)) >= 2048) p.steps *= 2;
  p.chunks = (int)((slots + 256 * p.steps - 1) / (256 * p.steps));
  if ((double)BH * p.chunks > 2147483647.0) return set_error(QFA_EUNSUPPORTED, "paged_weights: too many keys for one launch");
  if (!one) {
    const int64_t rows = x.B * x.H * x.N;
    int8_t *codes = static_cast<int8_t *>(x.workspace), *zero = codes + rows * (D + 8);
    float *scale = reinterpret_cast<float *>(codes + rows * D);
    int32_t *sum = reinterpret_cast<int32_t *>(codes + rows * (D + 4));
    if (int e = launch_quant(x.q, x.q_dtype, codes, scale, nullptr, 0, zero, sum, x.B, x.H, x.N, D, x.sq[0], x.sq[1], x.sq[2], x.H * x.N * D, x.N * D, D, st)) return e;
    p.q_codes = codes; p.q_scale = scale; p.q_zero = zero; p.q_sum = sum;
  }
  const dim3 grid((unsigned)(BH * p.chunks)), block(256);
  if (one) paged_weigh_kernel<S, D, true><<<grid, block, 0, st>>>(p);
  else paged_weigh_kernel<S, D, false><<<grid, block, 0, st>>>(p);
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
