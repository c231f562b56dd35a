// RMSNorm of every head's row and the position rotation, in one pass, and its gradient:
//     y = rot(x * r * w),   r = 1 / sqrt(mean(x^2) + eps)
//     g = rot^T(dy),  dw = sum over rows of g x r,  dx = r (g w - x r mean((g w) x r))
// Bound by memory: the forward reads and writes each row once, the backward reads x (with a weight) and dy and writes dx; r is computed again
// from x, which it reads anyway, so the forward keeps nothing.  4 x 64 heads x 4096 x 128 bf16: forward 102 us (5.3 TB/s), gradient
// 150 us (5.4 TB/s); a copy of that size 5.0.
//
// A row is held by D/16 lanes (RopeLane), a workgroup of 256 threads holds 4096/D tokens of one head at a time and walks over
// `heads_each` heads of these tokens, so that the angles (4 D bytes of fp32 per token against 2 D of a 16-bit row) are read once
// for all of them.  Queries and keys go out in one launch.  Everything in between is fp32, one rounding at the end.
//
// dw: a thread adds up what it sees in registers; the workgroup's threads meet in LDS and leave one row of partial sums, which
// a second small kernel adds up in a fixed order (no atomics: the same call gives the same bits): 8 us for 2 x 2048 rows of 128.
#include "qfa_rope_row.h"

namespace qfa {

struct NormRopeTensor {
  const void *x, *dy, *w;
  void *y;           // forward: y, backward: dx (nullable)
  float *dw_parts;   // backward: [groups][D], groups as dw_groups counts them
  int64_t H, sxb, sxh, sxn, syb, syh, syn, sgb, sgh, sgn;
  int64_t sw;        // elements between the heads' weights (0: one for all)
  int heads_each, head_groups;
};
struct NormRopeKernelArgs {
  NormRopeTensor t[2];
  const float *cos, *sin;
  const int32_t *pos;
  int64_t rows, spb, spn, B, N;
  float eps;
  int half, step, w_f32;
  unsigned blocks0, token_blocks;
};

template <typename T> __device__ __forceinline__ void load_weight(const void *w, int w_f32, int64_t at, float *v) {
  if (w_f32) load8<float>(static_cast<const float *>(w) + at, v);
  else load8<T>(static_cast<const T *>(w) + at, v);
}

template <typename T, int D, bool INTERLEAVED, bool BACK, bool ONCE>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeKernelArgs p) {
  constexpr int LPR = D / 16, TOK = 256 / LPR;
  const bool second = blockIdx.x >= p.blocks0;
  const NormRopeTensor &a = p.t[second];
  const unsigned id = second ? blockIdx.x - p.blocks0 : blockIdx.x;
  const unsigned tb = id / (unsigned)a.head_groups, hg = id % (unsigned)a.head_groups;
  const int tid = threadIdx.x, sub = tid % LPR;
  const int64_t tokens = p.B * p.N, t_raw = (int64_t)tb * TOK + tid / LPR, t = min(t_raw, tokens - 1);
  const bool live = t_raw < tokens;
  const int64_t b = index_div(t, p.N), n = t - b * p.N;
  RopeLane<D, INTERLEAVED> lane(sub, p.half);
  if (p.half) lane.angles(p.cos, p.sin, (p.pos ? (int64_t)p.pos[b * p.spb + n * p.spn] : 0) + n * p.step, p.rows, p.half);

  const int h0 = (int)hg * a.heads_each, h1 = min(h0 + a.heads_each, (int)a.H);
  float w[16];
  if (a.w && a.sw == 0) {
    load_weight<T>(a.w, p.w_f32, lane.a, w);
    load_weight<T>(a.w, p.w_f32, lane.b, w + 8);
  }
  float dw[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) dw[e] = 0.f;
  __shared__ __attribute__((aligned(16))) float meet[BACK ? 256 * 16 : 4];
  // what the workgroup's tokens give dw, to row `group` of the partial sums
  auto leave = [&](int64_t group) __attribute__((always_inline)) {
    __syncthreads();   // (what was there before is read)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<f32x4 *>(&meet[(tid / LPR) * D + (e < 8 ? lane.a + e : lane.b + e - 8)]) = f32x4{dw[e], dw[e + 1], dw[e + 2], dw[e + 3]};
    __syncthreads();
    if (tid < D) {
      float sum = 0.f;
#pragma unroll 8
      for (int i = 0; i < TOK; ++i) sum += meet[i * D + tid];
      a.dw_parts[group * D + tid] = sum;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) dw[e] = 0.f;
  };

  for (int h = h0; h < h1; ++h) {
    const T *x = static_cast<const T *>(a.x) + b * a.sxb + h * a.sxh + n * a.sxn;
    float v[16];
    load8<T>(x + lane.a, v);
    load8<T>(x + lane.b, v + 8);
    if (a.w && a.sw != 0) {
      load_weight<T>(a.w, p.w_f32, h * a.sw + lane.a, w);
      load_weight<T>(a.w, p.w_f32, h * a.sw + lane.b, w + 8);
    }
    if constexpr (!BACK) {
      if (a.w) {
        float k;
        const float r = row_inverse_rms<LPR>(v, p.eps, k);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = v[e] * r * w[e];
      }
      if (p.half) lane.template turn<false>(v);
    } else {
      const T *dy = static_cast<const T *>(a.dy) + b * a.sgb + h * a.sgh + n * a.sgn;
      float g[16];
      load8<T>(dy + lane.a, g);
      load8<T>(dy + lane.b, g + 8);
      if (p.half) lane.template turn<true>(g);
      if (a.w) {
        // xh = x r, and dx = r (g w - xh mean(g w xh)): every factor is of the size of what it stands for (r^3, and x times it, leave fp32's
        // range where dx does not)
        float k, dot = 0.f;
        const float r = row_inverse_rms<LPR>(v, p.eps, k);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          v[e] *= r;
          if (live) dw[e] += g[e] * v[e];
          g[e] *= w[e];
          dot += g[e] * v[e];
        }
        const float n = row_sum<LPR>(dot) * (1.0f / D), rk = r * k;
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = rk * (g[e] - v[e] * n);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = g[e];
      }
    }
    if (live && (!BACK || a.y)) {
      T *y = static_cast<T *>(a.y) + b * a.syb + h * a.syh + n * a.syn;
      store8<T, ONCE>(y + lane.a, v);
      store8<T, ONCE>(y + lane.b, v + 8);
    }
    if (BACK && a.dw_parts && a.sw != 0) leave((int64_t)h * p.token_blocks + tb);
  }
  if (BACK && a.dw_parts && a.sw == 0) leave((int64_t)hg * p.token_blocks + tb);
}

// dw[o][d] = sum over `parts` rows of partial sums.  A workgroup takes 16 columns: 16 threads side by side, 64 rows at a time.
struct SumPartsTensor { const float *parts; void *dw; int64_t outs, each; };   // outs: D or H * D values; each: rows of one sum
template <typename T> __global__ __launch_bounds__(1024) void norm_rope_dw_kernel(SumPartsTensor q, SumPartsTensor k, int D, int w_f32) {
  __shared__ float red[64][17];
  const bool second = (int64_t)blockIdx.x * 16 >= q.outs;
  const SumPartsTensor &a = second ? k : q;
  const int64_t o = ((int64_t)blockIdx.x - (second ? q.outs / 16 : 0)) * 16;
  const int col = threadIdx.x % 16, rg = threadIdx.x / 16;
  const float *p = a.parts + o / D * a.each * D + o % D + col;
  float s = 0.f;
#pragma unroll 4
  for (int64_t i = rg; i < a.each; i += 64) s += p[i * D];
  red[rg][col] = s;
  __syncthreads();
  if (threadIdx.x >= 16) return;
  s = 0.f;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) s += red[i][col];
  if (w_f32) static_cast<float *>(a.dw)[o + col] = s;
  else static_cast<T *>(a.dw)[o + col] = (T)s;
}

// Heads that a workgroup walks over: as many as leave the chip 512 workgroups, eight at most.  Forward, gradient and the weights' sums in
// us, of four sequences of 256, 512, 1024 and 2048 tokens, with 2048 workgroups and with 512: 32 + 8 heads of 128 in bf16 25 and 22, 35 and 30,
// 50 and 43, 85 and 95; 64 + 64 of 64 31 and 26, 46 and 39, 67 and 64, 128 and 126; 16 + 4 of 256 in fp32 31 and 30, 48 and 44, 83 and 81, 150
// and 152; 32 + 8 of 256 in fp16 37 and 31, 50 and 43, 88 and 89, 157 and 153: 2 to 16 % less up to 512 tokens, and 11 % more at one of the
// larger ones.  (64 heads of 128, 4 x 4096 tokens: eight heads 100 us forward and 162 backward, sixteen 115 and 178.)
static int heads_each(int64_t tokens, int64_t H, int D) {
  const int64_t blocks = (tokens + 4096 / D - 1) / (4096 / D) * H;
  int e = 1;
  while (e < 8 && e < H && blocks / (2 * e) >= 512) e *= 2;
  return e;
}
static int64_t token_blocks(int64_t tokens, int D) { return (tokens + 4096 / D - 1) / (4096 / D); }
// rows of partial sums of one tensor's dw
static int64_t dw_groups(int64_t tokens, int64_t H, int D, bool per_head) {
  const int e = heads_each(tokens, H, D);
  return token_blocks(tokens, D) * (per_head ? H : (H + e - 1) / e);
}
int64_t norm_rope_bwd_workspace_bytes(int64_t tokens, int64_t H0, int64_t H1, int D, bool per_head) {
  return 4 * D * (dw_groups(tokens, H0, D, per_head) + (H1 > 0 ? dw_groups(tokens, H1, D, per_head) : 0));
}

template <typename T, int D, bool INTERLEAVED> static int launch_typed(const NormRopeArgs &x, bool back, hipStream_t st) {
  NormRopeKernelArgs a;
  const int64_t tokens = x.B * x.N;
  float *parts = static_cast<float *>(x.workspace);
  int64_t blocks[2] = {0, 0};
  const int64_t tb = token_blocks(tokens, D);
  for (int i = 0; i < 2; ++i) {
    NormRopeTensor &t = a.t[i];
    const NormRopeArgs::Tensor &s = x.t[i];
    t = {s.x, s.dy, s.w, s.y, nullptr, s.H, s.sx[0], s.sx[1], s.sx[2], s.sy[0], s.sy[1], s.sy[2], s.sg[0], s.sg[1], s.sg[2],
         s.per_head ? (int64_t)D : 0, 1, 1};
    if (s.H <= 0) continue;
    if (back && !s.w) {   // a rotation's gradient does not need x: dy's lines once more, which the caches have (a branch around the loads
      t.x = t.dy;         // costs the others 2 %)
      t.sxb = t.sgb; t.sxh = t.sgh; t.sxn = t.sgn;
    }
    t.heads_each = heads_each(tokens, s.H, D);
    t.head_groups = (int)((s.H + t.heads_each - 1) / t.heads_each);
    blocks[i] = tb * t.head_groups;
    if (back && s.dw) {
      t.dw_parts = parts;
      parts += dw_groups(tokens, s.H, D, s.per_head) * D;
    }
  }
  if (blocks[0] + blocks[1] > 0x7fffffffLL || tokens > 0x7fffffffLL)
    return set_error(QFA_EUNSUPPORTED, "norm_rope: too many tokens for one launch");
  a.cos = x.cos; a.sin = x.sin; a.pos = x.pos; a.rows = x.rows; a.spb = x.spb; a.spn = x.spn; a.B = x.B; a.N = x.N;
  a.eps = x.eps; a.half = x.half; a.step = x.step; a.w_f32 = x.w_f32;
  a.blocks0 = (unsigned)blocks[0];
  a.token_blocks = (unsigned)tb;
  const dim3 grid((unsigned)(blocks[0] + blocks[1])), block(256);
  // Stores are non-temporal where what a launch touches outgrows the last-level cache, of the forward up to three times its size.  4 x 64
  // heads of 128 in bf16, forward + gradient, us with plain stores and with these: 512 tokens 15 + 24 and 14 + 23; 1024 (134 and 201 MB) 24
  // + 36 and 22 + 35; 2048 51 + 76 and 44 + 64; 4096 106 + 163 and 106 + 142; 8192 204 + 329 and 220 + 320; in fp32 512 tokens 22 + 33 and
  // 23 + 36, 1024 52 + 72 and 46 + 68, 2048 101 + 156 and 109 + 141, 4096 212 + 350 and 244 + 349.
  const double bytes = (back ? 3.0 : 2.0) * (double)(tokens * (x.t[0].H + (x.t[1].H > 0 ? x.t[1].H : 0))) * D * sizeof(T);
  const double last = (double)LAST_LEVEL_BYTES;
  const bool once = bytes >= last && (back || bytes < 3 * last);
  if (!back) {
    if (once) norm_rope_kernel<T, D, INTERLEAVED, false, true><<<grid, block, 0, st>>>(a);
    else norm_rope_kernel<T, D, INTERLEAVED, false, false><<<grid, block, 0, st>>>(a);
    return check_launch("qfa_norm_rope");
  }
  if (once) norm_rope_kernel<T, D, INTERLEAVED, true, true><<<grid, block, 0, st>>>(a);
  else norm_rope_kernel<T, D, INTERLEAVED, true, false><<<grid, block, 0, st>>>(a);
  if (int e = check_launch("qfa_norm_rope_bwd")) return e;
  SumPartsTensor s[2] = {};
  for (int i = 0; i < 2; ++i)
    if (a.t[i].dw_parts) {
      const bool ph = x.t[i].per_head;
      s[i] = {a.t[i].dw_parts, x.t[i].dw, ph ? x.t[i].H * D : D, ph ? tb : dw_groups(tokens, x.t[i].H, D, false)};
    }
  const int64_t outs = s[0].outs + s[1].outs;
  if (outs == 0) return 0;
  norm_rope_dw_kernel<T><<<dim3((unsigned)(outs / 16)), dim3(1024), 0, st>>>(s[0], s[1], D, x.w_f32);
  return check_launch("qfa_norm_rope_bwd (weights)");
}

template <typename T> static int launch_t(const NormRopeArgs &x, bool back, hipStream_t st) {
  if (x.interleaved) {
    if (x.D == 64) return launch_typed<T, 64, true>(x, back, st);
    if (x.D == 128) return launch_typed<T, 128, true>(x, back, st);
    return launch_typed<T, 256, true>(x, back, st);
  }
  if (x.D == 64) return launch_typed<T, 64, false>(x, back, st);
  if (x.D == 128) return launch_typed<T, 128, false>(x, back, st);
  return launch_typed<T, 256, false>(x, back, st);
}
int launch_norm_rope(const NormRopeArgs &x, bool back, hipStream_t st) {
  if (x.dtype == QFA_F32) return launch_t<float>(x, back, st);
  if (x.dtype == QFA_F16) return launch_t<_Float16>(x, back, st);
  return launch_t<__bf16>(x, back, st);
}

}  // namespace qfa
