// Rows into and out of a paged INT8 cache.
//
// Append: every token's keys (RMSNorm and rotation on the way, where asked for) and values are quantized by the quantizer's own
// arithmetic and go to the page and row of their position:  page_table[b, p / page], row p % page,  p = starts[b] + n.
// Read: rows of positions starts[b] .. as the values they stand for, (code - zero point) * scale, rounded once.
//
// Both are bound by memory: 2 D bytes (16-bit rows) against D + 3 in the cache; 4 x 32 heads x 4096 x 128: 87 and 74 us (4.6 and
// 5.5 TB/s).  A call whose sequences bring fewer tokens than it has room for computes the padding too and stores nothing of it (16 x 16
// heads, up to 517 tokens of 64, half of it padding: 16 us).  The work is dealt as in the kernel that norms and rotates
// (qfa_norm_rope.hip): D/16 lanes hold a row, a workgroup 4096/D tokens, and it walks over some heads of them with their angles and places
// in registers.  Nothing is written for a token that has no place (see qfa.h): position, page and angle are checked here, since the
// host does not see them.
#include "qfa_quant_row.h"
#include "qfa_rope_row.h"

namespace qfa {

struct PagedRowsKernelArgs {
  PagedRowsArgs x;
  unsigned blocks0, head_groups;
  int heads_each;
};

// Where a token's rows are: the first row of its page among all pages' rows of one head ([pages, H, page]); -1: nowhere
struct Place {
  int64_t page;
  int row;
  __device__ __forceinline__ Place(const PagedRowsArgs &x, int64_t b, int64_t n, int64_t pos) {
    page = -1;
    row = 0;
    if (pos < 0 || (x.counts && n >= x.counts[b])) return;
    const int64_t at = pos >> x.page_log2;
    if (at >= x.width) return;
    const int64_t id = x.page_table[b * x.stb + at * x.stw];
    if (id < 0 || id >= x.pages) return;
    page = id;
    row = (int)(pos & ((1 << x.page_log2) - 1));
  }
  __device__ __forceinline__ int64_t of_head(const PagedRowsArgs &x, int64_t h) const {
    return ((page * x.H + h) << x.page_log2) + row;
  }
};

__device__ __forceinline__ void store_scale(void *p, int dtype, int64_t at, float s) {
  if (dtype == QFA_F32) static_cast<float *>(p)[at] = s;
  else if (dtype == QFA_F16) static_cast<_Float16 *>(p)[at] = (_Float16)s;
  else static_cast<__bf16 *>(p)[at] = (__bf16)s;
}
__device__ __forceinline__ float load_scale(const void *p, int dtype, int64_t at) {
  if (dtype == QFA_F32) return static_cast<const float *>(p)[at];
  if (dtype == QFA_F16) return (float)static_cast<const _Float16 *>(p)[at];
  return (float)static_cast<const __bf16 *>(p)[at];
}

template <typename T, int D, bool INTERLEAVED, bool ONCE> __global__ __launch_bounds__(256) void paged_append_kernel(PagedRowsKernelArgs p) {
  constexpr int LPR = D / 16, TOK = 256 / LPR;
  const PagedRowsArgs &x = p.x;
  const bool values = blockIdx.x >= p.blocks0;
  const unsigned id = values ? blockIdx.x - p.blocks0 : blockIdx.x, tb = id / p.head_groups, hg = id % p.head_groups;
  const int tid = threadIdx.x, sub = tid % LPR;
  const int64_t tokens = x.B * x.N, t_raw = (int64_t)tb * TOK + tid / LPR, t = min(t_raw, tokens - 1);
  const int64_t b = index_div(t, x.N), n = t - b * x.N, pos = (int64_t)x.starts[b] + n;
  const Place place(x, b, n, pos);
  const bool turn = !values && x.half != 0, norm = !values && x.w != nullptr;
  const bool live = t_raw < tokens && place.page >= 0 && (x.half == 0 || pos < x.rope_rows);   // (the same tokens of both)
  RopeLane<D, INTERLEAVED> lane(sub, turn ? x.half : 0);
  if (turn) lane.angles(x.cos, x.sin, live ? pos : 0, x.rope_rows, x.half);
  const void *src = values ? x.v : x.k;
  const int64_t *st = values ? x.sv : x.sk;
  int8_t *codes = values ? x.cache.v_codes : x.cache.k_codes, *zero = values ? x.cache.v_zero : x.cache.k_zero;
  void *scale = values ? x.cache.v_scale : x.cache.k_scale;
  const int h0 = (int)hg * p.heads_each, h1 = min(h0 + p.heads_each, (int)x.H);
  for (int h = h0; h < h1; ++h) {
    const T *row = static_cast<const T *>(src) + b * st[0] + h * st[1] + n * st[2];
    float v[16];
    load8<T, ONCE>(row + lane.a, v);
    load8<T, ONCE>(row + lane.b, v + 8);
    if (norm) {
      float k, w[16];
      const float r = row_inverse_rms<LPR>(v, x.eps, k);
      const int64_t at = x.w_per_head ? (int64_t)h * D : 0;
      if (x.w_f32) {
        load8<float>(static_cast<const float *>(x.w) + at + lane.a, w);
        load8<float>(static_cast<const float *>(x.w) + at + lane.b, w + 8);
      } else {
        load8<T>(static_cast<const T *>(x.w) + at + lane.a, w);
        load8<T>(static_cast<const T *>(x.w) + at + lane.b, w + 8);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = v[e] * r * w[e];
    }
    if (turn) lane.template turn<false>(v);
    const QuantRow<16> q = quant_row<LPR, false, 16>(v, true);
    if (!live) continue;
    const int64_t to = place.of_head(x, h);
    *reinterpret_cast<u32x2 *>(codes + to * D + lane.a) = u32x2{q.codes[0], q.codes[1]};
    *reinterpret_cast<u32x2 *>(codes + to * D + lane.b) = u32x2{q.codes[2], q.codes[3]};
    if (sub == 0) {
      store_scale(scale, x.scale_dtype, to, q.scale);
      zero[to] = (int8_t)(int)q.zp;
    }
  }
}

template <typename T, int D, bool ONCE> __global__ __launch_bounds__(256) void paged_read_kernel(PagedRowsKernelArgs p) {
  constexpr int LPR = D / 16, TOK = 256 / LPR;
  const PagedRowsArgs &x = p.x;
  const bool values = blockIdx.x >= p.blocks0;
  const unsigned id = values ? blockIdx.x - p.blocks0 : blockIdx.x, tb = id / p.head_groups, hg = id % p.head_groups;
  const int tid = threadIdx.x, sub = tid % LPR;
  const int64_t tokens = x.B * x.N, t = (int64_t)tb * TOK + tid / LPR;
  if (t >= tokens) return;
  const int64_t b = index_div(t, x.N), n = t - b * x.N;
  const Place place(x, b, n, (int64_t)x.starts[b] + n);
  const int8_t *codes = values ? x.cache.v_codes : x.cache.k_codes, *zero = values ? x.cache.v_zero : x.cache.k_zero;
  const void *scale = values ? x.cache.v_scale : x.cache.k_scale;
  T *out = static_cast<T *>(values ? x.v_out : x.k_out) + (b * x.H * x.N + n) * D + 16 * sub;
  const int h0 = (int)hg * p.heads_each, h1 = min(h0 + p.heads_each, (int)x.H);
  for (int h = h0; h < h1; ++h) {
    float v[16];
    if (place.page >= 0) {
      const int64_t at = place.of_head(x, h);
      const u32x4 *from = reinterpret_cast<const u32x4 *>(codes + at * D + 16 * sub);
      const u32x4 w = ONCE ? __builtin_nontemporal_load(from) : *from;
      const float s = load_scale(scale, x.scale_dtype, at);
      const int z = zero[at];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = (float)((int)(signed char)(w[e / 4] >> (8 * (e % 4))) - z) * s;
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = 0.f;
    }
    store8<T>(out + (int64_t)h * x.N * D, v);
    store8<T>(out + (int64_t)h * x.N * D + 8, v + 8);
  }
}

// heads per workgroup: as many as leave the chip 2048 workgroups, eight at most (with 2048 and with 1024: 4 x 2048 tokens of 8 heads of 128 15 + 12.6 and
// 14.5 + 10.5 us for append and read, 1024 tokens of 16 heads of 256 23 + 17 and 24 + 20)
static int plan(PagedRowsKernelArgs &a, int64_t *grid) {
  const int64_t tb = (a.x.B * a.x.N + 4096 / a.x.D - 1) / (4096 / a.x.D);
  int e = 1;
  while (e < 8 && e < a.x.H && 2 * tb * a.x.H / (2 * e) >= 2048) e *= 2;
  a.heads_each = e;
  a.head_groups = (unsigned)((a.x.H + e - 1) / e);
  const int64_t blocks = tb * a.head_groups;
  if (a.x.B * a.x.N > 0x7fffffffLL || 2 * blocks > 0x7fffffffLL) return set_error(QFA_EUNSUPPORTED, "paged cache: too many tokens for one launch");
  a.blocks0 = (unsigned)blocks;
  *grid = 2 * blocks;
  return 0;
}

template <typename T, int D> static int launch_td(const PagedRowsArgs &x, bool read, hipStream_t st) {
  PagedRowsKernelArgs a;
  a.x = x;
  int64_t grid;
  if (int e = plan(a, &grid)) return e;
  // Non-temporal loads where what a launch touches outgrows the last-level cache.  4 x 32 heads of 128 in bf16, append and read in turn, us
  // with plain loads and with these: 101 MB each 21 + 17 and 24 + 18; 203 MB 45 + 41 and 45 + 37 (alone, again and again 41 and 47, 36
  // and 47); 405 MB 97 + 89 and 89 + 77; 811 MB 191 + 176 and 176 + 178.  Non-temporal stores of codes: 405 MB 104 + 86, of rows 80 + 85,
  // 203 MB 38 + 55.
  const bool once = 2.0 * (double)(x.B * x.N * x.H) * (D * (sizeof(T) + 1) + 3) >= (double)LAST_LEVEL_BYTES;
  const dim3 g((unsigned)grid), block(256);
  if (read && once) paged_read_kernel<T, D, true><<<g, block, 0, st>>>(a);
  else if (read) paged_read_kernel<T, D, false><<<g, block, 0, st>>>(a);
  else if (x.interleaved && once) paged_append_kernel<T, D, true, true><<<g, block, 0, st>>>(a);
  else if (x.interleaved) paged_append_kernel<T, D, true, false><<<g, block, 0, st>>>(a);
  else if (once) paged_append_kernel<T, D, false, true><<<g, block, 0, st>>>(a);
  else paged_append_kernel<T, D, false, false><<<g, block, 0, st>>>(a);
  return check_launch(read ? "qfa_paged_read" : "qfa_paged_append");
}
template <typename T> static int launch_t(const PagedRowsArgs &x, bool read, hipStream_t st) {
  if (x.D == 64) return launch_td<T, 64>(x, read, st);
  if (x.D == 128) return launch_td<T, 128>(x, read, st);
  return launch_td<T, 256>(x, read, st);
}
int launch_paged_rows(const PagedRowsArgs &x, bool read, hipStream_t st) {
  if (x.dtype == QFA_F32) return launch_t<float>(x, read, st);
  if (x.dtype == QFA_F16) return launch_t<_Float16>(x, read, st);
  return launch_t<__bf16>(x, read, st);
}

}  // namespace qfa
