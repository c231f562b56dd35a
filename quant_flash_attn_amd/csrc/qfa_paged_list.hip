// Attention of every token on a list of blocks (pages) of its sequence, those that a cheap score has selected (qfa_paged_select.hip):
//     O = softmax(sm_scale * Q^ K^^T) V^   over the keys of the listed blocks at or before the token,
// with the kernel and the arithmetic of attention on all keys (qfa_paged_attn.hip).  A token and key head are an item: the query heads that
// share the key head are its rows, the list's blocks one behind the other its keys.  A half of a tile lies in one block, so what the mask
// asks is where each half's keys begin; the list is read beside the page numbers, 32 tiles ahead.
#include "qfa_paged_block.h"

namespace qfa {

constexpr int LIST_WGS = 256 * 2;   // two on a CU
constexpr int LIST_EXTRA = 12;      // units of an item beside its tiles, as there

// O of the items that several workgroups share
struct PagedListMergeArgs {
  PagedWork work;
  void *o;
  int o_dtype;
};
template <int D> __global__ __launch_bounds__(256) void paged_list_merge_kernel(PagedListMergeArgs a) {
  constexpr int CL = D / 4, SLOTS = 256 / CL;
  __shared__ float red[SLOTS][D + 4];
  const int tid = threadIdx.x, d = 4 * (tid % CL), slot = tid / CL;
  const PagedListDeal deal(a.work, PAGED_ROWS, SKV_TILE);
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
struct PagedListPlan {
  unsigned tiles, each;
  int grid;
  bool cut;
};
static PagedListPlan list_plan(int64_t items, int64_t keep, int page_log2, int D) {
  PagedListPlan p;
  p.tiles = (unsigned)(((keep << page_log2) + SKV_TILE - 1) / SKV_TILE);
  const int64_t unit = p.tiles + LIST_EXTRA, total = items * unit, full = D == 256 ? 192 : 256;   // items that keep the chip busy
  p.cut = items < full && (int64_t)p.tiles * (full - items) > (D == 256 ? 20 : 32) * full;
  p.each = (unsigned)(p.cut ? max((int64_t)LIST_EXTRA, (total + LIST_WGS - 1) / LIST_WGS) : unit);
  p.grid = (int)((total + p.each - 1) / p.each);
  return p;
}
static int64_t list_items(int64_t B, int64_t N, int64_t Hk, int64_t G) { return B * N * Hk * ((G + PAGED_ROWS - 1) / PAGED_ROWS); }
int64_t paged_list_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t keep, int page_log2) {
  const PagedListPlan p = list_plan(list_items(B, N, Hk, H / Hk), keep, page_log2, D);
  return p.cut ? 2LL * p.grid * PAGED_ROWS * (D + 2) * 4 : 0;
}
double paged_list_units(int64_t B, int64_t H, int64_t Hk, int64_t N, int64_t keep, int page_log2) {
  return (double)list_items(B, N, Hk, H / Hk) * ((double)keep * (1 << page_log2) / SKV_TILE + 1 + LIST_EXTRA);
}

template <int D> static int launch_d(const PagedListArgs &l, hipStream_t st) {
  const PagedAttnArgs &x = l.x;
  const int G = (int)(x.H / x.Hk);
  const int64_t items = list_items(x.B, x.N, x.Hk, G);
  const PagedListPlan p = list_plan(items, l.keep, x.page_log2, D);
  PagedAttnKernelArgs a = {};
  a.q = x.q; a.kc = x.cache.k_codes; a.ks = x.cache.k_scale; a.kz = x.cache.k_zero;
  a.vc = x.cache.v_codes; a.vs = x.cache.v_scale; a.vz = x.cache.v_zero; a.o = x.o; a.page_table = x.page_table;
  a.pages = x.pages; a.stb = x.stb; a.stw = x.stw; a.sqb = x.sq[0]; a.sqh = x.sq[1]; a.sqn = x.sq[2];
  a.width = (int)x.width; a.page_log2 = x.page_log2; a.q_dtype = x.q_dtype;
  a.sm_scale_log2 = x.sm_scale * kLog2e;
  a.blocks = l.blocks; a.keep = (int)l.keep;
  float *slots = static_cast<float *>(x.workspace);
  a.work = {x.starts, x.counts, (int)x.B, (int)x.Hk, G, (int)x.N, 1, 0, (int)(x.width << x.page_log2), p.grid, PAGED_ROWS, SKV_TILE, LIST_EXTRA, nullptr,
            slots, p.cut ? slots + 2LL * p.grid * PAGED_ROWS * D : nullptr, nullptr, nullptr, p.tiles, p.each};
  const dim3 grid((unsigned)p.grid), block(256);
  if (x.scale_dtype == QFA_F32) paged_rows_kernel<float, D, PagedListDeal, false><<<grid, block, 0, st>>>(a);
  else if (x.scale_dtype == QFA_F16) paged_rows_kernel<_Float16, D, PagedListDeal, false><<<grid, block, 0, st>>>(a);
  else paged_rows_kernel<__bf16, D, PagedListDeal, false><<<grid, block, 0, st>>>(a);
  if (int e = check_launch("qfa_attn_paged_blocks")) return e;
  if (!p.cut) return 0;
  paged_list_merge_kernel<D><<<dim3((unsigned)items), block, 0, st>>>({a.work, x.o, x.q_dtype});
  return check_launch("qfa_attn_paged_blocks (merge)");
}
int launch_paged_list(const PagedListArgs &x, hipStream_t st) {
  if (x.x.D == 64) return launch_d<64>(x, st);
  if (x.x.D == 128) return launch_d<128>(x, st);
  return launch_d<256>(x, st);
}

}  // namespace qfa
