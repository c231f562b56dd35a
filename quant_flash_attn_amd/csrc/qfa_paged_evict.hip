// The heaviest rows of a paged INT8 cache, per sequence and key head, to new pages: eviction from a cache that has grown too long.
//
// Two launches.  A workgroup for each sequence and key head finds the `keep` slots with the largest weights (qfa_topk.h; the first and the last
// ones always, ties to the lowest slot) and writes down, in order, which they are and their weights.  Then the rows move, codes, scales
// and zero points of keys and values, each to its place in the new pages: what is kept stays in order, so the last slots are the newest
// ones again, and pages that other sequences share are not touched.
//
// The selection waits for its own steps (8 x 5120 slots 10.7 us, 512 x 3000 13.4), the rows are bound by HBM: 16 sequences, 32 heads of 128, 2000 rows of each,
// codes in and out 530 MB in 108 us (4.9 TB/s); 8 heads x 4096 rows 5.7 us, a launch with three loads that wait for each other.
#include "qfa_host.h"
#include "qfa_topk.h"

namespace qfa {

// Top: TopHeld, of T threads
template <typename Top, int T> __global__ __launch_bounds__(T) void evict_select_kernel(PagedEvictArgs x) {
  __shared__ Top top;
  const int64_t bh = blockIdx.x, b = index_div(bh, x.Hk);
  const int tid = threadIdx.x;
  const int64_t slots = x.width << x.page_log2, new_slots = x.new_width << x.page_log2;
  const int n = (int)max((int64_t)0, min((int64_t)x.lengths[b], slots)), keep = (int)x.keep, k = min(n, keep);
  const float *weights = x.weights + bh * slots;
  int32_t *kept = x.kept + bh * keep;
  float *new_weights = x.new_weights + bh * new_slots;
  if (bh == b * x.Hk && tid == 0) x.new_lengths[b] = k;
  if (n > k) {
    const int first = (int)x.first, last = n - (int)x.last;
    top.run(n, (unsigned)k, [&](int i) __attribute__((always_inline)) { return weights[i]; },
            [&](int i, float w) __attribute__((always_inline)) -> unsigned { return ((i < first) | (i >= last)) ? TOP_ALWAYS : top_key(w); },
            [&](unsigned place, int i, float w) __attribute__((always_inline)) {
              kept[place] = i;
              new_weights[place] = w;
            });
  } else {
    for (int i = tid; i < n; i += T) {
      kept[i] = i;
      new_weights[i] = weights[i];
    }
  }
  for (int64_t i = k + tid; i < keep; i += T) kept[i] = -1;
  for (int64_t i = k + tid; i < new_slots; i += T) new_weights[i] = 0.f;
}

// D/16 lanes hold a row; a workgroup moves some rows of one sequence and key head, of keys or of values
constexpr int EVICT_UNROLL = 2;   // rows of a thread (1 x 8 heads x 4096 and 16 x 32 x 1900 rows of 128, us: 2 5.7 and 108, 4 6.8 and 115, 8 11.2 and 128)
template <typename S, int D, bool ONCE> __global__ __launch_bounds__(256) void evict_move_kernel(PagedEvictArgs x, int chunks) {
  constexpr int LPR = D / 16, ROWS = 256 / LPR;
  unsigned id = blockIdx.x;
  const int chunk = (int)(id % (unsigned)chunks);
  id /= (unsigned)chunks;
  const bool values = id & 1;
  const int64_t bh = id >> 1, b = index_div(bh, x.Hk), h = bh - b * x.Hk;
  const int tid = threadIdx.x, sub = tid % LPR;
  const int64_t slots = x.width << x.page_log2;
  const int k = (int)max((int64_t)0, min(min((int64_t)x.lengths[b], slots), x.keep));
  int8_t *codes = values ? x.cache.v_codes : x.cache.k_codes, *zero = values ? x.cache.v_zero : x.cache.k_zero;
  S *scale = static_cast<S *>(values ? x.cache.v_scale : x.cache.k_scale);
  const int row_mask = (1 << x.page_log2) - 1;
  int64_t from[EVICT_UNROLL], to[EVICT_UNROLL];
#pragma unroll
  for (int u = 0; u < EVICT_UNROLL; ++u) {
    const int i = (chunk * EVICT_UNROLL + u) * ROWS + tid / LPR;
    from[u] = to[u] = -1;
    if (i >= k) continue;
    const int slot = x.kept[bh * x.keep + i];
    const int page = x.page_table[b * x.stb + (int64_t)(slot >> x.page_log2) * x.stw];
    const int new_page = x.new_table[b * x.ntb + (int64_t)(i >> x.page_log2) * x.ntw];
    if (page >= 0 && page < x.pages) from[u] = (((int64_t)page * x.Hk + h) << x.page_log2) + (slot & row_mask);
    if (new_page >= 0 && new_page < x.pages) to[u] = (((int64_t)new_page * x.Hk + h) << x.page_log2) + (i & row_mask);
  }
  u32x4 w[EVICT_UNROLL];
  S s[EVICT_UNROLL];
  int8_t z[EVICT_UNROLL];
#pragma unroll
  for (int u = 0; u < EVICT_UNROLL; ++u) {   // (a row without a page becomes zeros)
    w[u] = u32x4{0, 0, 0, 0};
    s[u] = (S)0.f;
    z[u] = 0;
    if (from[u] < 0 || to[u] < 0) continue;
    const u32x4 *at = reinterpret_cast<const u32x4 *>(codes + from[u] * D + 16 * sub);
    w[u] = ONCE ? __builtin_nontemporal_load(at) : *at;
    if (sub == 0) {
      s[u] = scale[from[u]];
      z[u] = zero[from[u]];
    }
  }
#pragma unroll
  for (int u = 0; u < EVICT_UNROLL; ++u) {
    if (to[u] < 0) continue;
    *reinterpret_cast<u32x4 *>(codes + to[u] * D + 16 * sub) = w[u];
    if (sub == 0) {
      scale[to[u]] = s[u];
      zero[to[u]] = z[u];
    }
  }
}

template <typename S, int D> static void launch_move_d(const PagedEvictArgs &x, dim3 grid, int chunks, hipStream_t st) {
  // Non-temporal loads of the old rows where what is moved, codes in and out, is 128 MiB or more: two caches in turn, 64, 128 and 256 elements, us with plain loads and
  // with these: 64 MiB 24, 22, 18 and 29, 25, 24; 128 MiB 51, 46, 41 and 47, 41, 38; 256 MiB 104, 83, 75 and 96, 75, 67; 512 MiB 197, 160, 140 and 196, 156, 138
  const int64_t rows = x.keep < x.width << x.page_log2 ? x.keep : x.width << x.page_log2;
  if (4.0 * (double)(x.B * x.Hk * rows) * D >= 128.0 * (1 << 20)) evict_move_kernel<S, D, true><<<grid, dim3(256), 0, st>>>(x, chunks);
  else evict_move_kernel<S, D, false><<<grid, dim3(256), 0, st>>>(x, chunks);
}
template <typename S> static int launch_move(const PagedEvictArgs &x, int64_t chunks, hipStream_t st) {
  const dim3 grid((unsigned)(x.B * x.Hk * 2 * chunks));
  if (x.D == 64) launch_move_d<S, 64>(x, grid, (int)chunks, st);
  else if (x.D == 128) launch_move_d<S, 128>(x, grid, (int)chunks, st);
  else launch_move_d<S, 256>(x, grid, (int)chunks, st);
  return check_launch("qfa_paged_evict (rows)");
}
template <typename Top, int T> static void launch_top(const PagedEvictArgs &x, hipStream_t st) {
  evict_select_kernel<Top, T><<<dim3((unsigned)(x.B * x.Hk)), dim3(T), 0, st>>>(x);
}
int launch_paged_evict(const PagedEvictArgs &x, hipStream_t st) {
  const int64_t most = x.keep < x.width << x.page_log2 ? x.keep : x.width << x.page_log2, rows = EVICT_UNROLL * 4096 / x.D;
  const int64_t chunks = (most + rows - 1) / rows;
  if ((double)x.B * (double)x.Hk * 2 * (double)chunks > 2147483647.0) return set_error(QFA_EUNSUPPORTED, "paged_evict: too many rows for one launch");
  const int64_t slots = x.width << x.page_log2;
  // More sequences and heads than CUs share one: 512 threads and the numbers that they hold leave room for more of them.  256, 1024, 2048 and 4096 slots, us with 512 threads:  512
  // sequences times heads 6.1, 7.2, 8.9, 12.0,  1024: 7.7, 9.6, 12.0, 16.2,  4096: 22.4, 27.9, 33.7, 48.5;  with 1024:  7.1, 9.5, 11.1, 12.0,  12.0, 15.8, 17.4, 21.0,  37.0, 51.2, 58.0, 69.0.
  // (512 x 3000: 13.4 and 12.5.)  Few of them want all threads: 8 x 5120 slots 12.5 with 512 and 10.9 with 1024.
  if (slots <= 4096 && x.B * x.Hk > 256) launch_top<TopHeld<512, 4096, 11>, 512>(x, st);
  else if (slots <= 16384) launch_top<TopHeld<1024, 16384, 11>, 1024>(x, st);
  else launch_top<TopHeld<1024, 0, 11>, 1024>(x, st);
  if (int e = check_launch("qfa_paged_evict")) return e;
  if (x.scale_dtype == QFA_F32) return launch_move<float>(x, chunks, st);
  if (x.scale_dtype == QFA_F16) return launch_move<_Float16>(x, chunks, st);
  return launch_move<__bf16>(x, chunks, st);
}

}  // namespace qfa
