// C entry points around a paged cache: argument validation, then dispatch to the kernel launchers (see qfa_api.cpp).
#include <math.h>
#include <string.h>

#include "qfa_check.h"

using namespace qfa;

static bool head_dim_ok(int D) { return D == 64 || D == 128 || D == 256; }

// The angles of a call: all of them or none
static int check_rope(const char *who, const float *cos, const float *sin, int64_t rows, int rotated, int D) {
  if (!cos && !sin && rotated == 0) return 0;
  if (!cos || !sin) return set_error(QFA_EINVAL, "%s: cos and sin go together with rotated > 0", who);
  if (rotated <= 0 || rotated > D || rotated % 16 != 0)
    return set_error(QFA_EUNSUPPORTED, "%s: %d rotated elements: a multiple of 16 up to head_dim %d is needed", who, rotated, D);
  if (rows <= 0) return set_error(QFA_EINVAL, "%s: the table of angles is empty", who);
  if (!aligned16(cos) || !aligned16(sin)) return set_error(QFA_EINVAL, "%s: cos and sin must be 16-byte aligned", who);
  return 0;
}
static int check_norm(const char *who, const void *w, int w_dtype, int dtype, float eps) {
  if (!w) return 0;
  if (w_dtype != QFA_F32 && w_dtype != dtype) return set_error(QFA_EINVAL, "%s: weights must be QFA_F32 or of the tensor's type", who);
  if (!aligned16(w)) return set_error(QFA_EINVAL, "%s: weights must be 16-byte aligned", who);
  if (!(eps >= 0.f) || isinf(eps)) return set_error(QFA_EINVAL, "%s: eps must be finite and not negative", who);
  return 0;
}

static int fill_norm_rope(const char *who, bool back, NormRopeArgs *a, const qfa_norm_rope_tensor *q, const qfa_norm_rope_tensor *k,
                          const float *cos, const float *sin, int64_t rope_rows, int rotated, int interleaved, const int32_t *positions,
                          int64_t spb, int64_t spn, int step, float eps, int dtype, int w_dtype, int64_t B, int64_t N, int D) {
  memset(a, 0, sizeof(*a));
  if (!q) return set_error(QFA_EINVAL, "%s: null tensor", who);
  if (!is_float_dtype(dtype)) return set_error(QFA_EINVAL, "%s: dtype %d is not QFA_F32/F16/BF16", who, dtype);
  if (B <= 0 || N <= 0) return set_error(QFA_EINVAL, "%s: B and N must be positive", who);
  if (!head_dim_ok(D)) return set_error(QFA_EUNSUPPORTED, "%s: head_dim %d not in {64, 128, 256}", who, D);
  if (int e = check_rope(who, cos, sin, rope_rows, rotated, D)) return e;
  if (step != 0 && step != 1) return set_error(QFA_EINVAL, "%s: step must be 0 or 1", who);
  const int es = elem_size(dtype);
  const qfa_norm_rope_tensor *side[2] = {q, k};
  for (int i = 0; i < 2; ++i) {
    const qfa_norm_rope_tensor *s = side[i];
    if (!s) continue;
    if (s->H <= 0) return set_error(QFA_EINVAL, "%s: H must be positive", who);
    const bool in = !back || s->weight, out = !back || s->y || !s->dweight;   // of the backward: x with a weight, dx unless dweight alone is wanted
    if ((in && !s->x) || (out && !s->y) || (back && !s->dy)) return set_error(QFA_EINVAL, "%s: null pointer argument", who);
    if ((in && !aligned16(s->x)) || (out && !aligned16(s->y)) || (back && !aligned16(s->dy)))
      return set_error(QFA_EINVAL, "%s: tensors must be 16-byte aligned", who);
    if ((in && !strides_ok(s->sx[0], s->sx[1], s->sx[2], D, es)) || (out && !strides_ok(s->sy[0], s->sy[1], s->sy[2], D, es)) ||
        (back && !strides_ok(s->sdy[0], s->sdy[1], s->sdy[2], D, es)))
      return set_error(QFA_EINVAL, "%s: strides must be positive multiples of 16 bytes, token stride >= D", who);
    if (int e = check_norm(who, s->weight, w_dtype, dtype, eps)) return e;
    if (back && s->dweight && (!s->weight || !aligned16(s->dweight)))
      return set_error(QFA_EINVAL, "%s: dweight needs a weight and 16-byte alignment", who);
    NormRopeArgs::Tensor &t = a->t[i];
    t.x = s->x; t.w = s->weight; t.y = s->y; t.dy = s->dy; t.dw = s->dweight; t.H = s->H; t.per_head = s->weight_per_head != 0;
    for (int j = 0; j < 3; ++j) { t.sx[j] = s->sx[j]; t.sy[j] = s->sy[j]; t.sg[j] = s->sdy[j]; }
  }
  a->cos = cos; a->sin = sin; a->pos = positions; a->rows = rope_rows; a->spb = spb; a->spn = spn; a->B = B; a->N = N;
  a->half = rotated / 2; a->step = step; a->interleaved = interleaved != 0; a->D = D; a->dtype = dtype; a->w_f32 = w_dtype == QFA_F32;
  a->eps = eps;
  return 0;
}

static int check_cache(const char *who, const qfa_paged_cache *c) {
  if (!c || !c->k_codes || !c->k_scale || !c->k_zero || !c->v_codes || !c->v_scale || !c->v_zero)
    return set_error(QFA_EINVAL, "%s: null cache pointer", who);
  if (!aligned16(c->k_codes) || !aligned16(c->v_codes)) return set_error(QFA_EINVAL, "%s: codes must be 16-byte aligned", who);
  if (!is_float_dtype(c->scale_dtype)) return set_error(QFA_EINVAL, "%s: scale_dtype %d is not QFA_F32/F16/BF16", who, c->scale_dtype);
  if (c->pages <= 0 || c->H <= 0) return set_error(QFA_EINVAL, "%s: pages and H must be positive", who);
  if (!head_dim_ok(c->D)) return set_error(QFA_EUNSUPPORTED, "%s: head_dim %d not in {64, 128, 256}", who, c->D);
  if ((double)c->pages * (double)c->H * (double)c->page_size > 4294967295.0)
    return set_error(QFA_EUNSUPPORTED, "%s: a cache holds fewer than 2^32 rows of keys", who);
  if (c->page_size < 16 || c->page_size > (1 << 20) || (c->page_size & (c->page_size - 1)))
    return set_error(QFA_EUNSUPPORTED, "%s: page size %d: a power of two from 16 on is needed", who, c->page_size);
  return 0;
}
static int log2_of(int x) { return __builtin_ctz((unsigned)x); }
static PagedCachePtrs ptrs_of(const qfa_paged_cache *c) { return {c->k_codes, c->k_scale, c->k_zero, c->v_codes, c->v_scale, c->v_zero}; }
static int check_places(const char *who, const qfa_paged_cache *c, const int32_t *table, const int32_t *starts, int64_t width, int64_t stb,
                        int64_t stw, int64_t B, int64_t N) {
  if (!table || !starts) return set_error(QFA_EINVAL, "%s: null page_table or starts", who);
  if (B <= 0 || N <= 0 || width <= 0) return set_error(QFA_EINVAL, "%s: B, N and the page table's width must be positive", who);
  if (stb < 0 || stw < 0) return set_error(QFA_EINVAL, "%s: page_table strides must not be negative", who);
  if (width > 0x7fffffffLL / c->page_size || N > (1LL << 28) || B > (1LL << 28))
    return set_error(QFA_EUNSUPPORTED, "%s: a sequence has room for 2^31 keys at most, a call for 2^28 sequences and tokens", who);
  return 0;
}

static bool keep_ok(int64_t keep) { return keep > 0 && keep <= (1LL << 30); }
static bool page_size_ok(int n) { return n >= 16 && n <= (1 << 20) && (n & (n - 1)) == 0; }
// Of what is kept some are always the first and last ones
static int check_keep(const char *who, int64_t keep, int64_t first, int64_t last) {
  if (!keep_ok(keep)) return set_error(QFA_EINVAL, "%s: keep must be positive and at most 2^30, got %lld", who, (long long)keep);
  if (first < 0 || last < 0 || first > keep || last > keep - first)
    return set_error(QFA_EINVAL, "%s: first %lld and last %lld must not be negative and fit into keep %lld together", who, (long long)first, (long long)last, (long long)keep);
  return 0;
}
// Tensors with a value for every slot that a page table has room for
static int check_slots(const char *who, const qfa_paged_cache *c, int64_t width) {
  return width <= (1LL << 30) / c->page_size ? 0 : set_error(QFA_EUNSUPPORTED, "%s: a page table has room for 2^30 keys at most", who);
}
// Bounds with zero points of 8 or 16 bits
struct Bounds {
  bool given;
  int8_t *codes; float *scale; void *zero;
  int bits;
};
template <typename T> static Bounds bounds_of(const T *b) {
  return b ? Bounds{true, b->codes, b->scale, b->zero, (int)sizeof(*b->zero) * 8} : Bounds{false, nullptr, nullptr, nullptr, 8};
}
static int check_bounds(const char *who, const Bounds &b) {
  if (!b.given || !b.codes || !b.scale || !b.zero) return set_error(QFA_EINVAL, "%s: null bounds pointer", who);
  if (!aligned16(b.codes) || !aligned8(b.scale) || reinterpret_cast<uintptr_t>(b.zero) % (unsigned)(b.bits / 4))
    return set_error(QFA_EINVAL, "%s: the bounds' codes must be 16-byte aligned, scales 8-byte and zero points %d-byte aligned", who, b.bits / 4);
  return 0;
}

// Checks a call of attention on a paged cache and fills in what all of them have
static int fill_attn(const char *who, PagedAttnArgs *a, const qfa_paged_cache *cache, const void *q, int q_dtype, int64_t sqb, int64_t sqh, int64_t sqn,
                     const int32_t *page_table, int64_t width, int64_t stb, int64_t stw, const int32_t *starts, const int32_t *counts, int64_t B, int64_t H,
                     int64_t N) {
  memset(a, 0, sizeof(*a));
  if (int e = check_cache(who, cache)) return e;
  if (int e = check_places(who, cache, page_table, starts, width, stb, stw, B, N)) return e;
  if (!q) return set_error(QFA_EINVAL, "%s: null pointer argument", who);
  if (!is_float_dtype(q_dtype)) return set_error(QFA_EINVAL, "%s: q_dtype %d is not QFA_F32/F16/BF16", who, q_dtype);
  if (!aligned16(q)) return set_error(QFA_EINVAL, "%s: q must be 16-byte aligned", who);
  if (!strides_ok(sqb, sqh, sqn, cache->D, elem_size(q_dtype)))
    return set_error(QFA_EINVAL, "%s: strides must be positive multiples of 16 bytes, token stride >= D", who);
  if (H <= 0 || H % cache->H != 0)
    return set_error(QFA_EINVAL, "%s: %lld query heads are no multiple of the cache's %lld", who, (long long)H, (long long)cache->H);
  if ((double)B * (double)H * (double)N > 1073741823.0) return set_error(QFA_EUNSUPPORTED, "%s: too many rows for one call", who);
  a->cache = ptrs_of(cache);
  a->page_table = page_table; a->starts = starts; a->counts = counts;
  a->pages = cache->pages; a->Hk = cache->H; a->width = width; a->stb = stb; a->stw = stw; a->B = B; a->H = H; a->N = N;
  a->page_log2 = log2_of(cache->page_size); a->scale_dtype = cache->scale_dtype; a->D = cache->D; a->q_dtype = q_dtype;
  a->q = q; a->sq[0] = sqb; a->sq[1] = sqh; a->sq[2] = sqn;
  return 0;
}
static int check_scale(const char *who, float sm_scale) {
  return sm_scale > 0.f && !isinf(sm_scale) ? 0 : set_error(QFA_EINVAL, "%s: sm_scale must be positive and finite", who);
}
static int check_workspace(const char *who, const char *query, const void *workspace, int64_t bytes, int64_t need) {
  if (need == 0 || (workspace && aligned16(workspace) && bytes >= need)) return 0;
  return set_error(QFA_EINVAL, "%s: workspace must be 16-byte aligned and hold %lld bytes (%s), got %lld", who, (long long)need, query, (long long)bytes);
}

static int attn_paged(const char *who, const char *query, bool with_lse, const qfa_paged_cache *cache, const void *q, int q_dtype, int64_t sqb, int64_t sqh, int64_t sqn,
                      const int32_t *page_table, int64_t width, int64_t stb, int64_t stw, const int32_t *starts, const int32_t *counts, void *o, float *lse,
                      int64_t B, int64_t H, int64_t N, int64_t prefix, float sm_scale, int causal, void *workspace, int64_t workspace_bytes, void *stream) {
  PagedAttnArgs a;
  if (int e = fill_attn(who, &a, cache, q, q_dtype, sqb, sqh, sqn, page_table, width, stb, stw, starts, counts, B, H, N)) return e;
  if (!o || (with_lse && !lse)) return set_error(QFA_EINVAL, "%s: null pointer argument", who);
  if (!aligned16(o)) return set_error(QFA_EINVAL, "%s: q and o must be 16-byte aligned", who);
  if (int e = check_scale(who, sm_scale)) return e;
  if (prefix < 0 || prefix > width * cache->page_size)
    return set_error(QFA_EINVAL, "%s: a prefix of %lld keys does not fit the page table", who, (long long)prefix);
  // rows, and units of work, are counted in 31 bits
  if (paged_attn_most_units(B, H, cache->H, N, cache->D, prefix, width * cache->page_size) > 2147483647.0)
    return set_error(QFA_EUNSUPPORTED, "%s: too many rows, or sequences times the keys that a page table has room for, for one call", who);
  if (int e = check_workspace(who, query, workspace, workspace_bytes, paged_attn_workspace_bytes(B, H, cache->H, N, cache->D, prefix, with_lse))) return e;
  a.o = o; a.lse = lse; a.prefix = prefix; a.sm_scale = sm_scale; a.causal = causal != 0; a.workspace = workspace;
  return launch_paged_attn(a, (hipStream_t)stream);
}

static int update_bounds(const char *who, const qfa_paged_cache *cache, const Bounds &bounds, const int32_t *page_table, int64_t width, int64_t stb, int64_t stw,
                         const int32_t *starts, const int32_t *counts, int64_t B, int64_t N, void *stream) {
  if (int e = check_cache(who, cache)) return e;
  if (int e = check_places(who, cache, page_table, starts, width, stb, stw, B, N)) return e;
  if (int e = check_bounds(who, bounds)) return e;
  PagedSelectArgs a;
  memset(&a, 0, sizeof(a));
  a.cache = ptrs_of(cache);
  a.codes = bounds.codes; a.scale = bounds.scale; a.zero = bounds.zero; a.zero_bits = bounds.bits;
  a.page_table = page_table; a.starts = starts; a.counts = counts;
  a.pages = cache->pages; a.Hk = cache->H; a.width = width; a.stb = stb; a.stw = stw; a.B = B; a.N = N;
  a.page_log2 = log2_of(cache->page_size); a.scale_dtype = cache->scale_dtype; a.D = cache->D;
  return launch_paged_bounds(a, (hipStream_t)stream);
}

static int select_blocks(const char *who, const qfa_paged_cache *cache, const Bounds &bounds, const void *q, int q_dtype, int64_t sqb, int64_t sqh, int64_t sqn,
                         const int32_t *page_table, int64_t width, int64_t stb, int64_t stw, const int32_t *starts, const int32_t *counts, int32_t *blocks,
                         float *scores, int64_t B, int64_t H, int64_t N, int64_t keep, int64_t first, int64_t last, void *workspace, int64_t workspace_bytes,
                         void *stream) {
  PagedAttnArgs x;
  if (int e = fill_attn(who, &x, cache, q, q_dtype, sqb, sqh, sqn, page_table, width, stb, stw, starts, counts, B, H, N)) return e;
  if (int e = check_bounds(who, bounds)) return e;
  if (!blocks) return set_error(QFA_EINVAL, "%s: null pointer argument", who);
  if (int e = check_keep(who, keep, first, last)) return e;
  if (!scores)
    if (int e = check_workspace(who, "qfa_paged_select_workspace_bytes", workspace, workspace_bytes, qfa_paged_select_workspace_bytes(B, cache->H, N, width)))
      return e;
  PagedSelectArgs a;
  memset(&a, 0, sizeof(a));
  a.cache = x.cache;
  a.codes = bounds.codes; a.scale = bounds.scale; a.zero = bounds.zero; a.zero_bits = bounds.bits;
  a.page_table = page_table; a.starts = starts; a.counts = counts;
  a.pages = x.pages; a.Hk = x.Hk; a.width = width; a.stb = stb; a.stw = stw; a.B = B; a.H = H; a.N = N;
  a.page_log2 = x.page_log2; a.scale_dtype = x.scale_dtype; a.D = x.D; a.q_dtype = q_dtype;
  a.q = q; a.sq[0] = sqb; a.sq[1] = sqh; a.sq[2] = sqn;
  a.blocks = blocks; a.scores = scores ? scores : static_cast<float *>(workspace); a.all_scores = scores != nullptr;
  a.keep = keep; a.first = first; a.last = last;
  return launch_paged_select(a, (hipStream_t)stream);
}

extern "C" {

int qfa_norm_rope(const qfa_norm_rope_tensor *q, const qfa_norm_rope_tensor *k, const float *cos, const float *sin, int64_t rope_rows,
                  int rotated, int interleaved, const int32_t *positions, int64_t spb, int64_t spn, int step, float eps, int dtype,
                  int w_dtype, int64_t B, int64_t N, int D, void *stream) {
  NormRopeArgs a;
  if (int e = fill_norm_rope("norm_rope", false, &a, q, k, cos, sin, rope_rows, rotated, interleaved, positions, spb, spn, step, eps, dtype, w_dtype, B, N, D))
    return e;
  return launch_norm_rope(a, false, (hipStream_t)stream);
}

int64_t qfa_norm_rope_bwd_workspace_bytes(int64_t B, int64_t N, int64_t Hq, int64_t Hk, int D, int weight_per_head) {
  if (B <= 0 || N <= 0 || Hq <= 0 || Hk < 0 || !head_dim_ok(D)) return 0;
  return norm_rope_bwd_workspace_bytes(B * N, Hq, Hk, D, weight_per_head != 0);
}

int qfa_norm_rope_bwd(const qfa_norm_rope_tensor *q, const qfa_norm_rope_tensor *k, const float *cos, const float *sin, int64_t rope_rows,
                      int rotated, int interleaved, const int32_t *positions, int64_t spb, int64_t spn, int step, float eps, int dtype,
                      int w_dtype, int64_t B, int64_t N, int D, void *workspace, int64_t workspace_bytes, void *stream) {
  NormRopeArgs a;
  if (int e = fill_norm_rope("norm_rope_bwd", true, &a, q, k, cos, sin, rope_rows, rotated, interleaved, positions, spb, spn, step, eps, dtype, w_dtype, B, N, D))
    return e;
  int64_t need = 0;
  for (int i = 0; i < 2; ++i)
    if (a.t[i].dw) need += norm_rope_bwd_workspace_bytes(B * N, a.t[i].H, 0, D, a.t[i].per_head);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return set_error(QFA_EINVAL, "norm_rope_bwd: workspace must be 16-byte aligned and hold %lld bytes (qfa_norm_rope_bwd_workspace_bytes), got %lld",
                     (long long)need, (long long)workspace_bytes);
  a.workspace = workspace;
  return launch_norm_rope(a, true, (hipStream_t)stream);
}

int qfa_paged_append(const qfa_paged_cache *cache, const void *k, const void *v, int dtype, int64_t skb, int64_t skh, int64_t skn, int64_t svb,
                     int64_t svh, int64_t svn, const int32_t *page_table, int64_t width, int64_t stb, int64_t stw, const int32_t *starts,
                     const int32_t *counts, const void *k_weight, int w_dtype, int weight_per_head, float eps, const float *cos, const float *sin,
                     int64_t rope_rows, int rotated, int interleaved, int64_t B, int64_t N, void *stream) {
  const char *who = "paged_append";
  if (int e = check_cache(who, cache)) return e;
  if (int e = check_places(who, cache, page_table, starts, width, stb, stw, B, N)) return e;
  if (!k || !v) return set_error(QFA_EINVAL, "%s: null pointer argument", who);
  if (!is_float_dtype(dtype)) return set_error(QFA_EINVAL, "%s: dtype %d is not QFA_F32/F16/BF16", who, dtype);
  if (!aligned16(k) || !aligned16(v)) return set_error(QFA_EINVAL, "%s: k and v must be 16-byte aligned", who);
  if (!strides_ok(skb, skh, skn, cache->D, elem_size(dtype)) || !strides_ok(svb, svh, svn, cache->D, elem_size(dtype)))
    return set_error(QFA_EINVAL, "%s: strides must be positive multiples of 16 bytes, token stride >= D", who);
  if (int e = check_norm(who, k_weight, w_dtype, dtype, eps)) return e;
  if (int e = check_rope(who, cos, sin, rope_rows, rotated, cache->D)) return e;
  PagedRowsArgs a;
  memset(&a, 0, sizeof(a));
  a.cache = ptrs_of(cache);
  a.page_table = page_table; a.starts = starts; a.counts = counts;
  a.pages = cache->pages; a.H = cache->H; a.width = width; a.stb = stb; a.stw = stw; a.B = B; a.N = N;
  a.page_log2 = log2_of(cache->page_size); a.scale_dtype = cache->scale_dtype; a.D = cache->D; a.dtype = dtype;
  a.k = k; a.v = v;
  a.sk[0] = skb; a.sk[1] = skh; a.sk[2] = skn; a.sv[0] = svb; a.sv[1] = svh; a.sv[2] = svn;
  a.w = k_weight; a.w_f32 = w_dtype == QFA_F32; a.w_per_head = weight_per_head != 0; a.eps = eps;
  a.cos = cos; a.sin = sin; a.rope_rows = rope_rows; a.half = rotated / 2; a.interleaved = interleaved != 0;
  return launch_paged_rows(a, false, (hipStream_t)stream);
}

int qfa_paged_read(const qfa_paged_cache *cache, const int32_t *page_table, int64_t width, int64_t stb, int64_t stw, const int32_t *starts,
                   const int32_t *counts, void *k_out, void *v_out, int dtype, int64_t B, int64_t N, void *stream) {
  const char *who = "paged_read";
  if (int e = check_cache(who, cache)) return e;
  if (int e = check_places(who, cache, page_table, starts, width, stb, stw, B, N)) return e;
  if (!k_out || !v_out) return set_error(QFA_EINVAL, "%s: null pointer argument", who);
  if (!is_float_dtype(dtype)) return set_error(QFA_EINVAL, "%s: dtype %d is not QFA_F32/F16/BF16", who, dtype);
  if (!aligned16(k_out) || !aligned16(v_out)) return set_error(QFA_EINVAL, "%s: outputs must be 16-byte aligned", who);
  PagedRowsArgs a;
  memset(&a, 0, sizeof(a));
  a.cache = ptrs_of(cache);
  a.page_table = page_table; a.starts = starts; a.counts = counts;
  a.pages = cache->pages; a.H = cache->H; a.width = width; a.stb = stb; a.stw = stw; a.B = B; a.N = N;
  a.page_log2 = log2_of(cache->page_size); a.scale_dtype = cache->scale_dtype; a.D = cache->D; a.dtype = dtype;
  a.k_out = k_out; a.v_out = v_out;
  return launch_paged_rows(a, true, (hipStream_t)stream);
}

int64_t qfa_attn_paged_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t prefix) {
  if (B <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || N <= 0 || !head_dim_ok(D) || prefix < 0) return 0;
  return paged_attn_workspace_bytes(B, H, Hk, N, D, prefix, false);
}

int64_t qfa_attn_paged_shared_prefix(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t prefix) {
  if (B <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || N <= 0 || !head_dim_ok(D) || prefix <= 0) return 0;
  return paged_attn_shared_prefix(B, H, Hk, N, D, prefix);
}

int qfa_attn_paged(const qfa_paged_cache *cache, const void *q, int q_dtype, int64_t sqb, int64_t sqh, int64_t sqn, const int32_t *page_table,
                   int64_t width, int64_t stb, int64_t stw, const int32_t *starts, const int32_t *counts, void *o, int64_t B, int64_t H, int64_t N,
                   int64_t prefix, float sm_scale, int causal, void *workspace, int64_t workspace_bytes, void *stream) {
  return attn_paged("attn_paged", "qfa_attn_paged_workspace_bytes", false, cache, q, q_dtype, sqb, sqh, sqn, page_table, width, stb, stw, starts, counts, o, nullptr, B, H,
                    N, prefix, sm_scale, causal, workspace, workspace_bytes, stream);
}

int64_t qfa_attn_paged_lse_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t prefix) {
  if (B <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || N <= 0 || !head_dim_ok(D) || prefix < 0) return 0;
  return paged_attn_workspace_bytes(B, H, Hk, N, D, prefix, true);
}

int qfa_attn_paged_lse(const qfa_paged_cache *cache, const void *q, int q_dtype, int64_t sqb, int64_t sqh, int64_t sqn, const int32_t *page_table,
                       int64_t width, int64_t stb, int64_t stw, const int32_t *starts, const int32_t *counts, void *o, float *lse, int64_t B, int64_t H, int64_t N,
                       int64_t prefix, float sm_scale, int causal, void *workspace, int64_t workspace_bytes, void *stream) {
  return attn_paged("attn_paged_lse", "qfa_attn_paged_lse_workspace_bytes", true, cache, q, q_dtype, sqb, sqh, sqn, page_table, width, stb, stw, starts, counts, o, lse, B,
                    H, N, prefix, sm_scale, causal, workspace, workspace_bytes, stream);
}

int qfa_paged_bounds(const qfa_paged_cache *cache, const qfa_page_bounds *bounds, const int32_t *page_table, int64_t width, int64_t stb, int64_t stw,
                     const int32_t *starts, const int32_t *counts, int64_t B, int64_t N, void *stream) {
  return update_bounds("paged_bounds", cache, bounds_of(bounds), page_table, width, stb, stw, starts, counts, B, N, stream);
}
int qfa_paged_bounds16(const qfa_paged_cache *cache, const qfa_page_bounds16 *bounds, const int32_t *page_table, int64_t width, int64_t stb, int64_t stw,
                       const int32_t *starts, const int32_t *counts, int64_t B, int64_t N, void *stream) {
  return update_bounds("paged_bounds16", cache, bounds_of(bounds), page_table, width, stb, stw, starts, counts, B, N, stream);
}

int64_t qfa_paged_select_workspace_bytes(int64_t B, int64_t Hk, int64_t N, int64_t width) {
  if (B <= 0 || Hk <= 0 || N <= 0 || width <= 0) return 0;
  return (B * Hk * N * width * 4 + 15) / 16 * 16;
}

int qfa_paged_select(const qfa_paged_cache *cache, const qfa_page_bounds *bounds, const void *q, int q_dtype, int64_t sqb, int64_t sqh, int64_t sqn,
                     const int32_t *page_table, int64_t width, int64_t stb, int64_t stw, const int32_t *starts, const int32_t *counts, int32_t *blocks,
                     float *scores, int64_t B, int64_t H, int64_t N, int64_t keep, int64_t first, int64_t last, void *workspace, int64_t workspace_bytes,
                     void *stream) {
  return select_blocks("paged_select", cache, bounds_of(bounds), q, q_dtype, sqb, sqh, sqn, page_table, width, stb, stw, starts, counts, blocks, scores, B, H, N, keep, first, last,
                       workspace, workspace_bytes, stream);
}
int qfa_paged_select16(const qfa_paged_cache *cache, const qfa_page_bounds16 *bounds, const void *q, int q_dtype, int64_t sqb, int64_t sqh, int64_t sqn,
                       const int32_t *page_table, int64_t width, int64_t stb, int64_t stw, const int32_t *starts, const int32_t *counts, int32_t *blocks,
                       float *scores, int64_t B, int64_t H, int64_t N, int64_t keep, int64_t first, int64_t last, void *workspace, int64_t workspace_bytes,
                       void *stream) {
  return select_blocks("paged_select16", cache, bounds_of(bounds), q, q_dtype, sqb, sqh, sqn, page_table, width, stb, stw, starts, counts, blocks, scores, B, H, N, keep, first, last,
                       workspace, workspace_bytes, stream);
}

int64_t qfa_attn_paged_blocks_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t keep, int page_size) {
  if (B <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || N <= 0 || !head_dim_ok(D) || !keep_ok(keep) || !page_size_ok(page_size)) return 0;
  if (keep > (1LL << 30) / page_size || paged_list_units(B, H, Hk, N, keep, log2_of(page_size)) > 2147483647.0) return 0;
  return paged_list_workspace_bytes(B, H, Hk, N, D, keep, log2_of(page_size));
}

int qfa_attn_paged_blocks(const qfa_paged_cache *cache, const void *q, int q_dtype, int64_t sqb, int64_t sqh, int64_t sqn, const int32_t *page_table,
                          int64_t width, int64_t stb, int64_t stw, const int32_t *starts, const int32_t *counts, const int32_t *blocks, int64_t keep, void *o,
                          int64_t B, int64_t H, int64_t N, float sm_scale, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "attn_paged_blocks";
  PagedListArgs a;
  if (int e = fill_attn(who, &a.x, cache, q, q_dtype, sqb, sqh, sqn, page_table, width, stb, stw, starts, counts, B, H, N)) return e;
  if (!o || !blocks) return set_error(QFA_EINVAL, "%s: null pointer argument", who);
  if (!aligned16(o)) return set_error(QFA_EINVAL, "%s: q and o must be 16-byte aligned", who);
  if (int e = check_scale(who, sm_scale)) return e;
  if (int e = check_keep(who, keep, 0, 0)) return e;
  if (keep > (1LL << 30) / cache->page_size) return set_error(QFA_EUNSUPPORTED, "%s: a list has room for 2^30 keys at most", who);
  if (paged_list_units(B, H, cache->H, N, keep, a.x.page_log2) > 2147483647.0)
    return set_error(QFA_EUNSUPPORTED, "%s: too many tokens times the keys of their lists for one call", who);
  if (int e = check_workspace(who, "qfa_attn_paged_blocks_workspace_bytes", workspace, workspace_bytes,
                              paged_list_workspace_bytes(B, H, cache->H, N, cache->D, keep, a.x.page_log2)))
    return e;
  a.x.o = o; a.x.sm_scale = sm_scale; a.x.causal = 1; a.x.workspace = workspace;
  a.blocks = blocks; a.keep = keep;
  return launch_paged_list(a, (hipStream_t)stream);
}

int64_t qfa_paged_weights_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int D) {
  if (B <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || N <= 0 || !head_dim_ok(D)) return 0;
  return paged_weigh_workspace_bytes(B, H, Hk, N, D);
}

int qfa_paged_weights(const qfa_paged_cache *cache, const void *q, int q_dtype, int64_t sqb, int64_t sqh, int64_t sqn, const float *lse,
                      const int32_t *page_table, int64_t width, int64_t stb, int64_t stw, const int32_t *starts, const int32_t *counts, const float *before,
                      float decay, float *out, int64_t B, int64_t H, int64_t N, float sm_scale, int causal, void *workspace, int64_t workspace_bytes,
                      void *stream) {
  const char *who = "paged_weights";
  PagedWeighArgs a;
  if (int e = fill_attn(who, &a.x, cache, q, q_dtype, sqb, sqh, sqn, page_table, width, stb, stw, starts, counts, B, H, N)) return e;
  if (!lse || !out) return set_error(QFA_EINVAL, "%s: null pointer argument", who);
  if (int e = check_scale(who, sm_scale)) return e;
  if (before && !(fabsf(decay) <= 3.402823466e38f)) return set_error(QFA_EINVAL, "%s: decay must be finite", who);
  if (int e = check_slots(who, cache, width)) return e;
  if (int e = check_workspace(who, "qfa_paged_weights_workspace_bytes", workspace, workspace_bytes, paged_weigh_workspace_bytes(B, H, cache->H, N, cache->D))) return e;
  a.x.sm_scale = sm_scale; a.x.causal = causal != 0; a.x.workspace = workspace;
  a.lse = lse; a.before = before; a.decay = decay; a.out = out;
  return launch_paged_weigh(a, (hipStream_t)stream);
}

int qfa_paged_evict(const qfa_paged_cache *cache, const int32_t *page_table, int64_t width, int64_t stb, int64_t stw, const int32_t *lengths,
                    const float *weights, const int32_t *new_table, int64_t new_width, int64_t ntb, int64_t ntw, int32_t *kept, float *new_weights,
                    int32_t *new_lengths, int64_t B, int64_t keep, int64_t first, int64_t last, void *stream) {
  const char *who = "paged_evict";
  if (int e = check_cache(who, cache)) return e;
  if (int e = check_places(who, cache, page_table, lengths, width, stb, stw, B, 1)) return e;
  if (int e = check_places(who, cache, new_table, lengths, new_width, ntb, ntw, B, 1)) return e;
  if (!weights || !kept || !new_weights || !new_lengths) return set_error(QFA_EINVAL, "%s: null pointer argument", who);
  if (int e = check_keep(who, keep, first, last)) return e;
  if (int e = check_slots(who, cache, width)) return e;
  if (int e = check_slots(who, cache, new_width)) return e;
  if (new_width * cache->page_size < (keep < width * cache->page_size ? keep : width * cache->page_size))
    return set_error(QFA_EINVAL, "%s: %lld new pages of %d rows do not hold %lld", who, (long long)new_width, cache->page_size, (long long)keep);
  PagedEvictArgs a;
  memset(&a, 0, sizeof(a));
  a.cache = ptrs_of(cache);
  a.page_table = page_table; a.new_table = new_table; a.lengths = lengths; a.weights = weights;
  a.kept = kept; a.new_lengths = new_lengths; a.new_weights = new_weights;
  a.pages = cache->pages; a.Hk = cache->H; a.width = width; a.stb = stb; a.stw = stw; a.new_width = new_width; a.ntb = ntb; a.ntw = ntw;
  a.B = B; a.keep = keep; a.first = first; a.last = last;
  a.page_log2 = log2_of(cache->page_size); a.scale_dtype = cache->scale_dtype; a.D = cache->D;
  return launch_paged_evict(a, (hipStream_t)stream);
}

}  // extern "C"
