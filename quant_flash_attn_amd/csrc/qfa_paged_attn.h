// Shared declarations of the kernels for attention on a paged cache: rows in blocks of 16 (qfa_paged_attn.hip), and many of
// them on tiles that a workgroup expands once (qfa_paged_tile.hip).
#pragma once
#include "qfa_paged_work.h"

namespace qfa {

struct PagedAttnKernelArgs {
  PagedWork work;
  const void *q; const int8_t *kc; const void *ks; const int8_t *kz; const int8_t *vc; const void *vs; const int8_t *vz;
  void *o;
  const int32_t *page_table;
  int64_t pages, stb, stw, sqb, sqh, sqn;
  const int8_t *q_codes; const float *q_scale; const int8_t *q_zero;   // the queries quantized, dense (for many rows)
  int width, page_log2, q_dtype;
  float sm_scale_log2;
  // of lists: [B, Hk, N, keep]; tiles of an item, units of a workgroup
  const int32_t *blocks;
  int keep;
  unsigned list_tiles, list_each;
};

// What lists need stands behind all else and not in PagedWork: eight bytes more there, and the compiler makes other code of the kernels that have no lists (20 rows of 256
// elements, 801 to 3001 keys of 8 sequences: 23.6 us in place of 23.0)
static_assert(sizeof(PagedWork) == 104, "measure attention on all keys before a field is added");

// log2 of the largest p' = p * scale_j at a new reference, and the p' past which the reference moves (see CACHE_P_REF in
// qfa_cache.hip): p' enters the P.V product as binary16, and the scales carry V's magnitude
constexpr float PAGED_P_REF = 7.0f, PAGED_P_MAX = 0x1p10f;
constexpr unsigned PAGED_P_MAX_BITS = 0x6400;   // that limit as a binary16 number

constexpr int PAGED_TILE = 64;   // keys of a tile there
// blocks of 64 or 128 rows: qw = 2 or 4 waves side by side; the workgroups of a launch, and the launch
// (three workgroups on a CU with 64 elements: 2 to 5 % over two)
inline int paged_tile_grid(int D) { return D == 256 ? 256 : D == 64 ? 768 : 512; }
int launch_paged_tile(const PagedAttnKernelArgs &a, bool shared, int D, int scale_dtype, int qw, hipStream_t st);

}  // namespace qfa
