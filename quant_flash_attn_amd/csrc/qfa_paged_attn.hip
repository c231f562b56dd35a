// Attention of the queries at the end of every sequence of a batch on the pages of an INT8 cache:
//     O = softmax(sm_scale * Q^ K^^T) V^,   X^ = scale * (codes - zero_point) per token,
// with the arithmetic of the kernel for a cache in one piece (qfa_cache.hip): queries quantized per token here, Q K^T on INT8
// MFMA with the exact zero-point term, V as its exact codes in binary16, softmax statistics and sums in fp32.
//
// Bound by reading the cache once (2 D + 6 bytes per key and key head): 64 sequences of 65 to 8192 keys, 8 key heads of 128, 550 MB in
// 99 us (5.6 TB/s); of short work the start, where lengths, page numbers and keys are three loads that wait for each other (4 us), and
// the kernel that joins the pieces (5 us): 16 heads of 16384 keys 22 us.  A workgroup = 4 waves = 16 rows (queries times the
// query heads that share a key head) of one sequence and key head, and a piece of its keys (qfa_paged_work.h); 32-key tiles are
// dealt to the waves, each with its own online softmax.  A tile lives in registers, double-buffered (but for 256 elements) as there.  A page holds 16
// keys or a multiple, so the two halves of a tile lie in one page each: their pages' numbers are fetched 32 tiles ahead, one
// lane per half, and read out of the lanes as scalars, so that no load of keys waits for the page table.
//
// What the mask hides may hold anything (pages that were never written): its scores are replaced, its probability is zero and
// zero wins over whatever its scale holds.
#include "qfa_paged_block.h"

namespace qfa {

// O from the pieces of its rows: a workgroup joins up to 16 rows of one sequence and key head, D/4 lanes of four columns each; with
// fewer rows than 1024/D the pieces of a row are dealt to several groups of lanes, which meet in LDS.  Rows that lie in one piece
// have been stored already (no shared prefix); rows that see no key become zeros.
struct PagedMergeArgs {
  PagedWork own, shared;   // shared.grid 0: none
  void *o;
  int o_dtype, chunks, chunk_rows;   // chunks of rows of a sequence and key head, a power of two that divides a block
  float *lse;                        // of LSE
};
template <int D, bool LSE> __global__ __launch_bounds__(256) void paged_merge_kernel(PagedMergeArgs a) {
  constexpr int CL = D / 4, SLOTS = 256 / CL;
  __shared__ float red[SLOTS][D + 4];
  const int tid = threadIdx.x, d = 4 * (tid % CL), slot = tid / CL;
  const PagedDeal<false, false> own(a.own, a.own.br, a.own.tk);
  const int bh = (int)(blockIdx.x / (unsigned)a.chunks), chunk = (int)(blockIdx.x % (unsigned)a.chunks), b = bh / a.own.Hk, h = bh % a.own.Hk;
  const int r0 = chunk * a.chunk_rows, n = min(a.chunk_rows, own.rows - r0), rb = r0 / own.BR;
  const unsigned *note = a.own.first + 2 * own.item_index(b, h, rb), first = note[0], each = max(note[1], 1u);   // (nobody's, without tiles)
  const PagedSeq seq = own.load(b);
  const PagedPieces mine(first, each, own.tiles(seq, rb), (int64_t)bh * own.rows + r0, r0 % own.BR);
  if (!a.own.whole && mine.whole >= 0) return;   // stored
  auto store = [&](int r, const PagedSum &x) __attribute__((always_inline)) {
    const int i = r / a.own.G;
    const float inv = i >= seq.tokens || x.l == 0.f ? 0.f : 1.0f / x.l;
    const int64_t row = ((int64_t)b * a.own.Hk * a.own.G + h * a.own.G + r % a.own.G) * a.own.N + i, off = row * D;
    if (LSE && d == 0) a.lse[row] = i >= seq.tokens || x.l == 0.f ? -INFINITY : (x.m + __log2f(x.l)) * kLn2;
    store4(static_cast<char *>(a.o) + off * (a.o_dtype == QFA_F32 ? 4 : 2), a.o_dtype, d,
           f32x4{mul_zero_wins(x.acc[0], inv), mul_zero_wins(x.acc[1], inv), mul_zero_wins(x.acc[2], inv), mul_zero_wins(x.acc[3], inv)});
  };
  if (n > SLOTS && a.shared.grid == 0) {   // two rows at a time
    for (int k = slot; k < n; k += 2 * SLOTS) {
      PagedSum x[2] = {{NO_KEY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}}, {NO_KEY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}}};
      PagedPieces p = mine;
      p.in_block += k;
      if (p.whole >= 0) p.whole += k;
      paged_add<D, 2>(a.own, p, d, 0, 1, x, k + SLOTS < n ? SLOTS : 0);
      store(r0 + k, x[0]);
      if (k + SLOTS < n) store(r0 + k + SLOTS, x[1]);
    }
    return;
  }
  const int groups = n >= SLOTS ? 1 : SLOTS / n;   // of pieces
  for (int first = 0; first < n; first += SLOTS) {
    const int k = groups == 1 ? first + slot : slot % n, group = groups == 1 ? 0 : slot / n;   // row of the chunk
    const bool live = k < n && group < groups;
    const int r = r0 + min(k, n - 1), i = r / a.own.G;
    PagedSum x[1] = {{NO_KEY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}}};
    if (live && i < seq.tokens) {
      PagedPieces p = mine;
      p.in_block += r - r0;
      if (p.whole >= 0) p.whole += r - r0;
      paged_add<D, 1>(a.own, p, d, group, groups, x, 0);
      if (a.shared.grid > 0) {
        const PagedDeal<true, false> all(a.shared, a.shared.br, a.shared.tk);
        const int rs = b * own.rows + r, item = h * all.blocks + rs / all.BR;
        const unsigned u = all.units({0, 0}, 0);
        const PagedPieces q((unsigned)item * u + (unsigned)a.shared.extra, all.each, all.tiles({0, 0}, 0), (int64_t)h * all.rows + rs, rs % all.BR);
        paged_add<D, 1>(a.shared, q, d, group, groups, x, 0);
      }
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
    store(r, x[0]);
  }
}

// Rows of a block, in a launch over `problems` (sequences times key heads) of that many rows: 16, or the tiles' 64 or 128 beyond.
// Two blocks of 16 read the keys twice but need no other launch and leave no wave without rows; 20 rows of 256 elements, 3000 keys
// of 8 sequences: 39 us against 47 on tiles; 32 rows, 8192 keys of one sequence, 128 elements: 23 against 29, of 64 sequences with
// 64 elements 167 against 193, but with 128 elements, where the keys no longer stay in the last cache, 313 against 250.
// (48 rows on three blocks: 68 us against 59.)
static int block_rows(int64_t rows, int D, int64_t problems) {
  if (rows <= PAGED_ROWS || (rows <= 2 * PAGED_ROWS && (D != 128 || problems <= 128))) return PAGED_ROWS;
  return rows <= 64 ? 64 : 128;
}
static int tile_keys(int br) { return br == PAGED_ROWS ? SKV_TILE : PAGED_TILE; }
static int item_units(int br) { return br == PAGED_ROWS ? 12 : 4; }   // beside its tiles, see qfa_paged_work.h
static int work_grid(int br, int D) { return br == PAGED_ROWS ? PAGED_WGS : paged_tile_grid(D); }
// bytes of a launch's slots, and of its whole items
static int64_t slots_bytes(int br, int D) { return 2LL * work_grid(br, D) * br * (D + 2) * 4; }
static int64_t whole_bytes(int64_t rows, int D) { return (rows * (D + 2) * 4 + 15) / 16 * 16; }
static int64_t first_bytes(int64_t problems, int64_t rows, int br) { return (8 * problems * ((rows + br - 1) / br) + 15) / 16 * 16; }
static int64_t quantized_bytes(int64_t rows, int D) { return (rows * D + 4 * rows + rows + 15) / 16 * 16; }
int64_t paged_attn_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t prefix, bool lse) {
  const int64_t rows = N * (H / Hk);
  const int own = block_rows(rows, D, B * Hk), shared = prefix > 0 ? block_rows(B * rows, D, Hk) : 0;
  int64_t bytes = slots_bytes(own, D) + first_bytes(B * Hk, rows, own);
  if (prefix > 0) bytes += slots_bytes(shared, D) + 2 * whole_bytes(B * H * N, D);
  else if (lse) bytes += whole_bytes(B * H * N, D);   // (the kernel that joins pieces writes it, of items in one piece also)
  if (own > PAGED_ROWS || shared > PAGED_ROWS) bytes += quantized_bytes(B * H * N, D);   // (blocks of 16 quantize their own)
  return bytes;
}

// Units of work (qfa_paged_work.h) that a launch of the call has at most, if every sequence fills its `keys` keys
double paged_attn_most_units(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t prefix, int64_t keys) {
  const auto most = [&](int64_t problems, int64_t rows, int64_t n) {
    const int br = block_rows(rows, D, problems);
    return (double)problems * (double)((rows + br - 1) / br) * ((double)n / tile_keys(br) + 2 + item_units(br));
  };
  const double own = most(B * Hk, N * (H / Hk), keys), shared = prefix > 0 ? most(Hk, B * N * (H / Hk), prefix) : 0.0;
  return own > shared ? own : shared;
}

// How long a pass over `keys` keys takes for problems * rows rows beside its start, in us: every block of rows reads them again, at the
// rate (TB/s, of a chip that is full) that its kernel has in its caches
static double pass_us(int64_t problems, int64_t rows, int64_t keys, int D) {
  const int br = block_rows(rows, D, problems);
  const double rate = br == PAGED_ROWS ? 11.0 : br == 64 ? (D == 128 ? 5.5 : 3.75) : (D == 128 ? 3.4 : 2.5);
  return (double)problems * (double)((rows + br - 1) / br) * (double)keys * 2 * D / (rate * 1e6);
}
// Whether a prefix gets a pass of its own.  That one has its start, its queries quantized and results of all rows written and joined
// again against it: where it saves less, every sequence reads the prefix from its own pages.  Of 240 calls timed both ways (4 to 64
// sequences, 1 to 300 rows, prefixes of 400, 2000 and 8000 keys, D 64, 128 and 256) 34 get one: 31 of them take 0.33 to 1.0 of the time
// without and three, of 256 elements, 1.09 to 1.29; of the others 201 take 1.01 to 2.4 of the time with it, five 0.78 to 0.95.
int64_t paged_attn_shared_prefix(int64_t B, int64_t H, int64_t Hk, int64_t N, int D, int64_t prefix) {
  const int64_t rows = N * (H / Hk);
  const double start = block_rows(B * rows, D, Hk) == PAGED_ROWS ? 6.0 + D / 64 : 13.0 + 3.5 * (D / 64);
  const double joined = (double)(B * H * N) * (D + 2) * 16 / 4.5e6;   // written twice, read twice
  return B > 1 && pass_us(B * Hk, rows, prefix, D) > pass_us(Hk, B * rows, prefix, D) + start + joined ? prefix : 0;
}

template <typename S, int D, bool SHARED> static int launch_rows(const PagedAttnKernelArgs &a, bool one, bool stream, hipStream_t st) {
  const dim3 grid((unsigned)a.work.grid), block(256);
  if (!one) paged_rows_kernel<S, D, PagedDeal<SHARED, false>, false><<<grid, block, 0, st>>>(a);
  else if (!SHARED && stream) paged_rows_kernel<S, D, PagedDeal<false, true>, true><<<grid, block, 0, st>>>(a);
  else paged_rows_kernel<S, D, PagedDeal<SHARED, true>, false><<<grid, block, 0, st>>>(a);
  return check_launch(SHARED ? "qfa_attn_paged (prefix)" : "qfa_attn_paged");
}
template <typename S, int D> static int launch_rows(const PagedAttnKernelArgs &a, bool shared, bool one, bool stream, hipStream_t st) {
  return shared ? launch_rows<S, D, true>(a, one, stream, st) : launch_rows<S, D, false>(a, one, stream, st);
}
template <int D> static int launch_d(const PagedAttnArgs &x, hipStream_t st) {
  PagedAttnKernelArgs a = {};
  a.q = x.q; a.kc = x.cache.k_codes; a.ks = x.cache.k_scale; a.kz = x.cache.k_zero;
  a.vc = x.cache.v_codes; a.vs = x.cache.v_scale; a.vz = x.cache.v_zero; a.o = x.o; a.page_table = x.page_table;
  a.pages = x.pages; a.stb = x.stb; a.stw = x.stw; a.sqb = x.sq[0]; a.sqh = x.sq[1]; a.sqn = x.sq[2];
  a.width = (int)x.width; a.page_log2 = x.page_log2; a.q_dtype = x.q_dtype;
  a.sm_scale_log2 = x.sm_scale * kLog2e;
  const int G = (int)(x.H / x.Hk);
  const int64_t rows = x.B * x.H * x.N, problem[2] = {x.N * G, x.B * x.N * G};
  PagedWork w[2];
  float *mem = static_cast<float *>(x.workspace);
  for (int i = 0; i < 2; ++i) {
    const int br = block_rows(problem[i], D, (i == 0 ? x.B : 1) * x.Hk), grid = x.prefix > 0 || i == 0 ? work_grid(br, D) : 0;
    w[i] = {x.starts, x.counts, (int)x.B, (int)x.Hk, G, (int)x.N, x.causal, (int)x.prefix, (int)(x.width << x.page_log2), grid, br,
            tile_keys(br), item_units(br), nullptr, nullptr, nullptr, nullptr, nullptr};
    if (grid == 0) continue;
    if (i == 0) {
      w[i].first = reinterpret_cast<unsigned *>(mem);
      mem += first_bytes(x.B * x.Hk, problem[0], br) / 4;
    }
    w[i].slots = mem;
    w[i].slots_ml = mem + 2LL * grid * br * D;
    mem += slots_bytes(br, D) / 4;
    if (x.prefix > 0 || x.lse) {
      w[i].whole = mem;
      w[i].whole_ml = mem + rows * D;
      mem += whole_bytes(rows, D) / 4;
    }
  }
  if (w[0].br > PAGED_ROWS || (w[1].grid > 0 && w[1].br > PAGED_ROWS)) {   // many rows: quantized once, every piece of keys needs them
    int8_t *codes = reinterpret_cast<int8_t *>(mem), *zero = codes + rows * (D + 4);
    float *scale = reinterpret_cast<float *>(codes + rows * D);
    // (one token each: a sequence's heads as tokens of one head, which fill the quantizer's workgroups)
    const bool one = x.N == 1;
    if (int e = launch_quant(x.q, x.q_dtype, codes, scale, nullptr, 0, zero, nullptr, x.B, one ? 1 : x.H, one ? x.H : x.N, D, x.sq[0], one ? x.sq[2] : x.sq[1],
                             one ? x.sq[1] : x.sq[2], x.H * x.N * D, one ? D : x.N * D, D, st))
      return e;
    a.q_codes = codes; a.q_scale = scale; a.q_zero = zero;
  }
  // Non-temporal loads (LOAD_ONCE) where the keys and values that a call may reach outgrow the last-level cache (256 MiB) for good.  One token
  // of 64 sequences, 8 key heads of 64, 128 and 256 elements, us with plain loads and with these: 128 MiB 29.1, 27.4, 28.4 and 28.8, 28.1,
  // 28.3; 256 MiB 49.2, 46.3, 47.4 and 49.7, 48.1, 47.7; 320 MiB 65.4, 61.5, 62.1 and 60.8, 58.1, 57.1; 512 MiB 105, 99, 100 and 93, 88, 87.
  // The lengths are not known here: short sequences under a table of 4 GiB are read with these too, 16 to 128 MiB of them in the same time
  // and 256 in 49.0 us in place of 46.7.  Two blocks of rows, which read every key twice, keep plain loads (20 rows, 512 MiB, 64, 128 and 256
  // elements: 200, 176 and 191 us; with these 180, 182 and 181).
  const bool stream = (double)(x.pages < x.B * x.width ? x.pages : x.B * x.width) * (double)(x.Hk << x.page_log2) * 2 * D >= 320.0 * (1 << 20);
  for (int i = 1; i >= 0; --i) {
    if (w[i].grid == 0) continue;
    a.work = w[i];
    int e;
    if (w[i].br > PAGED_ROWS) e = launch_paged_tile(a, i == 1, D, x.scale_dtype, w[i].br / 32, st);
    else if (x.scale_dtype == QFA_F32) e = launch_rows<float, D>(a, i == 1, problem[i] <= PAGED_ROWS, stream, st);
    else if (x.scale_dtype == QFA_F16) e = launch_rows<_Float16, D>(a, i == 1, problem[i] <= PAGED_ROWS, stream, st);
    else e = launch_rows<__bf16, D>(a, i == 1, problem[i] <= PAGED_ROWS, stream, st);
    if (e) return e;
  }
  // rows per workgroup: few, whose pieces many lanes share, while that leaves no more than 1024 workgroups (2048 rows one by one: 9.4 us
  // against 6.4 two by two, with a prefix 12.9 against 10.5; in 512 workgroups 5.7 and 11.4)
  int chunk_rows = 1;
  while (chunk_rows < 16 && x.B * x.Hk * ((problem[0] + chunk_rows - 1) / chunk_rows) > 1024) chunk_rows *= 2;
  const int chunks = (int)((problem[0] + chunk_rows - 1) / chunk_rows);
  const PagedMergeArgs m = {w[0], w[1], x.o, x.q_dtype, chunks, chunk_rows, x.lse};
  const dim3 grid((unsigned)(x.B * x.Hk * chunks));
  if (x.lse) paged_merge_kernel<D, true><<<grid, dim3(256), 0, st>>>(m);
  else paged_merge_kernel<D, false><<<grid, dim3(256), 0, st>>>(m);
  return check_launch("qfa_attn_paged (merge)");
}
int launch_paged_attn(const PagedAttnArgs &x, hipStream_t st) {
  if (x.D == 64) return launch_d<64>(x, st);
  if (x.D == 128) return launch_d<128>(x, st);
  return launch_d<256>(x, st);
}

}  // namespace qfa
