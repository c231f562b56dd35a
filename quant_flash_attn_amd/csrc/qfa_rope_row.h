// One token row of one head, as the kernels that norm and rotate hold it: D/16 adjacent lanes, 16 elements each, in two
// chunks of eight consecutive ones.  The chunks are chosen so that a lane holds both elements of every pair that the rotation
// mixes, so nothing is exchanged between lanes but the sums of the norm:
//   pairs (i, i + R/2): lane j < R/16 holds the chunks j and j + R/16 (and what is not rotated is dealt to the other lanes)
//   pairs (2i, 2i + 1): any chunk holds whole pairs; lane j takes the chunks j and j + D/16
// Either way the lanes of a row read whole lines together.
#pragma once
#include "qfa_device.h"
#include "qfa_host.h"

namespace qfa {

// eight consecutive elements of T as floats, and back with one rounding.  ONCE: non-temporal, for what nothing in the caches is to make
// room for
template <typename T, bool ONCE = false> __device__ __forceinline__ void load8(const T *p, float *v) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 *w = reinterpret_cast<const f32x4 *>(p);
    const f32x4 a = ONCE ? __builtin_nontemporal_load(w) : w[0], b = ONCE ? __builtin_nontemporal_load(w + 1) : w[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
  } else {
    const u32x4 *from = reinterpret_cast<const u32x4 *>(p), w = ONCE ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[2 * e] = lo_to_f32<T>(w[e]); v[2 * e + 1] = hi_to_f32<T>(w[e]); }
  }
}
template <typename V, bool ONCE> __device__ __forceinline__ void store_words(void *p, V x) {
  if constexpr (ONCE) __builtin_nontemporal_store(x, static_cast<V *>(p));
  else *static_cast<V *>(p) = x;
}
template <typename T, bool ONCE = false> __device__ __forceinline__ void store8(T *p, const float *v) {
  if constexpr (sizeof(T) == 4) {
    store_words<f32x4, ONCE>(p, f32x4{v[0], v[1], v[2], v[3]});
    store_words<f32x4, ONCE>(p + 4, f32x4{v[4], v[5], v[6], v[7]});
  } else {
    store_words<u32x4, ONCE>(p, u32x4{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])});
  }
}

// sum over the LPR adjacent lanes of a row, in every one of them
template <int LPR> __device__ __forceinline__ float row_sum(float x) {
  static_assert(LPR == 4 || LPR == 8 || LPR == 16, "rows of 64, 128 or 256 elements");
  x += dpp_f<0xB1>(x);
  x += dpp_f<0x4E>(x);
  if constexpr (LPR >= 8) x += dpp_f<0x141>(x);
  if constexpr (LPR >= 16) x += dpp_f<0x140>(x);
  return x;
}

// 1 / sqrt(mean(x^2) + eps) of a row of LPR lanes, for v[e] as it then stands: where the squares leave fp32's range (their mean is infinite, or
// below 2^-100, where what underflows begins to count) v, eps and the result are those of the row times `k`, a power of two, and x / rms is
// v * result all the same; 1 for any other row.  A row with an infinity or a NaN keeps it.
template <int LPR> __device__ __forceinline__ float row_inverse_rms(float (&v)[16], float eps, float &k) {
  constexpr float PART = 1.0f / (16 * LPR);
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) ss += v[e] * v[e];
  float mean = row_sum<LPR>(ss) * PART + eps;
  k = 1.f;
  if (!(mean >= 0x1p-100f && mean < INFINITY)) {   // (the same in all lanes of a row)
    k = mean < 1.f ? 0x1p100f : 0x1p-70f;
    ss = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      v[e] *= k;
      ss += v[e] * v[e];
    }
    mean = row_sum<LPR>(ss) * PART + eps * k * k;
  }
  return 1.0f / sqrtf(mean);
}

// What a lane holds of a row, and the angles of its token
template <int D, bool INTERLEAVED> struct RopeLane {
  static constexpr int LPR = D / 16;
  int a, b;          // first elements of its two chunks
  bool rot_a, rot_b; // whether they are rotated
  float c[8], s[8];
  // half: pairs of a row that are rotated, a multiple of 8 (0: none)
  __device__ __forceinline__ RopeLane(int sub, int half) {
    if constexpr (INTERLEAVED) {
      a = 8 * sub;
      b = 8 * (sub + LPR);
      rot_a = a < 2 * half;
      rot_b = b < 2 * half;
    } else {
      const int hc = half / 8;
      rot_a = rot_b = sub < hc;
      a = 8 * (rot_a ? sub : hc + sub);   // (the rest: chunks 2 hc .. 2 LPR - 1, its first half and its second)
      b = 8 * (rot_a ? sub + hc : LPR + sub);
    }
  }
  // Angles of a position.  One outside the table leaves NaN, which the row's rotated elements then are.
  __device__ __forceinline__ void angles(const float *cos, const float *sin, int64_t pos, int64_t rows, int half) {
    const bool in = pos >= 0 && pos < rows;
    const int at_a = INTERLEAVED ? a / 2 : a, at_b = INTERLEAVED ? b / 2 : a + 4;
    const bool go_a = rot_a, go_b = INTERLEAVED ? rot_b : rot_a;
    f32x4 x[4];
    const float nan = __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = f32x4{nan, nan, nan, nan};
    if (in) {
      const float *cp = cos + pos * half, *sp = sin + pos * half;
      if (go_a) {
        x[0] = *reinterpret_cast<const f32x4 *>(cp + at_a);
        x[2] = *reinterpret_cast<const f32x4 *>(sp + at_a);
      }
      if (go_b) {
        x[1] = *reinterpret_cast<const f32x4 *>(cp + at_b);
        x[3] = *reinterpret_cast<const f32x4 *>(sp + at_b);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) { c[e] = x[0][e]; c[4 + e] = x[1][e]; s[e] = x[2][e]; s[4 + e] = x[3][e]; }
  }
  // v[0..7] is chunk a, v[8..15] chunk b.  BACK: by the opposite angle (the transposed rotation).  Each product and sum is
  // rounded by itself where the file is compiled without contraction.
  template <bool BACK> __device__ __forceinline__ void turn(float (&v)[16]) const {
    if constexpr (INTERLEAVED) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = v[2 * e], y = v[2 * e + 1], sn = BACK ? -s[e] : s[e];
        const bool rot = e < 4 ? rot_a : rot_b;
        v[2 * e] = rot ? x * c[e] - y * sn : x;
        v[2 * e + 1] = rot ? y * c[e] + x * sn : y;
      }
    } else if (rot_a) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = v[e], y = v[8 + e], sn = BACK ? -s[e] : s[e];
        v[e] = x * c[e] - y * sn;
        v[8 + e] = y * c[e] + x * sn;
      }
    }
  }
};

}  // namespace qfa
