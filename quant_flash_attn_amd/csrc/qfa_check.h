// Argument checks that the C entry points share.
#pragma once
#include "qfa_host.h"

namespace qfa {

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned8(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }
inline bool is_float_dtype(int d) { return d == QFA_F32 || d == QFA_F16 || d == QFA_BF16; }
inline int elem_size(int d) { return d == QFA_F32 ? 4 : 2; }

// strides (elements) of a [B,H,N,D] tensor with element size `es`: positive, 16-byte multiples,
// and the token stride must at least span a row
inline bool strides_ok(int64_t sb, int64_t sh, int64_t sn, int D, int es) {
  if (sb <= 0 || sh <= 0 || sn < D) return false;
  return (sb * es) % 16 == 0 && (sh * es) % 16 == 0 && (sn * es) % 16 == 0;
}

}  // namespace qfa
