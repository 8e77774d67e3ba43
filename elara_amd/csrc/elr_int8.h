// Rows held in 8-bit integers: int8 values with one fp32 scale for each row or each group of columns; value = q * scale.
// Shared by the quantizer, the products and the norm's backward.
#pragma once

#include "elr_elem.h"

namespace elr {

// As many int8 elements as a 16-byte vector of E has.
template <class E>
struct Int8Raw {
  uint32_t v[Elem<E>::VE / 4];
};

// The elements at p of which `valid` (any number; <= 0: none) may be read; the others are 0.
template <class E>
__device__ __forceinline__ Int8Raw<E> int8_load(const int8_t* p, int64_t valid) {
  constexpr int VE = Elem<E>::VE;
  Int8Raw<E> r;
  if (valid >= VE) {
    typedef uint32_t uN __attribute__((ext_vector_type(VE / 4 > 1 ? VE / 4 : 2)));
    typedef uint32_t u1 __attribute__((aligned(1)));
    typedef uN uN_u __attribute__((aligned(1)));
    if constexpr (VE == 4) {
      r.v[0] = __builtin_nontemporal_load(reinterpret_cast<const u1*>(p));
    } else {
      const uN x = __builtin_nontemporal_load(reinterpret_cast<const uN_u*>(p));
#pragma unroll
      for (int i = 0; i < VE / 4; ++i) r.v[i] = x[i];
    }
    return r;
  }
#pragma unroll
  for (int i = 0; i < VE / 4; ++i) {
    r.v[i] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (4 * i + j < valid) r.v[i] |= (uint32_t)(uint8_t)p[4 * i + j] << (8 * j);
  }
  return r;
}

template <class E>
__device__ __forceinline__ Frag<E> int8_widen(const Int8Raw<E>& r, float scale) {
  Frag<E> f;
#pragma unroll
  for (int j = 0; j < Elem<E>::VE; ++j) f.v[j] = (float)(int8_t)(r.v[j / 4] >> (8 * (j & 3))) * scale;
  return f;
}

inline bool int8_group_ok(int64_t group) { return group == 0 || group == 32 || group == 64 || group == 128 || group == 256; }
// Scales of a row of D columns, and the shift from a column to its scale (a whole row's: every column to 0, D < 2^31).
inline int64_t int8_groups(int64_t D, int64_t group) { return group ? (D + group - 1) / group : 1; }
inline int int8_shift(int64_t group) {
  int s = 0;
  if (!group) return 31;
  while (((int64_t)1 << s) < group) ++s;
  return s;
}

}  // namespace elr
