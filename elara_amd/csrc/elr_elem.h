// Element types (fp32, fp16, bf16) in 16-byte vectors, and wave reductions, for the operators between the looked-up rows
// and their update (log probabilities, norms, gradient clipping).  All arithmetic is fp32: an element is widened when it
// is loaded and rounded once, to nearest even, when it is stored.
#pragma once

#include "elr_common.h"

namespace elr {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// A 16-byte vector at any element's address: gfx950 takes such accesses in one instruction (a row of an odd number of
// 16-bit elements then needs no peeled head; only the memory lines at its ends are touched twice).
typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_u __attribute__((ext_vector_type(2), aligned(2)));

// VE elements in 16 bytes; widen() and narrow() convert a whole vector.
template <class E>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int VE = 4, kType = ELR_F32;
  typedef f32x4 vec;
};
template <>
struct Elem<_Float16> {
  static constexpr int VE = 8, kType = ELR_F16;
  typedef f16x8 vec;
};
template <>
struct Elem<__bf16> {
  static constexpr int VE = 8, kType = ELR_BF16;
  typedef bf16x8 vec;
};

template <class E>
struct Frag {
  float v[Elem<E>::VE];
};

template <class E>
__device__ __forceinline__ Frag<E> widen(u32x4 raw) {
  constexpr int N = Elem<E>::VE;
  typedef float fN __attribute__((ext_vector_type(N)));
  const fN f = __builtin_convertvector(__builtin_bit_cast(typename Elem<E>::vec, raw), fN);
  Frag<E> r;
#pragma unroll
  for (int j = 0; j < N; ++j) r.v[j] = f[j];
  return r;
}

template <class E>
__device__ __forceinline__ u32x4 narrow(const Frag<E>& a) {
  constexpr int N = Elem<E>::VE;
  typedef float fN __attribute__((ext_vector_type(N)));
  fN f;
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = a.v[j];
  return __builtin_bit_cast(u32x4, __builtin_convertvector(f, typename Elem<E>::vec));
}

// The raw vector at p of which `valid` elements (any number; <= 0: none) may be read; the others are `fill`.  NT: read
// once, not kept in the caches.
template <class E, bool NT>
__device__ __forceinline__ u32x4 load_raw(const E* p, int64_t valid, float fill) {
  constexpr int N = Elem<E>::VE;
  if (valid >= N) {
    if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4_u*>(p));
    else return *reinterpret_cast<const u32x4_u*>(p);
  }
  typename Elem<E>::vec r;
#pragma unroll
  for (int j = 0; j < N; ++j) r[j] = j < valid ? p[j] : (E)fill;
  return __builtin_bit_cast(u32x4, r);
}

template <class E, bool NT>
__device__ __forceinline__ void store_raw(E* p, u32x4 x, int64_t valid) {
  constexpr int N = Elem<E>::VE;
  if (valid >= N) {
    if constexpr (NT) __builtin_nontemporal_store((u32x4_u)x, reinterpret_cast<u32x4_u*>(p));
    else *reinterpret_cast<u32x4_u*>(p) = (u32x4_u)x;
    return;
  }
  const typename Elem<E>::vec r = __builtin_bit_cast(typename Elem<E>::vec, x);
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < valid) p[j] = r[j];
}

// The raw vector at p[e], where elements outside [0, len) are `fill` and not read (e may be negative: a row or tensor walked
// from the memory line that it starts in, so that every wave's accesses are whole lines).
template <class E, bool NT>
__device__ __forceinline__ u32x4 load_part(const E* p, int64_t e, int64_t len, float fill) {
  constexpr int N = Elem<E>::VE;
  if (e >= 0 && e + N <= len) {
    if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4_u*>(p + e));
    else return *reinterpret_cast<const u32x4_u*>(p + e);
  }
  typename Elem<E>::vec r;
#pragma unroll
  for (int j = 0; j < N; ++j) r[j] = e + j >= 0 && e + j < len ? p[e + j] : (E)fill;
  return __builtin_bit_cast(u32x4, r);
}
template <class E, bool NT>
__device__ __forceinline__ void store_part(E* p, int64_t e, int64_t len, u32x4 x) {
  constexpr int N = Elem<E>::VE;
  if (e >= 0 && e + N <= len) {
    if constexpr (NT) __builtin_nontemporal_store((u32x4_u)x, reinterpret_cast<u32x4_u*>(p + e));
    else *reinterpret_cast<u32x4_u*>(p + e) = (u32x4_u)x;
    return;
  }
  const typename Elem<E>::vec r = __builtin_bit_cast(typename Elem<E>::vec, x);
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (e + j >= 0 && e + j < len) p[e + j] = r[j];
}
// Elements between p and the line of `bytes` that it lies in.
template <class E>
__host__ __device__ inline int line_shift(const void* p, int bytes) {
  return (int)(((uintptr_t)p & (uintptr_t)(bytes - 1)) / sizeof(E));
}

// Four elements (8 bytes of a 16-bit type, 16 of fp32) at p[e], where those outside [0, len) are 0 and not read.
template <class E, bool NT>
__device__ __forceinline__ f32x4 load4(const E* p, int64_t e, int64_t len) {
  typedef E v4 __attribute__((ext_vector_type(4)));
  if (e >= 0 && e + 4 <= len) {
    if constexpr (sizeof(E) == 4) {
      const u32x4_u* q = reinterpret_cast<const u32x4_u*>(p + e);
      const u32x4 r = NT ? __builtin_nontemporal_load(q) : *q;
      return __builtin_bit_cast(f32x4, r);
    } else {
      const u32x2_u* q = reinterpret_cast<const u32x2_u*>(p + e);
      const u32x2 r = NT ? __builtin_nontemporal_load(q) : *q;
      return __builtin_convertvector(__builtin_bit_cast(v4, r), f32x4);
    }
  }
  f32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = e + j >= 0 && e + j < len ? (float)p[e + j] : 0.0f;
  return r;
}

template <class E>
__device__ __forceinline__ float to_f32(E x) { return (float)x; }

// max(a, b) that is NaN if either is (torch's amax); __builtin_fmaxf drops a NaN.
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// x of the partner lane at distance 1, 2, 4, 8 (within a row of 16 lanes, for values that are alike below that distance),
// 16 and 32, moved within the vector unit (ds_bpermute, what a shuffle is, waits for LDS at each step).
template <int CTRL>
__device__ __forceinline__ float dpp_of(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xF, 0xF, true));
}
// op over aligned groups of `width` lanes (a power of two up to 64, the same in the whole wave); every lane gets the result.
// op is commutative, so both partners compute the same bits; the order is fixed.
template <class F>
__device__ __forceinline__ float lanes_op(float x, int width, const F& op) {
  if (width > 1) x = op(x, dpp_of<0xB1>(x));     // quad_perm 1, 0, 3, 2
  if (width > 2) x = op(x, dpp_of<0x4E>(x));     // quad_perm 2, 3, 0, 1
  if (width > 4) x = op(x, dpp_of<0x141>(x));    // row_half_mirror
  if (width > 8) x = op(x, dpp_of<0x140>(x));    // row_mirror
  if (width > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if (width > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return x;
}
__device__ __forceinline__ float lanes_sum(float x, int width) {
  return lanes_op(x, width, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float lanes_max_nan(float x, int width) {
  return lanes_op(x, width, [](float a, float b) { return max_nan(a, b); });
}

// Over the whole wave with data-parallel moves within it (no LDS), the same value in every lane; fixed order.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_or(float x, float none) {   // x of the lane that CTRL names; `none` where there is none
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)__float_as_uint(none), (int)__float_as_uint(x), CTRL,
                                                               ROWS, 0xF, false));
}
__device__ __forceinline__ float last_lane(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), 63));
}
__device__ __forceinline__ float wave_sum(float x) {
  x = x + dpp_or<0x111, 0xF>(x, 0.0f);   // row_shr 1, 2, 4, 8: each row of 16 lanes into its last
  x = x + dpp_or<0x112, 0xF>(x, 0.0f);
  x = x + dpp_or<0x114, 0xF>(x, 0.0f);
  x = x + dpp_or<0x118, 0xF>(x, 0.0f);
  x = x + dpp_or<0x142, 0xA>(x, 0.0f);   // row_bcast 15 into rows 1 and 3
  x = x + dpp_or<0x143, 0xC>(x, 0.0f);   // row_bcast 31 into rows 2 and 3
  return last_lane(x);
}
__device__ __forceinline__ float wave_max(float x) {   // (a NaN is dropped)
  constexpr float none = -__builtin_inff();
  x = __builtin_fmaxf(x, dpp_or<0x111, 0xF>(x, none));
  x = __builtin_fmaxf(x, dpp_or<0x112, 0xF>(x, none));
  x = __builtin_fmaxf(x, dpp_or<0x114, 0xF>(x, none));
  x = __builtin_fmaxf(x, dpp_or<0x118, 0xF>(x, none));
  x = __builtin_fmaxf(x, dpp_or<0x142, 0xA>(x, none));
  x = __builtin_fmaxf(x, dpp_or<0x143, 0xC>(x, none));
  return last_lane(x);
}

inline int64_t elem_size(int type) { return type == ELR_F32 ? 4 : 2; }
inline bool elem_type_ok(int type) { return type == ELR_F32 || type == ELR_F16 || type == ELR_BF16; }
inline bool elem_aligned(const void* p, int type) { return ((uintptr_t)p & (uintptr_t)(elem_size(type) - 1)) == 0; }

}  // namespace elr
