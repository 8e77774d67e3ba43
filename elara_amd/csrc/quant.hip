// Rows into 8-bit integers with scales, and back (HBM-bound).  No counterpart in the reference.
//
// Over a row, or over each group of g columns (the last one shorter where g does not divide D), with a = max|x|:
//   scale = a / 127 (1 where that rounds to 0), or, pow2, the smallest power of two s with 127 s >= a, 2^-126 at least (1 for
//   a = 0);   q = x / scale, rounded once to the nearest integer, ties to even;   back: x = q scale.
// A power of two makes the way back exact in bf16 and fp32: q has 7 bits, bf16 holds 8; what a backward pass multiplies is then
// the kept value itself, in whatever order scale and value meet.  It costs up to one bit of the 7 (half a bit on average).
// A group that holds a NaN or an infinity gets scale NaN and q = 0: the values read back are NaN, never finite.
//
// Rounding.  For a power of two x / scale is exact but for underflow, which rounds to 0 either way.  Else q0 = x RN(1 / s) rounded
// is off by one at most, x - q0 s is exact in one fma (a multiple of ulp(s) / 2 of no more than s), and comparing twice it with
// s settles q: the fp32 quotient would first be rounded to a tie.  Scales below 2^-96 are lifted by 2^64 first, with x.
// The sum with 1.5 2^23 rounds to an integer, to even, and leaves it in the low byte.
//
// Layout.  Groups: a thread a vector of 16 bytes, the vectors of a group in neighbouring lanes.  Rows: a team of lanes or a block
// holds the row in registers, as the norms do; longer rows are read twice.
//
// Measured, 16,384 rows of 4,096 bf16 (201 MB either way): groups of 128 with powers of two 40.6 us (5.0 TB/s), a scale a row 35.6 (5.7),
// back 36 (5.6); with scales of max / 127 63 and 51: the quotient settled by its remainder costs ten instructions a value.  fp32
// (336 MB): 60, 53 and 60; max / 127 75 and 53.  5,001 of 1,000 fp32 7 us and back 8, of which the call and launch are about 4.
#include "elr_int8.h"

namespace elr {

struct QuantArgs {
  const void* x;
  int64_t x_ld, n;
  int32_t D, group, groups, pow2;
  int8_t* q;
  float* scale;
};

struct Int8Scale {
  float s, inv, lift;   // inv: RN(1 / (s lift)); 0 for a group that is not finite
  bool exact;           // inv is the reciprocal itself
};

__device__ __forceinline__ Int8Scale int8_scale(float amax, int pow2) {
  Int8Scale k;
  k.lift = 1.0f;
  k.exact = pow2;
  if (!(amax < __builtin_inff())) {
    k.s = __builtin_nanf("");
    k.inv = 0.0f;
    k.exact = true;
    return k;
  }
  if (pow2) {
    // amax = m 2^e, m in [1, 2): 127 2^(e - 6) >= amax unless m > 127 / 64
    const uint32_t b = __float_as_uint(amax);
    int e = (int)(b >> 23) - 6 + ((b & 0x7FFFFFu) > 0x7E0000u);     // biased exponent of the scale
    e = e < 1 ? 1 : e;
    k.s = amax > 0.0f ? __uint_as_float((uint32_t)e << 23) : 1.0f;
    k.inv = amax > 0.0f ? __uint_as_float((uint32_t)(254 - e) << 23) : 1.0f;
    return k;
  }
  k.s = amax / 127.0f;
  if (k.s == 0.0f) k.s = 1.0f;
  if (k.s < 0x1p-96f) k.lift = 0x1p64f;
  k.inv = 1.0f / (k.s * k.lift);
  return k;
}

// x / scale as an integer in the low byte of the result.
__device__ __forceinline__ uint32_t int8_of(float x, const Int8Scale& k) {
  constexpr float kMagic = 12582912.0f;    // 1.5 2^23
  if (k.exact) return k.inv == 0.0f ? 0u : __float_as_uint(x * k.inv + kMagic);
  const float s = k.s * k.lift;
  x = x * k.lift;
  float q = (x * k.inv + kMagic) - kMagic;
  const float r = __builtin_fmaf(-q, s, x), r2 = __builtin_fabsf(r) * 2.0f;
  const bool odd = __float_as_uint(q + kMagic) & 1u;
  if (r2 > s || (r2 == s && odd)) q = q + __builtin_copysignf(1.0f, r);
  q = __builtin_fminf(__builtin_fmaxf(q, -127.0f), 127.0f);    // (a subnormal scale is rounded coarsely)
  return __float_as_uint(q + kMagic);
}

template <class E>
__device__ __forceinline__ void int8_store(int8_t* p, const Frag<E>& f, const Int8Scale& k, int64_t valid) {
  constexpr int VE = Elem<E>::VE;
  typedef uint32_t u1 __attribute__((aligned(1)));
  typedef u32x2 u2 __attribute__((aligned(1)));
  uint32_t w[VE / 4];
#pragma unroll
  for (int i = 0; i < VE / 4; ++i) {
    const uint32_t a = int8_of(f.v[4 * i], k), b = int8_of(f.v[4 * i + 1], k), c = int8_of(f.v[4 * i + 2], k),
                   d = int8_of(f.v[4 * i + 3], k);
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0C0C0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000C0Cu);
    w[i] = lo | hi;
  }
  if (valid >= VE) {
    if constexpr (VE == 4) *reinterpret_cast<u1*>(p) = w[0];
    else *reinterpret_cast<u2*>(p) = u32x2{w[0], w[1]};
    return;
  }
#pragma unroll
  for (int j = 0; j < VE; ++j)
    if (j < valid) p[j] = (int8_t)(w[j / 4] >> (8 * (j & 3)));
}

template <class E>
__device__ __forceinline__ float vec_amax(const Frag<E>& f) {
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < Elem<E>::VE; ++j) m = max_nan(m, __builtin_fabsf(f.v[j]));
  return m;
}

// Groups.  A row is `slots` vectors, whole groups of them (those past the row's end hold nothing).  Rows of at most 256 vectors: as many
// as a block's threads hold, else a row takes `per_row` blocks; a block does the work of U of them, all loads first.
template <class E, int U>
__global__ __launch_bounds__(256) void k_quant_groups(QuantArgs a, int32_t slots, int32_t per_row) {
  constexpr int VE = Elem<E>::VE;
  const int gl = a.group / VE;
  int64_t row[U];
  int32_t s[U];
  u32x4 raw[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t b = blockIdx.x * U + i;
    bool live;
    if (per_row > 1) {
      row[i] = b / (uint32_t)per_row;
      s[i] = (int32_t)(b - (uint32_t)row[i] * (uint32_t)per_row) * 256 + threadIdx.x;
      live = s[i] < slots && row[i] < a.n;
    } else {
      const int32_t rows = 256 / slots, r = (int32_t)threadIdx.x / slots;
      s[i] = (int32_t)threadIdx.x - r * slots;
      row[i] = (int64_t)b * rows + r;
      live = r < rows && row[i] < a.n;
    }
    if (!live) row[i] = -1;
    raw[i] = load_raw<E, true>((const E*)a.x + (live ? row[i] * a.x_ld + s[i] * VE : 0), live ? a.D - s[i] * VE : 0, 0.0f);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const Frag<E> f = widen<E>(raw[i]);
    const Int8Scale k = int8_scale(lanes_max_nan(vec_amax<E>(f), gl), a.pow2);
    const int32_t e = s[i] * VE;
    if (row[i] < 0 || e >= a.D) continue;
    int8_store<E>(a.q + row[i] * a.D + e, f, k, a.D - e);
    if ((s[i] & (gl - 1)) == 0) a.scale[row[i] * a.groups + s[i] / gl] = k.s;
  }
}

// A scale a row: T = 64: teams of 2^lg lanes of a wave; else a block of T threads a row; NV vectors a thread.
template <class E, int T, int NV>
__global__ __launch_bounds__(T > 256 ? T : 256) void k_quant_rows(QuantArgs a, int lg) {
  constexpr int VE = Elem<E>::VE;
  __shared__ float lds[T > 64 ? T / 64 : 1];
  const int team = T > 64 ? T : 1 << lg;
  const int l = T > 64 ? (int)threadIdx.x : (int)threadIdx.x & (team - 1);
  const int64_t row = T > 64 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (256 >> lg) + (threadIdx.x >> lg);
  const bool live = row < a.n;
  const E* x = (const E*)a.x + (live ? row : 0) * a.x_ld;
  Frag<E> f[NV];
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * team + l) * VE;
    const int64_t valid = live ? a.D - e : 0;
    f[i] = widen<E>(load_raw<E, true>(x + (valid > 0 ? e : 0), valid, 0.0f));
    m = max_nan(m, vec_amax<E>(f[i]));
  }
  m = lanes_max_nan(m, team < 64 ? team : 64);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 64; ++i) m = max_nan(m, lds[i]);
  }
  const Int8Scale k = int8_scale(m, a.pow2);
  if (!live) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * team + l) * VE;
    if (e < a.D) int8_store<E>(a.q + row * a.D + e, f[i], k, a.D - e);
  }
  if (l == 0) a.scale[row] = k.s;
}

// Rows too long for a block's registers: read again for the values.
template <class E>
__global__ __launch_bounds__(1024) void k_quant_long(QuantArgs a) {
  constexpr int VE = Elem<E>::VE, T = 1024;
  __shared__ float lds[T / 64];
  const int64_t row = blockIdx.x;
  const E* x = (const E*)a.x + row * a.x_ld;
  float m = 0.0f;
  for (int64_t e = threadIdx.x * VE; e < a.D; e += T * VE)
    m = max_nan(m, vec_amax<E>(widen<E>(load_raw<E, false>(x + e, a.D - e, 0.0f))));
  m = lanes_max_nan(m, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < T / 64; ++i) m = max_nan(m, lds[i]);
  const Int8Scale k = int8_scale(m, a.pow2);
  for (int64_t e = threadIdx.x * VE; e < a.D; e += T * VE)
    int8_store<E>(a.q + row * a.D + e, widen<E>(load_raw<E, false>(x + e, a.D - e, 0.0f)), k, a.D - e);
  if (threadIdx.x == 0) a.scale[row] = k.s;
}

struct DequantArgs {
  const int8_t* q;
  int64_t q_ld, n;
  int32_t D, groups, shift;
  const float* scale;
  void* x;
};

// A thread a vector; rows of at most 256 vectors several to a block, else `per_row` blocks a row.
template <class E>
__global__ __launch_bounds__(256) void k_dequant(DequantArgs a, int32_t slots, int32_t per_row) {
  constexpr int VE = Elem<E>::VE;
  int64_t row;
  int32_t s;
  if (per_row > 1) {
    row = blockIdx.x / (uint32_t)per_row;
    s = (int32_t)(blockIdx.x - (uint32_t)row * (uint32_t)per_row) * 256 + threadIdx.x;
    if (s >= slots) return;
  } else {
    const int32_t rows = 256 / slots, r = (int32_t)threadIdx.x / slots;
    s = (int32_t)threadIdx.x - r * slots;
    row = (int64_t)blockIdx.x * rows + r;
    if (r >= rows || row >= a.n) return;
  }
  const int32_t e = s * VE;
  const Frag<E> f = int8_widen<E>(int8_load<E>(a.q + row * a.q_ld + e, a.D - e), a.scale[row * a.groups + (e >> a.shift)]);
  store_raw<E, false>((E*)a.x + row * (int64_t)a.D + e, narrow<E>(f), a.D - e);
}

// ---- host side

// Blocks of vectors that a block of k_quant_groups takes: 16,384 rows of 4,096 bf16 in groups of 128 40.6 us with 2, 41.6 with 1, 40.3
// with 4; 1,024 of 20,480 15.6 with 2 and 16.7 with 4.
constexpr int kGroupWork = 2;

// Blocks of a launch (a grid has less than 2^32 threads), and of a row of `slots` vectors in blocks of 256.
constexpr int64_t kQuantBlocks = (int64_t)1 << 23;

// Rows in launches of at most kQuantBlocks blocks: go(first row, rows, blocks, blocks of a row).
template <class F>
static void row_launches(int64_t n, int64_t slots, const F& go) {
  const int64_t per_row = (slots + 255) / 256, rows_block = slots <= 256 ? 256 / slots : 1;
  const int64_t rows_launch = slots <= 256 ? kQuantBlocks * rows_block : per_row > kQuantBlocks ? 1 : kQuantBlocks / per_row;
  for (int64_t r = 0; r < n; r += rows_launch) {
    const int64_t m = n - r < rows_launch ? n - r : rows_launch;
    go(r, m, (unsigned)(slots <= 256 ? (m + rows_block - 1) / rows_block : m * per_row), (int32_t)per_row);
  }
}

template <class E>
static void quantize(const QuantArgs& b, hipStream_t st) {
  constexpr int VE = Elem<E>::VE;
  if (b.group) {
    const int64_t slots = (int64_t)b.groups * (b.group / VE);
    row_launches(b.n, slots, [&](int64_t r, int64_t m, unsigned blocks, int32_t per_row) {
      QuantArgs a = b;
      a.x = (const E*)b.x + r * b.x_ld, a.n = m, a.q = b.q + r * b.D, a.scale = b.scale + r * b.groups;
      k_quant_groups<E, kGroupWork><<<(blocks + kGroupWork - 1) / kGroupWork, 256, 0, st>>>(a, (int32_t)slots, per_row);
    });
    return;
  }
  const int64_t nvec = (b.D + VE - 1) / VE;
  int lg = 0;
  while (lg < 6 && ((int64_t)1 << lg) < nvec) ++lg;
  const int64_t most = (int64_t)1 << 21;
  for (int64_t r = 0; r < b.n; r += most) {
    QuantArgs a = b;
    a.n = b.n - r < most ? b.n - r : most;
    a.x = (const E*)b.x + r * b.x_ld, a.q = b.q + r * b.D, a.scale = b.scale + r;
    const unsigned rows = (unsigned)a.n, teams = (unsigned)((a.n + (256 >> lg) - 1) / (256 >> lg));
    if (nvec <= 64) k_quant_rows<E, 64, 1><<<teams, 256, 0, st>>>(a, lg);
    else if (nvec <= 128) k_quant_rows<E, 64, 2><<<teams, 256, 0, st>>>(a, 6);
    else if (nvec <= 256) k_quant_rows<E, 64, 4><<<teams, 256, 0, st>>>(a, 6);
    else if (nvec <= 1024) k_quant_rows<E, 256, 4><<<rows, 256, 0, st>>>(a, 6);
    else if (nvec <= 4096) k_quant_rows<E, 1024, 4><<<rows, 1024, 0, st>>>(a, 6);
    else k_quant_long<E><<<rows, 1024, 0, st>>>(a);
  }
}

template <class E>
static void dequantize(const DequantArgs& b, hipStream_t st) {
  const int64_t slots = (b.D + Elem<E>::VE - 1) / Elem<E>::VE;
  row_launches(b.n, slots, [&](int64_t r, int64_t m, unsigned blocks, int32_t per_row) {
    DequantArgs a = b;
    a.q = b.q + r * b.q_ld, a.n = m, a.scale = b.scale + r * b.groups, a.x = (E*)b.x + r * b.D;
    k_dequant<E><<<blocks, 256, 0, st>>>(a, (int32_t)slots, per_row);
  });
}

constexpr int64_t kQuantColumns = (int64_t)1 << 28;

}  // namespace elr

extern "C" int elr_quantize_int8(const void* x, int type, int64_t n, int64_t D, int64_t x_ld, int64_t group, int pow2, int8_t* q,
                                 float* scale, void* stream) {
  using namespace elr;
  if (n < 0 || D < 1 || x_ld < 0 || group < 0 || !elem_type_ok(type)) return ELR_EINVAL;
  if (!int8_group_ok(group) || D > kQuantColumns) return ELR_EUNSUPPORTED;
  if (n == 0) return ELR_OK;
  if (!x || !q || !scale || !elem_aligned(x, type) || ((uintptr_t)scale & 3u)) return ELR_EINVAL;
  const QuantArgs a{x, x_ld, n, (int32_t)D, (int32_t)group, (int32_t)int8_groups(D, group), pow2 != 0, q, scale};
  hipStream_t st = (hipStream_t)stream;
  if (type == ELR_F32) quantize<float>(a, st);
  else if (type == ELR_F16) quantize<_Float16>(a, st);
  else quantize<__bf16>(a, st);
  return launch_status();
}

extern "C" int elr_dequantize_int8(const int8_t* q, int64_t n, int64_t D, int64_t q_ld, int64_t group, const float* scale, void* x,
                                   int type, void* stream) {
  using namespace elr;
  if (n < 0 || D < 1 || q_ld < 0 || group < 0 || !elem_type_ok(type)) return ELR_EINVAL;
  if (!int8_group_ok(group) || D > kQuantColumns) return ELR_EUNSUPPORTED;
  if (n == 0) return ELR_OK;
  if (!x || !q || !scale || !elem_aligned(x, type) || ((uintptr_t)scale & 3u)) return ELR_EINVAL;
  const DequantArgs a{q, q_ld, n, (int32_t)D, (int32_t)int8_groups(D, group), int8_shift(group), scale, x};
  hipStream_t st = (hipStream_t)stream;
  if (type == ELR_F32) dequantize<float>(a, st);
  else if (type == ELR_F16) dequantize<_Float16>(a, st);
  else dequantize<__bf16>(a, st);
  return launch_status();
}
