// Root-mean-square norm with the residual's addition, output in the input's type or in fp8 (e4m3) with scales, and its
// backward (HBM-bound).  No counterpart in the reference.
//
// A row of D elements:  h = x + r;  c = 1 / sqrt(sum h^2 / D + eps);  y = h c w.
// fp8: over the row, or over each group of columns, scale = max|y| / 448 (1 where that rounds to 0) and q = e4m3(y / scale), round
// to nearest even; 448 is the largest finite e4m3 value.
// Backward, of y's gradient dy and the gradient dh that arrives on the residual stream, with u = w dy and xh = h c:
//   dx = c (u - xh sum(u xh) / D) + dh  (x's and r's alike);   dw = sum over the rows of dy xh.
//
// The norm is taken of the unrounded fp32 sum h; h itself is rounded once, when it is stored.  Sums are fp32.
//
// Layout.  A row lies in the registers of a team: 2^lg lanes of one wave (rows of up to 64 vectors of 16 bytes: several rows
// a wave), a wave, or a block, NV vectors a lane; vector j * team + lane.  It is read once and written once.  Rows too long
// for a block's registers (k_norm_long) are read again from the caches for the output.
//
// Loads are non-temporal (read once; plain ones 3 to 14 % slower on 537 MB).  16,384 rows of 4,096 bf16 with a residual (537
// MB) take 84 us (6.4 TB/s); their backward 85 us and 5 for the sum of the weight gradients (6.0 TB/s); that of 425,984 rows
// of 128 fp32 (656 MB) 109 and 5 (5.8 TB/s).  fp8 of 8,192 rows of 2,048 with groups of 128 (118 MB): 24 us (4.9 TB/s, of
// which a launch is 3 us); of 16,384 rows of 4,096 with a scale a row (470 MB) 82 us (5.8 TB/s).  An fp32 residual stream
// under bf16: 16,384 of 1,024 40 us forward (5.0 TB/s) and 51 backward (4.6), of 4,096 206 (3.9) and 243 (3.9).  bf16 rows of
// 20,480 (2,048 of them) 66 us (5.1 TB/s), and 245 backward (1.4), which reads such rows twice; of 100,000 (1,024), read twice
// either way, 256 (3.2) and 630 (1.3).  The backward from h kept in 8 bits (q s, a scale a row or for each group of columns, widened as
// it is loaded): 16,384 of 4,096 bf16 with groups of 128 and dh (472 MB) 77 us and 4 for the weight's sum (5.8 TB/s), 2,048 of 256 6.7
// and 3.5; of 20,480 (2,048 of them, with dh) 245, of 100,000 (1,024) 643 (1.1-1.2 TB/s, read twice).
#include "elr_int8.h"

#include <type_traits>

namespace elr {

constexpr float kFp8Max = 448.0f;

struct NormArgs {
  const void *x, *r, *w;       // r: residual or NULL; w: weight or NULL
  int64_t x_ld, r_ld;
  int64_t n;
  int32_t D, group;            // group: columns of a scale (0: the row)
  int w_f32;                   // the weight's type: 1 fp32, 0 the input's
  float eps;
  void *y, *h;                 // y: input's type, or e4m3 bytes; h: residual's type, NULL without a residual
  float *rstd, *scale;
  int nt;                      // 16-byte stores past the caches
};

// Weight elements [e, e + VE) as fp32 (1 without a weight).
template <class E>
__device__ __forceinline__ Frag<E> weight_at(const void* w, int w_f32, int64_t e, int64_t valid) {
  constexpr int VE = Elem<E>::VE;
  Frag<E> f;
  if (!w) {
#pragma unroll
    for (int j = 0; j < VE; ++j) f.v[j] = 1.0f;
  } else if (w_f32) {
    const float* p = (const float*)w + e;
#pragma unroll
    for (int q = 0; q < VE / 4; ++q) {
      const Frag<float> a = widen<float>(load_raw<float, false>(p + 4 * q, valid - 4 * q, 0.0f));
#pragma unroll
      for (int j = 0; j < 4; ++j) f.v[4 * q + j] = a.v[j];
    }
  } else {
    f = widen<E>(load_raw<E, false>((const E*)w + e, valid, 0.0f));
  }
  return f;
}

// Outputs that the last-level cache (256 MB) could not keep anyway are stored past it; smaller ones stay for what reads them
// next.  16,384 rows of 4,096 bf16 with a residual (268 MB out): 84 us against 89; their backward (134 MB out): 94 past the
// cache, 90 into it; 425,984 rows of 128 fp32, backward (218 MB out): 114 and 121.
constexpr int64_t kKeepBytes = (int64_t)192 << 20;
template <class E>
__device__ __forceinline__ void store_out(E* p, u32x4 x, int64_t valid, int nt) {
  if (nt) store_raw<E, true>(p, x, valid);
  else store_raw<E, false>(p, x, valid);
}

// VE fp32 or 16-bit residual elements at the same places as an input vector of type E.
template <class E, class R>
struct ResRaw {
  static constexpr int N = Elem<E>::VE / Elem<R>::VE;   // 1, or 2 for an fp32 residual of a 16-bit input
  u32x4 v[N];
};
template <class E, class R>
__device__ __forceinline__ ResRaw<E, R> res_load(const R* p, int64_t valid) {
  ResRaw<E, R> a;
#pragma unroll
  for (int q = 0; q < ResRaw<E, R>::N; ++q)
    a.v[q] = load_raw<R, true>(p + q * Elem<R>::VE, valid - q * Elem<R>::VE, 0.0f);
  return a;
}
template <class E, class R>
__device__ __forceinline__ Frag<E> res_widen(const ResRaw<E, R>& a) {
  Frag<E> f;
#pragma unroll
  for (int q = 0; q < ResRaw<E, R>::N; ++q) {
    const Frag<R> b = widen<R>(a.v[q]);
#pragma unroll
    for (int j = 0; j < Elem<R>::VE; ++j) f.v[q * Elem<R>::VE + j] = b.v[j];
  }
  return f;
}
template <class E, class R>
__device__ __forceinline__ void res_store(R* p, const Frag<E>& f, int64_t valid, int nt) {
#pragma unroll
  for (int q = 0; q < ResRaw<E, R>::N; ++q) {
    Frag<R> b;
#pragma unroll
    for (int j = 0; j < Elem<R>::VE; ++j) b.v[j] = f.v[q * Elem<R>::VE + j];
    store_out<R>(p + q * Elem<R>::VE, narrow<R>(b), valid - q * Elem<R>::VE, nt);
  }
}

// The scale of values up to m, and what divides by it.  The quotient is the correctly rounded one: q = y RN(1 / s) is within
// two ulps, its residual q s - y is exact in one fma, and a second fma takes it off (Markstein's theorem, for a correctly
// rounded reciprocal).  A product with the reciprocal alone takes values at e4m3's ties to the wrong side.  8,192 rows of 2,048
// take 24 us either way, and 27 with a division for each value.  A scale below 2^-80, whose residuals could underflow, and one
// that is infinite or NaN, divides.
struct Scale {
  float s, inv;
  bool exact;
};
constexpr float kLeastScale = 0x1.0p-80f;
__device__ __forceinline__ Scale scale_of(float m) {
  Scale r;
  r.s = m / kFp8Max;
  if (r.s == 0.0f) r.s = 1.0f;     // nothing but zeros, or values whose scale rounds to 0 (up to 3.1e-43)
  r.inv = 1.0f / r.s;
  r.exact = !(r.s >= kLeastScale && r.s < __builtin_inff());
  return r;
}
template <class E>
__device__ __forceinline__ void divide(Frag<E>& h, const Scale& k) {
  if (k.exact) {
#pragma unroll
    for (int j = 0; j < Elem<E>::VE; ++j) h.v[j] = h.v[j] / k.s;
  } else {
#pragma unroll
    for (int j = 0; j < Elem<E>::VE; ++j) {
      const float q = h.v[j] * k.inv;
      h.v[j] = __builtin_fmaf(-__builtin_fmaf(q, k.s, -h.v[j]), k.inv, q);   // (the signs keep -0)
    }
  }
}

// e4m3 of VE values already divided by their scale, at p.  The clamp takes what rounding may put above 448.
template <class E>
__device__ __forceinline__ void store_fp8(uint8_t* p, const Frag<E>& f, int64_t valid) {
  constexpr int VE = Elem<E>::VE;
  uint32_t q[VE / 4];
#pragma unroll
  for (int i = 0; i < VE / 4; ++i) {
    float c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c[j] = __builtin_elementwise_minimum(__builtin_elementwise_maximum(f.v[4 * i + j], -kFp8Max), kFp8Max);
    int b = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    q[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], b, true);
  }
  // (rows of an odd number of bytes: the store takes any address)
  typedef uint32_t u32x2_b __attribute__((ext_vector_type(2), aligned(1)));
  typedef uint32_t u32_b __attribute__((aligned(1)));
  if (valid >= VE) {
    if constexpr (VE == 8) __builtin_nontemporal_store((u32x2_b){q[0], q[1]}, (u32x2_b*)p);
    else *(u32_b*)p = q[0];
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j)
      if (j < valid) p[j] = (uint8_t)(q[j / 4] >> (8 * (j & 3)));
  }
}

// Sum (or NaN-keeping maximum) over a team: 2^lg lanes, or (T > 64) the whole block through LDS, T / 64 floats that no
// thread may still be reading from an earlier call.
template <int T>
__device__ __forceinline__ float team_sum(float x, int lg, float* lds) {
  x = lanes_sum(x, 1 << lg);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) x = x + lds[w];
  }
  return x;
}
template <int T>
__device__ __forceinline__ float team_max(float x, int lg, float* lds) {
  x = lanes_max_nan(x, 1 << lg);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) x = max_nan(x, lds[w]);
  }
  return x;
}

__device__ __forceinline__ float rstd_of(float sum, float D, float eps) { return 1.0f / sqrt_rn(sum / D + eps); }

// T = 64: blocks of four waves, each of 64 >> lg rows; else a block of T threads a row (lg = 6).
template <class E, class R, bool FP8, int T, int NV>
__global__ __launch_bounds__(T > 256 ? T : 256) void k_norm(NormArgs a, int lg) {
  constexpr int VE = Elem<E>::VE;
  __shared__ float lds[2][T > 64 ? T / 64 : 1];
  const int lane = threadIdx.x & 63;
  const int team = T > 64 ? T : 1 << lg;
  const int l = T > 64 ? (int)threadIdx.x : lane & (team - 1);
  const int64_t row = T > 64 ? (int64_t)blockIdx.x
                             : (((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) << (6 - lg)) + (lane >> lg);
  const bool live = row < a.n;
  if (T > 64 && !live) return;
  const int64_t at = live ? row : 0;      // (lanes of a row past the end take part in the shuffles)
  const E* x = (const E*)a.x + at * a.x_ld;
  u32x4 raw[NV];
  ResRaw<E, R> res[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * team + l) * VE;
    raw[i] = load_raw<E, true>(x + e, live ? a.D - e : 0, 0.0f);
  }
  if (a.r) {
    const R* r = (const R*)a.r + at * a.r_ld;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * team + l) * VE;
      res[i] = res_load<E, R>(r + e, live ? a.D - e : 0);
    }
  }
  Frag<E> h[NV];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    h[i] = widen<E>(raw[i]);
    if (a.r) {
      const Frag<E> q = res_widen<E, R>(res[i]);
#pragma unroll
      for (int j = 0; j < VE; ++j) h[i].v[j] = h[i].v[j] + q.v[j];
      const int e = (i * team + l) * VE;
      res_store<E, R>((R*)a.h + at * a.D + e, h[i], live ? a.D - e : 0, a.nt);
    }
#pragma unroll
    for (int j = 0; j < VE; ++j) ss = __builtin_fmaf(h[i].v[j], h[i].v[j], ss);
  }
  ss = team_sum<T>(ss, lg, lds[0]);
  const float c = rstd_of(ss, (float)a.D, a.eps);
  if (l == 0 && live) a.rstd[row] = c;
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * team + l) * VE;
    // (loaded with the row the weight costs 2 % more: 86 us for 84)
    const Frag<E> w = weight_at<E>(a.w, a.w_f32, e, a.D - e);
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      h[i].v[j] = h[i].v[j] * c * w.v[j];
      if (FP8 && e + j < a.D) amax = max_nan(amax, __builtin_fabsf(h[i].v[j]));
    }
    if constexpr (FP8) {
      if (a.group) {       // a group is an aligned run of lanes
        const int gl = a.group / VE;
        const float m = lanes_max_nan(amax, gl);
        const Scale k = scale_of(m);
        if (live && e < a.D) {
          if ((lane & (gl - 1)) == 0) a.scale[row * (a.D / a.group) + e / a.group] = k.s;
          divide<E>(h[i], k);
          store_fp8<E>((uint8_t*)a.y + row * a.D + e, h[i], a.D - e);
        }
        amax = 0.0f;
      }
    } else {
      store_out<E>((E*)a.y + at * a.D + e, narrow<E>(h[i]), live ? a.D - e : 0, a.nt);
    }
  }
  if constexpr (FP8) {
    if (a.group) return;
    amax = team_max<T>(amax, lg, lds[1]);
    const Scale k = scale_of(amax);
    if (l == 0 && live) a.scale[row] = k.s;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * team + l) * VE;
      divide<E>(h[i], k);
      store_fp8<E>((uint8_t*)a.y + at * a.D + e, h[i], live ? a.D - e : 0);
    }
  }
}

// Rows longer than a block's registers: the sum of squares in one pass, the output in another (and, in fp8 without
// groups, the maximum in one between), from x and r again.
template <class E, class R, bool FP8>
__global__ __launch_bounds__(256) void k_norm_long(NormArgs a) {
  constexpr int VE = Elem<E>::VE, T = 256;
  __shared__ float lds[2][T > 64 ? T / 64 : 1];
  const int64_t row = blockIdx.x;
  const E* x = (const E*)a.x + row * a.x_ld;
  const R* r = (const R*)a.r + row * a.r_ld;
  auto load = [&](int64_t e) {
    Frag<E> h = widen<E>(load_raw<E, false>(x + e, a.D - e, 0.0f));
    if (a.r) {
      ResRaw<E, R> q;
#pragma unroll
      for (int i = 0; i < ResRaw<E, R>::N; ++i)
        q.v[i] = load_raw<R, false>(r + e + i * Elem<R>::VE, a.D - e - i * Elem<R>::VE, 0.0f);
      const Frag<E> f = res_widen<E, R>(q);
#pragma unroll
      for (int j = 0; j < VE; ++j) h.v[j] = h.v[j] + f.v[j];
    }
    return h;
  };
  float ss = 0.0f;
  for (int64_t e = threadIdx.x * VE; e < a.D; e += T * VE) {
    const Frag<E> h = load(e);
#pragma unroll
    for (int j = 0; j < VE; ++j) ss = __builtin_fmaf(h.v[j], h.v[j], ss);
  }
  ss = team_sum<T>(ss, 6, lds[0]);
  const float c = rstd_of(ss, (float)a.D, a.eps);
  if (threadIdx.x == 0) a.rstd[row] = c;
  auto norm = [&](int64_t e) {
    Frag<E> h = load(e);
    const Frag<E> w = weight_at<E>(a.w, a.w_f32, e, a.D - e);
#pragma unroll
    for (int j = 0; j < VE; ++j) h.v[j] = h.v[j] * c * w.v[j];
    return h;
  };
  Scale k{1.0f, 1.0f, false};
  if constexpr (FP8) {
    if (!a.group) {
      float m = 0.0f;
      for (int64_t e = threadIdx.x * VE; e < a.D; e += T * VE) {
        const Frag<E> h = norm(e);
#pragma unroll
        for (int j = 0; j < VE; ++j)
          if (e + j < a.D) m = max_nan(m, __builtin_fabsf(h.v[j]));
      }
      m = team_max<T>(m, 6, lds[1]);
      k = scale_of(m);
      if (threadIdx.x == 0) a.scale[row] = k.s;
    }
  }
  const int64_t end = (a.D + T * VE - 1) / (T * VE) * (T * VE);    // whole blocks: the groups' shuffles
  for (int64_t e = threadIdx.x * VE; e < end; e += T * VE) {
    const int64_t valid = a.D - e;
    Frag<E> h = norm(e < a.D ? e : 0);
    if constexpr (FP8) {
      if (a.group) {
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < VE; ++j) m = max_nan(m, __builtin_fabsf(h.v[j]));
        const int gl = a.group / VE;
        m = lanes_max_nan(m, gl);
        k = scale_of(m);
        if (e < a.D && (threadIdx.x & (gl - 1)) == 0) a.scale[row * (a.D / a.group) + e / a.group] = k.s;
      }
      divide<E>(h, k);
      store_fp8<E>((uint8_t*)a.y + row * a.D + e, h, valid);
    } else {
      store_out<E>((E*)a.y + row * a.D + e, narrow<E>(h), valid, a.nt);
    }
    if (a.r) {
      const Frag<E> f = load(e < a.D ? e : 0);
      res_store<E, R>((R*)a.h + row * a.D + e, f, valid, a.nt);
    }
  }
}

struct NormBackArgs {
  const void *dy, *h, *dh, *w;    // dh: gradient on the residual stream, or NULL
  int64_t dy_ld, h_ld, dh_ld;
  const float* rstd;
  int64_t n;
  int32_t D;
  int w_f32;
  void* dx;                       // h's type, contiguous
  float* part;                    // [gridDim.x][D] weight gradient of each block's rows, or NULL
  int nt;
  const float* h_scale;           // int8 h: fp32 [n, groups], a scale for each 2^shift columns
  int32_t groups, shift;
};

// A vector of h: of the residual's type, or int8 with its scale (a vector lies within one group).
template <class E, class R, class H>
struct HRaw {
  ResRaw<E, R> v;
};
template <class E, class R>
struct HRaw<E, R, int8_t> {
  Int8Raw<E> q;
  float s;
};
template <class E, class R, class H>
__device__ __forceinline__ HRaw<E, R, H> h_load(const NormBackArgs& a, int64_t row, int64_t e, int64_t valid) {
  HRaw<E, R, H> r;
  if constexpr (sizeof(H) == 1) {
    r.q = int8_load<E>((const int8_t*)a.h + row * a.h_ld + e, valid);
    r.s = valid > 0 ? a.h_scale[row * a.groups + (e >> a.shift)] : 0.0f;
  } else {
    r.v = res_load<E, R>((const R*)a.h + row * a.h_ld + e, valid);
  }
  return r;
}
template <class E, class R, class H>
__device__ __forceinline__ Frag<E> h_widen(const HRaw<E, R, H>& r) {
  if constexpr (sizeof(H) == 1) return int8_widen<E>(r.q, r.s);
  else return res_widen<E, R>(r.v);
}

// E: dy's and the weight's type; R: dh's and dx's; H: h's, R or int8_t.  Each team walks U rows at a time, `teams` apart.  (With the next rows'
// loads in flight: 425,984 rows of 128 fp32 114 us either way, 16,384 of 4,096 bf16 95 us against 89.)  Its weight gradient
// stays in registers until the end, then the block's teams are added in a fixed order.
template <class E, class R, class H, int T, int NV, int U>
__global__ __launch_bounds__(T > 256 ? T : 256) void k_norm_back(NormBackArgs a, int lg) {
  constexpr int VE = Elem<E>::VE;
  extern __shared__ float dwsum[];     // [D], only with a.part
  __shared__ float lds[2][T > 64 ? T / 64 : 1];
  const int lane = threadIdx.x & 63;
  const int team = T > 64 ? T : 1 << lg;
  const int l = T > 64 ? (int)threadIdx.x : lane & (team - 1);
  const int64_t first = T > 64 ? (int64_t)blockIdx.x
                               : (((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) << (6 - lg)) + (lane >> lg);
  const int64_t teams = T > 64 ? (int64_t)gridDim.x : ((int64_t)gridDim.x * 4) << (6 - lg);
  const int64_t base = T > 64 ? first : first - (lane >> lg);     // the wave's first row: a wave's lanes loop alike
  const float inv_d = 1.0f / (float)a.D;
  Frag<E> w[NV], dw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * team + l) * VE;
    w[i] = weight_at<E>(a.w, a.w_f32, e, a.D - e);
#pragma unroll
    for (int j = 0; j < VE; ++j) dw[i].v[j] = 0.0f;
  }
  struct Rows {
    u32x4 dy[U][NV];
    HRaw<E, R, H> h[U][NV];
    ResRaw<E, R> dh[U][NV];
    float c[U];
  };
  const auto load = [&](Rows& x, int64_t b) {
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int64_t row = b + (first - base) + q * teams;
      const bool live = row < a.n;
      const int64_t at = live ? row : 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (i * team + l) * VE;
        const int valid = live ? a.D - e : 0;
        x.dy[q][i] = load_raw<E, true>((const E*)a.dy + at * a.dy_ld + e, valid, 0.0f);
        x.h[q][i] = h_load<E, R, H>(a, at, e, valid);
        if (a.dh) x.dh[q][i] = res_load<E, R>((const R*)a.dh + at * a.dh_ld + e, valid);
      }
      x.c[q] = live ? a.rstd[at] : 0.0f;
    }
  };
  int turn = 0;       // rows alternate between two places in LDS: one barrier a row
  const auto compute = [&](const Rows& x, int64_t b) {
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int64_t row = b + (first - base) + q * teams;
      const bool live = row < a.n;
      float dot = 0.0f;
      Frag<E> u[NV], xh[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        u[i] = widen<E>(x.dy[q][i]);
        xh[i] = h_widen<E, R, H>(x.h[q][i]);
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          xh[i].v[j] = xh[i].v[j] * x.c[q];
          dw[i].v[j] = __builtin_fmaf(u[i].v[j], xh[i].v[j], dw[i].v[j]);
          u[i].v[j] = u[i].v[j] * w[i].v[j];
          dot = __builtin_fmaf(u[i].v[j], xh[i].v[j], dot);
        }
      }
      dot = team_sum<T>(dot, lg, lds[turn]) * inv_d;
      turn ^= 1;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (i * team + l) * VE;
        Frag<E> f;
        if (a.dh) {
          f = res_widen<E, R>(x.dh[q][i]);
        } else {
#pragma unroll
          for (int j = 0; j < VE; ++j) f.v[j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < VE; ++j)
          f.v[j] = __builtin_fmaf(x.c[q], __builtin_fmaf(-xh[i].v[j], dot, u[i].v[j]), f.v[j]);
        res_store<E, R>((R*)a.dx + (live ? row : 0) * a.D + e, f, live ? a.D - e : 0, a.nt);
      }
    }
  };
  for (int64_t b = base; b < a.n; b += teams * U) {
    Rows x;
    load(x, b);
    compute(x, b);
  }
  if (!a.part) return;
  if constexpr (T == 64) {
    // teams of a wave, then the four waves one after another
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VE; ++j)
        for (int o = 1 << lg; o < 64; o <<= 1) dw[i].v[j] = dw[i].v[j] + __shfl_xor(dw[i].v[j], o, 64);
    for (int wv = 0; wv < 4; ++wv) {
      if ((int)(threadIdx.x >> 6) == wv && lane < team) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int e = (i * team + l) * VE;
#pragma unroll
          for (int j = 0; j < VE; ++j)
            if (e + j < a.D) dwsum[e + j] = wv == 0 ? dw[i].v[j] : dwsum[e + j] + dw[i].v[j];
        }
      }
      __syncthreads();
    }
    for (int e = threadIdx.x; e < a.D; e += 256) a.part[(int64_t)blockIdx.x * a.D + e] = dwsum[e];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * team + l) * VE;
#pragma unroll
      for (int j = 0; j < VE; ++j)
        if (e + j < a.D) a.part[(int64_t)blockIdx.x * a.D + e + j] = dw[i].v[j];
    }
  }
}

// Long rows: one block a row at a time, dx in a second pass; the weight gradient of a block's rows is accumulated in its
// own row of `part` (each element by one thread).
template <class E, class R, class H>
__global__ __launch_bounds__(256) void k_norm_back_long(NormBackArgs a) {
  constexpr int VE = Elem<E>::VE, T = 256;
  __shared__ float lds[2][T > 64 ? T / 64 : 1];
  const float inv_d = 1.0f / (float)a.D;
  float* part = a.part ? a.part + (int64_t)blockIdx.x * a.D : nullptr;
  bool fresh = true;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const E* dy = (const E*)a.dy + row * a.dy_ld;
    const R* dh = (const R*)a.dh + row * a.dh_ld;
    const float c = a.rstd[row];
    float dot = 0.0f;
    for (int64_t e = threadIdx.x * VE; e < a.D; e += T * VE) {
      const Frag<E> y = widen<E>(load_raw<E, false>(dy + e, a.D - e, 0.0f));
      const Frag<E> q = h_widen<E, R, H>(h_load<E, R, H>(a, row, e, a.D - e));
      const Frag<E> w = weight_at<E>(a.w, a.w_f32, e, a.D - e);
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float xh = q.v[j] * c;
        dot = __builtin_fmaf(y.v[j] * w.v[j], xh, dot);
        if (part && e + j < a.D) part[e + j] = __builtin_fmaf(y.v[j], xh, fresh ? 0.0f : part[e + j]);
      }
    }
    fresh = false;
    dot = team_sum<T>(dot, 6, lds[turn]) * inv_d;
    turn ^= 1;
    for (int64_t e = threadIdx.x * VE; e < a.D; e += T * VE) {
      const Frag<E> y = widen<E>(load_raw<E, false>(dy + e, a.D - e, 0.0f));
      const Frag<E> q = h_widen<E, R, H>(h_load<E, R, H>(a, row, e, a.D - e));
      const Frag<E> w = weight_at<E>(a.w, a.w_f32, e, a.D - e);
      Frag<E> f;
#pragma unroll
      for (int j = 0; j < VE; ++j) f.v[j] = 0.0f;
      if (a.dh) f = res_widen<E, R>(res_load<E, R>(dh + e, a.D - e));
#pragma unroll
      for (int j = 0; j < VE; ++j)
        f.v[j] = __builtin_fmaf(c, __builtin_fmaf(-(q.v[j] * c), dot, y.v[j] * w.v[j]), f.v[j]);
      res_store<E, R>((R*)a.dx + row * a.D + e, f, a.D - e, a.nt);
    }
  }
}

// dw[e] = sum over the blocks' partial rows, D apart, in a fixed order: 32 columns a block, 32 threads a column, each every 32nd
// row.
__global__ __launch_bounds__(1024) void k_norm_dw(const float* part, int rows, int32_t D, int32_t cols, float* dw) {
  __shared__ float s[32][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t e = (int64_t)blockIdx.x * 32 + c;
  float x = 0.0f;
  if (e < cols)
#pragma unroll 8
    for (int r = g; r < rows; r += 32) x = x + part[(int64_t)r * D + e];
  s[g][c] = x;
  __syncthreads();
  if (g == 0 && e < cols) {
    float t = s[0][c];
#pragma unroll
    for (int i = 1; i < 32; ++i) t = t + s[i][c];
    dw[e] = t;
  }
}

// ---- host side

// The team of a row of `nvec` vectors: 2^lg lanes (T = 64), or a block of T threads, of NV vectors each.  As many threads as
// vectors as far as a block goes (rows of 4,096 bf16: 512 threads of one vector 84 us, 256 of two 88, a wave of eight 93; of
// 2,048: 25 us against 28 for a wave of four).  NV = 0: the long kernels.
struct Team {
  int lg, T, NV;
};
static Team team_of(int64_t nvec, int most_nv) {
  int lg = 0;
  while (lg < 6 && ((int64_t)1 << lg) < nvec) ++lg;
  if (nvec <= 64) return {lg, 64, 1};
  if (nvec <= 128) return {6, 64, 2};
  if (nvec <= 256) return {6, 256, 1};
  if (nvec <= 512) return {6, 512, 1};
  if (nvec <= 1024) return {6, 1024, 1};
  if (nvec <= 2048) return {6, 1024, 2};
  if (nvec <= 4096 && most_nv >= 4) return {6, 1024, 4};
  return {6, 0, 0};
}

template <class E, class R, bool FP8>
static void launch_norm(const NormArgs& a, hipStream_t st) {
  const Team t = team_of((a.D + Elem<E>::VE - 1) / Elem<E>::VE, 4);
  const unsigned rows = (unsigned)a.n;
  const unsigned waves = (unsigned)(((a.n + (64 >> t.lg) - 1) / (64 >> t.lg) + 3) / 4);
  switch (t.T * 8 + t.NV) {
    case 64 * 8 + 1: k_norm<E, R, FP8, 64, 1><<<waves, 256, 0, st>>>(a, t.lg); break;
    case 64 * 8 + 2: k_norm<E, R, FP8, 64, 2><<<waves, 256, 0, st>>>(a, 6); break;
    case 256 * 8 + 1: k_norm<E, R, FP8, 256, 1><<<rows, 256, 0, st>>>(a, 6); break;
    case 512 * 8 + 1: k_norm<E, R, FP8, 512, 1><<<rows, 512, 0, st>>>(a, 6); break;
    case 1024 * 8 + 1: k_norm<E, R, FP8, 1024, 1><<<rows, 1024, 0, st>>>(a, 6); break;
    case 1024 * 8 + 2: k_norm<E, R, FP8, 1024, 2><<<rows, 1024, 0, st>>>(a, 6); break;
    case 1024 * 8 + 4: k_norm<E, R, FP8, 1024, 4><<<rows, 1024, 0, st>>>(a, 6); break;
    default: k_norm_long<E, R, FP8><<<rows, 256, 0, st>>>(a); break;
  }
}

constexpr int64_t kNormRowsPerLaunch = 1 << 21;   // (a grid has less than 2^32 threads)
constexpr int64_t kDwColumns = 1 << 26;

template <class E, class R>
static void norm_rows(NormArgs a, bool fp8, hipStream_t st) {
  const NormArgs b = a;
  for (int64_t r = 0; r < b.n; r += kNormRowsPerLaunch) {
    a.n = b.n - r < kNormRowsPerLaunch ? b.n - r : kNormRowsPerLaunch;
    a.x = (const E*)b.x + r * b.x_ld;
    if (b.r) a.r = (const R*)b.r + r * b.r_ld, a.h = (R*)b.h + r * b.D;
    a.y = (char*)b.y + r * b.D * (fp8 ? 1 : (int64_t)sizeof(E));
    a.rstd = b.rstd + r;
    if (fp8) {
      a.scale = b.scale + r * (b.group ? b.D / b.group : 1);
      launch_norm<E, R, true>(a, st);
    } else {
      launch_norm<E, R, false>(a, st);
    }
  }
}

// Blocks of the backward: enough to fill the chip, few enough that the partial weight gradients (written and read once, D
// fp32 a block) stay a small part of the rows' traffic.  bf16 but where said: a block of 1,024 threads fills a CU (4,000 rows
// of 8,192: 53 us with 256 blocks, 59 with 512; 8,192 of 5,120 69 and 75; 4,000 of 4,096 fp32 47 either way).  Blocks of 256,
// four a CU: 12,094 of 1,536 38 us with 1,024 blocks, 46 with 512, though 16,384 of 2,048 take 54 and 52, 5,000 of 1,024 fp32
// 21 and 20.  Two rows a block where they are few (822 of 1,000 fp16 12.5 us, 14.0 with one; 200 of 4,096 9.2 and 10.3), and
// one block, which needs no addition of partial sums, for what up to three would do (30 of 64 fp32 6.0 us, 8.2 with two; 3 of
// 4,096 6.1 and 8.5).
constexpr int64_t kBackBlocks = 512, kBackBlocksMost = 1024, kBackFew = 32, kBackOne = 3;
static int64_t back_blocks(int64_t n, int64_t D, int type) {
  const Team t = team_of((D + 16 / elem_size(type) - 1) / (16 / elem_size(type)), 2);
  const int64_t per = t.T == 64 ? 4 << (6 - t.lg) : 1;
  int64_t most = kBackBlocks;
  if (t.T == 1024) most = 256;
  else if (t.T == 256) most = kBackBlocksMost;
  else if (t.T == 64) most = n / 64 < most ? most : n / 64 < kBackBlocksMost ? n / 64 : kBackBlocksMost;
  int64_t b = (n + per - 1) / per;
  if (b > kBackFew) b = (b + 1) / 2;
  if (b <= kBackOne) b = 1;
  return b < most ? b : most;
}

template <class E, class R, class H>
static void launch_norm_back(const NormBackArgs& a, unsigned blocks, hipStream_t st) {
  const Team t = team_of((a.D + Elem<E>::VE - 1) / Elem<E>::VE, 2);
  const size_t lds = a.part ? (size_t)a.D * 4 : 0;
  switch (t.T * 8 + t.NV) {
    case 64 * 8 + 1: k_norm_back<E, R, H, 64, 1, 1><<<blocks, 256, lds, st>>>(a, t.lg); break;
    case 64 * 8 + 2: k_norm_back<E, R, H, 64, 2, 2><<<blocks, 256, lds, st>>>(a, 6); break;
    case 256 * 8 + 1: k_norm_back<E, R, H, 256, 1, 2><<<blocks, 256, 0, st>>>(a, 6); break;
    case 512 * 8 + 1: k_norm_back<E, R, H, 512, 1, 1><<<blocks, 512, 0, st>>>(a, 6); break;
    case 1024 * 8 + 1: k_norm_back<E, R, H, 1024, 1, 1><<<blocks, 1024, 0, st>>>(a, 6); break;
    case 1024 * 8 + 2:
      if constexpr (sizeof(E) == sizeof(R)) {
        k_norm_back<E, R, H, 1024, 2, 1><<<blocks, 1024, 0, st>>>(a, 6);
        break;
      }
      [[fallthrough]];   // (its registers would spill)
    default: k_norm_back_long<E, R, H><<<blocks, 256, 0, st>>>(a); break;
  }
}

// The backward behind both entry points, for checked rows: Q8 for h in int8, else of dx's type.
template <bool Q8>
static int norm_back(NormBackArgs a, int type, int x_type, float* dweight, void* scratch, int64_t scratch_bytes,
                     hipStream_t st) {
  const int64_t n = a.n, D = a.D;
  if (n == 0 && !dweight) return ELR_OK;
  const int64_t blocks = back_blocks(n, D, type);
  if (dweight && n > 0 && (!scratch || scratch_bytes < blocks * D * 4 || ((uintptr_t)scratch & 3u))) return ELR_ECAPACITY;
  a.part = !dweight ? nullptr : blocks == 1 ? dweight : (float*)scratch;
  a.nt = n * D * elem_size(x_type) > kKeepBytes;
  if (n > 0) {
    const auto go = [&](auto e, auto r) {
      typedef decltype(e) E;
      typedef decltype(r) R;
      launch_norm_back<E, R, typename std::conditional<Q8, int8_t, R>::type>(a, (unsigned)blocks, st);
    };
    const bool wide = x_type == ELR_F32;
    switch (type) {
      case ELR_F32: go(float(), float()); break;
      case ELR_F16: wide ? go(_Float16(), float()) : go(_Float16(), _Float16()); break;
      default: wide ? go(__bf16(), float()) : go(__bf16(), __bf16()); break;
    }
  }
  if (dweight && (n == 0 || blocks > 1)) {   // no rows: zeros
    for (int64_t e = 0; e < D; e += kDwColumns) {
      const int64_t m = D - e < kDwColumns ? D - e : kDwColumns;
      k_norm_dw<<<(unsigned)((m + 31) / 32), 1024, 0, st>>>(n > 0 ? (const float*)scratch + e : nullptr,
                                                           n > 0 ? (int)blocks : 0, (int32_t)D, (int32_t)m, dweight + e);
    }
  }
  return launch_status();
}

static int check_norm(int64_t n, int64_t D, int type, int res_type, int w_type) {
  if (n < 0 || D < 1 || !elem_type_ok(type) || !elem_type_ok(res_type) || !elem_type_ok(w_type)) return ELR_EINVAL;
  if (res_type != type && res_type != ELR_F32) return ELR_EUNSUPPORTED;
  if (w_type != type && w_type != ELR_F32) return ELR_EUNSUPPORTED;
  if (D > (int64_t)1 << 28) return ELR_EUNSUPPORTED;
  return ELR_OK;
}

}  // namespace elr

extern "C" int elr_rms_norm(const void* x, int type, int64_t n, int64_t D, int64_t x_ld, const void* residual,
                            int res_type, int64_t res_ld, const void* weight, int w_type, float eps, void* y, int fp8,
                            int64_t group, float* scale, void* h, float* rstd, void* stream) {
  using namespace elr;
  if (int rc = check_norm(n, D, type, res_type, w_type)) return rc;
  if (x_ld < 0 || res_ld < 0 || group < 0) return ELR_EINVAL;
  if (group && (!fp8 || D % group)) return ELR_EINVAL;
  if (group && group != 32 && group != 64 && group != 128 && group != 256) return ELR_EUNSUPPORTED;
  if (n == 0) return ELR_OK;
  if (!x || !y || !rstd || (residual && !h) || (fp8 && !scale)) return ELR_EINVAL;
  if (!elem_aligned(x, type) || !elem_aligned(residual, res_type) || !elem_aligned(h, res_type) ||
      !elem_aligned(weight, w_type) || (!fp8 && !elem_aligned(y, type)))
    return ELR_EINVAL;
  const NormArgs a{x, residual, weight, x_ld, res_ld, n, (int32_t)D, (int32_t)group, w_type == ELR_F32, eps,
                   y, h, rstd, scale,
                   n * D * ((fp8 ? 1 : elem_size(type)) + (residual ? elem_size(res_type) : 0)) > kKeepBytes};
  hipStream_t st = (hipStream_t)stream;
  const bool q = fp8 != 0, wide = residual && res_type == ELR_F32;
  switch (type) {
    case ELR_F32: norm_rows<float, float>(a, q, st); break;
    case ELR_F16: wide ? norm_rows<_Float16, float>(a, q, st) : norm_rows<_Float16, _Float16>(a, q, st); break;
    default: wide ? norm_rows<__bf16, float>(a, q, st) : norm_rows<__bf16, __bf16>(a, q, st); break;
  }
  return launch_status();
}

extern "C" int64_t elr_rms_norm_backward_scratch_bytes(int64_t n, int64_t D, int type) {
  if (n < 0 || D < 1 || !elr::elem_type_ok(type)) return -1;
  return elr::back_blocks(n, D, type) * D * 4;
}

extern "C" int elr_rms_norm_backward(const void* dy, int type, int64_t n, int64_t D, int64_t dy_ld, const void* h,
                                     int h_type, int64_t h_ld, const void* dh, int64_t dh_ld, const void* weight,
                                     int w_type, const float* rstd, void* dx, float* dweight, void* scratch,
                                     int64_t scratch_bytes, void* stream) {
  using namespace elr;
  if (int rc = check_norm(n, D, type, h_type, w_type)) return rc;
  if (dy_ld < 0 || h_ld < 0 || dh_ld < 0) return ELR_EINVAL;
  if (n > 0) {
    if (!dy || !h || !rstd || !dx) return ELR_EINVAL;
    if (!elem_aligned(dy, type) || !elem_aligned(h, h_type) || !elem_aligned(dh, h_type) || !elem_aligned(dx, h_type) ||
        !elem_aligned(weight, w_type))
      return ELR_EINVAL;
  }
  const NormBackArgs a{dy, h, dh, weight, dy_ld, h_ld, dh_ld, rstd, n, (int32_t)D, w_type == ELR_F32, dx,
                       nullptr, 0, nullptr, 1, 31};
  return norm_back<false>(a, type, h_type, dweight, scratch, scratch_bytes, (hipStream_t)stream);
}

extern "C" int elr_rms_norm_backward_int8(const void* dy, int type, int64_t n, int64_t D, int64_t dy_ld, const int8_t* h,
                                          int64_t h_ld, int64_t group, const float* h_scale, const void* dh, int x_type,
                                          int64_t dh_ld, const void* weight, int w_type, const float* rstd, void* dx,
                                          float* dweight, void* scratch, int64_t scratch_bytes, void* stream) {
  using namespace elr;
  if (int rc = check_norm(n, D, type, x_type, w_type)) return rc;
  if (dy_ld < 0 || h_ld < 0 || dh_ld < 0 || group < 0) return ELR_EINVAL;
  if (!int8_group_ok(group)) return ELR_EUNSUPPORTED;
  if (n > 0) {
    if (!dy || !h || !h_scale || !rstd || !dx) return ELR_EINVAL;
    if (!elem_aligned(dy, type) || !elem_aligned(dh, x_type) || !elem_aligned(dx, x_type) || !elem_aligned(weight, w_type) ||
        ((uintptr_t)h_scale & 3u))
      return ELR_EINVAL;
  }
  const NormBackArgs a{dy, h, dh, weight, dy_ld, h_ld, dh_ld, rstd, n, (int32_t)D, w_type == ELR_F32, dx,
                       nullptr, 0, h_scale, (int32_t)int8_groups(D, group), int8_shift(group)};
  return norm_back<true>(a, type, x_type, dweight, scratch, scratch_bytes, (hipStream_t)stream);
}
