// A token for each row of logits, drawn by temperature, top-k, top-p and min-p from a given uniform number, and its log probability in
// the distribution that it was drawn from.  No counterpart in the reference.
//
// A row x of V logits with maximum m, temperature T and a number u in [0, 1):
//   e_v = exp((x_v - m) / T);   order: larger x first, ties by the lower id (-0 equal to +0);
//   kept: the first top_k of the order; of these, those before whose place in the order the mass of e is less than top_p of the k's
//   mass (the first always); of these, those with e_v >= min_p;
//   token = the first kept id, in the order of ids, at which the sum of e over the kept ids exceeds u S, S their whole mass;
//   logprob = log(e_token / S).   T = 0: the first of the order, logprob 0.
//
// Exactness.  With one uniform number a row the draw is a search in a cumulative sum, and an error of 2^-24 of the mass moves it across
// a border in one of a few hundred rows of 100,000 ids.  So the weights are integers: e in fp64, times 2^s and rounded to 64 bits, with
// V 2^s < 2^63 and s at most 51.  Their sums are exact in any order (atomics and splits included), and the same for every launch shape; what
// is below 2^-(s + 1) of the largest has no weight (2^-46 at 131,072 ids).
//
// A row is a block's: read once for its maximum and, in registers or by the maxima of its steps, for the few elements that can matter.
// top_k of up to 192 (48 for a wave's short rows): the k-th largest of 256 threads' maxima bounds the k-th largest element from below;
// min_p: its own value.  What reaches the bound, a few dozen to a few hundred elements, is ranked pairwise in LDS with the mass before
// each, and the draw is a sum over the smaller ids.  Other rows: counts and masses by bins of distance from the maximum, the bin that the
// target falls into ranked the same way (or, where too many elements lie in it, a selection by digits of the key), then partial sums
// of the kept weights in the order of ids.
//
// Measured (bf16 but where said; the floor is the row read once at 5.3 TB/s).  4,096 rows of 32,768 (51 us): T = 0 51, top_k 50 88-98,
// with top_p 0.9 too 87-93, min_p 0.05 119-132, no restriction 156-180, top_k 1,000 260-273, top_p 0.9 alone 360-405, settings by row 178.  301 of
// 50,021 fp32 (11): none 47.  1,024 of 100,003 fp32 (77): T = 0 81, top_k 50 101, none 190.  1 of 131,072: T = 0 9, top_k 50 17-18, none 42,
// top_p alone 106-110: one CU's work.  8,192 of 1,000 (3): 14, 39, none 25.  What bounds them: T = 0 memory; a bound's rows the
// chain of barriers behind the reading, about 10 us a row on a CU with four at once; the others about 25 instructions of fp64 an
// element and pass, two passes of it with top_p, and LDS atomics for the bins.
#include "elr_elem.h"

namespace elr {

typedef unsigned long long u64;

// What a block of T threads keeps in LDS.  (A wave by itself works on rows of up to 2,048 elements: LDS bounds how many run at once.)
template <int T>
struct Shape {
  static constexpr int kSegs = T > 64 ? 512 : 64;      // partial sums of a row in the order of ids
  static constexpr int kDigit = T > 64 ? 11 : 8;       // bits of a selection pass
  static constexpr int kList = T > 64 ? 512 : 256;     // candidates that are ranked among themselves
  static constexpr int kBins = T > 64 ? 1024 : 256;    // bins of a row by distance from its maximum, up to 2^-32 in e
};
constexpr int kWeightBits = 51;      // of the largest weight

struct SampleArgs {
  const void* x;
  int64_t ld, n;
  int32_t V, shift;                  // weights are e 2^shift
  int32_t per_seg;                   // steps of a wave (64 vectors) in a segment
  const float* u;
  double temperature, top_p, min_p;  // where the pointers are NULL
  int64_t top_k;
  const float *temperature_rows, *top_p_rows, *min_p_rows;
  const void* top_k_rows;
  int top_k_64;
  int64_t* token;
  float* logprob;
};

// An unsigned order of the values of a type in kKeyBits bits: larger value, larger key; -0 as +0.  (NaN rows are refused before.)
template <class E>
constexpr int kKeyBits = Elem<E>::kType == ELR_F32 ? 32 : Elem<E>::kType == ELR_BF16 ? 16 : 19;
template <class E>
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return ((b & 0x80000000u) ? ~b : (b | 0x80000000u)) >> (32 - kKeyBits<E>);
}
__device__ __forceinline__ uint32_t order_of_value(float x) {      // (of fp32: the next value is the next number)
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of_order(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
template <class E>
__device__ __forceinline__ float value_of_key(uint32_t key) {
  constexpr int kDrop = 32 - kKeyBits<E>;
  const uint32_t o = key << kDrop;
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o >> kDrop << kDrop);
}

// a b + c with c in scalar registers (left to itself the compiler copies each constant into vector registers and overwrites the copy).
__device__ __forceinline__ double fma_const(double a, double b, double c) {
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
}

// 2^(z + shift) for z <= 0, rounded to an integer below 2^52.  2^f, |f| <= 1/2, by the polynomial through the ten Chebyshev points
// (within 3.8e-14 of the value, 2^-44.6, at the ends); the sum with 1.5 2^52 rounds z, the one with 2^52 the result.  About 20 instructions of fp64, which runs at
// the rate of fp32 here; a NaN (0 times infinity: an infinite temperature) counts as no weight.
__device__ __forceinline__ u64 weight_of(double z, int shift) {
  constexpr double kRound = 0x1.8p52;
  z = __builtin_fmax(z, -200.0);
  const double t = z + kRound, f = z - (t - kRound);
  const int n = (int)(uint32_t)__builtin_bit_cast(uint64_t, t);
  double p = 0x1.b6571d9fbc782p-24;
  p = fma_const(p, f, 0x1.63ef9699f65f0p-20);
  p = fma_const(p, f, 0x1.ffcb7678dfe12p-17);
  p = fma_const(p, f, 0x1.43088e257f900p-13);
  p = fma_const(p, f, 0x1.5d87fe908f6f7p-10);
  p = fma_const(p, f, 0x1.3b2ab72b175e9p-7);
  p = fma_const(p, f, 0x1.c6b08d704411ap-5);
  p = fma_const(p, f, 0x1.ebfbdff8149f2p-3);
  p = fma_const(p, f, 0x1.62e42fefa39f7p-1);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_bit_cast(uint64_t, __builtin_ldexp(p, n + shift) + 0x1p52) & 0xFFFFFFFFFFFFFu;
}

struct Candidate {
  u64 at;        // key in the high half, ~id in the low: larger comes first
  u64 w;
};
template <int T>
struct SampleShared {
  static constexpr int kSegs = Shape<T>::kSegs, kDigit = Shape<T>::kDigit, kList = Shape<T>::kList, kBins = Shape<T>::kBins;
  union {
    struct {
      uint32_t count[1 << kDigit];
      u64 mass[1 << kDigit];
    } radix;
    struct {
      u64 mass[kBins];
      uint32_t count[kBins];
      Candidate list[kList];
    } bins;
    float step_max[kSegs];      // of a wave's vectors at a time (before the bins are filled)
  };
  u64 seg[kSegs];
  float fmax[16];
  u64 sums[16];
  uint32_t bin, bin_count, listed, bound;
  u64 above, bin_mass, total, rest;
  uint32_t id, thr_id;
  float thr;
  int seg_at;
};

__device__ __forceinline__ u64 wave_sum_u64(u64 x) {
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}
// Inclusive sums over the lanes.
__device__ __forceinline__ u64 wave_scan_u64(u64 x, int lane) {
  for (int o = 1; o < 64; o <<= 1) {
    const u64 y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  return x;
}

// One row by a block of T threads.  NV > 0: the row's vectors of a thread stay in registers for the search of candidates; the passes that
// some rows need beyond it read the row again (from the caches).
template <class E, int T, int NV>
__global__ __launch_bounds__(T, T == 256 ? 4 : 1) void k_sample(SampleArgs a) {
  constexpr int VE = Elem<E>::VE, W = T / 64;
  constexpr int kSegs = Shape<T>::kSegs, kDigit = Shape<T>::kDigit, kList = Shape<T>::kList, kBins = Shape<T>::kBins;
  __shared__ SampleShared<T> sh;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const E* x = (const E*)a.x + row * a.ld;
  constexpr float kNone = -__builtin_inff();
  const int nseg = (int)(((int64_t)a.V + (int64_t)64 * VE * a.per_seg - 1) / ((int64_t)64 * VE * a.per_seg));
  // The vector from id e on, and its values: unconditional loads (a branch around a load ends in a wait for it).  The row's last vector, and
  // those past it, are the last VE elements, of which those before e count as -inf: no candidates, without weight.
  constexpr bool kTiny = T == 64 && NV == 1;         // rows of less than a vector come here
  const auto base = [&](int32_t e) { return e < a.V - VE ? e : a.V - VE < 0 ? 0 : a.V - VE; };
  const auto load = [&](int32_t e) -> u32x4 {
    if constexpr (kTiny)
      if (a.V < VE) return load_raw<E, false>(x, e == 0 ? a.V : 0, kNone);
    return *reinterpret_cast<const u32x4_u*>(x + base(e));
  };
  const auto values = [&](u32x4 r, int32_t e) {
    Frag<E> f = widen<E>(r);
    if (__builtin_amdgcn_readfirstlane(e - lane * VE) + 64 * VE > a.V) {      // (lanes hold neighbouring vectors)
      const int32_t b = base(e);
#pragma unroll
      for (int j = 0; j < VE; ++j)
        if (b + j < e) f.v[j] = kNone;
    }
    return f;
  };
  // f(segment, first id, VE values) over the wave's vectors; the segments are in the order of ids.
  const auto each = [&](const auto& f) {
    int s = wave, j = 0;
    if (s >= nseg) return;
    int32_t e = (s * a.per_seg * 64 + lane) * VE;
    u32x4 next = load(e);
    while (s < nseg) {                 // (the next vector on its way)
      const u32x4 now = next;
      const int seg = s;
      const int32_t at = e;
      if (++j == a.per_seg) j = 0, s += W;
      e = ((s * a.per_seg + j) * 64 + lane) * VE;
      next = load(e);                  // (past the row: its end again)
      f(seg, base(at), values(now, at));
    }
  };
  // the row's maximum (NaN or +inf in the row show in it), and the thread's
  [[maybe_unused]] u32x4 raw[NV > 0 ? NV : 1];
  [[maybe_unused]] float vec_max[NV > 0 ? NV : 1], own_max = kNone;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      raw[i] = load((i * T + threadIdx.x) * VE);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Frag<E> f = values(raw[i], (i * T + threadIdx.x) * VE);
      vec_max[i] = f.v[0];
#pragma unroll
      for (int j = 1; j < VE; ++j) vec_max[i] = max_nan(vec_max[i], f.v[j]);
      asm volatile("" : "+v"(vec_max[i]));    // (taken here: put off, all vectors' values would take the registers)
      own_max = max_nan(own_max, vec_max[i]);
    }
  } else {
    for (int s = wave; s * 64 * VE < a.V;) {          // eight vectors on their way
      u32x4 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = load(((s + i * W) * 64 + lane) * VE);
#pragma unroll
      for (int i = 0; i < 8; ++i, s += W) {
        const Frag<E> f = values(v[i], (s * 64 + lane) * VE);
        float vm = f.v[0];
#pragma unroll
        for (int j = 1; j < VE; ++j) vm = max_nan(vm, f.v[j]);
        own_max = max_nan(own_max, vm);
        vm = lanes_max_nan(vm, 64);
        if (lane == 0 && s < kSegs) sh.step_max[s] = vm;
      }
    }
  }
  float m = lanes_max_nan(own_max, 64);
  if constexpr (T > 64) {
    if (lane == 0) sh.fmax[wave] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) m = max_nan(m, sh.fmax[i]);
  }
  const double temp = a.temperature_rows ? (double)a.temperature_rows[row] : a.temperature;
  const double top_p = a.top_p_rows ? (double)a.top_p_rows[row] : a.top_p;
  const double min_p = a.min_p_rows ? (double)a.min_p_rows[row] : a.min_p;
  const double u = (double)a.u[row];
  if (!(m < __builtin_inff()) || !(temp >= 0.0) || u != u || m == kNone) {
    if (threadIdx.x == 0) {
      a.token[row] = -1;
      a.logprob[row] = m == kNone && temp >= 0.0 && u == u ? kNone : __builtin_nanf("");
    }
    return;
  }
  const bool greedy = temp == 0.0;
  int64_t top_k = !a.top_k_rows ? a.top_k
                  : a.top_k_64 ? ((const int64_t*)a.top_k_rows)[row] : ((const int32_t*)a.top_k_rows)[row];
  if (greedy) top_k = 1;
  const bool by_k = top_k > 0 && top_k < a.V, by_p = !greedy && top_p < 1.0;
  // (1 / T at most 2^1000: already there any smaller value has no weight, and the maximum's own difference times it stays 0)
  const double inv_t = greedy ? 0.0 : __builtin_fmin(1.0 / temp, 0x1p1000), per_e = inv_t * 0x1.71547652b82fep+0;      // to powers of two
  const auto weight = [&](float v) -> u64 { return weight_of(((double)v - (double)m) * per_e, a.shift); };
  const double low = greedy || !(min_p > 0.0) ? -__builtin_inf() : log(min_p < 1.0 ? min_p : 1.0) * temp;
  // the smallest value that min_p lets through: m itself at most
  float low_v = kNone;
  if (low > -__builtin_inf()) {
    low_v = (float)((double)m + low);
    const auto step = [](float v, int by) { return value_of_order(order_of_value(v) + by); };
    for (int i = 0; i < 4 && (double)low_v - (double)m < low; ++i) low_v = step(low_v, 1);
    for (int i = 0; i < 4 && !((double)step(low_v, -1) - (double)m < low); ++i) low_v = step(low_v, -1);
    low_v = low_v < m ? low_v : m;
  }
  const auto near = [&](float v) { return v >= low_v; };
  float thr = kNone;                           // kept: a larger value, or this value and no larger id
  uint32_t thr_id = 0xFFFFFFFFu;
  const auto in_order = [&](float v, uint32_t id) { return (v > thr) | ((v == thr) & (id <= thr_id)); };

  // The sum of one value a thread; every thread gets it.
  const auto block_sum = [&](u64 v) {
    v = wave_sum_u64(v);
    if constexpr (T == 64) return v;
    __syncthreads();
    if (lane == 0) sh.sums[wave] = v;
    __syncthreads();
    u64 all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) all += sh.sums[i];
    return all;
  };
  const auto share = [](double part, u64 all) {      // the least whole mass that reaches the part of `all`
    const u64 t = (u64)__builtin_ceil((part > 0.0 ? part : 0.0) * (double)all);
    return t < 1 ? (u64)1 : t > all ? all : t;
  };
  const auto place = [&](u64 all) {                  // u of `all`, below it
    const u64 t = u > 0.0 ? (u64)__builtin_floor(u * (double)all) : 0;
    return t < all ? t : all - 1;
  };
  const auto answer = [&](uint32_t id, float v, u64 all) {
    a.token[row] = id;
    a.logprob[row] = greedy ? 0.0f
                            : (float)(((double)v - (double)m) * inv_t - log((double)all * __builtin_ldexp(1.0, -a.shift)));
  };

  // The elements for which f(value, id) holds into the list, in any order; their number (more than kList: not all of them are there).
  const auto take = [&](float v, uint32_t id) {
    const uint32_t at = atomicAdd(&sh.listed, 1u);
    if (at < kList) sh.bins.list[at].at = (u64)key_of<E>(v) << 32 | (uint32_t)~id;
  };
  const auto list_begin = [&] {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
  };
  const auto list_end = [&]() -> int {
    __syncthreads();
    const int n = (int)(sh.listed < kList ? sh.listed : kList + 1);
    if (n <= kList)
      for (int i = threadIdx.x; i < n; i += T) sh.bins.list[i].w = weight(value_of_key<E>((uint32_t)(sh.bins.list[i].at >> 32)));
    __syncthreads();
    return n;
  };
  constexpr int kOwn = (kList + T - 1) / T;          // of the list, a thread's
  // Places in the order and mass before each of a thread's candidates, among the list's.
  const auto rank = [&](int n, uint32_t (&before)[kOwn], u64 (&mass)[kOwn]) {
    u64 at[kOwn];
#pragma unroll
    for (int q = 0; q < kOwn; ++q) {
      at[q] = (int)threadIdx.x + q * T < n ? sh.bins.list[threadIdx.x + q * T].at : ~0ull;
      before[q] = 0, mass[q] = 0;
    }
    for (int j = 0; j < n; ++j) {
      const Candidate c = sh.bins.list[j];
#pragma unroll
      for (int q = 0; q < kOwn; ++q)
        if (kOwn == 1 || q * T < n) {
          before[q] += c.at > at[q];
          mass[q] += c.at > at[q] ? c.w : 0;
        }
    }
  };

  // ---- rows whose candidates a bound leaves few of: the k-th largest of 256 threads' maxima (a lower bound of the k-th largest
  // element), or the smallest value that min_p lets through
  const bool few = by_k && top_k <= (T >= 256 ? 192 : 48);
  if (few || (low > -__builtin_inf() && !(by_k && by_p))) {
    float bound = kNone;
    if (few) {
      constexpr int N = T >= 256 ? 4 : 1;            // maxima a lane of the first wave looks at
      constexpr int G = T > 256 ? T / 256 : 1;       // threads of one
      float g = own_max;
      if constexpr (G > 1) g = lanes_max_nan(g, G);
      uint32_t* const maxima = (uint32_t*)sh.seg;
      if (threadIdx.x % G == 0) maxima[threadIdx.x / G] = key_of<E>(g);
      __syncthreads();
      if (wave == 0) {
        uint32_t o[N], t = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = maxima[i * 64 + lane];
#pragma unroll
        for (int b = kKeyBits<E> - 1; b >= 0; --b) {
          const uint32_t c = t | 1u << b;
          int n = 0;
#pragma unroll
          for (int i = 0; i < N; ++i) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(o[i] >= c));
          if (n >= (int)top_k) t = c;
        }
        if (lane == 0) sh.bound = t;
      }
      __syncthreads();
      bound = value_of_key<E>(sh.bound);
    }
    // (a row that top_p cuts without top_k needs min_p's candidates alone, but the mass of all)
    u64 all = 0;
    if (by_p && !by_k) {
      each([&](int, int, const Frag<E>& v) {
#pragma unroll
        for (int j = 0; j < VE; ++j) all += weight(v.v[j]);
      });
      all = block_sum(all);
    }
    list_begin();
    if (!few) bound = low_v;
    const auto looked = [&](float v, uint32_t id) {
      if ((v >= bound) & (v > kNone)) take(v, id);
    };
    if constexpr (NV > 0) {
      int32_t tid = threadIdx.x;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (vec_max[i] >= bound) {
          asm("" : "+v"(raw[i]), "+v"(tid));      // (widened again: what the first pass made would take the registers)
          const int32_t e = (i * T + tid) * VE;
          const Frag<E> f = values(raw[i], e);
#pragma unroll
          for (int j = 0; j < VE; ++j) looked(f.v[j], (uint32_t)(base(e) + j));
        }
      }
    } else {
      for (int s = wave; s * 64 * VE < a.V; s += W)    // (the steps whose maximum reaches the bound are read again)
        if (s >= kSegs || sh.step_max[s] >= bound) {
          const int32_t e = (s * 64 + lane) * VE;
          const Frag<E> f = values(load(e), e);
#pragma unroll
          for (int j = 0; j < VE; ++j) looked(f.v[j], (uint32_t)(base(e) + j));
        }
    }
    const int n = list_end();
    if (n <= kList) {
      uint32_t before[kOwn];
      u64 mass[kOwn], w[kOwn], at[kOwn];
      rank(n, before, mass);
      u64 sum = 0;
#pragma unroll
      for (int q = 0; q < kOwn; ++q) {
        const int i = threadIdx.x + q * T;
        at[q] = i < n ? sh.bins.list[i].at : 0, w[q] = i < n ? sh.bins.list[i].w : 0;
        if (i >= n || (by_k && before[q] >= (uint64_t)top_k)) before[q] = 0xFFFFFFFFu, w[q] = 0;
        sum += w[q];
      }
      if (by_p) {
        const u64 target = share(top_p, by_k ? block_sum(sum) : all);
        sum = 0;
#pragma unroll
        for (int q = 0; q < kOwn; ++q) {
          if (mass[q] >= target) w[q] = 0;
          sum += w[q];
        }
      }
      if (low > -__builtin_inf()) {
        sum = 0;
#pragma unroll
        for (int q = 0; q < kOwn; ++q) {
          if (!near(value_of_key<E>((uint32_t)(at[q] >> 32)))) w[q] = 0;
          sum += w[q];
        }
      }
      sum = block_sum(sum);
      __syncthreads();
#pragma unroll
      for (int q = 0; q < kOwn; ++q)
        if ((int)threadIdx.x + q * T < n) sh.bins.list[threadIdx.x + q * T].w = w[q];
      __syncthreads();
      const u64 t = place(sum);
      u64 upto[kOwn];
#pragma unroll
      for (int q = 0; q < kOwn; ++q) upto[q] = 0;
      for (int j = 0; j < n; ++j) {
        const Candidate c = sh.bins.list[j];
#pragma unroll
        for (int q = 0; q < kOwn; ++q)
          if (kOwn == 1 || q * T < n) upto[q] += (uint32_t)c.at > (uint32_t)at[q] ? c.w : 0;      // (a smaller id)
      }
#pragma unroll
      for (int q = 0; q < kOwn; ++q)
        if (w[q] > 0 && upto[q] <= t && t - upto[q] < w[q]) answer(~(uint32_t)at[q], value_of_key<E>((uint32_t)(at[q] >> 32)), sum);
      return;
    }
  }

  // ---- the other rows
  // The first id at which the running sum of f over the ids exceeds t (t below the whole sum); sh.total holds the whole sum, from which
  // t_of makes t.
  const auto locate = [&](const auto& f, const auto& t_of) {
    __syncthreads();
    for (int i = threadIdx.x; i < kSegs; i += T) sh.seg[i] = 0;
    if (threadIdx.x == 0) sh.seg_at = 0, sh.id = 0, sh.rest = 0;
    __syncthreads();
    u64 acc = 0;
    int at = -1;
    each([&](int s, int e, const Frag<E>& v) {
      if (s != at && at >= 0) {
        const u64 r = wave_sum_u64(acc);
        if (lane == 0) sh.seg[at] = r;
        acc = 0;
      }
      at = s;
#pragma unroll
      for (int j = 0; j < VE; ++j) acc += f(v.v[j], (uint32_t)(e + j));
    });
    if (at >= 0) {
      const u64 r = wave_sum_u64(acc);
      if (lane == 0) sh.seg[at] = r;
    }
    __syncthreads();
    if (wave == 0) {
      constexpr int N = kSegs / 64;
      u64 own = 0;
      for (int i = 0; i < N; ++i) own += sh.seg[lane * N + i];
      const u64 upto = wave_scan_u64(own, lane), all = __shfl(upto, 63, 64);
      if (lane == 0) sh.total = all;
      const u64 t = t_of(all);
      if (upto > t && upto - own <= t) {
        u64 before = upto - own;
        int s = lane * N;
        while (before + sh.seg[s] <= t) before += sh.seg[s++];
        sh.seg_at = s;
        sh.rest = t - before;
      }
    }
    __syncthreads();
    const int s = sh.seg_at;
    if (wave == 0) {
      u64 rest = sh.rest;
      for (int j = 0; j < a.per_seg; ++j) {
        int32_t e = ((s * a.per_seg + j) * 64 + lane) * VE;
        const Frag<E> v = values(load(e), e);
        e = base(e);
        u64 own = 0, w[VE];
#pragma unroll
        for (int q = 0; q < VE; ++q) {
          w[q] = f(v.v[q], (uint32_t)(e + q));
          own += w[q];
        }
        const u64 upto = wave_scan_u64(own, lane), all = __shfl(upto, 63, 64);
        if (rest < all) {
          if (upto > rest && upto - own <= rest) {
            u64 before = upto - own;
            int q = 0;
#pragma unroll
            for (int i = 0; i < VE - 1; ++i)
              if (q == i && before + w[i] <= rest) before += w[i], q = i + 1;
            sh.id = (uint32_t)(e + q);
          }
          break;
        }
        rest -= all;
      }
    }
    __syncthreads();
    const uint32_t id = sh.id;
    __syncthreads();      // (the next call clears it)
    return id;
  };

  // The threshold (thr, thr_id) at which the order, from its largest on and within the present threshold, has reached `target`: places,
  // or mass.  By digits of the key, whatever the row holds.
  const auto search = [&](bool by_mass, u64 target) {
    uint32_t prefix = 0;
    u64 above = 0;
    int bits = kKeyBits<E>;
    while (bits > 0) {
      const int take_bits = bits < kDigit ? bits : kDigit, shift = bits - take_bits;
      __syncthreads();
      for (int i = threadIdx.x; i < 1 << kDigit; i += T) sh.radix.count[i] = 0, sh.radix.mass[i] = 0;
      __syncthreads();
      each([&](int, int e, const Frag<E>& v) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const uint32_t key = key_of<E>(v.v[j]);
          if ((bits == kKeyBits<E> || key >> bits == prefix) && in_order(v.v[j], (uint32_t)(e + j))) {
            const uint32_t d = key >> shift & ((1u << take_bits) - 1);
            atomicAdd(&sh.radix.count[d], 1u);
            if (by_mass) atomicAdd(&sh.radix.mass[d], weight(v.v[j]));
          }
        }
      });
      __syncthreads();
      if (wave == 0) {      // lane 0 the largest digits
        constexpr int N = (1 << kDigit) / 64;
        u64 own = 0;
        for (int i = 0; i < N; ++i) {
          const int d = (1 << kDigit) - 1 - (lane * N + i);
          own += by_mass ? sh.radix.mass[d] : sh.radix.count[d];
        }
        const u64 upto = wave_scan_u64(own, lane) + above;
        if (upto >= target && upto - own < target) {
          u64 before = upto - own;
          for (int i = 0; i < N; ++i) {
            const int d = (1 << kDigit) - 1 - (lane * N + i);
            const u64 v = by_mass ? sh.radix.mass[d] : sh.radix.count[d];
            if (before + v >= target) {
              sh.bin = (uint32_t)d, sh.bin_count = sh.radix.count[d], sh.bin_mass = v, sh.above = before;
              break;
            }
            before += v;
          }
        }
      }
      __syncthreads();
      prefix = prefix << take_bits | sh.bin;
      above = sh.above;
      bits = shift;
    }
    // ties at the threshold: the first `need` of them by id
    const u64 of = sh.bin_mass, n_ties = sh.bin_count;
    const u64 each_w = by_mass ? of / n_ties : 1;
    const u64 need = (target - above + each_w - 1) / each_w;
    const float at = value_of_key<E>(prefix);
    uint32_t id = 0xFFFFFFFFu;
    if (need < n_ties)
      id = locate([&](float v, uint32_t i) -> u64 { return (v == at) & in_order(v, i); }, [&](u64) { return need - 1; });
    else if (at == thr) id = thr_id;
    thr = at, thr_id = id;
  };

  // Counts and masses by bins of distance from the maximum; then the bin in which places or mass reach a target, and the threshold from
  // that bin's elements alone, ranked among themselves.
  const float to_bin = (float)(per_e * -(kBins / 32));
  const auto bin_of = [&](float v) {
    const float d = (v - m) * to_bin;
    return d < (float)kBins ? (int)d : kBins - 1;      // (a NaN, of an infinite temperature: the last)
  };
  const auto bins = [&](bool with_mass) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += T) sh.bins.count[i] = 0, sh.bins.mass[i] = 0;
    __syncthreads();
    each([&](int, int, const Frag<E>& v) {
#pragma unroll
      for (int j = 0; j < VE; ++j)
        if (v.v[j] > kNone) {
          const int b = bin_of(v.v[j]);
          if (by_k) atomicAdd(&sh.bins.count[b], 1u);
          if (with_mass) {
            const u64 w = weight(v.v[j]);
            if (w) atomicAdd(&sh.bins.mass[b], w);
          }
        }
    });
    __syncthreads();
  };
  // False where too many elements lie in the bin.  A target beyond all there is leaves the threshold.
  u64 kept_mass = 0;                               // of the present threshold
  const auto refine = [&](bool by_mass, u64 target) -> bool {
    if (wave == 0) {
      constexpr int N = kBins / 64;
      u64 own = 0, own_mass = 0;
      for (int i = 0; i < N; ++i) own += by_mass ? sh.bins.mass[lane * N + i] : sh.bins.count[lane * N + i];
      for (int i = 0; i < N; ++i) own_mass += sh.bins.mass[lane * N + i];
      const u64 upto = wave_scan_u64(own, lane), upto_mass = wave_scan_u64(own_mass, lane);
      if (lane == 63) sh.bin = kBins, sh.bin_mass = upto_mass;
      if (upto >= target && upto - own < target) {
        u64 before = upto - own, mass = upto_mass - own_mass;
        for (int i = 0; i < N; ++i) {
          const int b = lane * N + i;
          const u64 v = by_mass ? sh.bins.mass[b] : sh.bins.count[b];
          if (before + v >= target) {
            sh.bin = (uint32_t)b, sh.above = before, sh.bin_mass = mass;
            break;
          }
          before += v, mass += sh.bins.mass[b];
        }
      }
    }
    __syncthreads();
    const int b = (int)sh.bin;
    const u64 above = sh.above, above_mass = sh.bin_mass;
    if (b == kBins) {
      __syncthreads();      // (the next call writes what every wave has just read; the way below has barriers of its own)
      kept_mass = above_mass;
      return true;
    }
    list_begin();
    each([&](int, int e, const Frag<E>& v) {
#pragma unroll
      for (int j = 0; j < VE; ++j)
        if ((v.v[j] > kNone) & (bin_of(v.v[j]) == b) & in_order(v.v[j], (uint32_t)(e + j))) take(v.v[j], (uint32_t)(e + j));
    });
    const int n = list_end();
    if (n > kList) return false;
    uint32_t before[kOwn];
    u64 mass[kOwn], part = 0;
    rank(n, before, mass);
#pragma unroll
    for (int q = 0; q < kOwn; ++q) {
      const int i = threadIdx.x + q * T;
      if (i >= n) continue;
      const Candidate c = sh.bins.list[i];
      const u64 from = above + (by_mass ? mass[q] : before[q]), size = by_mass ? c.w : 1;
      if (from < target) part += c.w;
      if (from < target && target - from <= size) sh.thr = value_of_key<E>((uint32_t)(c.at >> 32)), sh.thr_id = ~(uint32_t)c.at;
    }
    kept_mass = above_mass + block_sum(part);
    __syncthreads();
    thr = sh.thr, thr_id = sh.thr_id;
    return true;
  };

  if (by_k || by_p) {
    bins(by_p);
    if (by_k) {
      if (!refine(false, (u64)top_k)) {
        search(false, (u64)top_k);
        kept_mass = ~0ull;
      }
    } else {
      u64 part = 0;
      for (int i = threadIdx.x; i < kBins; i += T) part += sh.bins.mass[i];
      kept_mass = block_sum(part);
    }
    if (by_p) {
      bool done = false;
      if (kept_mass != ~0ull) {
        done = refine(true, share(top_p, kept_mass));
      } else {                                     // (the bins gave way to the search's)
        u64 part = 0;
        each([&](int, int e, const Frag<E>& v) {
#pragma unroll
          for (int j = 0; j < VE; ++j) part += weight(in_order(v.v[j], (uint32_t)(e + j)) ? v.v[j] : kNone);
        });
        kept_mass = block_sum(part);
      }
      if (!done) search(true, share(top_p, kept_mass));
    }
  }
  const auto kept = [&](float v, uint32_t id) { return weight(near(v) & in_order(v, id) ? v : kNone); };
  const uint32_t id = locate(kept, place);
  if (threadIdx.x == 0) answer(id, to_f32(x[id]), sh.total);
}

// ---- host side

constexpr int64_t kSampleRows = (int64_t)1 << 21;

template <class E, int T, int NV>
static void launch_sample(SampleArgs& a, int64_t nvec, hipStream_t st) {
  a.per_seg = (int32_t)(((nvec + 63) / 64 + Shape<T>::kSegs - 1) / Shape<T>::kSegs);
  k_sample<E, T, NV><<<(unsigned)a.n, T, 0, st>>>(a);
}

// A block a row: a wave for rows of up to 256 vectors, four for up to 4,096 where there are rows enough to fill the chip with them, else
// sixteen.
template <class E>
static void sample(const SampleArgs& b, hipStream_t st) {
  constexpr int VE = Elem<E>::VE;
  const int64_t nvec = ((int64_t)b.V + VE - 1) / VE;
  for (int64_t r = 0; r < b.n; r += kSampleRows) {
    SampleArgs a = b;
    a.n = b.n - r < kSampleRows ? b.n - r : kSampleRows;
    a.x = (const E*)b.x + r * b.ld, a.u = b.u + r, a.token = b.token + r, a.logprob = b.logprob + r;
    if (b.temperature_rows) a.temperature_rows = b.temperature_rows + r;
    if (b.top_p_rows) a.top_p_rows = b.top_p_rows + r;
    if (b.min_p_rows) a.min_p_rows = b.min_p_rows + r;
    if (b.top_k_rows) a.top_k_rows = (const char*)b.top_k_rows + r * (b.top_k_64 ? 8 : 4);
    const bool many = a.n >= 512;
    if (nvec <= 64) launch_sample<E, 64, 1>(a, nvec, st);
    else if (nvec <= 256) launch_sample<E, 64, 4>(a, nvec, st);
    else if (nvec <= 1024) launch_sample<E, 256, 4>(a, nvec, st);
    else if (nvec <= 4096 && many) launch_sample<E, 256, 16>(a, nvec, st);
    else if (nvec <= 4096) launch_sample<E, 1024, 4>(a, nvec, st);
    else if (a.n > 256) launch_sample<E, 512, 0>(a, nvec, st);
    else if (nvec <= 16384) launch_sample<E, 1024, 16>(a, nvec, st);
    else launch_sample<E, 1024, 0>(a, nvec, st);
  }
}

}  // namespace elr

extern "C" int elr_sample_tokens(const void* logits, int type, int64_t n, int64_t V, int64_t ld, const float* u, double temperature,
                                 const float* temperature_rows, int64_t top_k, const void* top_k_rows, int top_k_64, double top_p,
                                 const float* top_p_rows, double min_p, const float* min_p_rows, int64_t* token, float* logprob,
                                 void* stream) {
  using namespace elr;
  if (n < 0 || V < 1 || ld < 0 || !elem_type_ok(type)) return ELR_EINVAL;
  if (V > (int64_t)1 << 30) return ELR_EUNSUPPORTED;
  if (!temperature_rows && !(temperature >= 0.0 && temperature < __builtin_inf())) return ELR_EINVAL;
  if (!top_k_rows && top_k < 0) return ELR_EINVAL;
  if (!top_p_rows && !(top_p >= 0.0 && top_p <= 1.0)) return ELR_EINVAL;
  if (!min_p_rows && !(min_p >= 0.0 && min_p <= 1.0)) return ELR_EINVAL;
  if (n == 0) return ELR_OK;
  if (!logits || !u || !token || !logprob || !elem_aligned(logits, type)) return ELR_EINVAL;
  int lg = 0;
  while (((int64_t)1 << lg) < V) ++lg;
  const SampleArgs a{logits, ld, n, (int32_t)V, 62 - lg < kWeightBits ? 62 - lg : kWeightBits, 1, u, temperature, top_p, min_p, top_k,
                     temperature_rows, top_p_rows, min_p_rows, top_k_rows, top_k_64, token, logprob};
  hipStream_t st = (hipStream_t)stream;
  if (type == ELR_F32) sample<float>(a, st);
  else if (type == ELR_F16) sample<_Float16>(a, st);
  else sample<__bf16>(a, st);
  return launch_status();
}
