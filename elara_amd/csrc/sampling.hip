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
// V 2^s < 2^63.  Their sums are exact in any order (atomics and splits included), and the same for every launch shape.
#include "elr_elem.h"

namespace elr {

constexpr int kSegs = 1024;          // partial sums of a row in the order of ids
constexpr int kDigit = 11;           // bits of a selection pass

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

struct SampleShared {
  uint32_t count[1 << kDigit];
  unsigned long long mass[1 << kDigit];
  unsigned long long seg[kSegs];
  float fmax[16];
  uint32_t bin, bin_count;
  unsigned long long above_count, above_mass, bin_mass;
  unsigned long long total;
  uint32_t id;
  unsigned long long rest;
  int seg_at;
};

__device__ __forceinline__ unsigned long long wave_sum_u64(unsigned long long x) {
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}
// Inclusive sums over the lanes.
__device__ __forceinline__ unsigned long long wave_scan_u64(unsigned long long x, int lane) {
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned long long y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  return x;
}

// One row by a block of T threads; every pass reads it again (from the caches).
template <class E, int T>
__global__ __launch_bounds__(T) void k_sample(SampleArgs a) {
  constexpr int VE = Elem<E>::VE, W = T / 64;
  typedef unsigned long long u64;
  __shared__ SampleShared sh;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const E* x = (const E*)a.x + row * a.ld;
  constexpr float kNone = -__builtin_inff();
  const int nseg = (int)(((int64_t)a.V + (int64_t)64 * VE * a.per_seg - 1) / ((int64_t)64 * VE * a.per_seg));
  // f(segment, first id, VE values) over the wave's vectors; the segments are in the order of ids.
  const auto each = [&](const auto& f) {
    for (int s = wave; s < nseg; s += W)
      for (int j = 0; j < a.per_seg; ++j) {
        const int64_t e = (((int64_t)s * a.per_seg + j) * 64 + lane) * VE;
        f(s, (int)(e < a.V ? e : a.V), widen<E>(load_raw<E, false>(x + (e < a.V ? e : 0), a.V - e, kNone)));
      }
  };
  // the row's maximum; NaN or +inf in the row show in it
  float m = kNone;
  each([&](int, int, const Frag<E>& f) {
#pragma unroll
    for (int j = 0; j < VE; ++j) m = max_nan(m, f.v[j]);
  });
  m = lanes_max_nan(m, 64);
  if (lane == 0) sh.fmax[wave] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; ++i) m = max_nan(m, sh.fmax[i]);
  const double temp = a.temperature_rows ? (double)a.temperature_rows[row] : a.temperature;
  const double top_p = a.top_p_rows ? (double)a.top_p_rows[row] : a.top_p;
  const double min_p = a.min_p_rows ? (double)a.min_p_rows[row] : a.min_p;
  const int64_t top_k = !a.top_k_rows ? a.top_k
                        : a.top_k_64 ? ((const int64_t*)a.top_k_rows)[row] : ((const int32_t*)a.top_k_rows)[row];
  const double u = (double)a.u[row];
  if (!(m < __builtin_inff()) || !(temp >= 0.0) || u != u || m == kNone) {
    if (threadIdx.x == 0) {
      a.token[row] = -1;
      a.logprob[row] = m == kNone && temp >= 0.0 && u == u ? kNone : __builtin_nanf("");
    }
    return;
  }
  const bool greedy = temp == 0.0;
  const double inv_t = greedy ? 0.0 : 1.0 / temp, unit = __builtin_ldexp(1.0, a.shift);
  const auto weight = [&](float v) -> u64 {
    if (v == kNone) return 0;
    return (u64)__builtin_rint(exp(((double)v - (double)m) * inv_t) * unit);
  };
  uint32_t thr = 0, thr_id = 0xFFFFFFFFu;     // kept: a larger key, or this key and no larger id
  const auto in_order = [&](uint32_t key, uint32_t id) { return key > thr || (key == thr && id <= thr_id); };

  // The first id at which the running sum of f over the ids exceeds t (t below the whole sum), and the sum before it; sh.total holds
  // the whole sum when t_of is called.
  const auto locate = [&](const auto& f, const auto& t_of) {
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
      for (int j = 0; j < VE; ++j)
        if (e + j < a.V) acc += f(v.v[j], (uint32_t)(e + j));
    });
    if (at >= 0) {
      const u64 r = wave_sum_u64(acc);
      if (lane == 0 && at < kSegs) sh.seg[at] = r;
    }
    __syncthreads();
    if (wave == 0) {
      u64 own = 0;
      for (int i = 0; i < kSegs / 64; ++i) own += sh.seg[lane * (kSegs / 64) + i];
      const u64 upto = wave_scan_u64(own, lane);
      const u64 all = __shfl(upto, 63, 64);
      if (lane == 0) sh.total = all;
      const u64 t = t_of(all);
      if (upto > t && upto - own <= t) {
        u64 before = upto - own;
        int s = lane * (kSegs / 64);
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
        const int64_t e = (((int64_t)s * a.per_seg + j) * 64 + lane) * VE;
        const Frag<E> v = widen<E>(load_raw<E, false>(x + (e < a.V ? e : 0), a.V - e, kNone));
        u64 own = 0, w[VE];
#pragma unroll
        for (int q = 0; q < VE; ++q) {
          w[q] = e + q < a.V ? f(v.v[q], (uint32_t)(e + q)) : 0;
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
  // or mass.  t_of gives the target from the whole mass.
  const auto search = [&](bool by_mass, u64 target) {
    uint32_t prefix = 0;
    u64 above = 0;
    int bits = kKeyBits<E>;
    while (bits > 0) {
      const int take = bits < kDigit ? bits : kDigit, low = bits - take;
      __syncthreads();
      for (int i = threadIdx.x; i < 1 << kDigit; i += T) sh.count[i] = 0, sh.mass[i] = 0;
      __syncthreads();
      each([&](int, int e, const Frag<E>& v) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const uint32_t key = key_of<E>(v.v[j]);
          if (e + j < a.V && (bits == kKeyBits<E> || key >> bits == prefix) && in_order(key, (uint32_t)(e + j))) {
            const uint32_t d = key >> low & ((1u << take) - 1);
            atomicAdd(&sh.count[d], 1u);
            if (by_mass) atomicAdd(&sh.mass[d], weight(v.v[j]));
          }
        }
      });
      __syncthreads();
      if (wave == 0) {      // lane 0 the largest digits
        constexpr int N = (1 << kDigit) / 64;
        u64 own = 0;
        for (int i = 0; i < N; ++i) {
          const int d = (1 << kDigit) - 1 - (lane * N + i);
          own += by_mass ? sh.mass[d] : sh.count[d];
        }
        const u64 upto = wave_scan_u64(own, lane) + above;
        if (upto >= target && upto - own < target) {
          u64 before = upto - own;
          int i = 0;
          for (;; ++i) {
            const int d = (1 << kDigit) - 1 - (lane * N + i);
            const u64 v = by_mass ? sh.mass[d] : sh.count[d];
            if (before + v >= target) {
              sh.bin = (uint32_t)d, sh.bin_count = sh.count[d], sh.bin_mass = v, sh.above_mass = before;
              break;
            }
            before += v;
          }
        }
      }
      __syncthreads();
      prefix = prefix << take | sh.bin;
      above = sh.above_mass;
      bits = low;
    }
    // ties at the threshold: the first `need` of them by id
    const u64 of = sh.bin_mass, n_ties = sh.bin_count;
    const u64 each_w = by_mass ? of / n_ties : 1;
    const u64 need = (target - above + each_w - 1) / each_w;
    __syncthreads();
    uint32_t id = 0xFFFFFFFFu;
    if (need < n_ties)
      id = locate([&](float v, uint32_t i) -> u64 { const uint32_t k = key_of<E>(v); return k == prefix && in_order(k, i); },
                  [&](u64) { return need - 1; });
    else if (prefix == thr) id = thr_id;
    thr = prefix, thr_id = id;
  };

  if (greedy) {
    search(false, 1);
    const uint32_t id = locate([&](float v, uint32_t i) -> u64 { return in_order(key_of<E>(v), i); }, [](u64) { return (u64)0; });
    if (threadIdx.x == 0) a.token[row] = id, a.logprob[row] = 0.0f;
    return;
  }
  if (top_k > 0 && top_k < a.V) search(false, (u64)top_k);
  if (top_p < 1.0) {
    u64 part = 0;
    each([&](int, int e, const Frag<E>& v) {
#pragma unroll
      for (int j = 0; j < VE; ++j)
        if (e + j < a.V && in_order(key_of<E>(v.v[j]), (uint32_t)(e + j))) part += weight(v.v[j]);
    });
    part = wave_sum_u64(part);
    __syncthreads();
    if (lane == 0) sh.seg[wave] = part;
    __syncthreads();
    u64 all = 0;
    for (int i = 0; i < W; ++i) all += sh.seg[i];
    u64 target = (u64)__builtin_ceil((top_p > 0.0 ? top_p : 0.0) * (double)all);
    target = target < 1 ? 1 : target > all ? all : target;
    __syncthreads();
    search(true, target);
  }
  const double low = min_p > 0.0 ? log(min_p < 1.0 ? min_p : 1.0) * temp : -__builtin_inf();
  const auto kept = [&](float v, uint32_t id) -> u64 {
    return in_order(key_of<E>(v), id) && !((double)v - (double)m < low) ? weight(v) : 0;
  };
  const uint32_t id = locate(kept, [&](u64 all) {
    const u64 t = u > 0.0 ? (u64)__builtin_floor(u * (double)all) : 0;
    return t < all ? t : all - 1;
  });
  if (threadIdx.x == 0) {
    a.token[row] = id;
    const double z = ((double)to_f32(x[id]) - (double)m) * inv_t;
    a.logprob[row] = (float)(z - log((double)sh.total * __builtin_ldexp(1.0, -a.shift)));
  }
}

// ---- host side

constexpr int64_t kSampleRows = (int64_t)1 << 21;

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
    const int64_t steps = (nvec + 63) / 64;
    a.per_seg = (int32_t)((steps + kSegs - 1) / kSegs);
    const unsigned rows = (unsigned)a.n;
    if (nvec <= 64 * 4) k_sample<E, 64><<<rows, 64, 0, st>>>(a);
    else if (nvec <= 256 * 8) k_sample<E, 256><<<rows, 256, 0, st>>>(a);
    else k_sample<E, 1024><<<rows, 1024, 0, st>>>(a);
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
  const SampleArgs a{logits, ld, n, (int32_t)V, 62 - lg < 52 ? 62 - lg : 52, 1, u, temperature, top_p, min_p, top_k,
                     temperature_rows, top_p_rows, min_p_rows, top_k_rows, top_k_64, token, logprob};
  hipStream_t st = (hipStream_t)stream;
  if (type == ELR_F32) sample<float>(a, st);
  else if (type == ELR_F16) sample<_Float16>(a, st);
  else sample<__bf16>(a, st);
  return launch_status();
}
