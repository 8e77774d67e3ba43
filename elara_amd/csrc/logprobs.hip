// Log probabilities of given tokens over rows of logits, with the entropy and the k likeliest ids, and their gradient to
// the logits (HBM-bound).  No counterpart in the reference.
//
// A row x of V logits and its token a:
//   m = max x, s = sum e^(x_v - m), t = sum e^(x_v - m) (x_v - m);
//   lse = m + log s, logprob = x_a - lse, entropy = log s - t / s (both terms are >= 0, nothing cancels).
// The row is read once: each thread keeps a running (m, s, t) and rescales it when a chunk of its elements brings a larger
// maximum: with d = m_old - m_new, s' = s e^d and t' = (t + s d) e^d.
//
// Masked places.  -inf and a type's lowest value both give e = 0; the exponent is clamped at -10,000 (e^-10000 is 0 in
// fp32), so that e * (x - m) is 0 there too and not 0 * inf.  A row of nothing but -inf has s = 0: lse and logprob are
// -inf, entropy 0, and no gradient.  A NaN (or +inf) anywhere gives NaN, as the formula does: the clamp keeps a NaN.
//
// The k likeliest (k <= 32) need no second pass over the row, but for a few of its places.  Among the maxima of 64 disjoint
// parts of it (the lanes', taken anyway) the k-th largest is a lower bound of the row's k-th largest element; about
// 64 ln(64 / (64 - k)) elements of a random row reach it.  A part that fits the block's registers is searched there.  A longer one keeps the maximum of each
// thread's chunks in LDS, and only chunks whose maximum reaches the bound are read again, a vector per lane.  The elements
// found are ranked.  Where the bound's own value is too frequent for its list (equal values, masked ones) its first places
// are taken in index order; where too many elements lie above it (the large ones all with a few threads) four counting
// passes over the row find the k-th largest itself.
// Order: larger first, ties by the lower id; -0 equals +0; a NaN ranks as -inf.
//
// Measured (bf16 but where said): 4,096 rows of 32,768 47 us (5.7 TB/s), with k = 5 52; 1,024 of 131,072 46 (5.8 TB/s);
// 1,024 of 100,003 fp32 63 (6.5 TB/s); one row of 131,072 in 64 splits 4.4, with k = 20 10.  An element costs ten
// instructions, one of them an exponential, about 42 cycles of a SIMD for 64 of them: 36 of the 47 us above.  (The exponent
// as one fma, with another path for rows at a type's lowest value, gained nothing: 45.5 and 52.)  Many shorter rows pay more for
// the k likeliest, which one wave or block of each row selects and ranks while its lanes are idle: 16,384 of 4,096 24 us without,
// 41, 44 and 48 with k = 5, 20 and 32; 60,000 of 1,000 25, and 86 with 20; 200,000 of 100 19, and 158, 281 and 296.
// Backward: 4,096 of 131,072 (1 GB in, 1 GB out) 338 to 344 us (6.3 TB/s), 301 of 50,021 fp32 21 us (5.6 TB/s); a wave a row
// at least: 60,000 of 1,000 66 us (3.7 TB/s), 200,000 of 100 78 (1.1).
#include "elr_elem.h"

namespace elr {

constexpr float kLog2e = 0x1.715476p+0f;
constexpr float kExpFloor = -1e4f;
constexpr int kMaxTop = ELR_TOPK_MAX;
constexpr int kVecs = 4;        // 16-byte vectors a thread loads at a time (one chunk's step)
constexpr int kChunks = 16;     // chunk maxima a thread keeps
// Candidate lists, and vectors or chunks that hold candidates: of a block, and of a wave by itself (whose LDS bounds how many
// run at once: 10.5 KB a wave was 4 waves a SIMD).
template <int T>
constexpr int kAbove = T > 128 ? 448 : T > 64 ? 192 : 128;
constexpr int kTies = 64;
template <int T>
constexpr int kHits = T > 128 ? 256 : T > 64 ? 128 : 80;
constexpr uint32_t kFloorOrd = 0x007FFFFFu;   // order_of(-inf)
constexpr int kMaxSplits = 64;

__device__ __forceinline__ float exp_nat(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }
__device__ __forceinline__ float clamp_low(float d) { return max_nan(d, kExpFloor); }
// The value subtracted in the exponents: a maximum of -inf (nothing unmasked so far) is replaced by 0.
__device__ __forceinline__ float exp_ref(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// An unsigned order of fp32 values: larger value, larger number; NaN as -inf, -0 as +0.  Never 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  x = x + 0.0f;
  if (x != x) x = -__builtin_inff();
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}

struct Sums {
  float m, s, t;
};

// (m, s, t) of two parts of a row put together.
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  Sums r;
  r.m = __builtin_fmaxf(a.m, b.m);
  const float ref = exp_ref(r.m);
  const float da = clamp_low(a.m - ref), db = clamp_low(b.m - ref);
  const float fa = exp_nat(da), fb = exp_nat(db);
  r.s = a.s * fa + b.s * fb;
  r.t = (a.t + a.s * da) * fa + (b.t + b.s * db) * fb;
  return r;
}

struct LpArgs {
  const void* x;
  int64_t ld;
  int64_t n;
  int32_t V, splits, seg;      // seg: elements of a split (a multiple of the vector)
  int32_t per_chunk;           // steps of T * kVecs vectors that share a chunk maximum
  const void* tokens;
  int idx64, k;
  float *logprob, *lse, *entropy, *top_logprob;
  int64_t* top_id;
  float* part;                 // [n * splits][4] partial (m, s, t) and the token's logit, if the split holds it
  uint64_t* part_top;          // [n * splits][k] candidates: order in the high half, ~id in the low
};

__device__ __forceinline__ int64_t token_at(const LpArgs& a, int64_t row) {
  return a.idx64 ? ((const int64_t*)a.tokens)[row] : (int64_t)((const int32_t*)a.tokens)[row];
}

// A row's results from its joined sums; x_tok is the token's logit (has: the row has a token).
__device__ __forceinline__ void write_row(const LpArgs& a, int64_t row, const Sums& r, bool has, float x_tok) {
  const float logs = __builtin_logf(r.s);
  const bool empty = r.s == 0.0f;
  a.lse[row] = empty ? -__builtin_inff() : r.m + logs;
  a.entropy[row] = empty ? 0.0f : logs - r.t / r.s;
  a.logprob[row] = !has ? 0.0f : empty ? -__builtin_inff() : (x_tok - r.m) - logs;
}

// Bits of an order that tell values of the type apart (the others are all 0 or all 1).
template <class E>
constexpr uint32_t kBits = sizeof(E) == 4 ? ~0u : Elem<E>::kType == ELR_BF16 ? 0xFFFF0000u : 0xFFFFE000u;

// The k-th largest of the 64 lanes' N orders each, bit by bit (its low bits 0 where kBits has none).
template <class E, int N>
__device__ __forceinline__ uint32_t wave_kth(const uint32_t (&o)[N], int k) {
  uint32_t t = 0;
#pragma unroll
  for (int b = 31; b >= __builtin_ctz(kBits<E>); --b) {
    const uint32_t c = t | 1u << b;
    int n = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(o[j] >= c));
    if (n >= k) t = c;
  }
  return t;
}
__device__ __forceinline__ uint64_t lane_of(uint64_t x, int j) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), j) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)x, j);
}

// Candidates of one block: order and id packed so that a larger number comes first (ties: the lower id).
__device__ __forceinline__ uint64_t pack_cand(uint32_t o, uint32_t id) { return (uint64_t)o << 32 | (uint32_t)~id; }

template <int T>
struct TopShared {
  float gmax[T];                  // thread maxima
  uint64_t above[kAbove<T>], ties[kTies];
  int n_above, n_ties, n_hits;
  uint32_t thr;
  uint32_t hits[kHits<T>];        // a vector's number, or chunk * T + thread
  union {
    u32x4 vecs[kHits<T>];         // the vectors themselves (parts held in registers)
    uint32_t hist[256];           // of the radix selection, when they are done with
  };
  int scan[T / 64 + 1];
};

template <class E, int T>
struct RowPart {
  const E* p;           // the split's first element
  int32_t first, len;   // its place in the row and its length
  int32_t shift;        // elements between the start of p's memory line and p: vectors are laid from there
};

// f(order, id) for every element of the part, in no order.
template <class E, int T, class F>
__device__ __forceinline__ void each_elem(const RowPart<E, T>& r, const F& f) {
  constexpr int VE = Elem<E>::VE;
  for (int32_t e = threadIdx.x * VE; e < r.len; e += T * VE) {
    const Frag<E> x = widen<E>(load_raw<E, false>(r.p + e, r.len - e, 0.0f));
#pragma unroll
    for (int j = 0; j < VE; ++j)
      if (e + j < r.len) f(order_of(x.v[j]), (uint32_t)(r.first + e + j));
  }
}

// The first `want` (at most kTies) elements of order `o` in index order into ties[0 ..]; sets n_ties.
template <class E, int T>
__device__ void ordered_ties(const RowPart<E, T>& r, TopShared<T>& sh, uint32_t o, int want) {
  constexpr int VE = Elem<E>::VE;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int found = 0;   // the same in every thread
  for (int32_t e0 = 0; e0 < r.len && found < want; e0 += T * VE) {
    const int32_t e = e0 + threadIdx.x * VE;
    const Frag<E> x = widen<E>(load_raw<E, false>(r.p + e, r.len - e, 0.0f));
    int mine = 0;
#pragma unroll
    for (int j = 0; j < VE; ++j) mine += e + j < r.len && order_of(x.v[j]) == o;
    int inc = mine;   // inclusive sum over the wave's lanes
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(inc, d, 64);
      if (lane >= d) inc += y;
    }
    __syncthreads();
    if (lane == 63) sh.scan[wave] = inc;
    __syncthreads();
    int at = found + inc - mine, total = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
      if (w < wave) at += sh.scan[w];
      total += sh.scan[w];
    }
#pragma unroll
    for (int j = 0; j < VE; ++j)
      if (e + j < r.len && order_of(x.v[j]) == o) {
        if (at < want) sh.ties[at] = pack_cand(o, (uint32_t)(r.first + e + j));
        ++at;
      }
    found += total;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.n_ties = found < want ? found : want;
  __syncthreads();
}

// The order of the part's k-th largest element (k <= r.len), by four counting passes of 8 bits.
template <class E, int T>
__device__ uint32_t radix_kth(const RowPart<E, T>& r, TopShared<T>& sh, int k) {
  uint32_t prefix = 0;
  int left = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += T) sh.hist[i] = 0;
    __syncthreads();
    each_elem<E, T>(r, [&](uint32_t o, uint32_t) {
      if (shift == 24 || (o >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&sh.hist[(o >> shift) & 255u], 1u);
    });
    __syncthreads();
    int d = 255;      // every thread walks the counts alike
    for (; d > 0 && (int)sh.hist[d] < left; --d) left -= (int)sh.hist[d];
    prefix |= (uint32_t)d << shift;
    __syncthreads();
  }
  return prefix;
}

// The order of a lower bound of the block's k-th largest element (the bits of kBits), the same in every thread, from the
// threads' maxima m; most: the block's maximum.
template <class E, int T>
__device__ __forceinline__ uint32_t lower_bound(TopShared<T>& sh, float m, float most, int k) {
  const int lane = threadIdx.x & 63;
  if (threadIdx.x == 0) sh.n_above = sh.n_ties = sh.n_hits = 0;
  uint32_t thr = order_of(most) & kBits<E>;
  if (k > 1) {
    if constexpr (T > 64) {
      sh.gmax[threadIdx.x] = m;
      __syncthreads();
      if (threadIdx.x < 64) {
#pragma unroll
        for (int w = 1; w < T / 64; ++w) m = __builtin_fmaxf(m, sh.gmax[w * 64 + lane]);
      }
    }
    if (T == 64 || threadIdx.x < 64) {
      const uint32_t o[1] = {order_of(m)};
      thr = wave_kth<E, 1>(o, k);
      if (T > 64 && lane == 0) sh.thr = thr;
    }
  }
  __syncthreads();
  return T > 64 && k > 1 ? sh.thr : thr;
}

// The elements of a vector that reach the bound (thr_f) into the lists: above the bound's order, or equal to it.  Every
// place in a list is taken before the first is written, so that the waits for them overlap.
template <class E, int T>
__device__ __forceinline__ void push_vec(TopShared<T>& sh, const Frag<E>& x, uint32_t thr, float thr_f, int32_t id) {
  constexpr int VE = Elem<E>::VE;
  int at[VE];
#pragma unroll
  for (int j = 0; j < VE; ++j) {
    at[j] = -1;
    if (x.v[j] >= thr_f) {
      const uint32_t o = order_of(x.v[j]);
      at[j] = atomicAdd((o & kBits<E>) > thr ? &sh.n_above : &sh.n_ties, 1);
    }
  }
#pragma unroll
  for (int j = 0; j < VE; ++j) {
    if (at[j] < 0) continue;
    const uint32_t o = order_of(x.v[j]);
    const uint64_t c = pack_cand(o, (uint32_t)(id + j));
    if ((o & kBits<E>) > thr) {
      if (at[j] < kAbove<T>) sh.above[at[j]] = c;
    } else {
      if (at[j] < kTies) sh.ties[at[j]] = c;
    }
  }
}

// The nc candidates (distinct) of `at` ranked by one wave if they fit it, else by the block; out(rank, candidate) of the
// first k.
template <int T, class At, class Out>
__device__ __forceinline__ void rank_cands(int nc, int k, const At& at, const Out& out) {
  if (nc <= 64) {
    if (threadIdx.x >= 64) return;
    const uint64_t c = (int)threadIdx.x < nc ? at(threadIdx.x) : 0;
    int rank = 0;
    for (int j = 0; j < nc; j += 8) {   // (the lanes past the last hold 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) rank += lane_of(c, j + i) > c;
    }
    if ((int)threadIdx.x < nc && rank < k) out(rank, c);
    return;
  }
  for (int i = threadIdx.x; i < nc; i += T) {
    const uint64_t c = at(i);
    int rank = 0;
    for (int j = 0; j < nc; ++j) rank += at(j) > c;
    if (rank < k) out(rank, c);
  }
}

// The k likeliest of a part from the lists, in order, through out(rank, packed); thr: the bound they were filled by (of -inf:
// with what lies above it).  Too many hits: the elements above the bound are collected from the whole part.  Too many of
// those: above the k-th largest itself, which fewer than k are.  The rest are ties of that one value, in index order.
template <class E, int T, class Out>
__device__ __forceinline__ void finish_top(int k, const RowPart<E, T>& r, TopShared<T>& sh, uint32_t thr, const Out& out) {
  __syncthreads();
  int na = sh.n_above, nt = sh.n_ties;
  const bool lost = sh.n_hits > kHits<T>;
  if (lost || na > kAbove<T> || nt > kTies || thr <= kFloorOrd) {
    const int want = min(k, r.len);
    uint32_t kth = thr < 0x80000000u ? thr | ~kBits<E> : thr;   // (a negative value's order has ones there)
    for (int pass = 0; pass < 2 && (na > kAbove<T> || (pass == 0 && lost)); ++pass) {
      if (pass || !lost) kth = radix_kth<E, T>(r, sh, want);
      __syncthreads();
      if (threadIdx.x == 0) sh.n_above = 0;
      __syncthreads();
      each_elem<E, T>(r, [&](uint32_t o, uint32_t id) {
        if (o > kth) {
          const int i = atomicAdd(&sh.n_above, 1);
          if (i < kAbove<T>) sh.above[i] = pack_cand(o, id);
        }
      });
      __syncthreads();
      na = sh.n_above;
    }
    if (na < want) ordered_ties<E, T>(r, sh, kth, want - na);
    nt = na < want ? sh.n_ties : 0;
  }
  const int nc = na + nt;
  rank_cands<T>(nc, k, [&](int i) { return i < na ? sh.above[i] : sh.ties[i - na]; }, out);
  for (int i = nc + threadIdx.x; i < k; i += T) out(i, (uint64_t)0);   // a part shorter than k
}

__device__ __forceinline__ void write_top(const LpArgs& a, int64_t row, int rank, uint64_t c, float m, float logs,
                                          bool empty) {
  const float x = value_of((uint32_t)(c >> 32));
  a.top_logprob[row * a.k + rank] = empty ? -__builtin_inff() : (x - m) - logs;
  a.top_id[row * a.k + rank] = (int64_t)(uint32_t)~(uint32_t)c;
}

// A wave's lanes' sums put together, the same in every lane.
__device__ __forceinline__ Sums wave_join(const Sums& q) {
  Sums r;
  r.m = wave_max(q.m);
  const float d = clamp_low(q.m - exp_ref(r.m)), f = exp_nat(d);
  r.s = wave_sum(q.s * f);
  r.t = wave_sum((q.t + q.s * d) * f);
  return r;
}
template <int T>
__device__ __forceinline__ Sums block_join(Sums q, Sums* waves) {
  q = wave_join(q);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = q;
    __syncthreads();
    q = waves[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) q = join(q, waves[w]);
  }
  return q;
}

template <class E, int T>
__device__ __forceinline__ RowPart<E, T> part_of(const LpArgs& a, int64_t row, int split) {
  RowPart<E, T> r;
  r.first = split * a.seg;
  r.len = min(a.seg, a.V - r.first);
  r.p = (const E*)a.x + row * a.ld + r.first;
  r.shift = line_shift<E>(r.p, 128);
  return r;
}

// The part's results: the row's if it is not split.  bound(thr): the bound to use, given the one from the threads' maxima.
template <class E, int T, bool TOP, class Bound, class Fill>
__device__ __forceinline__ void part_done(const LpArgs& a, int64_t row, int64_t unit, const RowPart<E, T>& r,
                                          TopShared<TOP ? T : 64>& sh, const Sums& q, bool has, float x_tok,
                                          float mine, const Bound& bound, const Fill& fill) {
  if (a.splits == 1) {
    if (threadIdx.x == 0) write_row(a, row, q, has, x_tok);
  } else if (threadIdx.x == 0) {
    *(f32x4*)(a.part + unit * 4) = (f32x4){q.m, q.s, q.t, x_tok};
  }
  if constexpr (TOP) {
    const uint32_t thr = bound(lower_bound<E, T>(sh, mine, q.m, a.k));
    const float thr_f = thr <= kFloorOrd ? -0x1.fffffep+127f : value_of(thr);   // -inf: what is above it
    fill(thr, thr_f);
    const float logs = __builtin_logf(q.s);
    finish_top<E, T>(a.k, r, sh, thr, [&](int rank, uint64_t c) {
      if (a.splits == 1) write_top(a, row, rank, c, q.m, logs, q.s == 0.0f);
      else a.part_top[unit * a.k + rank] = c;
    });
  }
}

// Whether the part holds the row's token, and its logit: loaded by the first thread while the row is on its way.
template <class E, int T>
__device__ __forceinline__ bool token_logit(const LpArgs& a, int64_t row, const RowPart<E, T>& r, float& x) {
  x = 0.0f;
  if (threadIdx.x != 0) return false;
  const int64_t tok = token_at(a, row) - r.first;
  if (tok < 0 || tok >= r.len) return false;
  x = to_f32(r.p[tok]);
  return true;
}

// A part of up to T * NV vectors: it stays in registers, and no sum is rescaled.
template <class E, int T, int NV, bool TOP>
__global__ __launch_bounds__(T) void k_lp_one(LpArgs a) {
  constexpr int VE = Elem<E>::VE;
  __shared__ Sums waves[T / 64];
  __shared__ float wmax[T / 64];
  __shared__ TopShared<TOP ? T : 64> sh;
  const int64_t unit = blockIdx.x;
  const int64_t row = a.splits == 1 ? unit : unit / a.splits;
  const RowPart<E, T> r = part_of<E, T>(a, row, a.splits == 1 ? 0 : (int)(unit - row * a.splits));
  const int64_t e0 = (int64_t)threadIdx.x * VE - r.shift;
  u32x4 raw[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u)
    raw[u] = load_part<E, true>(r.p, e0 + (int64_t)u * T * VE, r.len, -__builtin_inff());
  float x_tok;
  const bool has = token_logit<E, T>(a, row, r, x_tok);
  Frag<E> x[NV];
  float vmax[NV];
  Sums q{-__builtin_inff(), 0.0f, 0.0f};
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    x[u] = widen<E>(raw[u]);
    vmax[u] = x[u].v[0];
#pragma unroll
    for (int j = 1; j < VE; ++j) vmax[u] = __builtin_fmaxf(vmax[u], x[u].v[j]);
    q.m = __builtin_fmaxf(q.m, vmax[u]);
  }
  const float mine = q.m;
  q.m = wave_max(q.m);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) wmax[threadIdx.x >> 6] = q.m;
    __syncthreads();
    q.m = wmax[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) q.m = __builtin_fmaxf(q.m, wmax[w]);
  }
  const float ref = exp_ref(q.m);
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const float d = clamp_low(x[u].v[j] - ref);
      const float e = exp_nat(d);
      q.s = q.s + e;
      q.t = __builtin_fmaf(e, d, q.t);
    }
  q.s = wave_sum(q.s);
  q.t = wave_sum(q.t);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = q;
    __syncthreads();
    q = waves[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) {
      q.s = q.s + waves[w].s;
      q.t = q.t + waves[w].t;
    }
  }
  const auto bound = [&](uint32_t thr) {
    if constexpr (T == 64 && NV == 1 && TOP) {
      // fewer vectors than k: that bound is -inf, so the k-th largest itself
      if (thr > kFloorOrd || (r.len + r.shift) > a.k * VE) return thr;
      uint32_t o[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const int64_t e = e0 + j;
        o[j] = e >= 0 && e < r.len ? order_of(x[0].v[j]) : 0;
      }
      return wave_kth<E, VE>(o, min(a.k, r.len));
    }
    return thr;
  };
  part_done<E, T, TOP>(a, row, unit, r, sh, q, has, x_tok, mine, bound, [&](uint32_t thr, float thr_f) {
    if constexpr (TOP) {
      // the vectors that reach the bound to LDS, then a vector per thread
#pragma unroll
      for (int u = 0; u < NV; ++u)
        if (vmax[u] >= thr_f) {
          const int i = atomicAdd(&sh.n_hits, 1);
          if (i < kHits<T>) {
            sh.hits[i] = (uint32_t)(u * T) + threadIdx.x;
            sh.vecs[i] = raw[u];
          }
        }
      __syncthreads();
      const int nh = sh.n_hits;
      if (nh > kHits<T>) return;
      for (int i = threadIdx.x; i < nh; i += T)
        push_vec<E, T>(sh, widen<E>(sh.vecs[i]), thr, thr_f, r.first + (int32_t)sh.hits[i] * VE - r.shift);
    }
  });
}

// Short rows without alternatives: 2^lg lanes a row, kVecs vectors a lane, several rows a wave, so that a row's share of the
// reductions is small (200,000 rows of 100 bf16: 74 us with a wave a row, 19 here; 60,000 of 1,000: 42 and 26).
template <class E>
__global__ __launch_bounds__(256) void k_lp_small(LpArgs a, int lg) {
  constexpr int VE = Elem<E>::VE;
  const int lane = threadIdx.x & 63, team = 1 << lg, l = lane & (team - 1);
  const int64_t row = (((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) << (6 - lg)) + (lane >> lg);
  const bool live = row < a.n;            // (lanes past the last row take part in the reductions)
  const E* p = (const E*)a.x + (live ? row : 0) * a.ld;
  u32x4 raw[kVecs];
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int e = (u * team + l) * VE;
    raw[u] = load_raw<E, true>(p + e, live ? a.V - e : 0, -__builtin_inff());
  }
  bool has = false;
  float x_tok = 0.0f;
  if (live && l == 0) {
    const int64_t tok = token_at(a, row);
    has = tok >= 0 && tok < a.V;
    if (has) x_tok = to_f32(p[tok]);
  }
  Frag<E> x[kVecs];
  Sums q{-__builtin_inff(), 0.0f, 0.0f};
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    x[u] = widen<E>(raw[u]);
#pragma unroll
    for (int j = 0; j < VE; ++j) q.m = __builtin_fmaxf(q.m, x[u].v[j]);
  }
  q.m = lanes_op(q.m, team, [](float b, float c) { return __builtin_fmaxf(b, c); });
  const float ref = exp_ref(q.m);
#pragma unroll
  for (int u = 0; u < kVecs; ++u)
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const float d = clamp_low(x[u].v[j] - ref);
      const float e = exp_nat(d);
      q.s = q.s + e;
      q.t = __builtin_fmaf(e, d, q.t);
    }
  q.s = lanes_sum(q.s, team);
  q.t = lanes_sum(q.t, team);
  if (live && l == 0) write_row(a, row, q, has, x_tok);
}

// A longer part, T * kVecs vectors at a time.
template <class E, int T, bool TOP>
__global__ __launch_bounds__(T) void k_lp_rows(LpArgs a) {
  constexpr int VE = Elem<E>::VE;
  constexpr int64_t kStep = (int64_t)T * kVecs * VE;
  __shared__ float cmax[TOP ? kChunks * T : 1];
  __shared__ Sums waves[T / 64];
  __shared__ TopShared<TOP ? T : 64> sh;
  const int64_t unit = blockIdx.x;
  const int64_t row = a.splits == 1 ? unit : unit / a.splits;
  const RowPart<E, T> r = part_of<E, T>(a, row, a.splits == 1 ? 0 : (int)(unit - row * a.splits));
  const int steps = (int)((r.len + r.shift + kStep - 1) / kStep);
  float x_tok;
  const bool has = token_logit<E, T>(a, row, r, x_tok);
  Sums q{-__builtin_inff(), 0.0f, 0.0f};
  float ck = -__builtin_inff();   // the current chunk's maximum
  int in_chunk = 0, chunk = 0;
  for (int it = 0; it < steps; ++it) {
    const int64_t s0 = it * kStep - r.shift, e0 = s0 + (int64_t)threadIdx.x * VE;
    u32x4 raw[kVecs];
    if (s0 >= 0 && s0 + kStep <= r.len) {
#pragma unroll
      for (int u = 0; u < kVecs; ++u) raw[u] = load_raw<E, true>(r.p + e0 + (int64_t)u * T * VE, VE, 0.0f);
    } else {
#pragma unroll
      for (int u = 0; u < kVecs; ++u)
        raw[u] = load_part<E, true>(r.p, e0 + (int64_t)u * T * VE, r.len, -__builtin_inff());
    }
    Frag<E> x[kVecs];
    float c = -__builtin_inff();
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      x[u] = widen<E>(raw[u]);
#pragma unroll
      for (int j = 0; j < VE; ++j) c = __builtin_fmaxf(c, x[u].v[j]);
    }
    const float mn = __builtin_fmaxf(q.m, c);
    const float ref = exp_ref(mn);
    const float d0 = clamp_low(q.m - ref), f0 = exp_nat(d0);
    q.t = (q.t + q.s * d0) * f0;
    q.s = q.s * f0;
    q.m = mn;
#pragma unroll
    for (int u = 0; u < kVecs; ++u)
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float d = clamp_low(x[u].v[j] - ref);
        const float e = exp_nat(d);
        q.s = q.s + e;
        q.t = __builtin_fmaf(e, d, q.t);
      }
    if constexpr (TOP) {
      ck = __builtin_fmaxf(ck, c);
      if (++in_chunk == a.per_chunk || it + 1 == steps) {
        cmax[chunk * T + threadIdx.x] = ck;
        ++chunk;
        in_chunk = 0;
        ck = -__builtin_inff();
      }
    }
  }
  const float mine = q.m;
  q = block_join<T>(q, waves);
  const auto bound = [](uint32_t thr) { return thr; };
  part_done<E, T, TOP>(a, row, unit, r, sh, q, has, x_tok, mine, bound, [&](uint32_t thr, float thr_f) {
    if constexpr (TOP) {
      // the chunks that reach the bound ...
      if (mine >= thr_f)
        for (int c = 0; c < chunk; ++c)
          if (cmax[c * T + threadIdx.x] >= thr_f) {
            const int i = atomicAdd(&sh.n_hits, 1);
            if (i < kHits<T>) sh.hits[i] = (uint32_t)(c * T) + threadIdx.x;
          }
      __syncthreads();
      const int nh = sh.n_hits;
      if (nh > kHits<T>) return;
      // ... read again, one vector a thread at a time
      const int per = a.per_chunk * kVecs, tasks = nh * per;
      for (int i = threadIdx.x; i < tasks; i += T) {
        const int h = i / per, v = i - h * per;
        const uint32_t hit = sh.hits[h];
        const int64_t vec = ((int64_t)(hit / T) * per + v) * T + hit % T;
        const int64_t e = vec * VE - r.shift;
        const Frag<E> x = widen<E>(load_part<E, false>(r.p, e, r.len, -__builtin_inff()));
        push_vec<E, T>(sh, x, thr, thr_f, r.first + (int32_t)e);
      }
    }
  });
}

// The splits of a row joined: lane i holds split i's sums.  The splits' sorted candidates fall into up to 64 runs, at least k,
// and a candidate below the k-th largest of the runs' first ones cannot be among the row's k; of k candidates a run, that
// leaves at most k (k - 1) + 1.
constexpr int kJoinThreads = 256;
__global__ __launch_bounds__(kJoinThreads) void k_lp_join(LpArgs a) {
  constexpr int kMost = kMaxTop * (kMaxTop - 1) + 1, kEach = kMaxSplits * kMaxTop / kJoinThreads;
  __shared__ uint64_t cand[kMost];
  __shared__ int count;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, S = a.splits, all = S * a.k;
  const uint64_t* top = a.part_top + row * S * a.k;
  uint64_t mine[kEach], head = 0;
  float x_tok = 0.0f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = i * kJoinThreads + threadIdx.x;
    mine[i] = j < all ? top[j] : 0;
  }
  const int runs = kMaxSplits / S, each = (a.k + runs - 1) / runs;   // of a split
  const int sp = lane / runs, in = (lane - sp * runs) * each;
  if (sp < S && in < a.k) head = top[sp * a.k + in];
  Sums q{-__builtin_inff(), 0.0f, 0.0f};
  if (lane < S) {
    const f32x4 p = *(const f32x4*)(a.part + (row * S + lane) * 4);
    q = Sums{p[0], p[1], p[2]};
    x_tok = p[3];
  }
  const int64_t tok = token_at(a, row);
  const bool has = tok >= 0 && tok < a.V;
  x_tok = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x_tok), has ? (int)(tok / a.seg) : 0));
  if (threadIdx.x == 0) count = 0;
  q = wave_join(q);
  if (threadIdx.x == 0) write_row(a, row, q, has, x_tok);
  if (a.k == 0) return;
  __syncthreads();
  int rank = 0;      // distinct, but for those of no run, which are 0
#pragma unroll 8
  for (int j = 0; j < 64; ++j) rank += lane_of(head, j) > head;
  const uint64_t at = __builtin_amdgcn_ballot_w64(rank == a.k - 1);
  const uint64_t thr = at ? lane_of(head, __builtin_ctzll(at)) : 0;   // fewer than k runs: every candidate
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (mine[i] != 0 && mine[i] >= thr) cand[atomicAdd(&count, 1)] = mine[i];
  __syncthreads();
  const float logs = __builtin_logf(q.s);
  rank_cands<kJoinThreads>(count, a.k, [&](int i) { return cand[i]; }, [&](int r, uint64_t c) {
    write_top(a, row, r, c, q.m, logs, q.s == 0.0f);
  });
}

// d x_v = [v = a] g + p_v (z - g - h (log p_v + H)), p = e^(x - lse): one read and one write of the logits, in place too.
struct LpBackArgs {
  const void* x;
  int64_t ld;
  int64_t n;
  int32_t V, chunks;           // chunks: waves that share a row
  const void* tokens;
  int idx64;
  const float *lse, *entropy, *d_logprob, *d_entropy, *d_lse;
  void* out;
  int64_t out_ld;
};

constexpr int kBackVecs = 4;
// A row whose mask left nothing: all -inf, or all at a type's lowest value, where lse, -3.4e38 in fp32, has no digits left
// for log V and e^(x - lse) would be 1 for each of the V.  Such a row gets no gradient.
constexpr float kEmptyLse = -0x1.0p+100f;

// From here on half an ulp of lse (2^-17 and more) is what p = e^(x - lse) would err by, and at a common offset of 10^9 lse has
// no digit of log V left.  The sum of such a wide row's e^(x - lse), which should be 1, is taken then.
constexpr float kWideLse = 256.0f;

// What a row's gradient needs; logp = (x - ref) - sub.
struct RowGrad {
  int64_t tok;
  float g, h, c0, ref, sub;
  bool has, empty, wide;
};
__device__ __forceinline__ RowGrad row_grad(const LpBackArgs& a, int64_t row) {
  RowGrad r;          // (no load waits for the token: 200,000 rows of 100 in 80 us, 84 where that of g did)
  r.ref = a.lse[row];
  const float g = a.d_logprob ? a.d_logprob[row] : 0.0f;
  r.h = a.d_entropy ? a.d_entropy[row] : 0.0f;
  const float z = a.d_lse ? a.d_lse[row] : 0.0f;
  const float ent = a.d_entropy ? a.entropy[row] : 0.0f;
  r.tok = a.idx64 ? ((const int64_t*)a.tokens)[row] : (int64_t)((const int32_t*)a.tokens)[row];
  r.has = r.tok >= 0 && r.tok < a.V;
  r.g = r.has ? g : 0.0f;
  r.c0 = (z - r.g) - r.h * ent;
  r.sub = 0.0f;
  r.empty = r.ref < kEmptyLse;
  const float size = __builtin_fabsf(r.ref);
  r.wide = size >= kWideLse && size < __builtin_inff() && !r.empty;
  return r;
}
// A wide row's gradient by its own sum, s = sum e^(x - lse): p = e^((x - lse) - log s).  lse is no less than any x, and x - lse
// has all the digits that x has.  An lse from which the row's own is further than its rounding (it may be of more logits than
// these) is used as it is.
__device__ __forceinline__ void use_sum(RowGrad& r, float s) {
  const float rest = __builtin_logf(s);
  if (__builtin_fabsf(rest) <= __builtin_fabsf(r.ref) * 0x1.0p-22f) r.sub = rest;
}
// The gradients of the vector at element e of the row.  SUB: r.sub may be other than 0.
template <class E, bool SUB>
__device__ __forceinline__ u32x4 grad_vec(const RowGrad& r, u32x4 raw, int64_t e) {
  constexpr int VE = Elem<E>::VE;
  Frag<E> y = widen<E>(raw);
  const int at = r.has && r.tok >= e && r.tok < e + VE ? (int)(r.tok - e) : -1;
#pragma unroll
  for (int j = 0; j < VE; ++j) {
    const float d0 = y.v[j] - r.ref;
    const float logp = clamp_low(SUB ? d0 - r.sub : d0);
    const float d = exp_nat(logp) * __builtin_fmaf(-r.h, logp, r.c0);
    y.v[j] = r.empty ? 0.0f : j == at ? d + r.g : d;
  }
  return narrow<E>(y);
}

// s with e^(x - ref) of a vector's elements (those outside the row are -inf: nothing).
template <class E>
__device__ __forceinline__ float add_vec(float s, u32x4 raw, float ref) {
  const Frag<E> y = widen<E>(raw);
#pragma unroll
  for (int j = 0; j < Elem<E>::VE; ++j) s = s + exp_nat(clamp_low(y.v[j] - ref));
  return s;
}

// A wave's vectors of a row, from element e0 of lane 0 on; ALL: every one lies within the row.  False: a wide row of more than
// this chunk, of which nothing is written.
template <class E, int U, bool ALL>
__device__ __forceinline__ bool back_vecs(const LpBackArgs& a, int64_t row, const E* x, E* out, int64_t s0) {
  constexpr int VE = Elem<E>::VE;
  const int lane = threadIdx.x & 63;
  const int64_t e0 = s0 + lane * VE;
  u32x4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if constexpr (ALL) raw[u] = load_raw<E, true>(x + e0 + u * 64 * VE, VE, 0.0f);
    else raw[u] = load_part<E, true>(x, e0 + u * 64 * VE, a.V, -__builtin_inff());
  }
  RowGrad r = row_grad(a, row);
  if (r.wide) {
    if constexpr (U > 1) return false;
    use_sum(r, wave_sum(add_vec<E>(0.0f, raw[0], r.ref)));     // (the row is this chunk)
    store_part<E, true>(out, e0, a.V, grad_vec<E, true>(r, raw[0], e0));
    return true;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t e = e0 + u * 64 * VE;
    const u32x4 y = grad_vec<E, false>(r, raw[u], e);
    if constexpr (ALL) store_raw<E, true>(out + e, y, VE);
    else store_part<E, true>(out, e, a.V, y);
  }
  return true;
}

// A whole wide row by one wave, or by the `waves` of a block of which all are the row's.  In place none may write before the sum
// is taken, so the row's other waves leave it alone.  4,096 rows of 131,072 bf16, all wide, take 752 us (344 where none is), one
// such row alone 36 (a wave a row: 1,133 and 130); 200,000 of 100, each in its wave's registers, 95 (78).
template <class E>
__device__ __forceinline__ void back_wide(const LpBackArgs& a, int64_t row, const E* x, E* out, int waves, float* sums) {
  constexpr int VE = Elem<E>::VE, U = 16 / VE;      // (more vectors a step would cost the other rows' waves registers)
  constexpr int64_t kStep = 64 * U * VE;
  const int lane = threadIdx.x & 63, w = waves > 1 ? (int)(threadIdx.x >> 6) : 0;
  const int64_t first = w * kStep - line_shift<E>(out, 128);
  const auto load = [&](u32x4 (&raw)[U], int64_t e0) {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_part<E, false>(x, e0 + u * 64 * VE, a.V, -__builtin_inff());
  };
  RowGrad r = row_grad(a, row);
  float s = 0.0f;
  for (int64_t s0 = first; s0 < a.V; s0 += waves * kStep) {
    u32x4 raw[U];
    load(raw, s0 + lane * VE);
#pragma unroll
    for (int u = 0; u < U; ++u) s = add_vec<E>(s, raw[u], r.ref);
  }
  s = wave_sum(s);
  if (waves > 1) {
    if (lane == 0) sums[w] = s;
    __syncthreads();
    s = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
  use_sum(r, s);
  for (int64_t s0 = first; s0 < a.V; s0 += waves * kStep) {
    u32x4 raw[U];
    load(raw, s0 + lane * VE);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t e = s0 + lane * VE + u * 64 * VE;
      store_part<E, true>(out, e, a.V, grad_vec<E, true>(r, raw[u], e));
    }
  }
}

// Chunks of 64 * U vectors, one wave each, laid from the memory line in which the output's row starts.  U = 1: a row is one.
template <class E, int U>
__global__ __launch_bounds__(256) void k_lp_back(LpBackArgs a, int64_t row0) {
  constexpr int VE = Elem<E>::VE;
  constexpr int64_t kChunk = 64 * U * VE;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4u + (threadIdx.x >> 6)));
  const uint32_t in = wave / (uint32_t)a.chunks;
  const int64_t row = row0 + in;
  if (row >= a.n) return;
  const E* x = (const E*)a.x + row * a.ld;
  E* out = (E*)a.out + row * a.out_ld;
  const uint32_t chunk = wave - in * (uint32_t)a.chunks;
  const int64_t s0 = (int64_t)chunk * kChunk - line_shift<E>(out, 128);
  const bool done = s0 >= 0 && s0 + kChunk <= a.V ? back_vecs<E, U, true>(a, row, x, out, s0)
                                                  : back_vecs<E, U, false>(a, row, x, out, s0);
  if constexpr (U > 1) {
    // (another chunk for each row: with the first one always, all of them fell to one of the chip's eight parts)
    __shared__ float sums[4];
    const uint32_t chunks = (uint32_t)a.chunks;
    if (done) return;
    if (chunks % 4 == 0) {                           // every block is one row's: all four waves come here
      if (chunk / 4 == in % (chunks / 4)) back_wide<E>(a, row, x, out, 4, sums);
    } else if (chunk == in * 4u % chunks) {
      back_wide<E>(a, row, x, out, 1, sums);
    }
  }
}

// ---- host side

constexpr int kThreads = 256;
constexpr int64_t kSplitMin = 2048;       // elements of a split, at least (8,192: one row of 131,072 with k = 20 in 12.5 us, not 11.2)
constexpr int64_t kSplitBlocks = 1024;    // blocks that splitting aims at

static int lp_splits(int64_t n, int64_t V) {
  int64_t s = kSplitBlocks / n;
  if (s > V / kSplitMin) s = V / kSplitMin;
  if (s > kMaxSplits) s = kMaxSplits;
  return s < 1 ? 1 : (int)s;
}

constexpr int64_t kRowsPerLaunch = 1 << 22;

// A row's or split's kernel by the vectors that it holds (`most` elements with the start of its line).  16,384 rows of 4,096
// bf16, k = 20: 128 threads of four vectors 43 us, 256 of two 55.
template <class E, bool TOP>
static void launch_part(const LpArgs& a, int64_t most, unsigned blocks, hipStream_t st) {
  constexpr int64_t VE = Elem<E>::VE;
  if constexpr (TOP) {   // (without alternatives k_lp_small has them)
    if (a.splits == 1 && most <= 256 * VE) {
      if (most <= 64 * VE) k_lp_one<E, 64, 1, TOP><<<blocks, 64, 0, st>>>(a);
      else if (most <= 128 * VE) k_lp_one<E, 64, 2, TOP><<<blocks, 64, 0, st>>>(a);
      else k_lp_one<E, 64, 4, TOP><<<blocks, 64, 0, st>>>(a);
      return;
    }
  }
  if (a.splits == 1 && most <= 512 * VE) k_lp_one<E, 128, 4, TOP><<<blocks, 128, 0, st>>>(a);
  else if (most <= kThreads * VE) k_lp_one<E, kThreads, 1, TOP><<<blocks, kThreads, 0, st>>>(a);
  else if (most <= kThreads * 2 * VE) k_lp_one<E, kThreads, 2, TOP><<<blocks, kThreads, 0, st>>>(a);
  else if (most <= kThreads * 4 * VE) k_lp_one<E, kThreads, 4, TOP><<<blocks, kThreads, 0, st>>>(a);
  else k_lp_rows<E, kThreads, TOP><<<blocks, kThreads, 0, st>>>(a);
}

template <class E>
static void launch_rows(LpArgs a, hipStream_t st) {
  constexpr int VE = Elem<E>::VE;
  constexpr int64_t line = 128 / sizeof(E);
  a.seg = (int32_t)(((a.V + a.splits - 1) / a.splits + line - 1) / line * line);
  a.splits = (a.V + a.seg - 1) / a.seg;
  // a part's vectors start at its memory line: up to a line less one element more than its own
  const bool lines = line_shift<E>(a.x, 128) == 0 && (a.n == 1 || a.ld % line == 0);
  const int64_t most = a.seg + (lines ? 0 : line - 1);
  const int64_t steps = (most + kThreads * kVecs * VE - 1) / (kThreads * kVecs * VE);
  a.per_chunk = (int)((steps + kChunks - 1) / kChunks);
  const unsigned blocks = (unsigned)(a.n * a.splits);
  if (a.k == 0 && a.V <= 64 * kVecs * VE) {      // never split
    int lg = 0;
    while ((VE * kVecs << lg) < a.V) ++lg;
    k_lp_small<E><<<(unsigned)((((a.n - 1) >> (6 - lg)) >> 2) + 1), 256, 0, st>>>(a, lg);
    return;
  }
  if (a.k) launch_part<E, true>(a, most, blocks, st);
  else launch_part<E, false>(a, most, blocks, st);
  if (a.splits > 1) k_lp_join<<<(unsigned)a.n, kJoinThreads, 0, st>>>(a);
}

template <class E>
static void launch_back(const LpBackArgs& a0, hipStream_t st) {
  constexpr int VE = Elem<E>::VE;
  LpBackArgs a = a0;
  const bool lines = a.out_ld * (int64_t)sizeof(E) % 128 == 0 && line_shift<E>(a.out, 128) == 0;
  const int64_t most = (int64_t)a.V + (lines ? 0 : 128 / sizeof(E) - 1);
  const bool one = most <= 64 * VE;
  const int64_t per = 64 * VE * (one ? 1 : kBackVecs);
  a.chunks = (int32_t)((most + per - 1) / per);
  if (a.chunks > 16) a.chunks = (a.chunks + 3) / 4 * 4;     // whole blocks, which can share a wide row
  const int64_t rows = (int64_t)1 << 25;          // waves of a launch (a grid has less than 2^32 threads)
  const int64_t step = rows / a.chunks < 1 ? 1 : rows / a.chunks;
  for (int64_t r = 0; r < a.n; r += step) {
    const int64_t m = a.n - r < step ? a.n - r : step;
    const unsigned blocks = (unsigned)((m * a.chunks + 3) / 4);
    LpBackArgs b = a;
    b.n = r + m;
    if (one) k_lp_back<E, 1><<<blocks, 256, 0, st>>>(b, r);
    else k_lp_back<E, kBackVecs><<<blocks, 256, 0, st>>>(b, r);
  }
}

static int check_rows(const void* x, int type, int64_t n, int64_t V, int64_t ld) {
  if (!elem_type_ok(type) || n < 0 || V < 1 || ld < 0) return ELR_EINVAL;
  if (V > (int64_t)1 << 30) return ELR_EUNSUPPORTED;
  if (n > 0 && (!x || !elem_aligned(x, type))) return ELR_EINVAL;
  return ELR_OK;
}

}  // namespace elr

extern "C" int64_t elr_token_logprobs_scratch_bytes(int64_t n, int64_t V, int k) {
  if (n < 0 || V < 1 || k < 0 || k > ELR_TOPK_MAX) return -1;
  if (n == 0) return 0;
  const int64_t s = elr::lp_splits(n, V);
  if (s == 1) return 0;
  return n * s * (16 + k * 8);
}

extern "C" int elr_token_logprobs(const void* logits, int type, int64_t n, int64_t V, int64_t ld, const void* tokens,
                                  int idx64, int k, float* logprob, float* lse, float* entropy, float* top_logprob,
                                  int64_t* top_id, void* scratch, int64_t scratch_bytes, void* stream) {
  using namespace elr;
  if (int rc = check_rows(logits, type, n, V, ld)) return rc;
  if (k < 0 || k > V) return ELR_EINVAL;
  if (k > ELR_TOPK_MAX) return ELR_EUNSUPPORTED;
  if (n == 0) return ELR_OK;
  if (!tokens || !logprob || !lse || !entropy || (k && (!top_logprob || !top_id))) return ELR_EINVAL;
  const int64_t need = elr_token_logprobs_scratch_bytes(n, V, k);
  if (need > 0 && (!scratch || scratch_bytes < need || ((uintptr_t)scratch & 15u))) return ELR_ECAPACITY;
  LpArgs a{};
  a.x = logits, a.ld = ld, a.n = n, a.V = (int32_t)V, a.splits = lp_splits(n, V);
  a.tokens = tokens, a.idx64 = idx64, a.k = k;
  a.logprob = logprob, a.lse = lse, a.entropy = entropy, a.top_logprob = top_logprob, a.top_id = top_id;
  a.part = (float*)scratch;
  a.part_top = (uint64_t*)((char*)scratch + n * a.splits * 16);
  hipStream_t st = (hipStream_t)stream;
  for (int64_t r = 0; r < n; r += kRowsPerLaunch) {   // one launch unless n is huge (then a row is no longer split)
    a.n = n - r < kRowsPerLaunch ? n - r : kRowsPerLaunch;
    a.x = (const char*)logits + r * ld * elem_size(type);
    a.tokens = (const char*)tokens + r * (idx64 ? 8 : 4);
    a.logprob = logprob + r, a.lse = lse + r, a.entropy = entropy + r;
    if (k) a.top_logprob = top_logprob + r * k, a.top_id = top_id + r * k;
    switch (type) {
      case ELR_F32: launch_rows<float>(a, st); break;
      case ELR_F16: launch_rows<_Float16>(a, st); break;
      default: launch_rows<__bf16>(a, st); break;
    }
  }
  return launch_status();
}

extern "C" int elr_token_logprobs_backward(const void* logits, int type, int64_t n, int64_t V, int64_t ld,
                                           const void* tokens, int idx64, const float* lse, const float* entropy,
                                           const float* d_logprob, const float* d_entropy, const float* d_lse,
                                           void* d_logits, int64_t out_ld, void* stream) {
  using namespace elr;
  if (int rc = check_rows(logits, type, n, V, ld)) return rc;
  if (out_ld < 0 || (n > 1 && out_ld < V)) return ELR_EINVAL;
  if (n == 0) return ELR_OK;
  if (!tokens || !lse || !d_logits || !elem_aligned(d_logits, type) || (d_entropy && !entropy)) return ELR_EINVAL;
  const LpBackArgs a{logits, ld, n, (int32_t)V, 0, tokens, idx64, lse, entropy, d_logprob, d_entropy, d_lse,
                     d_logits, out_ld};
  hipStream_t st = (hipStream_t)stream;
  switch (type) {
    case ELR_F32: launch_back<float>(a, st); break;
    case ELR_F16: launch_back<_Float16>(a, st); break;
    default: launch_back<__bf16>(a, st); break;
  }
  return launch_status();
}
