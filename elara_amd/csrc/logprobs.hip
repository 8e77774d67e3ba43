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
// The k likeliest (k <= 32) need no second pass over the row.  Each thread remembers the maximum of each of its chunks (in
// LDS).  Among the 64 maxima of disjoint parts of the row the k-th largest is a lower bound of the row's k-th largest
// element, so only chunks whose maximum reaches it are read again (about 64 ln(64 / (64 - k)) elements of a random row
// reach it), and their elements that reach it are ranked.  Rows with more such elements than the lists hold (many
// equal values, few unmasked ones) take the radix selection below: four counting passes, then the ties in index order.
// Order: larger first, ties by the lower id; -0 equals +0; a NaN ranks as -inf.
#include "elr_elem.h"

#include <cmath>

namespace elr {

constexpr float kLog2e = 0x1.715476p+0f;
constexpr float kExpFloor = -1e4f;
constexpr int kMaxTop = ELR_TOPK_MAX;
constexpr int kVecs = 4;        // 16-byte vectors a thread loads at a time (one chunk's step)
constexpr int kChunks = 16;     // chunk maxima a thread keeps
constexpr int kAbove = 448, kTies = 64;   // candidate lists
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
  float* part;                 // [n * splits][3] partial (m, s, t)
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

// A rank among the 64 lanes' distinct keys (0: the largest).
__device__ __forceinline__ int lane_rank(uint32_t key) {
  int rank = 0;
#pragma unroll
  for (int j = 0; j < 64; ++j) rank += (uint32_t)__builtin_amdgcn_readlane((int)key, j) > key;
  return rank;
}

// Candidates of one block: order and id packed so that a larger number comes first (ties: the lower id).
__device__ __forceinline__ uint64_t pack_cand(uint32_t o, uint32_t id) { return (uint64_t)o << 32 | (uint32_t)~id; }

template <int T>
struct TopShared {
  float gmax[T];                  // thread maxima
  uint64_t above[kAbove], ties[kTies];
  int n_above, n_ties;
  uint32_t hist[256];
  int scan[T / 64 + 1];
};

template <class E, int T>
struct RowPart {
  const E* p;        // the split's first element
  int32_t first, len;   // its place in the row and its length
};

// The elements of the part that satisfy `pred(order)`, counted over the whole block into *count, in no order.
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

// The k likeliest of a part, in order, through out(rank, packed).  cm: the thread's chunk maxima (column threadIdx.x of
// [kChunks][T]); m: the thread's maximum.
template <class E, int T, class Out>
__device__ void top_of(const LpArgs& a, const RowPart<E, T>& r, TopShared<T>& sh, const float* cm, int steps, float m,
                       const Out& out) {
  constexpr int VE = Elem<E>::VE;
  const int k = a.k, lane = threadIdx.x & 63;
  sh.gmax[threadIdx.x] = m;
  if (threadIdx.x == 0) sh.n_above = sh.n_ties = 0;
  __syncthreads();
  float g = sh.gmax[lane];
#pragma unroll
  for (int w = 1; w < T / 64; ++w) g = __builtin_fmaxf(g, sh.gmax[w * 64 + lane]);
  // the low 6 bits make the keys distinct; what they cut off only lowers the bound
  const uint32_t key = (order_of(g) & ~63u) | (uint32_t)(63 - lane);
  const uint64_t at = __builtin_amdgcn_ballot_w64(lane_rank(key) == k - 1);
  const uint32_t thr = (uint32_t)__builtin_amdgcn_readlane((int)key, __builtin_ctzll(at)) & ~63u;
  const uint32_t floor_ord = 0x007FFFFFu;   // order_of(-inf)
  const float thr_f = thr <= floor_ord ? -__builtin_inff() : value_of(thr);
  for (int c = 0; c * a.per_chunk < steps; ++c) {
    if (!(cm[c * T] >= thr_f)) continue;
    const int end = min(steps, (c + 1) * a.per_chunk);
    for (int it = c * a.per_chunk; it < end; ++it) {
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        const int64_t e = ((int64_t)(it * kVecs + u) * T + threadIdx.x) * VE;
        if (e >= r.len) break;
        const Frag<E> x = widen<E>(load_raw<E, false>(r.p + e, r.len - e, 0.0f));
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const uint32_t o = order_of(x.v[j]);
          if (o < thr || e + j >= r.len) continue;
          if ((o & ~63u) > thr) {
            const int i = atomicAdd(&sh.n_above, 1);
            if (i < kAbove) sh.above[i] = pack_cand(o, (uint32_t)(r.first + e + j));
          } else {
            const int i = atomicAdd(&sh.n_ties, 1);
            if (i < kTies) sh.ties[i] = pack_cand(o, (uint32_t)(r.first + e + j));
          }
        }
      }
    }
  }
  __syncthreads();
  int na = sh.n_above, nt = sh.n_ties;
  if (na > kAbove || nt > kTies) {
    // 16-bit types and -inf: the bound is one value, so its ties in index order complete the list
    const int want = min(k, r.len);
    uint32_t kth = thr < 0x80000000u ? thr | 63u : thr;   // (a negative value's order has ones there)
    if (na > kAbove || (sizeof(E) == 4 && thr > floor_ord)) {
      kth = radix_kth<E, T>(r, sh, want);
      if (threadIdx.x == 0) sh.n_above = 0;
      __syncthreads();
      each_elem<E, T>(r, [&](uint32_t o, uint32_t id) {   // fewer than k elements
        if (o > kth) sh.above[atomicAdd(&sh.n_above, 1)] = pack_cand(o, id);
      });
      __syncthreads();
      na = sh.n_above;
    }
    ordered_ties<E, T>(r, sh, kth, want);
    nt = sh.n_ties;
  }
  const int nc = na + nt;
  for (int i = threadIdx.x; i < nc; i += T) {
    const uint64_t c = i < na ? sh.above[i] : sh.ties[i - na];
    int rank = 0;
    for (int j = 0; j < na; ++j) rank += sh.above[j] > c;
    for (int j = 0; j < nt; ++j) rank += sh.ties[j] > c;
    if (rank < k) out(rank, c);
  }
  for (int i = nc + threadIdx.x; i < k; i += T) out(i, (uint64_t)0);   // a part shorter than k
}

__device__ __forceinline__ void write_top(const LpArgs& a, int64_t row, int rank, uint64_t c, float m, float logs,
                                          bool empty) {
  const float x = value_of((uint32_t)(c >> 32));
  a.top_logprob[row * a.k + rank] = empty ? -__builtin_inff() : (x - m) - logs;
  a.top_id[row * a.k + rank] = (int64_t)(uint32_t)~(uint32_t)c;
}

// One block of T threads per (row, split).
template <class E, int T, bool TOP>
__global__ __launch_bounds__(T) void k_lp_rows(LpArgs a) {
  constexpr int VE = Elem<E>::VE;
  __shared__ float cmax[TOP ? kChunks * T : 1];
  __shared__ Sums waves[T / 64];
  __shared__ TopShared<TOP ? T : 64> sh;
  const int64_t unit = blockIdx.x;
  const int64_t row = a.splits == 1 ? unit : unit / a.splits;
  const int split = a.splits == 1 ? 0 : (int)(unit - row * a.splits);
  RowPart<E, T> r;
  r.first = split * a.seg;
  r.len = min(a.seg, a.V - r.first);
  r.p = (const E*)a.x + row * a.ld + r.first;
  const int steps = (int)(((int64_t)r.len + (int64_t)T * kVecs * VE - 1) / ((int64_t)T * kVecs * VE));
  Sums q{-__builtin_inff(), 0.0f, 0.0f};
  float ck = -__builtin_inff();   // the current chunk's maximum
  int in_chunk = 0, chunk = 0;
  for (int it = 0; it < steps; ++it) {
    const int64_t e0 = ((int64_t)it * kVecs * T + threadIdx.x) * VE;
    u32x4 raw[kVecs];
    if ((int64_t)(it + 1) * kVecs * T * VE <= r.len) {
#pragma unroll
      for (int u = 0; u < kVecs; ++u) raw[u] = load_raw<E, true>(r.p + e0 + (int64_t)u * T * VE, VE, 0.0f);
    } else {
#pragma unroll
      for (int u = 0; u < kVecs; ++u)
        raw[u] = load_raw<E, true>(r.p + e0 + (int64_t)u * T * VE, r.len - e0 - (int64_t)u * T * VE,
                                   -__builtin_inff());
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
  for (int o = 1; o < 64; o <<= 1) {
    Sums b;
    b.m = __shfl_xor(q.m, o, 64);
    b.s = __shfl_xor(q.s, o, 64);
    b.t = __shfl_xor(q.t, o, 64);
    q = join(q, b);
  }
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = q;
    __syncthreads();
    q = waves[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) q = join(q, waves[w]);
  }
  if (a.splits == 1) {
    if (threadIdx.x == 0) {
      const int64_t tok = token_at(a, row);
      const bool has = tok >= 0 && tok < a.V;
      write_row(a, row, q, has, has ? to_f32(((const E*)a.x)[row * a.ld + tok]) : 0.0f);
    }
    if constexpr (TOP) {
      const float logs = __builtin_logf(q.s);
      top_of<E, T>(a, r, sh, cmax + threadIdx.x, steps, mine, [&](int rank, uint64_t c) {
        write_top(a, row, rank, c, q.m, logs, q.s == 0.0f);
      });
    }
  } else {
    if (threadIdx.x == 0) {
      a.part[unit * 3] = q.m;
      a.part[unit * 3 + 1] = q.s;
      a.part[unit * 3 + 2] = q.t;
    }
    if constexpr (TOP)
      top_of<E, T>(a, r, sh, cmax + threadIdx.x, steps, mine,
                   [&](int rank, uint64_t c) { a.part_top[unit * a.k + rank] = c; });
  }
}

// The splits of a row joined: lane i holds split i's sums and its sorted candidates.  A candidate below the k-th largest
// of the splits' first candidates cannot be among the row's k, which leaves at most k (k - 1) + 1.
constexpr int kJoinThreads = 256;
template <class E>
__global__ __launch_bounds__(kJoinThreads) void k_lp_join(LpArgs a) {
  __shared__ uint64_t cand[kMaxTop * (kMaxTop - 1) + 1];
  __shared__ uint64_t heads[kMaxSplits];
  __shared__ int count;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, S = a.splits;
  Sums q{-__builtin_inff(), 0.0f, 0.0f};
  if (lane < S) {
    const float* p = a.part + (row * S + lane) * 3;
    q = Sums{p[0], p[1], p[2]};
  }
  for (int o = 1; o < 64; o <<= 1) {
    Sums b;
    b.m = __shfl_xor(q.m, o, 64);
    b.s = __shfl_xor(q.s, o, 64);
    b.t = __shfl_xor(q.t, o, 64);
    q = join(q, b);
  }
  if (threadIdx.x == 0) {
    const int64_t tok = token_at(a, row);
    const bool has = tok >= 0 && tok < a.V;
    write_row(a, row, q, has, has ? to_f32(((const E*)a.x)[row * a.ld + tok]) : 0.0f);
    count = 0;
  }
  if (a.k == 0) return;
  const uint64_t* top = a.part_top + row * S * a.k;
  if (threadIdx.x < kMaxSplits) heads[threadIdx.x] = threadIdx.x < S ? top[(int64_t)threadIdx.x * a.k] : 0;
  __syncthreads();
  const uint64_t mine = heads[lane];
  int rank = 0;      // ties (absent heads are 0) by the lane
  for (int j = 0; j < S; ++j) rank += heads[j] > mine || (heads[j] == mine && j < lane);
  const uint64_t at = __builtin_amdgcn_ballot_w64(rank == a.k - 1 && lane < S);
  const uint64_t thr = at ? heads[__builtin_ctzll(at)] : 0;   // fewer than k splits: every candidate
  const int all = S * a.k;
  for (int i = threadIdx.x; i < all; i += kJoinThreads) {
    const uint64_t c = top[i];
    if (c != 0 && c >= thr) cand[atomicAdd(&count, 1)] = c;
  }
  __syncthreads();
  const int nc = count;
  const float logs = __builtin_logf(q.s);
  for (int i = threadIdx.x; i < nc; i += kJoinThreads) {
    const uint64_t c = cand[i];
    int r = 0;
    for (int j = 0; j < nc; ++j) r += cand[j] > c;
    if (r < a.k) write_top(a, row, r, c, q.m, logs, q.s == 0.0f);
  }
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

template <class E, int U>
__global__ __launch_bounds__(256) void k_lp_back(LpBackArgs a, int64_t row0) {
  constexpr int VE = Elem<E>::VE;
  const int lane = threadIdx.x & 63;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4u + (threadIdx.x >> 6)));
  const uint32_t in = wave / (uint32_t)a.chunks;
  const int chunk = (int)(wave - in * (uint32_t)a.chunks);
  const int64_t row = row0 + in;
  if (row >= a.n) return;
  const E* x = (const E*)a.x + row * a.ld;
  E* out = (E*)a.out + row * a.out_ld;
  const int64_t e0 = (int64_t)chunk * 64 * U * VE + lane * VE;
  u32x4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    raw[u] = load_raw<E, true>(x + e0 + u * 64 * VE, a.V - e0 - u * 64 * VE, -__builtin_inff());
  const int64_t tok = a.idx64 ? ((const int64_t*)a.tokens)[row] : (int64_t)((const int32_t*)a.tokens)[row];
  const bool has = tok >= 0 && tok < a.V;
  const float g = has && a.d_logprob ? a.d_logprob[row] : 0.0f;
  const float h = a.d_entropy ? a.d_entropy[row] : 0.0f;
  const float z = a.d_lse ? a.d_lse[row] : 0.0f;
  const float lse = a.lse[row];
  const float c0 = (z - g) - (a.d_entropy ? h * a.entropy[row] : 0.0f);
  const bool empty = lse < kEmptyLse;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t e = e0 + u * 64 * VE;
    if (e >= a.V) break;
    Frag<E> y = widen<E>(raw[u]);
    const int at = has && tok >= e && tok < e + VE ? (int)(tok - e) : -1;
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const float logp = clamp_low(y.v[j] - lse);
      const float d = exp_nat(logp) * __builtin_fmaf(-h, logp, c0);
      y.v[j] = empty ? 0.0f : j == at ? d + g : d;
    }
    store_raw<E, true>(out + e, narrow<E>(y), a.V - e);
  }
}

// ---- host side

constexpr int64_t kSplitMin = 8192;       // elements of a split, at least
constexpr int64_t kSplitBlocks = 1024;    // blocks that splitting aims at

static int lp_splits(int64_t n, int64_t V) {
  int64_t s = kSplitBlocks / n;
  if (s > V / kSplitMin) s = V / kSplitMin;
  if (s > kMaxSplits) s = kMaxSplits;
  return s < 1 ? 1 : (int)s;
}

constexpr int64_t kRowsPerLaunch = 1 << 22;

template <class E>
static void launch_rows(LpArgs a, hipStream_t st) {
  constexpr int VE = Elem<E>::VE;
  a.seg = ((a.V + a.splits - 1) / a.splits + VE - 1) / VE * VE;
  a.splits = (a.V + a.seg - 1) / a.seg;
  const bool small = a.V <= 64 * VE * kVecs;
  const int64_t T = small ? 64 : 256;
  const int64_t steps = (a.seg + T * kVecs * VE - 1) / (T * kVecs * VE);
  a.per_chunk = (int)((steps + kChunks - 1) / kChunks);
  const unsigned blocks = (unsigned)(a.n * a.splits);
  if (small) {
    if (a.k) k_lp_rows<E, 64, true><<<blocks, 64, 0, st>>>(a);
    else k_lp_rows<E, 64, false><<<blocks, 64, 0, st>>>(a);
  } else {
    if (a.k) k_lp_rows<E, 256, true><<<blocks, 256, 0, st>>>(a);
    else k_lp_rows<E, 256, false><<<blocks, 256, 0, st>>>(a);
  }
  if (a.splits > 1) k_lp_join<E><<<(unsigned)a.n, kJoinThreads, 0, st>>>(a);
}

template <class E>
static void launch_back(const LpBackArgs& a0, hipStream_t st) {
  constexpr int VE = Elem<E>::VE;
  LpBackArgs a = a0;
  const bool one = a.V <= 64 * VE;
  const int64_t per = 64 * VE * (one ? 1 : kBackVecs);
  a.chunks = (int32_t)((a.V + per - 1) / per);
  const int64_t rows = (int64_t)1 << 28;          // waves of a launch
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
  return (n * s * 12 + 7) / 8 * 8 + n * s * k * 8;
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
  if (need > 0 && (!scratch || scratch_bytes < need || ((uintptr_t)scratch & 7u))) return ELR_ECAPACITY;
  LpArgs a{};
  a.x = logits, a.ld = ld, a.n = n, a.V = (int32_t)V, a.splits = lp_splits(n, V);
  a.tokens = tokens, a.idx64 = idx64, a.k = k;
  a.logprob = logprob, a.lse = lse, a.entropy = entropy, a.top_logprob = top_logprob, a.top_id = top_id;
  a.part = (float*)scratch;
  a.part_top = (uint64_t*)((char*)scratch + (n * a.splits * 12 + 7) / 8 * 8);
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
