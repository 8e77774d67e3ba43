// The global norm of many gradients, and clipping by it (HBM-bound).  No counterpart in the reference, whose training
// step updates without clipping.
//
//   N = (sum |g|^p)^(1/p) over every element of every tensor, p = 1, 2 or inf;  c = min(1, max_norm / (N + eps));
//   out = c g.
//
// The first launches leave one partial sum per block.  A list of few chunks is then scaled by one launch whose blocks each
// add the same partials in the same order; a longer one has a launch for the addition and then a block per chunk.  In place
// with c = 1 the scaling ends there and writes nothing.  No atomics: the order of the additions depends on the sizes and
// alignments alone.
//
// Sums are fp64: no overflow or underflow of squares, and the norm is exact to its one rounding to fp32.  It costs nothing
// (fp32 sums: 131 us against 133 for 717 MB).  A NaN gives a NaN norm; a norm of +inf gives c = 0 (so inf * 0 = NaN where a
// gradient was inf), as dividing by it does, unless max_norm is +inf too; no gradient and eps = 0 gives c = 1.
//
// The tensors travel in the kernel arguments, kList of them a launch: nothing is copied to the device ahead, and a captured
// graph holds its own list.  Each is cut into chunks of 16 KB.  A tensor that is not one run of memory has launches of its own,
// a thread an element with a 64-bit division for its place: 8,192 x 8,192 in rows 8,256 apart fp32 105 us for the norm and 234
// with the scaling (48 and 130 as one run), bf16 102 and 206 (28 and 74).
//
// Measured: 641 MB of bf16 gradients packed next to one another and 77 MB of fp32 rows, into fp32 (240 tensors): sum 125 us
// (5.7 TB/s), scaling 322 us (6.4 TB/s; the sum's last reads are still in the last-level cache when the scaling, which goes
// backwards, begins).  What brought it there from 928 us: whole memory lines (451 -> 385 us of scaling with aligned stores
// and a chunk a block), lines of 256 bytes for the widened output (-> 365), and a chunk's bounds tested once instead of at
// each access (-> 322).
#include "elr_elem.h"

#include <algorithm>

namespace elr {

constexpr int kList = 136;
constexpr int kGradThreads = 256;
constexpr int kGradVecs = 4;                 // 16-byte vectors of a thread in a chunk
constexpr int64_t kPartBlocks = 8192;        // blocks (and partial sums) over all launches of a call, about (2048: 12 % slower)
constexpr int64_t kScaleBlocks = 1 << 22;    // blocks of one scaling launch, at most
constexpr int64_t kOwnBlocks = 1024;         // chunks up to which the scaling's blocks add the partials themselves
constexpr int64_t kMostElems = (int64_t)1 << 31;   // elements of one list entry

// Entries of 4 and 8 bytes only.  With a byte array here the compiler formed (arguments + i) + 7 i as the address of in[i]
// for a scalar load, which drops the two low bits of each part and so read half of one pointer and half of the next (a
// memory violation): every part of such an address has to be a multiple of four.
struct GradList {
  const void* in[kList];
  void* out[kList];
  uint32_t len[kList];           // elements
  uint32_t end[kList];           // chunks up to and with this tensor
  uint32_t type[kList];          // input's element type | 4 if the output is fp32 and the input is not
  int32_t count;
};
static_assert(sizeof(GradList) + 64 <= 4096, "kernel arguments");

template <class E>
constexpr int chunk_elems() { return kGradThreads * kGradVecs * Elem<E>::VE; }
static int64_t chunk_of(int type) { return type == ELR_F32 ? chunk_elems<float>() : chunk_elems<__bf16>(); }

// P: 1, 2, or 0 for the maximum, which needs no more than fp32.
template <int P>
struct AccOf {
  typedef double type;
};
template <>
struct AccOf<0> {
  typedef float type;
};
template <int P>
using Acc = typename AccOf<P>::type;

template <int P>
__device__ __forceinline__ Acc<P> accum(Acc<P> acc, float x) {
  if constexpr (P == 2) return __builtin_fma((double)x, (double)x, acc);
  else if constexpr (P == 1) return acc + (double)__builtin_fabsf(x);
  else return max_nan(acc, __builtin_fabsf(x));
}
template <int P>
__device__ __forceinline__ Acc<P> merge(Acc<P> a, Acc<P> b) {
  if constexpr (P == 0) return max_nan(a, b);
  else return a + b;
}

// A block's result in every thread; fixed order.
template <int P>
__device__ __forceinline__ Acc<P> block_merge(Acc<P> x, Acc<P>* lds) {
  for (int o = 1; o < 64; o <<= 1) x = merge<P>(x, __shfl_xor(x, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  x = lds[0];
#pragma unroll
  for (int w = 1; w < kGradThreads / 64; ++w) x = merge<P>(x, lds[w]);
  return x;
}

// The list entry that holds chunk c: every lane compares its share of the chunk ends (one load's latency, where a binary
// search would be eight loads, one after another).
__device__ __forceinline__ int entry_of(const GradList& g, uint32_t c) {
  const int lane = threadIdx.x & 63;
  int n = 0;
#pragma unroll
  for (int q = 0; q < (kList + 63) / 64; ++q) {
    const int i = q * 64 + lane;
    const uint32_t end = i < g.count ? g.end[i] : UINT32_MAX;
    n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(end <= c));
  }
  return n;
}

// Chunks are laid from a memory line's start, the sum's from the input's and the scaling's from the output's: with a wave's
// 16-byte accesses off the lines by the tensor's own offset, tensors packed next to one another were 5 to 18 % slower than
// padded ones (160 M bf16 elements into fp32: 163 and 177 us against 150).
constexpr int kInLine = 128, kOutLine = 256;   // (256: 16-bit input then starts on 128 too when it widens to fp32)

template <int P, class E>
__device__ __forceinline__ Acc<P> chunk_sum(const void* in, int64_t chunk, int64_t len, Acc<P> acc) {
  constexpr int VE = Elem<E>::VE;
  const E* p = (const E*)in;
  const int64_t c0 = chunk * chunk_elems<E>() - line_shift<E>(in, kInLine), e0 = c0 + (int)threadIdx.x * VE;
  u32x4 raw[kGradVecs];
  if (c0 >= 0 && c0 + chunk_elems<E>() <= len) {
#pragma unroll
    for (int u = 0; u < kGradVecs; ++u) raw[u] = load_raw<E, false>(p + e0 + u * kGradThreads * VE, VE, 0.0f);
  } else {
#pragma unroll
    for (int u = 0; u < kGradVecs; ++u) raw[u] = load_part<E, false>(p, e0 + u * kGradThreads * VE, len, 0.0f);
  }
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const Frag<E> x = widen<E>(raw[u]);
#pragma unroll
    for (int j = 0; j < VE; ++j) acc = accum<P>(acc, x.v[j]);
  }
  return acc;
}

template <int P>
__global__ __launch_bounds__(kGradThreads) void k_grad_sum(GradList g, double* part) {
  __shared__ Acc<P> lds[kGradThreads / 64];
  const uint32_t chunks = g.end[g.count - 1];
  Acc<P> acc = 0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = entry_of(g, c);
    const int64_t in = c - (i ? g.end[i - 1] : 0u);
    const int64_t len = g.len[i];
    switch (g.type[i] & 3u) {
      case ELR_F32: acc = chunk_sum<P, float>(g.in[i], in, len, acc); break;
      case ELR_F16: acc = chunk_sum<P, _Float16>(g.in[i], in, len, acc); break;
      default: acc = chunk_sum<P, __bf16>(g.in[i], in, len, acc); break;
    }
  }
  acc = block_merge<P>(acc, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = (double)acc;
}

// rows x cols elements at strides ld and cs (elements): tensors that are not one run of memory.
struct Strided {
  const void* in;
  void* out;
  int64_t rows, cols, ld, cs, out_ld, out_cs;
  int type, out_f32;
};

__device__ __forceinline__ float elem_at(const Strided& s, int64_t i) {
  const int64_t r = i / s.cols, at = r * s.ld + (i - r * s.cols) * s.cs;
  return s.type == ELR_F32   ? ((const float*)s.in)[at]
         : s.type == ELR_F16 ? to_f32(((const _Float16*)s.in)[at])
                             : to_f32(((const __bf16*)s.in)[at]);
}

template <int P>
__global__ __launch_bounds__(kGradThreads) void k_grad_sum_strided(Strided s, double* part) {
  __shared__ Acc<P> lds[kGradThreads / 64];
  const int64_t n = s.rows * s.cols;
  Acc<P> acc = 0;
  for (int64_t i = (int64_t)blockIdx.x * kGradThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kGradThreads)
    acc = accum<P>(acc, elem_at(s, i));
  acc = block_merge<P>(acc, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = (double)acc;
}

// The norm from the partials, the same in every thread of every block.
template <int P>
__device__ __forceinline__ float norm_of(const double* part, int parts, Acc<P>* lds) {
  Acc<P> x = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < parts; i += kGradThreads) x = merge<P>(x, (Acc<P>)part[i]);
  x = block_merge<P>(x, lds);
  if constexpr (P == 2) return (float)__builtin_sqrt(x);
  else return (float)x;
}

template <int P>
__global__ __launch_bounds__(kGradThreads) void k_grad_norm(const double* part, int parts, float* norm) {
  __shared__ Acc<P> lds[kGradThreads / 64];
  const float x = norm_of<P>(part, parts, lds);
  if (threadIdx.x == 0) *norm = x;
}

struct Clip {
  const double* part;
  int parts;             // 0: *norm is there already
  float max_norm, eps;
  float* norm;
  int write;             // outputs other than the inputs: written also where c = 1
};

// c of every thread.  With parts, each block adds them up and the first writes the norm.
template <int P>
__device__ __forceinline__ float coef_of(const Clip& k, Acc<P>* lds) {
  float x;
  if (k.parts) {
    x = norm_of<P>(k.part, k.parts, lds);
    if (blockIdx.x == 0 && threadIdx.x == 0) *k.norm = x;
  } else {
    x = *k.norm;
  }
  const float d = x + k.eps;
  if (d == 0.0f || (d == __builtin_inff() && k.max_norm == d)) return 1.0f;   // nothing to scale, or no bound: not 0/0, inf/inf
  const float c = k.max_norm / d;
  return c > 1.0f ? 1.0f : c;    // NaN stays
}

template <class E, class O, bool ALL>
__device__ __forceinline__ void scale_vecs(const E* p, O* o, int64_t e0, int64_t len, float c) {
  constexpr int N = Elem<O>::VE, V = chunk_elems<E>() / (kGradThreads * N);   // elements of a store, stores of a thread
  Frag<O> x[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int64_t e = e0 + v * kGradThreads * N;
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
      const f32x4 a = load4<E, true>(p + (ALL ? e + 4 * q : 0), ALL ? 0 : e + 4 * q, ALL ? 4 : len);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[v].v[4 * q + j] = a[j];
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int64_t e = e0 + v * kGradThreads * N;
#pragma unroll
    for (int j = 0; j < N; ++j) x[v].v[j] = x[v].v[j] * c;
    if constexpr (ALL) store_raw<O, true>(o + e, narrow<O>(x[v]), N);
    else store_part<O, true>(o, e, len, narrow<O>(x[v]));
  }
}

template <class E, class O>
__device__ __forceinline__ void chunk_scale(const void* in, void* out, int64_t chunk, int64_t len, float c) {
  const int64_t c0 = chunk * chunk_elems<E>() - line_shift<O>(out, kOutLine);
  const int64_t e0 = c0 + (int)threadIdx.x * Elem<O>::VE;
  if (c0 >= 0 && c0 + chunk_elems<E>() <= len) scale_vecs<E, O, true>((const E*)in, (O*)out, e0, len, c);
  else scale_vecs<E, O, false>((const E*)in, (O*)out, e0, len, c);
}

// The chunks in the reverse of the sum's order (the lists come reversed): what it read last may still be in the last-level
// cache.
template <int P>
__global__ __launch_bounds__(kGradThreads) void k_grad_scale(GradList g, Clip k) {
  __shared__ Acc<P> lds[kGradThreads / 64];
  const float c = coef_of<P>(k, lds);
  if (c == 1.0f && !k.write) return;
  const uint32_t chunks = g.end[g.count - 1];
  for (uint32_t at = blockIdx.x; at < chunks; at += gridDim.x) {
    const int i = entry_of(g, at);
    const int64_t in = g.end[i] - 1 - at;
    const int64_t len = g.len[i];
    switch (g.type[i]) {
      case ELR_F32: chunk_scale<float, float>(g.in[i], g.out[i], in, len, c); break;
      case ELR_F16: chunk_scale<_Float16, _Float16>(g.in[i], g.out[i], in, len, c); break;
      case ELR_BF16: chunk_scale<__bf16, __bf16>(g.in[i], g.out[i], in, len, c); break;
      case ELR_F16 | 4: chunk_scale<_Float16, float>(g.in[i], g.out[i], in, len, c); break;
      default: chunk_scale<__bf16, float>(g.in[i], g.out[i], in, len, c); break;
    }
  }
}

template <int P>
__global__ __launch_bounds__(kGradThreads) void k_grad_scale_strided(Strided s, Clip k) {
  __shared__ Acc<P> lds[kGradThreads / 64];
  const float c = coef_of<P>(k, lds);
  if (c == 1.0f && !k.write) return;
  const int64_t n = s.rows * s.cols;
  for (int64_t i = (int64_t)blockIdx.x * kGradThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kGradThreads) {
    const int64_t r = i / s.cols, at = r * s.out_ld + (i - r * s.cols) * s.out_cs;
    const float y = elem_at(s, i) * c;
    if (s.out_f32 || s.type == ELR_F32) ((float*)s.out)[at] = y;
    else if (s.type == ELR_F16) ((_Float16*)s.out)[at] = (_Float16)y;
    else ((__bf16*)s.out)[at] = (__bf16)y;
  }
}

// ---- host side

static bool one_run(const elr_grad& g) {
  auto run = [&](int64_t ld, int64_t cs) { return (g.cols == 1 || cs == 1) && (g.rows == 1 || ld == g.cols); };
  return run(g.ld, g.cs) && (!g.out || run(g.out_ld, g.out_cs));
}

// The call's launches: lists of contiguous tensors (filled one at a time) and strided ones.  visit(list or NULL,
// strided or NULL, chunks) for each.  back: from the last tensor to the first.
template <class F>
static void each_launch(const elr_grad* g, int64_t n, bool back, const F& visit) {
  GradList l;
  l.count = 0;
  uint32_t chunks = 0;
  auto flush = [&] {
    if (l.count) visit((const GradList*)&l, (const Strided*)nullptr, (int64_t)chunks);
    l.count = 0;
    chunks = 0;
  };
  for (int64_t q = 0; q < n; ++q) {
    const elr_grad& t = g[back ? n - 1 - q : q];
    const int64_t total = t.rows * t.cols;
    if (total == 0) continue;
    const int64_t ie = elem_size(t.type), oe = elem_size(t.out_type);
    if (!one_run(t)) {
      const Strided s{t.data, t.out, t.rows, t.cols, t.ld, t.cs, t.out_ld, t.out_cs, t.type, t.out_type == ELR_F32};
      visit((const GradList*)nullptr, &s, (total + chunk_of(t.type) - 1) / chunk_of(t.type));
      continue;
    }
    const int64_t parts = (total + kMostElems - 1) / kMostElems;
    for (int64_t p = 0; p < parts; ++p) {
      const int64_t a = (back ? parts - 1 - p : p) * kMostElems, m = std::min(total - a, kMostElems);
      const char* out = t.out ? (const char*)t.out + a * oe : nullptr;
      const char* in = (const char*)t.data + a * ie;
      const int64_t shift = std::max(line_shift<char>(in, kInLine) / ie, line_shift<char>(out, kOutLine) / oe);
      const int64_t c = (m + shift + chunk_of(t.type) - 1) / chunk_of(t.type);
      if (l.count == kList || (int64_t)chunks + c > INT32_MAX) flush();
      l.in[l.count] = in;
      l.out[l.count] = (void*)out;
      l.len[l.count] = (uint32_t)m;
      l.type[l.count] = (uint32_t)(t.type | (t.out_type == ELR_F32 && t.type != ELR_F32 ? 4 : 0));
      chunks += (uint32_t)c;
      l.end[l.count++] = chunks;
    }
  }
  flush();
}

static int check_grads(const elr_grad* g, int64_t n, bool outs) {
  if (n < 0 || (n && !g)) return ELR_EINVAL;
  for (int64_t i = 0; i < n; ++i) {
    const elr_grad& t = g[i];
    if (t.rows < 0 || t.cols < 0 || !elem_type_ok(t.type) || !elem_type_ok(t.out_type)) return ELR_EINVAL;
    if (t.rows == 0 || t.cols == 0) continue;
    if (t.rows > INT64_MAX / 8 / t.cols) return ELR_EINVAL;
    if (!t.data || !elem_aligned(t.data, t.type)) return ELR_EINVAL;
    if (t.out_type != t.type && t.out_type != ELR_F32) return ELR_EUNSUPPORTED;
    if (outs && (!t.out || !elem_aligned(t.out, t.out_type) || (t.out == t.data && t.out_type != t.type)))
      return ELR_EINVAL;
  }
  return ELR_OK;
}

struct GradPlan {
  int64_t chunks = 0, launches = 0;
  int64_t blocks(int64_t c) const {   // of a launch of c chunks: its share of kPartBlocks
    const int64_t b = chunks <= kPartBlocks ? c : (c * kPartBlocks + chunks - 1) / chunks;
    return std::max<int64_t>(1, std::min(b, c));
  }
  int64_t parts() const { return std::min(chunks, kPartBlocks) + launches; }   // at most
};
static GradPlan grad_plan(const elr_grad* g, int64_t n) {
  GradPlan p;
  each_launch(g, n, false, [&](const GradList*, const Strided*, int64_t c) { p.chunks += c, p.launches += 1; });
  return p;
}

template <int P>
static int run_grads(const elr_grad* g, int64_t n, bool scale, int write, float max_norm, float eps, float* norm,
                     void* scratch, int64_t bytes, hipStream_t st) {
  const GradPlan plan = grad_plan(g, n);
  double* part = (double*)scratch;
  if (bytes < plan.parts() * 8 || (plan.chunks && !scratch) || ((uintptr_t)scratch & 7u)) return ELR_ECAPACITY;
  int64_t at = 0;
  each_launch(g, n, false, [&](const GradList* l, const Strided* s, int64_t c) {
    const unsigned b = (unsigned)plan.blocks(c);
    if (l) k_grad_sum<P><<<b, kGradThreads, 0, st>>>(*l, part + at);
    else k_grad_sum_strided<P><<<b, kGradThreads, 0, st>>>(*s, part + at);
    at += b;
  });
  // Where the partials are few, every scaling block adds them up by itself; otherwise that is a launch.
  const bool own = scale && plan.launches > 0 && plan.chunks <= kOwnBlocks;
  if (!own) k_grad_norm<P><<<1, kGradThreads, 0, st>>>(part, (int)at, norm);
  if (!scale) return launch_status();
  const Clip k{part, own ? (int)at : 0, max_norm, eps, norm, write};
  each_launch(g, n, true, [&](const GradList* l, const Strided* s, int64_t c) {
    const unsigned b = (unsigned)std::min(c, kScaleBlocks);
    if (l) k_grad_scale<P><<<b, kGradThreads, 0, st>>>(*l, k);
    else k_grad_scale_strided<P><<<b, kGradThreads, 0, st>>>(*s, k);
  });
  return launch_status();
}

static int grads_by_norm(const elr_grad* g, int64_t n, int p, bool scale, int write, float max_norm, float eps,
                         float* norm, void* scratch, int64_t bytes, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (!norm || !(max_norm >= 0.0f) || !(eps >= 0.0f)) return ELR_EINVAL;
  if (int rc = check_grads(g, n, scale)) return rc;
  switch (p) {
    case 0: return run_grads<0>(g, n, scale, write, max_norm, eps, norm, scratch, bytes, st);
    case 1: return run_grads<1>(g, n, scale, write, max_norm, eps, norm, scratch, bytes, st);
    case 2: return run_grads<2>(g, n, scale, write, max_norm, eps, norm, scratch, bytes, st);
    default: return ELR_EUNSUPPORTED;
  }
}

}  // namespace elr

extern "C" int64_t elr_grad_norm_scratch_bytes(const elr_grad* grads, int64_t n) {
  if (elr::check_grads(grads, n, false) != ELR_OK) return -1;
  return elr::grad_plan(grads, n).parts() * 8;
}

extern "C" int elr_grad_norm(const elr_grad* grads, int64_t n, int p, float* norm, void* scratch,
                             int64_t scratch_bytes, void* stream) {
  return elr::grads_by_norm(grads, n, p, false, 0, 0.0f, 0.0f, norm, scratch, scratch_bytes, stream);
}

extern "C" int elr_clip_grad_norm(const elr_grad* grads, int64_t n, int p, float max_norm, float eps, float* norm,
                                  void* scratch, int64_t scratch_bytes, void* stream) {
  bool in_place = true;
  for (int64_t i = 0; grads && i < n; ++i) in_place = in_place && (grads[i].out == grads[i].data || !grads[i].rows || !grads[i].cols);
  return elr::grads_by_norm(grads, n, p, true, !in_place, max_norm, eps, norm, scratch, scratch_bytes, stream);
}
