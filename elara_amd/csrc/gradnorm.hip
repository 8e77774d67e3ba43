// The global norm of many gradients, and clipping by it (HBM-bound).  No counterpart in the reference, whose training
// step updates without clipping.
//
//   N = (sum |g|^p)^(1/p) over every element of every tensor, p = 1, 2 or inf;  c = min(1, max_norm / (N + eps));
//   out = c g.
//
// Two launches: the first leaves one partial sum per block, the second adds the partials (every block the same ones in the
// same order, so there is no launch between that does only this) and scales.  In place with c = 1 the second ends there
// and writes nothing.  No atomics: the order of the additions depends on the sizes alone.
//
// Sums are fp64 (fp64 fma runs at fp32's rate on this chip): no overflow or underflow of squares, and the norm is exact to
// its one rounding to fp32.  A NaN gives a NaN norm; a norm of +inf gives c = 0 (so inf * 0 = NaN where a gradient was
// inf), as dividing by it does.
//
// The tensors travel in the kernel arguments, kList of them a launch: nothing is copied to the device ahead, and a captured
// graph holds its own list.  Each is cut into chunks of 16 KB; a block finds its chunk's tensor by binary search.
#include "elr_elem.h"

#include <algorithm>

namespace elr {

constexpr int kList = 144;
constexpr int kGradThreads = 256;
constexpr int kGradVecs = 4;                 // 16-byte vectors of a thread in a chunk
constexpr int64_t kPartBlocks = 2048;        // blocks (and partial sums) over all launches of a call, about
constexpr int64_t kMostElems = (int64_t)1 << 31;   // elements of one list entry

struct GradList {
  const void* in[kList];
  void* out[kList];
  uint32_t len[kList];           // elements
  uint32_t end[kList];           // chunks up to and with this tensor
  uint8_t type[kList];           // input's element type | 4 if the output is fp32 and the input is not
  int32_t count;
};

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

// The list entry that holds chunk c (wave-uniform).
__device__ __forceinline__ int entry_of(const GradList& g, uint32_t c) {
  int lo = 0, hi = g.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (c < g.end[mid]) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

template <int P, class E>
__device__ __forceinline__ Acc<P> chunk_sum(const E* p, int64_t left, Acc<P> acc) {
  constexpr int VE = Elem<E>::VE;
  u32x4 raw[kGradVecs];
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const int e = (u * kGradThreads + (int)threadIdx.x) * VE;
    raw[u] = load_raw<E, false>(p + e, left - e, 0.0f);
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
    const int type = g.type[i] & 3;
    if (type == ELR_F32) {
      const int64_t e = in * chunk_elems<float>();
      acc = chunk_sum<P>((const float*)g.in[i] + e, (int64_t)g.len[i] - e, acc);
    } else {
      const int64_t e = in * chunk_elems<__bf16>();
      if (type == ELR_F16) acc = chunk_sum<P>((const _Float16*)g.in[i] + e, (int64_t)g.len[i] - e, acc);
      else acc = chunk_sum<P>((const __bf16*)g.in[i] + e, (int64_t)g.len[i] - e, acc);
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
  int parts;
  float max_norm, eps;
  float* norm;
  int write;             // outputs other than the inputs: written also where c = 1
};

// c of every thread; the first block of the first launch writes the norm.
template <int P>
__device__ __forceinline__ float coef_of(const Clip& k, Acc<P>* lds) {
  const float x = norm_of<P>(k.part, k.parts, lds);
  if (k.norm && blockIdx.x == 0 && threadIdx.x == 0) *k.norm = x;
  const float c = k.max_norm / (x + k.eps);
  return c > 1.0f ? 1.0f : c;    // NaN stays
}

template <class E, class O>
__device__ __forceinline__ void chunk_scale(const E* p, O* o, int64_t left, float c) {
  constexpr int VE = Elem<E>::VE, VO = Elem<O>::VE;
  u32x4 raw[kGradVecs];
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const int e = (u * kGradThreads + (int)threadIdx.x) * VE;
    raw[u] = load_raw<E, true>(p + e, left - e, 0.0f);
  }
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const int e = (u * kGradThreads + (int)threadIdx.x) * VE;
    const Frag<E> x = widen<E>(raw[u]);
#pragma unroll
    for (int q = 0; q < VE / VO; ++q) {
      Frag<O> y;
#pragma unroll
      for (int j = 0; j < VO; ++j) y.v[j] = x.v[q * VO + j] * c;
      store_raw<O, true>(o + e + q * VO, narrow<O>(y), left - e - q * VO);
    }
  }
}

// The chunks in the reverse of the first launch's order: what it read last may still be in the last-level cache.
template <int P>
__global__ __launch_bounds__(kGradThreads) void k_grad_scale(GradList g, Clip k) {
  __shared__ Acc<P> lds[kGradThreads / 64];
  const float c = coef_of<P>(k, lds);
  if (c == 1.0f && !k.write) return;
  const uint32_t chunks = g.end[g.count - 1];
  for (uint32_t b = blockIdx.x; b < chunks; b += gridDim.x) {
    const uint32_t at = chunks - 1 - b;
    const int i = entry_of(g, at);
    const int64_t in = at - (i ? g.end[i - 1] : 0u);
    const int type = g.type[i];
    const int64_t e = in * ((type & 3) == ELR_F32 ? chunk_elems<float>() : chunk_elems<__bf16>());
    const int64_t left = (int64_t)g.len[i] - e;
    switch (type) {
      case ELR_F32: chunk_scale((const float*)g.in[i] + e, (float*)g.out[i] + e, left, c); break;
      case ELR_F16: chunk_scale((const _Float16*)g.in[i] + e, (_Float16*)g.out[i] + e, left, c); break;
      case ELR_BF16: chunk_scale((const __bf16*)g.in[i] + e, (__bf16*)g.out[i] + e, left, c); break;
      case ELR_F16 | 4: chunk_scale((const _Float16*)g.in[i] + e, (float*)g.out[i] + e, left, c); break;
      default: chunk_scale((const __bf16*)g.in[i] + e, (float*)g.out[i] + e, left, c); break;
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
// strided or NULL, chunks) for each.
template <class F>
static void each_launch(const elr_grad* g, int64_t n, const F& visit) {
  GradList l;
  l.count = 0;
  uint32_t chunks = 0;
  auto flush = [&] {
    if (l.count) visit(&l, (const Strided*)nullptr, (int64_t)chunks);
    l.count = 0;
    chunks = 0;
  };
  for (int64_t i = 0; i < n; ++i) {
    const elr_grad& t = g[i];
    const int64_t total = t.rows * t.cols;
    if (total == 0) continue;
    const int64_t ie = elem_size(t.type), oe = elem_size(t.out_type);
    if (!one_run(t)) {
      const Strided s{t.data, t.out, t.rows, t.cols, t.ld, t.cs, t.out_ld, t.out_cs, t.type, t.out_type == ELR_F32};
      visit((GradList*)nullptr, &s, (total + chunk_of(t.type) - 1) / chunk_of(t.type));
      continue;
    }
    for (int64_t a = 0; a < total; a += kMostElems) {
      const int64_t m = std::min(total - a, kMostElems), c = (m + chunk_of(t.type) - 1) / chunk_of(t.type);
      if (l.count == kList || (int64_t)chunks + c > INT32_MAX) flush();
      l.in[l.count] = (const char*)t.data + a * ie;
      l.out[l.count] = t.out ? (char*)t.out + a * oe : nullptr;
      l.len[l.count] = (uint32_t)m;
      l.type[l.count] = (uint8_t)(t.type | (t.out_type == ELR_F32 && t.type != ELR_F32 ? 4 : 0));
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
  each_launch(g, n, [&](const GradList*, const Strided*, int64_t c) { p.chunks += c, p.launches += 1; });
  return p;
}

template <int P>
static int run_grads(const elr_grad* g, int64_t n, bool scale, int write, float max_norm, float eps, float* norm,
                     void* scratch, int64_t bytes, hipStream_t st) {
  const GradPlan plan = grad_plan(g, n);
  double* part = (double*)scratch;
  if (bytes < plan.parts() * 8 || (plan.chunks && !scratch) || ((uintptr_t)scratch & 7u)) return ELR_ECAPACITY;
  int64_t at = 0;
  each_launch(g, n, [&](const GradList* l, const Strided* s, int64_t c) {
    const unsigned b = (unsigned)plan.blocks(c);
    if (l) k_grad_sum<P><<<b, kGradThreads, 0, st>>>(*l, part + at);
    else k_grad_sum_strided<P><<<b, kGradThreads, 0, st>>>(*s, part + at);
    at += b;
  });
  if (!scale || plan.launches == 0) {
    k_grad_norm<P><<<1, kGradThreads, 0, st>>>(part, (int)at, norm);
    return launch_status();
  }
  Clip k{part, (int)at, max_norm, eps, norm, write};
  each_launch(g, n, [&](const GradList* l, const Strided* s, int64_t c) {
    const unsigned b = (unsigned)plan.blocks(c);
    if (l) k_grad_scale<P><<<b, kGradThreads, 0, st>>>(*l, k);
    else k_grad_scale_strided<P><<<b, kGradThreads, 0, st>>>(*s, k);
    k.norm = nullptr;
  });
  return launch_status();
}

static int grads_by_norm(const elr_grad* g, int64_t n, int p, bool scale, int write, float max_norm, float eps,
                         float* norm, void* scratch, int64_t bytes, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (!norm) return ELR_EINVAL;
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
