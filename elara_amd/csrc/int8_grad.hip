// A linear layer's weight gradient from its input kept in 8-bit integers:  dW[j, k] = sum_i dy[i, j] x[i, k],  x = q scale, with a scale
// for each row of x or each group of its columns; dW in fp32, [N, K] or transposed.  No counterpart in the reference.
//
// x = q scale in bf16 is exact where the scale is a power of two (q has 7 bits, bf16 holds 8), else rounded once to it.  dy in bf16 goes
// into the products as it is; fp16 values are the sum of two bf16 parts (8 and 3 bits), fp32 values of three (8 bits each), each part
// what the ones before leave of the value, exactly; so the products are exact and only the fp32 sums round.  Parts of a value that is
// not finite: the value first, then zeros.
#include "elr_int8.h"

namespace elr {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

struct WgradArgs {
  const void* dy;
  const int8_t* q;
  const float* scale;
  int64_t dy_ld, q_ld, n, per_split;
  int32_t N, K, groups, shift;
  float* out;                  // [splits][N * K]
  int transposed;
};

template <class E>
constexpr int kParts = Elem<E>::kType == ELR_F32 ? 3 : Elem<E>::kType == ELR_F16 ? 2 : 1;

// The bf16 parts of x, each cut off (not rounded: the largest fp32 values would become infinite); their sum is x.
template <int P>
__device__ __forceinline__ void split_bf16(float x, __bf16 (&p)[P]) {
  if constexpr (P == 1) {
    p[0] = (__bf16)x;
  } else {
    const bool finite = __builtin_fabsf(x) < __builtin_inff();
    p[0] = finite ? __builtin_bit_cast(__bf16, (uint16_t)(__float_as_uint(x) >> 16)) : (__bf16)x;
    float rest = x;
#pragma unroll
    for (int i = 1; i < P; ++i) {
      rest = finite ? rest - (float)p[i - 1] : 0.0f;
      p[i] = __builtin_bit_cast(__bf16, (uint16_t)(__float_as_uint(rest) >> 16));
    }
  }
}

// Tiles of 64 x 64 of dW, 32 tokens at a time; four waves, a 32 x 32 part each.
template <class E>
__global__ __launch_bounds__(256) void k_wgrad(WgradArgs a) {
  constexpr int P = kParts<E>;
  __shared__ __bf16 ly[P][32][64 + 2], lx[32][64 + 2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int32_t m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  const int64_t from = (int64_t)blockIdx.z * a.per_split, to = from + a.per_split < a.n ? from + a.per_split : a.n;
  f32x16 acc{};
  const int c = threadIdx.x & 63;
  for (int64_t i0 = from; i0 < to; i0 += 32) {
    __syncthreads();
    for (int r = wave; r < 32; r += 4) {
      const int64_t i = i0 + r;
      __bf16 p[P];
      split_bf16<P>(i < to && m0 + c < a.N ? (float)((const E*)a.dy)[i * a.dy_ld + m0 + c] : 0.0f, p);
#pragma unroll
      for (int t = 0; t < P; ++t) ly[t][r][c] = p[t];
      const bool in = i < to && n0 + c < a.K;
      lx[r][c] = (__bf16)(in ? (float)a.q[i * a.q_ld + n0 + c] * a.scale[i * a.groups + ((n0 + c) >> a.shift)] : 0.0f);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 fx;
      const int k = h * 16 + (lane >> 5) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) fx[j] = lx[k + j][wn + (lane & 31)];
#pragma unroll
      for (int t = 0; t < P; ++t) {
        bf16x8 fy;
#pragma unroll
        for (int j = 0; j < 8; ++j) fy[j] = ly[t][k + j][wm + (lane & 31)];
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fy, fx, acc, 0, 0, 0);
      }
    }
  }
  float* out = a.out + (int64_t)blockIdx.z * a.N * a.K;
  const int32_t col = n0 + wn + (lane & 31);
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const int32_t row = m0 + wm + (q >> 2) * 8 + (lane >> 5) * 4 + (q & 3);
    if (row < a.N && col < a.K) out[a.transposed ? (int64_t)col * a.N + row : (int64_t)row * a.K + col] = acc[q];
  }
}

// out = the sum of the splits' parts, in their order.
__global__ __launch_bounds__(256) void k_wgrad_join(const float* part, int splits, int64_t count, float* out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    float s = part[i];
    for (int z = 1; z < splits; ++z) s = s + part[z * count + i];
    out[i] = s;
  }
}

// ---- host side

static int64_t wgrad_splits(int64_t n, int64_t N, int64_t K) {
  const int64_t tiles = ((N + 63) / 64) * ((K + 63) / 64);
  int64_t s = (512 + tiles - 1) / tiles, most = n / 256;
  if (s > most) s = most;
  return s < 1 ? 1 : s > 64 ? 64 : s;
}

template <class E>
static void wgrad(const WgradArgs& a, int splits, hipStream_t st) {
  k_wgrad<E><<<dim3((unsigned)((a.K + 63) / 64), (unsigned)((a.N + 63) / 64), (unsigned)splits), 256, 0, st>>>(a);
}

}  // namespace elr

extern "C" int64_t elr_int8_weight_grad_scratch_bytes(int64_t n, int64_t N, int64_t K, int type) {
  if (n < 0 || N < 0 || K < 0 || !elr::elem_type_ok(type)) return -1;
  if (N == 0 || K == 0) return 0;
  const int64_t s = elr::wgrad_splits(n, N, K);
  return s > 1 ? s * N * K * 4 : 0;
}

extern "C" int elr_int8_weight_grad(const void* dy, int type, int64_t n, int64_t N, int64_t dy_ld, const int8_t* q, int64_t K,
                                    int64_t q_ld, int64_t group, const float* scale, float* dw, int transposed, void* scratch,
                                    int64_t scratch_bytes, void* stream) {
  using namespace elr;
  if (n < 0 || N < 0 || K < 0 || dy_ld < 0 || q_ld < 0 || group < 0 || !elem_type_ok(type)) return ELR_EINVAL;
  if (!int8_group_ok(group) || N > 1 << 22 || K > 1 << 22) return ELR_EUNSUPPORTED;
  if (N == 0 || K == 0) return ELR_OK;
  if (!dw || ((uintptr_t)dw & 3u) || (n > 0 && (!dy || !q || !scale || !elem_aligned(dy, type) || ((uintptr_t)scale & 3u))))
    return ELR_EINVAL;
  const int64_t splits = wgrad_splits(n, N, K);
  if (splits > 1 && (!scratch || scratch_bytes < splits * N * K * 4 || ((uintptr_t)scratch & 3u))) return ELR_ECAPACITY;
  const WgradArgs a{dy, q, scale, dy_ld, q_ld, n, ((n + splits - 1) / splits + 31) / 32 * 32, (int32_t)N, (int32_t)K,
                    (int32_t)int8_groups(K, group), int8_shift(group), splits > 1 ? (float*)scratch : dw, transposed};
  hipStream_t st = (hipStream_t)stream;
  if (type == ELR_F32) wgrad<float>(a, (int)splits, st);
  else if (type == ELR_F16) wgrad<_Float16>(a, (int)splits, st);
  else wgrad<__bf16>(a, (int)splits, st);
  if (splits > 1) k_wgrad_join<<<grid_for(N * K, 256), 256, 0, st>>>((const float*)scratch, (int)splits, N * K, dw);
  return launch_status();
}
