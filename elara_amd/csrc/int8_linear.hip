// The product of rows in 8-bit integers with a weight in 8-bit integers:  y[i, j] = sx_i sw_j sum_k x[i, k] w[j, k], a scale for each
// row of x (token) and of w (output channel).  No counterpart in the reference.
//
// The sum is exact: int32 holds K products of at most 2^14 each for K < 2^17, which the entry point asks for.  It is widened to fp32
// (one rounding), multiplied by sx_i and by sw_j and rounded to the output's type.
#include "elr_int8.h"

namespace elr {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef u32x4 u32x4_b __attribute__((aligned(1)));

struct LinearArgs {
  const int8_t *x, *w;
  int64_t x_ld, w_ld;
  const float *x_scale, *w_scale;
  int64_t n, N;
  int32_t K;
  void* y;
};

// 16 bytes of a row at k, of which those up to K may be read; the rest are 0.
__device__ __forceinline__ u32x4 load_k(const int8_t* row, int32_t k, int32_t K) {
  if (k + 16 <= K) return *reinterpret_cast<const u32x4_b*>(row + k);
  u32x4 r{0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (k + j < K) r[j / 4] |= (uint32_t)(uint8_t)row[k + j] << (8 * (j & 3));
  return r;
}

// 16 bytes a lane from p into LDS, one lane's after the other's from `to` (the same in the wave) on; loads_done waits for them.
__device__ __forceinline__ void to_lds(const int8_t* p, int8_t* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p, (__attribute__((address_space(3))) void*)to, 16,
                                   0, 0);
}
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// What a wave's lanes wrote to LDS before is there for its own reads after.
__device__ __forceinline__ void wave_lds() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <class O>
__device__ __forceinline__ O scaled(int32_t acc, float sx, float sw) {
  return (O)((float)acc * sx * sw);
}

// A wave's outputs, MT x NT blocks of 32 tokens (a lane each) x 32 channels (four neighbouring ones a register quad), scaled and stored.
// They pass through LDS, 32 tokens at a time in a part of the wave's own, so that memory gets rows of NT * 32 channels in pieces of 16 bytes
// (stored from the registers, two bytes a lane, 8,192 x 16,384 outputs took 150 us longer than their bytes).
template <class O, int MT, int NT>
struct Outputs {
  static constexpr int kRow = NT * 32 * (int)sizeof(O) + 16, kBytes = 32 * kRow;      // LDS of a wave
  __device__ static __forceinline__ void store(const LinearArgs& a, int64_t m0, int64_t n0, const i32x16 (&acc)[MT][NT], int8_t* lds) {
    constexpr int VO = 16 / (int)sizeof(O), PIECES = NT * 32 / VO;    // outputs of a piece, pieces of a row
    typedef O O4 __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63, ch = (lane >> 5) * 4;
    f32x4 sw[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t c = n0 + j * 32 + q * 8 + ch;
#pragma unroll
        for (int t = 0; t < 4; ++t) sw[j][q][t] = a.w_scale[c + t < a.N ? c + t : a.N - 1];
      }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t row = m0 + i * 32 + (lane & 31);
      const float sx = a.x_scale[row < a.n ? row : a.n - 1];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          O4 v;
#pragma unroll
          for (int t = 0; t < 4; ++t) v[t] = scaled<O>(acc[i][j][4 * q + t], sx, sw[j][q][t]);
          *reinterpret_cast<O4*>(lds + (lane & 31) * kRow + (j * 32 + q * 8 + ch) * (int)sizeof(O)) = v;
        }
      wave_lds();
#pragma unroll
      for (int p = 0; p < 32 * PIECES / 64; ++p) {
        const int at = p * 64 + lane, r = at / PIECES, c = at % PIECES * VO;
        const int64_t to = m0 + i * 32 + r;
        const u32x4 v = *reinterpret_cast<const u32x4*>(lds + r * kRow + c * (int)sizeof(O));
        if (to < a.n) store_raw<O, false>((O*)a.y + to * a.N + n0 + c, v, a.N - n0 - c);
      }
      wave_lds();
    }
  }
};

// Tiles of BM tokens x BN channels, 64 bytes of K at a time through LDS; four waves, each a quarter of the tile in matrix instructions of
// 32 x 32 x 32.  Rows of any alignment.
template <class O, int BM, int BN>
__global__ __launch_bounds__(256) void k_linear(LinearArgs a) {
  constexpr int PITCH = 80, MT = BM / 64, NT = BN / 64;
  constexpr int kTile = (BM + BN) * PITCH, kOut = 4 * Outputs<O, MT, NT>::kBytes;
  __shared__ __attribute__((aligned(16))) int8_t lds[kTile > kOut ? kTile : kOut];
  int8_t *const lx = lds, *const lw = lds + BM * PITCH;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m0 = (int64_t)blockIdx.y * BM, n0 = (int64_t)blockIdx.x * BN;
  const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
  i32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = i32x16{};
  const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
  for (int32_t k = 0; k < a.K; k += 64) {
    u32x4 gx[MT], gw[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t row = m0 + r + i * 64;
      gx[i] = row < a.n ? load_k(a.x + row * a.x_ld, k + c, a.K) : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t row = n0 + r + j * 64;
      gw[j] = row < a.N ? load_k(a.w + row * a.w_ld, k + c, a.K) : u32x4{0, 0, 0, 0};
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i) *reinterpret_cast<u32x4*>(lx + (r + i * 64) * PITCH + c) = gx[i];
#pragma unroll
    for (int j = 0; j < NT; ++j) *reinterpret_cast<u32x4*>(lw + (r + j * 64) * PITCH + c) = gw[j];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      i32x4 fx[MT], fw[NT];
      const int at = (lane & 31) * PITCH + q * 32 + (lane >> 5) * 16;
#pragma unroll
      for (int i = 0; i < MT; ++i) fx[i] = *reinterpret_cast<const i32x4*>(lx + (wm + i * 32) * PITCH + at);
#pragma unroll
      for (int j = 0; j < NT; ++j) fw[j] = *reinterpret_cast<const i32x4*>(lw + (wn + j * 32) * PITCH + at);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[j], fx[i], acc[i][j], 0, 0, 0);
    }
  }
  __syncthreads();
  Outputs<O, MT, NT>::store(a, m0 + wm, n0 + wn, acc, lds + wave * Outputs<O, MT, NT>::kBytes);
}

// The tile of a block.  Blocks go to the 8 XCDs in turn, each with an L2 of its own: an XCD gets a compact part of the tiles, bands of 8 rows
// of tiles one column after another, so that its blocks share rows of both operands.
__device__ __forceinline__ int64_t tile_of(uint32_t b, uint32_t tiles_m, uint32_t tiles_n, uint32_t& n) {
  const uint32_t count = tiles_m * tiles_n, full = count / 8 * 8;
  const uint32_t i = b < full ? b % 8 * (count / 8) + b / 8 : b;
  const uint32_t band = 8 * tiles_n, first = i / band * 8;
  const uint32_t rows = tiles_m - first < 8 ? tiles_m - first : 8, in = i % band;
  n = in / rows;
  return first + in % rows;
}

// What rows past an end are read from, in pieces of 16 bytes.
__device__ const u32x4 kZeros = {0, 0, 0, 0};

// Tiles of BM x BN, 128 bytes of K a step, two LDS buffers.  The rows come straight from memory into LDS, 16 bytes a lane, for the next
// step while this one is multiplied; WM x WN waves, each a part of the tile in products of 32 x 32 x 32.
// A wave's load fills 8 rows of 128 bytes.  Piece c of row r lies in place c ^ (r / 2 % 8) of its row in LDS, so that the 16 lanes that read
// a piece of 16 rows at a time find them in different banks (r % 8 instead: half of LDS's cycles were conflicts).  Rows past an end repeat the last (their outputs are not stored); pieces past K
// are read from zeros.  Rows and strides are multiples of 16 bytes.
template <class O, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void k_linear_tiles(LinearArgs a, uint32_t tiles_m, uint32_t tiles_n) {
  constexpr int W = WM * WN, BK = 128, MT = BM / WM / 32, NT = BN / WN / 32;
  constexpr int LX = BM / 8 / W, LW = BN / 8 / W;          // loads of a wave for each operand
  static_assert(W * Outputs<O, MT, NT>::kBytes <= 2 * (BM + BN) * BK, "the outputs' LDS");
  extern __shared__ __attribute__((aligned(16))) int8_t tile_lds[];    // [2][BM + BN][BK]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t tn;
  const int64_t m0 = tile_of(blockIdx.x, tiles_m, tiles_n, tn) * BM, n0 = (int64_t)tn * BN;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  i32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = i32x16{};
  static_assert(W % 2 == 0, "a wave's rows: 8 of 16");
  const int piece = ((lane & 7) ^ ((wave & 1) * 4 + (lane >> 4))) * 16;      // this lane's piece of the row that it loads
  const int8_t *const x = a.x + m0 * a.x_ld, *const w = a.w + n0 * a.w_ld;
  uint32_t ox[LX], ow[LW];                                  // its rows' places behind these
#pragma unroll
  for (int l = 0; l < LX; ++l) {
    const int64_t r = (l * W + wave) * 8 + (lane >> 3);
    ox[l] = (uint32_t)((m0 + r < a.n ? r : a.n - 1 - m0) * a.x_ld) + piece;
  }
#pragma unroll
  for (int l = 0; l < LW; ++l) {
    const int64_t r = (l * W + wave) * 8 + (lane >> 3);
    ow[l] = (uint32_t)((n0 + r < a.N ? r : a.N - 1 - n0) * a.w_ld) + piece;
  }
  const auto load = [&](int32_t k, int buf) {
    int8_t* const to = tile_lds + buf * (BM + BN) * BK + wave * 8 * BK;
    if (k + BK <= a.K) {
#pragma unroll
      for (int l = 0; l < LX; ++l) to_lds(x + k + ox[l], to + l * W * 8 * BK);
#pragma unroll
      for (int l = 0; l < LW; ++l) to_lds(w + k + ow[l], to + (BM + l * W * 8) * BK);
    } else {
      const uintptr_t in = k + piece < a.K ? ~(uintptr_t)0 : 0, zeros = (uintptr_t)&kZeros & ~in;
#pragma unroll
      for (int l = 0; l < LX; ++l) to_lds((const int8_t*)(((uintptr_t)(x + k + ox[l]) & in) | zeros), to + l * W * 8 * BK);
#pragma unroll
      for (int l = 0; l < LW; ++l)
        to_lds((const int8_t*)(((uintptr_t)(w + k + ow[l]) & in) | zeros), to + (BM + l * W * 8) * BK);
    }
  };
  load(0, 0);
  int buf = 0;
  for (int32_t k = 0; k < a.K; k += BK, buf ^= 1) {
    loads_done();
    __syncthreads();
    if (k + BK < a.K) load(k + BK, buf ^ 1);
    const int8_t* const from = tile_lds + buf * (BM + BN) * BK + (lane & 31) * BK;
#pragma unroll
    for (int q = 0; q < BK / 32; ++q) {
      const int at = ((q * 2 + (lane >> 5)) ^ (lane >> 1 & 7)) * 16;
      i32x4 fx[MT], fw[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) fx[i] = *reinterpret_cast<const i32x4*>(from + (wm + i * 32) * BK + at);
#pragma unroll
      for (int j = 0; j < NT; ++j) fw[j] = *reinterpret_cast<const i32x4*>(from + (BM + wn + j * 32) * BK + at);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[j], fx[i], acc[i][j], 0, 0, 0);
    }
    // the first operands, then one of the next ones' reads behind each product
    __builtin_amdgcn_sched_group_barrier(0x100, MT + NT, 0);
#pragma unroll
    for (int q = 0; q < BK / 32 * MT * NT; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
  }
  __syncthreads();
  Outputs<O, MT, NT>::store(a, m0 + wm, n0 + wn, acc, tile_lds + wave * Outputs<O, MT, NT>::kBytes);
}

// ---- host side

constexpr int64_t kNearRows = 1 << 23;      // strides of rows whose 256 lie within 32-bit offsets

template <class O>
static void linear(const LinearArgs& b, hipStream_t st) {
  constexpr int64_t kRows = 65535 * (int64_t)128;      // gridDim.y
  for (int64_t r = 0; r < b.n; r += kRows) {
    LinearArgs a = b;
    a.n = b.n - r < kRows ? b.n - r : kRows;
    a.x = b.x + r * b.x_ld, a.x_scale = b.x_scale + r, a.y = (O*)b.y + r * b.N;
    const bool whole = a.K % 16 == 0 && a.K > 0 && (a.x_ld | a.w_ld) % 16 == 0 && (((uintptr_t)a.x | (uintptr_t)a.w) & 15u) == 0 &&
                       a.x_ld <= kNearRows && a.w_ld <= kNearRows;
    const auto tiles = [](int64_t x, int64_t t) { return (unsigned)((x + t - 1) / t); };
    if (whole && a.n > 64) {
      if (tiles(a.n, 256) * (uint64_t)tiles(a.N, 256) >= 192)
        k_linear_tiles<O, 256, 256, 2, 4><<<tiles(a.n, 256) * tiles(a.N, 256), 512, 2 * 512 * 128, st>>>(a, tiles(a.n, 256),
                                                                                                         tiles(a.N, 256));
      else
        k_linear_tiles<O, 128, 128, 2, 2><<<tiles(a.n, 128) * tiles(a.N, 128), 256, 2 * 256 * 128, st>>>(a, tiles(a.n, 128),
                                                                                                         tiles(a.N, 128));
    } else if (a.n <= 64) {
      k_linear<O, 64, 128><<<dim3(tiles(a.N, 128), 1), 256, 0, st>>>(a);
    } else {
      k_linear<O, 128, 128><<<dim3(tiles(a.N, 128), tiles(a.n, 128)), 256, 0, st>>>(a);
    }
  }
}

}  // namespace elr

extern "C" int64_t elr_int8_linear_scratch_bytes(int64_t n, int64_t N, int64_t K) {
  if (n < 0 || N < 0 || K < 0) return -1;
  return 0;
}

extern "C" int elr_int8_linear(const int8_t* x, int64_t n, int64_t K, int64_t x_ld, const float* x_scale, const int8_t* w, int64_t N,
                               int64_t w_ld, const float* w_scale, void* y, int type, void* scratch, int64_t scratch_bytes,
                               void* stream) {
  using namespace elr;
  if (n < 0 || N < 0 || K < 0 || x_ld < 0 || w_ld < 0 || !elem_type_ok(type)) return ELR_EINVAL;
  if (K >= 1 << 17 || N > (int64_t)1 << 31) return ELR_EUNSUPPORTED;
  if (n == 0 || N == 0) return ELR_OK;
  if (!x_scale || !w_scale || !y || (K > 0 && (!x || !w)) || !elem_aligned(y, type) ||
      (((uintptr_t)x_scale | (uintptr_t)w_scale) & 3u))
    return ELR_EINVAL;
  const LinearArgs a{x, w, x_ld, w_ld, x_scale, w_scale, n, N, (int32_t)K, y};
  hipStream_t st = (hipStream_t)stream;
  if (type == ELR_F32) linear<float>(a, st);
  else if (type == ELR_F16) linear<_Float16>(a, st);
  else linear<__bf16>(a, st);
  return launch_status();
}
