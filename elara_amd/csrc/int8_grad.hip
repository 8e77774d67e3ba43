// A linear layer's weight gradient from its input kept in 8-bit integers:  dW[j, k] = sum_i dy[i, j] x[i, k],  x = q scale, with a scale
// for each row of x or each group of its columns; dW in fp32, [N, K] or transposed.  No counterpart in the reference.
//
// x = q scale in bf16 is exact where the scale is a power of two (q has 7 bits, bf16 holds 8), else rounded once to it: by 2^-8 of |x| at most,
// where q itself is off by up to half a step, max / 254, so by no more than x has lost already; a second part of x would double the
// products.  dy in bf16 goes into the products as it is; fp16 values are the sum of two bf16 parts (8 and 3 bits), fp32 values of three (8 bits each), so the products
// are exact and only the fp32 sums round.  (Bits of fp32 values below 2^-133 are lost; an infinity makes its outputs NaN.)
//
// Measured, tokens x N x K with groups of 128.  16,384 x 4,096 x 4,096 bf16 512-530 us, 1.05 PFLOP/s (torch's library product of two bf16
// matrices that are already wide 470-475): the matrix units are busy 46 % of the cycles, a wave waits 29 % of its time for memory, LDS or
// the barrier and 39 % for its turn to issue.  Fewer barriers (64 tokens a step instead of 32) and rows two steps ahead instead of one
// changed nothing, LDS reads have no bank conflicts.  4,096 x 4,096 x 4,096 fp16 294 us, fp32 420-450 (two and three products).
// 5,001 x 500 x 1,000 fp32 34 us: 30 for 512 blocks of ten steps and 7 to join 16 parts.  2,048 x 512 x 256 bf16 14 us.
#include "elr_int8.h"

#include <type_traits>

namespace elr {

typedef float f32x16 __attribute__((ext_vector_type(16)));

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

// Eight values in P bf16 parts, each cut off (not rounded: the largest fp32 values would become infinite) from what the ones before leave;
// the parts' sum is the value.  (An infinity leaves a NaN.)
template <int P>
__device__ __forceinline__ void split_bf16(const float (&x)[8], bf16x8 (&p)[P]) {
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = x[j];
#pragma unroll
  for (int k = 0; k < P; ++k) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j)      // the high halves of two
      w[j] = __builtin_amdgcn_perm(__float_as_uint(r[2 * j + 1]), __float_as_uint(r[2 * j]), 0x07060302u);
    p[k] = __builtin_bit_cast(bf16x8, w);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + 1 < P) r[j] = r[j] - __uint_as_float(__float_as_uint(r[j]) & 0xFFFF0000u);
  }
}

// The tile of a block.  Blocks go to the 8 XCDs in turn, each with an L2 of its own: an XCD gets a compact part of the tiles, columns of
// at most 8 tiles one after another, so that its blocks share rows of both operands.
__device__ __forceinline__ int32_t tile_of(uint32_t b, int32_t tiles_m, int32_t tiles_n) {
  const uint32_t count = (uint32_t)tiles_m * (uint32_t)tiles_n;
  const uint32_t full = count / 8 * 8;
  const uint32_t i = b < full ? b % 8 * (count / 8) + b / 8 : b;      // the i-th in the order of tiles
  const uint32_t band = 8 * (uint32_t)tiles_n, first = i / band * 8;  // bands of 8 rows of tiles, each by columns
  const uint32_t rows = (uint32_t)tiles_m - first < 8 ? (uint32_t)tiles_m - first : 8, in = i % band;
  return (int32_t)((first + in % rows) * (uint32_t)tiles_n + in / rows);
}

// Staged loads.  A token's row of a tile lies in LDS as it lies in memory (PITCH elements apart, so that four tokens' rows fall into
// different banks); the products' operands, eight tokens of a column a lane, come from LDS by its transposing read, which gives lane i of
// 16 the four tokens of column i.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

__device__ __forceinline__ bf16x8 tokens_of(const __bf16* p, int pitch) {   // p: this lane's place in the first four of eight rows
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p + 4 * pitch));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// 8 elements of a row from e on, those outside [0, valid) as 0.
template <class E>
struct Row8 {
  u32x4 v[8 / Elem<E>::VE];
};
template <class E>
__device__ __forceinline__ Row8<E> load8(const E* p, int64_t valid) {
  Row8<E> r;
#pragma unroll
  for (int i = 0; i < 8 / Elem<E>::VE; ++i) r.v[i] = load_raw<E, false>(p + i * Elem<E>::VE, valid - i * Elem<E>::VE, 0.0f);
  return r;
}

// Order of half a step: the first reads of operands, then between any two products some of the conversions for the next step (the matrix
// unit works on a product for 32 cycles, of which its issue takes 4) and of the remaining reads.
template <int PRODUCTS, int READS, int VALU>
__device__ __forceinline__ void interleave() {
  constexpr int kVmem = 0x20, kMfma = 0x8, kValu = 0x2, kRead = 0x100;
  constexpr int kFirst = READS / 2 < 12 ? READS / 2 : 12, kEach = (READS - kFirst + PRODUCTS - 1) / PRODUCTS;
  __builtin_amdgcn_sched_group_barrier(kVmem, 64, 0);
  __builtin_amdgcn_sched_group_barrier(kRead, kFirst, 0);
#pragma unroll
  for (int i = 0; i < PRODUCTS; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    if constexpr (VALU > 0) __builtin_amdgcn_sched_group_barrier(kValu, VALU, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, kEach, 0);
  }
}

// Tiles of BM x BN of dW, BT tokens a step, two LDS buffers; the rows of the next AHEAD steps are on their way into registers, from where
// they go, in bf16, into the buffer that is not multiplied.  WM x WN waves, each a part of the tile in products of 32 x 32 x 16.
// Rows in LDS are 64 bytes longer than the tile's: two neighbouring blocks of 4 tokens x 16 columns then take all 64 banks once.
//
// Edges.  No load in the loop is conditional (a branch around a load ends in a wait for it).  A piece of 8 columns that the matrix ends
// within is loaded from 8 columns before the end on, and its own columns are then stored again in their place; pieces past the end are
// loaded from there too: what LDS holds in their place reaches outputs past the end alone.  Tokens past the end are loaded from the last one and zeroed.
// NARROW: a matrix of less than 8 columns, or with rows far apart, loaded with checks.
template <class E, int BM, int BN, int BT, int WM, int WN, int AHEAD, bool NARROW>
__global__ __launch_bounds__(WM * WN * 64, BM == 128 && WM * WN == 8 ? 4 : 1) void k_wgrad(WgradArgs a, int32_t tiles_m, int32_t tiles_n) {
  constexpr int P = kParts<E>, T = WM * WN * 64, PM = BM + 32, PN = BN + 32;
  constexpr int MT = BM / WM / 32, NT = BN / WN / 32;
  constexpr int RY = BT * BM / 8 / T, RX = BT * BN / 8 / T;       // row pieces of 8 of a thread
  static_assert(RY >= 1 && RX >= 1 && RY * T * 8 == BT * BM && RX * T * 8 == BT * BN, "whole pieces");
  extern __shared__ __attribute__((aligned(16))) __bf16 lds[];     // [2][P][BT][PM], then [2][BT][PN]
  __bf16* const ly = lds;
  __bf16* const lx = lds + 2 * P * BT * PM;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int32_t tile = tile_of(blockIdx.x, tiles_m, tiles_n);
  const int32_t m0 = tile / tiles_n * BM, n0 = tile % tiles_n * BN;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const int64_t from = (int64_t)blockIdx.z * a.per_split, to = from + a.per_split < a.n ? from + a.per_split : a.n;
  f32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x16{};
  struct Step {
    Row8<E> y[RY];
    u32x2 x[RX];
    float s[RX];
  };
  const int32_t last = (int32_t)(to - from) - 1;                   // of the split's tokens, by their number in it
  // the first column of the piece at c of a matrix of `cols` columns, as it is loaded
  const auto piece = [](int32_t c, int32_t cols) { return NARROW ? (c < cols ? c : 0) : c < cols - 8 ? c : cols - 8; };
  // Places of this thread's pieces from a step's first token on: 32 bits beside an address that the step's waves share (NARROW: 64).
  typedef typename std::conditional<NARROW, int64_t, uint32_t>::type off_t;
  off_t oy[RY], ox[RX], os[RX];
  const auto places = [&](int32_t most) {      // tokens past the most-th: that one
#pragma unroll
    for (int r = 0; r < RY; ++r) {
      const int at = r * T + threadIdx.x, t = at / (BM / 8), c = m0 + at % (BM / 8) * 8;
      oy[r] = ((off_t)(t < most ? t : most) * (off_t)a.dy_ld + (off_t)piece(c, a.N)) * (off_t)sizeof(E);
    }
#pragma unroll
    for (int r = 0; r < RX; ++r) {
      const int at = r * T + threadIdx.x, t = at / (BN / 8), c = n0 + at % (BN / 8) * 8, tt = t < most ? t : most;
      ox[r] = (off_t)tt * (off_t)a.q_ld + (off_t)piece(c, a.K);
      os[r] = ((off_t)tt * (off_t)a.groups + (off_t)((c < a.K ? c : 0) >> a.shift)) * 4;      // (8 columns lie within one group)
    }
  };
  places(BT);
  const auto load = [&](Step& g, int32_t i0) {
    if (i0 + BT - 1 > last) {                  // the last steps
      i0 = i0 < last ? i0 : last;
      places(last - i0);
    }
    const char* const dy = (const char*)a.dy + (from + i0) * a.dy_ld * (int64_t)sizeof(E);
    const char* const q = (const char*)a.q + (from + i0) * a.q_ld;
    const char* const scale = (const char*)(a.scale + (from + i0) * a.groups);
#pragma unroll
    for (int r = 0; r < RY; ++r) {
      if constexpr (NARROW) {
        const int c = m0 + (r * T + threadIdx.x) % (BM / 8) * 8;
        g.y[r] = load8<E>((const E*)(dy + oy[r]), a.N - c);
      } else {
#pragma unroll
        for (int k = 0; k < 8 / Elem<E>::VE; ++k) g.y[r].v[k] = *reinterpret_cast<const u32x4_u*>(dy + oy[r] + 16 * k);
      }
    }
#pragma unroll
    for (int r = 0; r < RX; ++r) {
      if constexpr (NARROW) {
        const int c = n0 + (r * T + threadIdx.x) % (BN / 8) * 8;
        const Int8Raw<__bf16> v = int8_load<__bf16>((const int8_t*)(q + ox[r]), a.K - c);
        g.x[r] = u32x2{v.v[0], v.v[1]};
      } else {
        typedef u32x2 u32x2_b __attribute__((aligned(1)));
        g.x[r] = *reinterpret_cast<const u32x2_b*>(q + ox[r]);
      }
      g.s[r] = *reinterpret_cast<const float*>(scale + os[r]);
    }
  };
  // A step's rows in bf16, tokens past the end zero.
  struct Rows {
    bf16x8 y[RY][P], x[RX];
  };
  const auto convert = [&](Step& g, int32_t i0) {
    Rows w;
    if (i0 + BT - 1 > last) {
#pragma unroll
      for (int r = 0; r < RY; ++r)
        if (i0 + (int)(r * T + threadIdx.x) / (BM / 8) > last)
#pragma unroll
          for (int k = 0; k < 8 / Elem<E>::VE; ++k) g.y[r].v[k] = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int r = 0; r < RX; ++r)
        if (i0 + (int)(r * T + threadIdx.x) / (BN / 8) > last) g.s[r] = 0.0f;
    }
#pragma unroll
    for (int r = 0; r < RY; ++r) {
      if constexpr (P == 1) {
        w.y[r][0] = __builtin_bit_cast(bf16x8, g.y[r].v[0]);
      } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8 / Elem<E>::VE; ++i) {
          const Frag<E> f = widen<E>(g.y[r].v[i]);
#pragma unroll
          for (int j = 0; j < Elem<E>::VE; ++j) v[i * Elem<E>::VE + j] = f.v[j];
        }
        split_bf16<P>(v, w.y[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < RX; ++r) {
      f32x8 f;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = (float)(int8_t)(g.x[r][j / 4] >> (8 * (j & 3))) * g.s[r];
      w.x[r] = __builtin_convertvector(f, bf16x8);
    }
    return w;
  };
  const bool ends = !NARROW && ((m0 + BM > a.N && a.N % 8) || (n0 + BN > a.K && a.K % 8));   // a piece that a matrix ends within
  const auto store = [&](const Rows& w, int buf) {
#pragma unroll
    for (int r = 0; r < RY; ++r) {
      const int at = r * T + threadIdx.x, t = at / (BM / 8), c = at % (BM / 8) * 8;
#pragma unroll
      for (int k = 0; k < P; ++k) *reinterpret_cast<bf16x8*>(ly + ((buf * P + k) * BT + t) * PM + c) = w.y[r][k];
    }
#pragma unroll
    for (int r = 0; r < RX; ++r) {
      const int at = r * T + threadIdx.x, t = at / (BN / 8), c = at % (BN / 8) * 8;
      *reinterpret_cast<bf16x8*>(lx + (buf * BT + t) * PN + c) = w.x[r];
    }
    if (!ends) return;
    const auto again = [](__bf16* row, int c, int end, bf16x8 v) {      // columns c..end of a piece that was loaded from end - 8 on
      if (c < end && c + 8 > end)
#pragma unroll
        for (int j = 1; j < 8; ++j)
          if (end - 8 + j >= c) row[end - 8 + j] = v[j];
    };
#pragma unroll
    for (int r = 0; r < RY; ++r) {
      const int at = r * T + threadIdx.x, t = at / (BM / 8), c = at % (BM / 8) * 8;
#pragma unroll
      for (int k = 0; k < P; ++k) again(ly + ((buf * P + k) * BT + t) * PM, c, a.N - m0, w.y[r][k]);
    }
#pragma unroll
    for (int r = 0; r < RX; ++r) {
      const int at = r * T + threadIdx.x, t = at / (BN / 8), c = at % (BN / 8) * 8;
      again(lx + (buf * BT + t) * PN, c, a.K - n0, w.x[r]);
    }
  };
  // this lane's place in a 16 x 32 block of tokens and columns
  const int tr = (lane >> 5) * 8 + ((lane & 15) >> 2), tc = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
  const auto multiply = [&](int buf, int half) {
#pragma unroll
    for (int h = half * (BT / 32); h < (half + 1) * (BT / 32); ++h) {
      bf16x8 fx[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) fx[j] = tokens_of(lx + (buf * BT + h * 16 + tr) * PN + wn + j * 32 + tc, PN);
#pragma unroll
      for (int q = P - 1; q >= 0; --q) {      // the smallest parts first
        bf16x8 fy[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) fy[i] = tokens_of(ly + ((buf * P + q) * BT + h * 16 + tr) * PM + wm + i * 32 + tc, PM);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fy[i], fx[j], acc[i][j], 0, 0, 0);
      }
    }
  };
  if (from < to) {
    Step g[AHEAD];
    load(g[0], 0);
    store(convert(g[0], 0), 0);
#pragma unroll
    for (int s = 1; s < AHEAD; ++s) load(g[s], s * BT);
    __syncthreads();
    constexpr int kProducts = MT * NT * P * BT / 32, kReads = (MT * P + NT) * BT / 16;      // of half a step
    int buf = 0;
    for (int32_t i0 = 0; i0 <= last; i0 += AHEAD * BT) {
#pragma unroll
      for (int s = 0; s < AHEAD; ++s, buf ^= 1) {      // (steps past the end multiply zeros)
        const int32_t i = i0 + s * BT;
        load(g[s], i + AHEAD * BT);
        multiply(buf, 0);
        interleave<kProducts, kReads, 0>();
        Step& next = g[(s + 1) % AHEAD];
        const Rows w = convert(next, i + BT);
        multiply(buf, 1);
        interleave<kProducts, kReads, (RX * 28 + (P > 1 ? RY * 16 * P : 0) + kProducts - 1) / kProducts>();
        store(w, buf ^ 1);
        __syncthreads();
      }
    }
  }
  float* out = a.out + (int64_t)blockIdx.z * a.N * a.K;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int32_t col = n0 + wn + j * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int32_t row = m0 + wm + i * 32 + q * 8 + (lane >> 5) * 4;
        if (col >= a.K) continue;
        if (a.transposed) {
          store_raw<float, false>(out + (int64_t)col * a.N + row,
                                  __builtin_bit_cast(u32x4, f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                                                                  acc[i][j][4 * q + 3]}), a.N - row);
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (row + t < a.N) out[(int64_t)(row + t) * a.K + col] = acc[i][j][4 * q + t];
        }
      }
    }
}

// out = the sum of the splits' parts: G threads an output, each every G-th part of them in order (eight loads at a time on their way), and
// these sums one after another.  (G = 4 from 16 splits on: 16,384 tokens into 64 x 64 16 us with it, 32 with one thread an output; 512 into
// 512 x 1,024, two splits, 18 with one thread, 21 with four.)
template <int G>
__global__ __launch_bounds__(256) void k_wgrad_join(const float* part, int splits, int64_t count, float* out) {
  constexpr int C = 256 / G;
  __shared__ float sums[G][C];
  const int c = threadIdx.x % C, g = threadIdx.x / C;
  for (int64_t first = (int64_t)blockIdx.x * C; first < count; first += (int64_t)gridDim.x * C) {
    const int64_t i = first + c < count ? first + c : count - 1;
    float s = 0.0f;
    for (int z = g; z < splits; z += 8 * G) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = z + k * G < splits ? part[(int64_t)(z + k * G) * count + i] : 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s = s + v[k];
    }
    if constexpr (G > 1) {
      sums[g][c] = s;
      __syncthreads();
#pragma unroll
      for (int k = 1; k < G; ++k) s = s + sums[k][c];
    }
    if (g == 0 && first + c < count) out[i] = s;
    if constexpr (G > 1) __syncthreads();
  }
}

// ---- host side

// Tiles and splits of the tokens.  256 x 256 where such tiles alone nearly fill the chip (4,096 x 4,096 x 4,096 bf16 1,000 TFLOP/s, 128 x
// 128 about 690), bf16 gradients only: two or three parts of a step's rows do not fit the registers beside that tile's sums.  Else 128 x
// 128 with the tokens split so that about two blocks a CU run, of 256 tokens at least (5,001 x 500 x 1,000 fp32 41 us so, 46 with one
// block a CU; 20,480 x 512 x 1,024 86 and 104; 128 tokens at least: 512 x 512 x 1,024 fp32 16.5 instead of 18, 1,024 of them 22 instead
// of 21).
struct WgradPlan {
  int tile;
  int64_t tiles_m, tiles_n, splits;
};
static WgradPlan wgrad_plan(int64_t n, int64_t N, int64_t K, int type) {
  const auto tiles = [](int64_t x, int64_t t) { return (x + t - 1) / t; };
  if (type == ELR_BF16 && tiles(N, 256) * tiles(K, 256) >= 192) return {256, tiles(N, 256), tiles(K, 256), 1};
  const int64_t m = tiles(N, 128), k = tiles(K, 128), most = n / 256 < 64 ? n / 256 : 64;
  int64_t s = 512 / (m * k);
  s = s > most ? most : s;
  return {128, m, k, s < 1 ? 1 : s};
}

constexpr int64_t kNearRows = 1 << 24;      // strides of rows whose 32 lie within 32-bit offsets

template <class E, int B, int BT>
constexpr int kWgradLds = 2 * (kParts<E> + 1) * BT * (B + 32) * 2;

template <class E, int B, int BT, int WM, int WN, int AHEAD>
static void launch_wgrad(const WgradArgs& a, const WgradPlan& p, hipStream_t st) {
  static_assert(kWgradLds<E, B, BT> <= 160 << 10, "LDS of a CU");
  const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), 1, (unsigned)p.splits);
  k_wgrad<E, B, B, BT, WM, WN, AHEAD, false><<<grid, WM * WN * 64, kWgradLds<E, B, BT>, st>>>(a, (int32_t)p.tiles_m, (int32_t)p.tiles_n);
}

template <class E>
static void wgrad(const WgradArgs& a, const WgradPlan& p, hipStream_t st) {
  constexpr int AH = 2;
  if (a.N < 8 || a.K < 8 || a.dy_ld > kNearRows || a.q_ld > kNearRows)
    k_wgrad<E, 128, 128, 32, 2, 2, 1, true><<<dim3((unsigned)(p.tiles_m * p.tiles_n), 1, (unsigned)p.splits), 256, kWgradLds<E, 128, 32>, st>>>(
        a, (int32_t)p.tiles_m, (int32_t)p.tiles_n);
  else if constexpr (kParts<E> == 1)
    p.tile == 256 ? launch_wgrad<E, 256, 64, 2, 4, 1>(a, p, st) : launch_wgrad<E, 128, 32, 2, 2, AH>(a, p, st);
  else launch_wgrad<E, 128, 32, 4, 2, AH>(a, p, st);
}

}  // namespace elr

extern "C" int64_t elr_int8_weight_grad_scratch_bytes(int64_t n, int64_t N, int64_t K, int type) {
  if (n < 0 || N < 0 || K < 0 || !elr::elem_type_ok(type)) return -1;
  if (N == 0 || K == 0) return 0;
  const int64_t s = elr::wgrad_plan(n, N, K, type).splits;
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
  const WgradPlan plan = wgrad_plan(n, N, K, type);
  const int64_t splits = plan.splits;
  if (n / splits >= (int64_t)1 << 30) return ELR_EUNSUPPORTED;
  if (splits > 1 && (!scratch || scratch_bytes < splits * N * K * 4 || ((uintptr_t)scratch & 3u))) return ELR_ECAPACITY;
  const WgradArgs a{dy, q, scale, dy_ld, q_ld, n, ((n + splits - 1) / splits + 31) / 32 * 32, (int32_t)N, (int32_t)K,
                    (int32_t)int8_groups(K, group), int8_shift(group), splits > 1 ? (float*)scratch : dw, transposed};
  hipStream_t st = (hipStream_t)stream;
  if (type == ELR_F32) wgrad<float>(a, plan, st);
  else if (type == ELR_F16) wgrad<_Float16>(a, plan, st);
  else wgrad<__bf16>(a, plan, st);
  if (splits >= 16) k_wgrad_join<4><<<grid_for(N * K, 64), 256, 0, st>>>((const float*)scratch, (int)splits, N * K, dw);
  else if (splits > 1) k_wgrad_join<1><<<grid_for(N * K, 256), 256, 0, st>>>((const float*)scratch, (int)splits, N * K, dw);
  return launch_status();
}
