// The product of rows in 8-bit integers with a weight in 8-bit integers:  y[i, j] = sx_i sw_j sum_k x[i, k] w[j, k], a scale for each
// row of x (token) and of w (output channel).  No counterpart in the reference.
//
// The sum is exact: int32 holds K products of at most 2^14 each for K < 2^17, which the entry point asks for.  It is widened to fp32
// (one rounding), multiplied by sx_i and by sw_j and rounded to the output's type.
//
// Measured (bf16 out but where said).  8,192 x 4,096 x 16,384 (tokens, K, channels) 515-527 us, 2.1 P operations/s, of which the outputs
// through memory are about 50: a longer K adds 2.6 P/s (each 4,096 of it 0.42 ms), near what this card's clock leaves of the matrix units'
// 5 P/s under that load; the library's own int8 product takes 550-575 us for the int32 sums alone.  Operands of zeros: 440 us, so the
// clock is part of it.  64 tokens x 4,096 x 16,384 26-27 us, 128 28-29; 301 x 1,000 x 20,011 (rows of no multiple of 16 bytes) into fp32 23 us, 1,024
// columns instead 16.  4 tokens x 4,096 x 16,384 15-18 us (67 MB of weight: 4.4 TB/s in turn over three weights), x 4,096 x 4,096 7, of
// which a call and its launch are 4-5.
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

// 16 bytes of a row at k, of which those up to K may be read; the rest are 0.  A row's end: its last 16 bytes, shifted (no branch, no
// loads byte by byte but for rows of less than 16).
__device__ __forceinline__ u32x4 load_k(const int8_t* row, int32_t k, int32_t K) {
  if (K >= 16) {
    const int32_t at = k < K - 16 ? k : K - 16, s = k - at;
    const unsigned __int128 v = __builtin_bit_cast(unsigned __int128, *reinterpret_cast<const u32x4_b*>(row + at));
    return __builtin_bit_cast(u32x4, s < 16 ? v >> (8 * s) : (unsigned __int128)0);
  }
  u32x4 r{0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 15; ++j)
    if (k + j < K) r[j / 4] |= (uint32_t)(uint8_t)row[k + j] << (8 * (j & 3));
  return r;
}

// 16 bytes a lane from p into LDS, one lane's after the other's from `to` (the same in the wave) on; loads_done waits for all of the
// wave's.
__device__ __forceinline__ void to_lds(const int8_t* p, int8_t* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p, (__attribute__((address_space(3))) void*)to, 16,
                                   0, 0);
}
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }      // vmcnt(0)

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

// Tiles of BM tokens x BN channels for rows of any alignment, 128 bytes of K a step, two LDS buffers; the next step's rows are on their
// way into registers while this one is multiplied.  Four waves, each a quarter of the tile in products of 32 x 32 x 32.  Rows past an end repeat
// the last (their outputs are not stored).
template <class O, int BM, int BN>
__global__ __launch_bounds__(256) void k_linear(LinearArgs a) {
  constexpr int BK = 128, PITCH = BK + 16, MT = BM / 64, NT = BN / 64;
  constexpr int kTile = (BM + BN) * PITCH, kOut = 4 * Outputs<O, MT, NT>::kBytes;
  __shared__ __attribute__((aligned(16))) int8_t lds[2 * kTile > kOut ? 2 * kTile : kOut];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m0 = (int64_t)blockIdx.y * BM, n0 = (int64_t)blockIdx.x * BN;
  const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
  i32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = i32x16{};
  const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 16;
  constexpr int LX = BM / 32, LW = BN / 32;
  const int8_t* p[LX + LW];
#pragma unroll
  for (int i = 0; i < LX; ++i) p[i] = a.x + (m0 + r + i * 32 < a.n ? m0 + r + i * 32 : a.n - 1) * a.x_ld;
#pragma unroll
  for (int j = 0; j < LW; ++j) p[LX + j] = a.w + (n0 + r + j * 32 < a.N ? n0 + r + j * 32 : a.N - 1) * a.w_ld;
  u32x4 g[LX + LW];
  const auto load = [&](int32_t k) {
    if (k + BK <= a.K) {
#pragma unroll
      for (int i = 0; i < LX + LW; ++i) g[i] = *reinterpret_cast<const u32x4_b*>(p[i] + k + c);
    } else {
#pragma unroll
      for (int i = 0; i < LX + LW; ++i) g[i] = load_k(p[i], k + c, a.K);
    }
  };
  const auto store = [&](int8_t* to) {
#pragma unroll
    for (int i = 0; i < LX + LW; ++i) *reinterpret_cast<u32x4*>(to + (r + i * 32) * PITCH + c) = g[i];
  };
  load(0);
  store(lds);
  int8_t* buf = lds;
  for (int32_t k = 0; k < a.K; k += BK) {
    __syncthreads();
    const bool more = k + BK < a.K;
    if (more) load(k + BK);
#pragma unroll
    for (int q = 0; q < BK / 32; ++q) {
      i32x4 fx[MT], fw[NT];
      const int8_t* const at = buf + (lane & 31) * PITCH + q * 32 + (lane >> 5) * 16;
#pragma unroll
      for (int i = 0; i < MT; ++i) fx[i] = *reinterpret_cast<const i32x4*>(at + (wm + i * 32) * PITCH);
#pragma unroll
      for (int j = 0; j < NT; ++j) fw[j] = *reinterpret_cast<const i32x4*>(at + (BM + wn + j * 32) * PITCH);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[j], fx[i], acc[i][j], 0, 0, 0);
    }
    buf = buf == lds ? lds + kTile : lds;
    if (more) store(buf);
  }
  __syncthreads();
  Outputs<O, MT, NT>::store(a, m0 + wm, n0 + wn, acc, lds + wave * Outputs<O, MT, NT>::kBytes);
}

// Few tokens (16 TB at most): the weight is read once, straight into registers, and there are no tiles to share.  Eight waves a block: `kw` of
// them take turns at 64 U bytes of K for the same 16 C channels, the others take further channels; the weight's rows are the products'
// first operand (16 x 16 x 64), so that a lane holds four neighbouring channels of a token.  The waves' sums, of whole numbers, are added in
// LDS.  Rows of any alignment; those past an end repeat the last.
template <class O, int TB, int C>
__global__ __launch_bounds__(512) void k_linear_few(LinearArgs a, int32_t kw) {
  constexpr int U = 8 / C;                       // steps of K in flight
  __shared__ __attribute__((aligned(16))) int32_t sums[8 * 16 * C * 16 * TB];      // [channels of the block][16 TB]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int group = wave / kw, channels = 16 * C * (8 / kw);
  const int64_t n0 = (int64_t)blockIdx.x * channels;
  for (int i = threadIdx.x; i < channels * 16 * TB; i += 512) sums[i] = 0;
  __syncthreads();
  const int32_t c = (lane >> 4) * 16;
  const int8_t *pw[C], *px[TB];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int64_t row = n0 + group * 16 * C + i * 16 + (lane & 15);
    pw[i] = a.w + (row < a.N ? row : a.N - 1) * a.w_ld + c;
  }
#pragma unroll
  for (int t = 0; t < TB; ++t) px[t] = a.x + (t * 16 + (lane & 15) < a.n ? t * 16 + (lane & 15) : a.n - 1) * a.x_ld + c;
  i32x4 acc[C][TB];
#pragma unroll
  for (int i = 0; i < C; ++i)
#pragma unroll
    for (int t = 0; t < TB; ++t) acc[i][t] = i32x4{0, 0, 0, 0};
  const auto multiply = [&](const i32x4 (&w)[C], const i32x4 (&x)[TB]) {
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
      for (int t = 0; t < TB; ++t) acc[i][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], x[t], acc[i][t], 0, 0, 0);
  };
  for (int32_t k = wave % kw * U * 64; k < a.K; k += kw * U * 64) {
    if (k + U * 64 <= a.K) {
      i32x4 w[U][C], x[U][TB];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < C; ++i) w[u][i] = __builtin_bit_cast(i32x4, *(const u32x4_b*)(pw[i] + k + u * 64));
#pragma unroll
        for (int t = 0; t < TB; ++t) x[u][t] = __builtin_bit_cast(i32x4, *(const u32x4_b*)(px[t] + k + u * 64));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) multiply(w[u], x[u]);
    } else {
      for (int32_t e = k; e < a.K; e += 64) {
        i32x4 w[C], x[TB];
#pragma unroll
        for (int i = 0; i < C; ++i) w[i] = __builtin_bit_cast(i32x4, load_k(pw[i] - c, e + c, a.K));
#pragma unroll
        for (int t = 0; t < TB; ++t) x[t] = __builtin_bit_cast(i32x4, load_k(px[t] - c, e + c, a.K));
        multiply(w, x);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < C; ++i)
#pragma unroll
    for (int t = 0; t < TB; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        atomicAdd(&sums[(t * 16 + (lane & 15)) * channels + group * 16 * C + i * 16 + (lane >> 4) * 4 + q], acc[i][t][q]);
  __syncthreads();
  typedef O O4 __attribute__((ext_vector_type(4)));
  typedef O4 O4_u __attribute__((aligned(sizeof(O))));
  for (int i = threadIdx.x; i < 16 * TB * channels / 4; i += 512) {
    const int row = i / (channels / 4), ch = i % (channels / 4) * 4;
    const int64_t col = n0 + ch;
    if (row >= a.n || col >= a.N) continue;
    const float sx = a.x_scale[row];
    O* y = (O*)a.y + row * a.N + col;
    O4 v;
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = scaled<O>(sums[row * channels + ch + q], sx, a.w_scale[col + q < a.N ? col + q : a.N - 1]);
    if (col + 4 <= a.N) {
      *reinterpret_cast<O4_u*>(y) = v;
    } else {
#pragma unroll
      for (int q = 0; q < 3; ++q)
        if (col + q < a.N) y[q] = v[q];
    }
  }
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

// Tiles of BM x BN, 128 bytes of K a step, NB LDS buffers.  The rows come straight from memory into LDS, 16 bytes a lane, NB - 1 steps ahead
// of the one that is multiplied; WM x WN waves, each a part of the tile in products of 32 x 32 x 32.  A step waits for all loads that are on
// their way, the later steps' too (the barrier would by itself: the compiler lets it wait for direct loads), so what hides a load is the time
// of one step however many buffers there are.  Four only start the first three steps together, and go without a branch around the
// loads (weights from memory: 64 x 4,096 x 4,096 23.7 us, with two buffers 25.9, with the branch 25.2; 128 x 4,096 x 16,384 28.0, 29.2, 29.0).
// A wave's load fills 8 rows of 128 bytes.  Piece c of row r lies in place c ^ (r / 2 % 8) of its row in LDS, so that the 16 lanes that read
// a piece of 16 rows at a time find them in different banks (r % 8 instead: half of LDS's cycles were conflicts).  Rows past an end repeat the last (their outputs are not stored); pieces past K
// are read from zeros.  Rows and strides are multiples of 16 bytes.
template <class O, int BM, int BN, int WM, int WN, int NB>
__global__ __launch_bounds__(WM * WN * 64) void k_linear_tiles(LinearArgs a, uint32_t tiles_m, uint32_t tiles_n) {
  constexpr int W = WM * WN, BK = 128, MT = BM / WM / 32, NT = BN / WN / 32;
  constexpr int LX = BM / 8 / W, LW = BN / 8 / W;          // loads of a wave for each operand
  static_assert(W * Outputs<O, MT, NT>::kBytes <= NB * (BM + BN) * BK, "the outputs' LDS");
  extern __shared__ __attribute__((aligned(16))) int8_t tile_lds[];    // [NB][BM + BN][BK]
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
#pragma unroll
  for (int i = 0; i < NB - 1; ++i) load(i * BK, i);
  int buf = 0;
  for (int32_t k = 0; k < a.K; k += BK, buf = buf + 1 < NB ? buf + 1 : 0) {
    loads_done();
    __syncthreads();
    if (NB > 2 || k + BK < a.K) load(k + (NB - 1) * BK, buf > 0 ? buf - 1 : NB - 1);     // (past K: zeros)
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
  loads_done();      // (zeros past K, on their way into the buffers that the outputs take)
  __syncthreads();
  Outputs<O, MT, NT>::store(a, m0 + wm, n0 + wn, acc, tile_lds + wave * Outputs<O, MT, NT>::kBytes);
}

// ---- host side

// Few tokens: waves that share channels, so that each has a few steps of K; channels a wave.
template <class O, int TB>
static void few(const LinearArgs& a, hipStream_t st) {
  int kw = 8;
  while (kw > 1 && a.K < kw * 256) kw /= 2;
  const auto blocks = [&](int c) { return (a.N + 16 * c * (8 / kw) - 1) / (16 * c * (8 / kw)); };
  if (blocks(4 / TB) >= 512) k_linear_few<O, TB, 4 / TB><<<(unsigned)blocks(4 / TB), 512, 0, st>>>(a, kw);
  else if (blocks(2 / TB) >= 512) k_linear_few<O, TB, 2 / TB><<<(unsigned)blocks(2 / TB), 512, 0, st>>>(a, kw);
  else k_linear_few<O, TB, 1><<<(unsigned)blocks(1), 512, 0, st>>>(a, kw);
}

constexpr int64_t kNearRows = 1 << 23;      // strides of rows whose 256 lie within 32-bit offsets

template <class O, int B, int WM, int WN, int NB>
static void launch_tiles(const LinearArgs& a, hipStream_t st) {
  const uint32_t m = (uint32_t)((a.n + B - 1) / B), n = (uint32_t)((a.N + B - 1) / B);
  k_linear_tiles<O, B, B, WM, WN, NB><<<m * n, WM * WN * 64, NB * 2 * B * 128, st>>>(a, m, n);
}

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
    if (a.n <= 32) {
      a.n <= 16 ? few<O, 1>(a, st) : few<O, 2>(a, st);
    } else if (whole) {
      // Tiles of 256 where they alone nearly fill the chip (160 x 4,096 x 131,072 150 us, with 128 176), but 128 for up to 128 tokens, which
      // are half of one at most (64 x 4,096 x 49,152 48 us, with 256 57; 128 x 4,096 x 131,072 138 and 146; 64 x 1,024 x 65,536 18 and 22).
      // Else 128 where there is one for each CU (300 x 4,096 x 16,384 37, with 64 73), else 64 (128 x 4,096 x 16,384 28, with 128 35; more
      // than 512 of them wait for each other's LDS, two to a CU: 300 x 4,096 x 8,192 47, with 128 33).
      if (tiles(a.n, 256) * (uint64_t)tiles(a.N, 256) >= 192)
        a.n > 128 ? launch_tiles<O, 256, 2, 4, 2>(a, st) : launch_tiles<O, 128, 2, 2, 2>(a, st);
      else if (a.n > 64 && tiles(a.n, 128) * (uint64_t)tiles(a.N, 128) >= 256) launch_tiles<O, 128, 2, 2, 2>(a, st);
      else launch_tiles<O, 64, 2, 2, 4>(a, st);
    } else if (a.n <= 64) {
      k_linear<O, 64, 128><<<dim3(tiles(a.N, 128), 1), 256, 0, st>>>(a);
    } else {
      k_linear<O, 128, 128><<<dim3(tiles(a.N, 128), tiles(a.n, 128)), 256, 0, st>>>(a);
    }
  }
}

}  // namespace elr

extern "C" int elr_int8_linear(const int8_t* x, int64_t n, int64_t K, int64_t x_ld, const float* x_scale, const int8_t* w, int64_t N,
                               int64_t w_ld, const float* w_scale, void* y, int type, void* stream) {
  using namespace elr;
  if (n < 0 || N < 0 || K < 0 || x_ld < 0 || w_ld < 0 || !elem_type_ok(type)) return ELR_EINVAL;
  if (K >= 1 << 17 || N > (int64_t)1 << 30) return ELR_EUNSUPPORTED;
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
