// ftm_w8a8.hip -- int8 activations x int8 weights: the per-token quantiser and
// the integer product with one scale per token and one per output channel,
// dense or grouped by expert (rows sorted by expert, one weight per expert).
//
//   s_m = fp32(max_k |x_mk| / 127), q_mk = the whole number nearest x_mk / s_m
//   y_mn = (sum_k q_mk w_nk) s_m t_n (+ b_n), optionally h = act(gate) * up
//
// The sum is exact in int32 (K <= 131071, checked by the callers), so its order
// is free: every kernel here returns the same bits whatever its tile and
// however it splits K.  One rounding of the sum to fp32, one for each scale and
// for the bias, one to the output dtype.
//
// Operands of v_mfma_i32_16x16x64_i8 (lane l): A[i][k] i = l % 16, B[k][j] j =
// l % 16, both k = 16 (l / 16) + 0..15; D[i][j] j = l % 16, i = 4 (l / 16) +
// 0..3.  The weights are A and the tokens B, so a lane's results are
// neighbouring output channels of one token.
#include <type_traits>

#include "ftm_layer.h"

namespace ftm {

typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ i32x4 mfma_i8(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// ------------------------------------------------------------------ quantiser
// Largest |x| of a wave as fp32 bits (unsigned order: NaN above infinity above
// every finite value, so a row with either is recognised).
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
  auto up = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  v = up(v, (uint32_t)dpp_i<kDppXor1>((int)v));
  v = up(v, (uint32_t)dpp_i<kDppXor2>((int)v));
  v = up(v, (uint32_t)dpp_i<kDppHalfMirror>((int)v));
  v = up(v, (uint32_t)dpp_i<kDppMirror>((int)v));
  auto at = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
  return up(up(at(0), at(16)), up(at(32), at(48)));
}

// A row's scale and the factor of its first guess; a row with a value that is
// not finite gets the scale NaN and codes 0, so its outputs are NaN and no
// other row's change.
struct QuantScale {
  float s, inv;
};
__device__ __forceinline__ QuantScale quant_scale(uint32_t max_bits) {
  if (max_bits >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.0f};
  const float s = fmaxf(__uint_as_float(max_bits), 1e-12f) / 127.0f;
  return {s, 1.0f / s};
}
// The whole number nearest x / s, ties to even, for the exact quotient: the
// guess rint(x * (1 / s)) is at most one off, and the remainder x - q s, which
// an fma gives exactly wherever it is near s / 2 (x and s have 24 bits, q 7),
// tells which side of the border x lies on.
__device__ __forceinline__ int quant_code(float x, QuantScale c) {
  const float q = rintf(x * c.inv);
  const float e2 = 2.0f * fmaf(-q, c.s, x);
  const float a = fabsf(e2);
  const int qi = (int)q;
  const bool step = a > c.s || (a == c.s && (qi & 1) != 0);
  const int r = qi + (step ? (e2 > 0.0f ? 1 : -1) : 0);
  return r > 127 ? 127 : r < -127 ? -127 : r;
}
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return ((uint32_t)a & 255u) | (((uint32_t)b & 255u) << 8) | (((uint32_t)c & 255u) << 16) | ((uint32_t)d << 24);
}

template <int DT>
struct QuantVec {  // the values of one 16-byte load
  static constexpr int kN = DT == FTM_DT_F32 ? 4 : 8;
  __device__ __forceinline__ static float at(u32x4 v, int i) {
    if constexpr (DT == FTM_DT_F32) return __uint_as_float(v[i]);
    const uint32_t h = (v[i >> 1] >> (16 * (i & 1))) & 0xffffu;
    return DT == FTM_DT_F16 ? f16_to_f32((uint16_t)h) : __uint_as_float(h << 16);
  }
  __device__ __forceinline__ static uint32_t max_bits(u32x4 v) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const uint32_t b = __float_as_uint(at(v, i)) & 0x7fffffffu;
      m = b > m ? b : m;
    }
    return m;
  }
  __device__ __forceinline__ static void store(int8_t* q, u32x4 v, QuantScale c) {
    uint32_t w[kN / 4];
#pragma unroll
    for (int i = 0; i < kN / 4; ++i)
      w[i] = pack4(quant_code(at(v, 4 * i), c), quant_code(at(v, 4 * i + 1), c), quant_code(at(v, 4 * i + 2), c),
                   quant_code(at(v, 4 * i + 3), c));
    if constexpr (kN == 8) *(u32x2*)q = (u32x2){w[0], w[1]};
    else *(uint32_t*)q = w[0];
  }
};

// One row per WPR waves, its values in registers between the maximum and the
// codes (NV 16-byte loads a lane), so x is read once.  Bound by HBM.
template <int DT, int WPR, int NV>
__global__ __launch_bounds__(256) void k_quant_int8(const char* x, int64_t x_stride, int64_t rows, int K, int8_t* q,
                                                    int64_t q_stride, float* scale) {
  using V = QuantVec<DT>;
  constexpr int kRows = 4 / WPR;
  __shared__ uint32_t wmax[4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * kRows + wave / WPR;
  const int first = (wave % WPR) * 64 + lane;  // of this lane's vectors, WPR * 64 apart
  const bool live = row < rows;
  const char* src = x + (live ? row : 0) * x_stride;
  u32x4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = (first + i * WPR * 64) * V::kN;
    v[i] = live && k < K ? *(const u32x4*)(src + (size_t)k * (16 / V::kN)) : (u32x4){0, 0, 0, 0};
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t b = V::max_bits(v[i]);
    m = b > m ? b : m;
  }
  m = wave_max_bits(m);
  if constexpr (WPR > 1) {
    if (lane == 0) wmax[wave] = m;
    __syncthreads();
    m = wmax[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = wmax[w] > m ? wmax[w] : m;
  }
  if (!live) return;
  const QuantScale c = quant_scale(m);
  int8_t* dst = q + row * q_stride;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = (first + i * WPR * 64) * V::kN;
    if (k < K) V::store(dst + k, v[i], c);
  }
  if (first == 0) scale[row] = c.s;
}

// Any row length, stride and alignment: one workgroup per row, x read twice.
template <int DT>
__global__ __launch_bounds__(256) void k_quant_int8_any(const char* x, int64_t x_stride, int K, int8_t* q,
                                                        int64_t q_stride, float* scale) {
  __shared__ uint32_t wmax[4];
  const int64_t row = blockIdx.x;
  const void* src = x + row * x_stride;
  uint32_t m = 0;
  for (int k = threadIdx.x; k < K; k += 256) {
    const uint32_t b = __float_as_uint(load_scalar(src, k, DT)) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  m = wave_max_bits(m);
  if ((threadIdx.x & 63) == 0) wmax[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) m = wmax[w] > m ? wmax[w] : m;
  const QuantScale c = quant_scale(m);
  for (int k = threadIdx.x; k < K; k += 256) q[row * q_stride + k] = (int8_t)quant_code(load_scalar(src, k, DT), c);
  if (threadIdx.x == 0) scale[row] = c.s;
}

template <int DT>
hipError_t quant_dt(const char* x, int64_t x_stride, int64_t rows, int K, int8_t* q, int64_t q_stride, float* scale,
                    hipStream_t st) {
  constexpr int kN = QuantVec<DT>::kN;
  const bool aligned = ((uintptr_t)x & 15u) == 0 && (x_stride & 15) == 0 && K % kN == 0 &&
                       ((uintptr_t)q & 7u) == 0 && (q_stride & 7) == 0;
  const int vecs = K / kN;
  if (!aligned || vecs > 8 * 256) {
    k_quant_int8_any<DT><<<dim3((unsigned)rows), dim3(256), 0, st>>>(x, x_stride, K, q, q_stride, scale);
    return hipGetLastError();
  }
  const dim3 by4((unsigned)((rows + 3) / 4)), by1((unsigned)rows), wg(256);
  // one wave a row up to four loads a lane, else a workgroup a row
  if (vecs <= 64) k_quant_int8<DT, 1, 1><<<by4, wg, 0, st>>>(x, x_stride, rows, K, q, q_stride, scale);
  else if (vecs <= 128) k_quant_int8<DT, 1, 2><<<by4, wg, 0, st>>>(x, x_stride, rows, K, q, q_stride, scale);
  else if (vecs <= 256) k_quant_int8<DT, 1, 4><<<by4, wg, 0, st>>>(x, x_stride, rows, K, q, q_stride, scale);
  else if (vecs <= 512) k_quant_int8<DT, 4, 2><<<by1, wg, 0, st>>>(x, x_stride, rows, K, q, q_stride, scale);
  else if (vecs <= 1024) k_quant_int8<DT, 4, 4><<<by1, wg, 0, st>>>(x, x_stride, rows, K, q, q_stride, scale);
  else k_quant_int8<DT, 4, 8><<<by1, wg, 0, st>>>(x, x_stride, rows, K, q, q_stride, scale);
  return hipGetLastError();
}

hipError_t launch_quant_int8(const void* x, int dt, int64_t rows, int K, int64_t x_stride, int8_t* q,
                             int64_t q_stride, float* scale, hipStream_t st) {
  const char* p = (const char*)x;
  if (dt == FTM_DT_F32) return quant_dt<FTM_DT_F32>(p, x_stride, rows, K, q, q_stride, scale, st);
  if (dt == FTM_DT_F16) return quant_dt<FTM_DT_F16>(p, x_stride, rows, K, q, q_stride, scale, st);
  return quant_dt<FTM_DT_BF16>(p, x_stride, rows, K, q, q_stride, scale, st);
}

// ------------------------------------------------------------------ tiles
// Rows of one tile: `cnt` (up to the tile's height) from output row `row0` on,
// of expert `e`; e < 0: rows behind (or before) every expert's, written as
// zeros; cnt 0: nothing to do.
struct RowTile {
  int64_t row0;
  int cnt, e;
};

// Row tile `t` of height BM.  Dense: the t-th BM rows.  Grouped: the experts'
// row tiles in order of the experts, then tiles over the rows of no expert.
// Every wave finds it by itself: eight experts a lane, one prefix sum over the
// wave.  The offsets are clamped to [0, rows], so a bad table reads and writes
// no other memory.
template <int BM>
__device__ __forceinline__ RowTile row_tile(const ftm_w8a8& c, int t) {
  RowTile r;
  if (c.offsets == nullptr) {
    r.row0 = (int64_t)t * BM;
    const int64_t left = c.rows - r.row0;
    r.cnt = left < BM ? (int)left : BM;
    r.e = 0;
    return r;
  }
  const int lane = threadIdx.x & 63, E = c.num_experts, P = (int)c.rows;
  int lo[9], tiles[8], sum = 0;
#pragma unroll
  for (int i = 0; i < 9; ++i) {
    const int e = 8 * lane + i;
    const int o = c.offsets[e < E ? e : E];
    lo[i] = o < 0 ? 0 : o > P ? P : o;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = lo[i + 1] - lo[i];
    tiles[i] = n > 0 ? (n + BM - 1) / BM : 0;
    sum += tiles[i];
  }
  int upto = sum;  // inclusive prefix sum over the lanes
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(upto, d);
    upto += lane >= d ? v : 0;
  }
  const int total = __builtin_amdgcn_readlane(upto, 63);
  const uint64_t in = __ballot(t >= upto - sum && t < upto);
  if (in != 0) {
    const int src = __builtin_ctzll(in);
    int before = upto - sum, e = 0, m = 0, begin = 0, end = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool here = t >= before && t < before + tiles[i];
      e = here ? 8 * lane + i : e;
      m = here ? t - before : m;
      begin = here ? lo[i] : begin;
      end = here ? lo[i + 1] : end;
      before += tiles[i];
    }
    e = __builtin_amdgcn_readlane(e, src);
    m = __builtin_amdgcn_readlane(m, src);
    begin = __builtin_amdgcn_readlane(begin, src) + m * BM;
    end = __builtin_amdgcn_readlane(end, src);
    r.row0 = begin;
    r.cnt = end - begin < BM ? end - begin : BM;
    r.e = e;
    return r;
  }
  // the rows of no expert: before the first offset and behind the last
  const int head = __builtin_amdgcn_readlane(lo[0], 0), tail = __builtin_amdgcn_readlane(lo[8], 63);
  const int head_tiles = (head + BM - 1) / BM;
  const int u = t - total;
  const int begin = u < head_tiles ? u * BM : tail + (u - head_tiles) * BM;
  const int end = u < head_tiles ? head : P;
  r.row0 = begin;
  r.cnt = end - begin < BM ? (end > begin ? end - begin : 0) : BM;
  r.e = -1;
  return r;
}

// Row tiles that row_tile<BM> can name: each expert ends in one partly filled
// tile at most, and so do the rows before and behind them.
inline int64_t row_tiles(const ftm_w8a8& c, int BM) {
  if (c.offsets == nullptr) return (c.rows + BM - 1) / BM;
  const int64_t e = c.rows < c.num_experts ? c.rows : c.num_experts;
  return c.rows / BM + e + 2;
}

// Source row of output row `row` (inside an expert's rows), or -1 where the
// index names none.
__device__ __forceinline__ int64_t source_row(const ftm_w8a8& c, int64_t row) {
  if (c.row_index == nullptr) return row;
  const int i = c.row_index[row];
  return i >= 0 && i < c.x_rows ? i : -1;
}

// Output channels: with an activation the weight rows [0, N/2) are gate and
// [N/2, N) up.
__host__ __device__ inline int out_cols(const ftm_w8a8& c) { return c.act >= 0 ? c.N / 2 : c.N; }

// One result: the sum(s) of channel `col` with the token's scale.
struct Channel {
  float t, b;
};
__device__ __forceinline__ Channel channel(const ftm_w8a8& c, int e, int n) {
  const int64_t i = (int64_t)e * c.N + n;
  return {load_scalar(c.w_scale, i, c.w_scale_dtype), c.bias != nullptr ? load_scalar(c.bias, i, c.bias_dtype) : 0.0f};
}
__device__ __forceinline__ float scaled(int sum, float s, Channel ch) {
  return fmaf((float)sum * s, ch.t, ch.b);
}

// ------------------------------------------------------------------ K split over the waves
// A workgroup's tile of 16 MT tokens x 16 NT weight rows (with an activation:
// NT / 2 blocks of gate rows and the up rows that belong to them); each of the
// NW waves takes a part of K over the whole tile, straight from memory into
// registers, and the waves' sums meet in LDS.  No barrier in the K loop, so a
// wave keeps its loads in flight; the tokens are read once a column of tiles,
// from L2.  For few rows (weights bound it) and for grids too small for the
// LDS tiles.
template <int MT, int NT, int NW, bool PACKED>
__global__ __launch_bounds__(64 * NW) void k_w8a8_split(ftm_w8a8 c, int mtiles, int ntiles) {
  constexpr int BM = 16 * MT;
  constexpr int U = MT * NT >= 8 ? 2 : 4;  // K steps of 64 in a register set
  extern __shared__ int red[];            // [NW][MT * NT * 4][64]
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const RowTile rt = row_tile<BM>(c, item / ntiles);
  if (rt.cnt <= 0) return;
  const bool act = c.act >= 0;
  const int NO = out_cols(c);
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cols = act ? 8 * NT : 16 * NT;  // output channels of the tile
  const int n0 = (item % ntiles) * cols;
  const int ncol = NO - n0 < cols ? NO - n0 : cols;
  i32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};
  if (rt.e >= 0) {
    const int K = c.K;
    const int per = ((K + 64 * NW - 1) / (64 * NW)) * 64;  // K of a wave
    const int k_lo = wave * per, k_hi = k_lo + per < K ? k_lo + per : K;
    // rows past the tile read a row inside it (their results are dropped)
    const char* xrow[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int r = 16 * i + m;
      const int64_t s = source_row(c, rt.row0 + (r < rt.cnt ? r : 0));
      xrow[i] = (const char*)c.x + (s < 0 ? 0 : s) * c.x_stride;
    }
    // the tile's weight rows, from n0 (and, with an activation, N/2 + n0) on;
    // rows past the last read zeros
    const char* wbase = (const char*)c.w + (int64_t)rt.e * c.w_stride;
    const uint32_t bytes = (uint32_t)ncol * (uint32_t)K;
    const Rsrc w0 = make_rsrc(wbase + (int64_t)n0 * K, bytes);
    const Rsrc w1 = make_rsrc(wbase + (int64_t)((act ? NO : 0) + n0) * K, bytes);
    struct Set {
      u32x4 x[U][MT], w[U][NT];
    };
    auto load = [&](Set& s, int k) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int kk = k + 64 * u + 16 * g;
        const bool in = kk < k_hi;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const bool up = j >= NT / 2 && NT > 1;
          const int jr = (act && up ? j - NT / 2 : j) * 16 + m;
          s.w[u][j] = bload16(act && up ? w1 : w0, in ? (uint32_t)jr * (uint32_t)K + (uint32_t)kk : kOOB);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) s.x[u][i] = *(const u32x4*)(xrow[i] + (in ? kk : 0));
      }
    };
    auto mma = [&](const Set& s, int k) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // packed bytes are offset by 128; past K both forms have to be zero
        const uint32_t flip = PACKED && k + 64 * u + 16 * g < k_hi ? 0x80808080u : 0u;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          u32x4 w = s.w[u][j];
          if constexpr (PACKED) w ^= flip;
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i][j] = mfma_i8(w, s.x[u][i], acc[i][j]);
        }
      }
    };
    Set s0, s1;
    load(s0, k_lo);
    for (int k = k_lo; k < k_hi; k += 128 * U) {
      load(s1, k + 64 * U);
      mma(s0, k);
      load(s0, k + 128 * U);
      mma(s1, k + 64 * U);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[((wave * MT * NT + i * NT + j) * 4 + r) * 64 + lane] = acc[i][j][r];
  __syncthreads();
  // sum of (token row, weight row) of the tile over the waves
  auto total = [&](int row, int n) {
    const int at = (((row >> 4) * NT + (n >> 4)) * 4 + (n & 3)) * 64 + (row & 15) + 16 * ((n >> 2) & 3);
    int v = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += red[w * MT * NT * 256 + at];
    return v;
  };
  for (int i = threadIdx.x; i < rt.cnt * cols; i += 64 * NW) {
    const int row = i / cols, n = i % cols;
    if (n >= ncol) continue;
    const int64_t orow = rt.row0 + row;
    float y = 0.0f;
    const int64_t src = rt.e >= 0 ? source_row(c, orow) : -1;
    if (src >= 0) {
      const float s = c.x_scale[src];
      y = scaled(total(row, n), s, channel(c, rt.e, n0 + n));
      if (act)
        y = act_fn(c.act, y, scaled(total(row, n + 8 * NT), s, channel(c, rt.e, NO + n0 + n)), c.act_alpha, c.act_limit);
    }
    store_scalar(c.out, orow * NO + n0 + n, c.out_dtype, y);
  }
}

// ------------------------------------------------------------------ any K and alignment
// 16 tokens x 16 output channels a workgroup, bytes through LDS: for K not a
// multiple of 16 and rows that are not 16-byte aligned.
__global__ __launch_bounds__(256) void k_w8a8_any(ftm_w8a8 c, int mtiles, int ntiles) {
  constexpr int KC = 64;
  __shared__ int8_t xs[16][KC + 4], ws[2][16][KC + 4];
  const int item = blockIdx.x;
  const RowTile rt = row_tile<16>(c, item / ntiles);
  if (rt.cnt <= 0) return;
  const bool act = c.act >= 0;
  const int NO = out_cols(c), n0 = (item % ntiles) * 16;
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4;
  int a = 0, b = 0;
  if (rt.e >= 0) {
    const int8_t* wp = (const int8_t*)c.w + (int64_t)rt.e * c.w_stride;
    const int flip = c.w_packed ? 0x80 : 0;
    for (int k0 = 0; k0 < c.K; k0 += KC) {
      for (int i = threadIdx.x; i < 16 * KC; i += 256) {
        const int r = i / KC, k = i % KC;
        const bool in = k0 + k < c.K;
        const int64_t s = r < rt.cnt ? source_row(c, rt.row0 + r) : -1;
        xs[r][k] = in && s >= 0 ? ((const int8_t*)c.x)[s * c.x_stride + k0 + k] : (int8_t)0;
        const bool wn = in && n0 + r < NO;
        ws[0][r][k] = wn ? (int8_t)(wp[(int64_t)(n0 + r) * c.K + k0 + k] ^ flip) : (int8_t)0;
        if (act) ws[1][r][k] = wn ? (int8_t)(wp[(int64_t)(NO + n0 + r) * c.K + k0 + k] ^ flip) : (int8_t)0;
      }
      __syncthreads();
      for (int k = 0; k < KC; ++k) {
        a += (int)xs[row][k] * (int)ws[0][col][k];
        if (act) b += (int)xs[row][k] * (int)ws[1][col][k];
      }
      __syncthreads();
    }
  }
  if (row >= rt.cnt || n0 + col >= NO) return;
  const int64_t orow = rt.row0 + row;
  const int64_t src = rt.e >= 0 ? source_row(c, orow) : -1;
  float y = 0.0f;
  if (src >= 0) {
    const float s = c.x_scale[src];
    y = scaled(a, s, channel(c, rt.e, n0 + col));
    if (act) y = act_fn(c.act, y, scaled(b, s, channel(c, rt.e, NO + n0 + col)), c.act_alpha, c.act_limit);
  }
  store_scalar(c.out, orow * NO + n0 + col, c.out_dtype, y);
}

namespace {

template <int MT, int NT, int NW>
hipError_t split(const ftm_w8a8& c, hipStream_t st) {
  const int NO = out_cols(c);
  const int cols = c.act >= 0 ? 8 * NT : 16 * NT;
  const int64_t mt = row_tiles(c, 16 * MT), nt = (NO + cols - 1) / cols;
  if (mt * nt > 0x7fffffff) return hipErrorInvalidValue;
  const size_t lds = (size_t)NW * MT * NT * 1024;
  const dim3 grid((unsigned)(mt * nt)), wg(64 * NW);
  if (c.w_packed) k_w8a8_split<MT, NT, NW, true><<<grid, wg, lds, st>>>(c, (int)mt, (int)nt);
  else k_w8a8_split<MT, NT, NW, false><<<grid, wg, lds, st>>>(c, (int)mt, (int)nt);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_w8a8(const ftm_w8a8& c, hipStream_t st) {
  const bool aligned = c.K % 16 == 0 && (((uintptr_t)c.x | (uintptr_t)c.w) & 15u) == 0 && (c.x_stride & 15) == 0 &&
                       (c.offsets == nullptr || (c.w_stride & 15) == 0);
  if (!aligned) {
    const int64_t mt = row_tiles(c, 16), nt = (out_cols(c) + 15) / 16;
    if (mt * nt > 0x7fffffff) return hipErrorInvalidValue;
    k_w8a8_any<<<dim3((unsigned)(mt * nt)), dim3(256), 0, st>>>(c, (int)mt, (int)nt);
    return hipGetLastError();
  }
  // rows an expert gets on average
  const int64_t seg = c.offsets == nullptr ? c.rows : c.rows / (c.rows < c.num_experts ? c.rows : c.num_experts);
  if (seg <= 16) return split<1, 2, 4>(c, st);
  if (seg <= 32) return split<2, 2, 4>(c, st);
  return split<4, 2, 4>(c, st);
}

}  // namespace ftm
