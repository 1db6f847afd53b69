// ftm_w4a4.hip -- MXFP4 activations x MXFP4 weights: the quantiser, and the product
// of two operands in blocks of 32 four-bit codes with one power of two each, dense
// or grouped by expert (rows sorted by expert, one weight per expert).
//
//   block of x: a = max(max |x|, 1e-12), e the least whole number with a <= 6 2^e
//   code: the nearest of 0 .5 1 1.5 2 3 4 6 to |x| / 2^e, ties to the smaller
//   y_mn = sum over blocks of 2^(ex_mb + ew_nb) sum_k x_mk w_nk (+ b_n), optionally h = act(gate) * up
//
// The products of two codes are multiples of 1/4 up to 36, so a block's sum is
// exact; the blocks are added in fp32.  One rounding for the bias and one to the
// output dtype.
//
// Operands of v_mfma_scale_f32_16x16x128_f8f6f4 with 4-bit types (lane l): A[i][k] i = l % 16,
// B[k][j] j = l % 16, both k = 32 (l / 16) + 0..31, so a lane's 16 bytes are one block,
// and its scale operand is that block's byte; D[i][j] j = l % 16, i = 4 (l / 16) +
// 0..3.
#include "ftm_rows.h"

namespace ftm {

// Scale bytes: byte OA of `sa` and OB of `sb`.
template <int OA = 0, int OB = 0>
__device__ __forceinline__ f32x4 mfma_fp4(u32x4 a, u32x4 b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8 bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, OA, (int)sa, OB, (int)sb);
}

// ------------------------------------------------------------------ quantiser
// Eight neighbouring values of one lane in fp32.
template <int DT>
struct Vec8 {
  static constexpr int kBytes = DT == FTM_DT_F32 ? 32 : 16;
  u32x4 raw[kBytes / 16];
  __device__ __forceinline__ void load(const char* p) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) raw[i] = *(const u32x4*)(p + 16 * i);
  }
  __device__ __forceinline__ void load_any(const void* p) {  // any alignment of whole elements
    uint32_t w[kBytes / 4];
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i)
      w[i] = DT == FTM_DT_F32 ? ((const uint32_t*)p)[i]
                              : (uint32_t)((const uint16_t*)p)[2 * i] | (uint32_t)((const uint16_t*)p)[2 * i + 1] << 16;
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) raw[i] = (u32x4){w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) raw[i] = (u32x4){0, 0, 0, 0};
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (DT == FTM_DT_F32) return __uint_as_float(raw[i >> 2][i & 3]);
    const uint32_t w = raw[0][i >> 1];
    if constexpr (DT == FTM_DT_F16) return f16_to_f32((uint16_t)(i & 1 ? w >> 16 : w & 0xffffu));
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
  __device__ __forceinline__ uint32_t max_bits() const {  // unsigned order: NaN above infinity above the finite
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = __float_as_uint(at(i)) & 0x7fffffffu;
      m = b > m ? b : m;
    }
    return m;
  }
};

// A block's scale byte from the bits of its largest |x|: 6 2^e has the mantissa 1.5, so
// the exponent alone and one comparison give e.  1e-12 has 85.  A block with an
// infinity or NaN gets 255, the format's NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t max_bits) {
  const int e = (int)(max_bits >> 23) - 2 + ((max_bits & 0x7fffffu) > 0x400000u ? 1 : 0);
  return max_bits >= 0x7f800000u ? 255u : (uint32_t)(e > 85 ? e : 85);
}

// Eight codes, low nibble first, of values / 2^(byte - 127).  The conversion rounds ties to
// even; the product with 1 - 2^-24 is the next value towards zero (the remainder
// x 2^-24 is over half a step of x, or half of it where x is a power of two and the steps below are half as
// large), which turns ties down and moves nothing else over a border: borders have at
// most two mantissa bits, so of fp32 values only those with the other bits zero are moved.
template <int DT>
__device__ __forceinline__ float towards_zero(float x) {
  const float y = x * 0x1.fffffep-1f;
  if constexpr (DT == FTM_DT_F32) return (__float_as_uint(x) & 0x1fffffu) == 0 ? y : x;
  return y;
}
// No code is -0.
__device__ __forceinline__ uint32_t positive_zeros(uint32_t w) {
  const uint32_t size = w & 0x77777777u;
  return size | (w & (((size | size >> 1 | size >> 2) & 0x11111111u) << 3));
}
template <int DT>
__device__ __forceinline__ uint32_t mx_codes(const Vec8<DT>& v, uint32_t byte) {
  const float s = __uint_as_float(byte << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, towards_zero<DT>(v.at(0)), towards_zero<DT>(v.at(1)), s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, towards_zero<DT>(v.at(2)), towards_zero<DT>(v.at(3)), s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, towards_zero<DT>(v.at(4)), towards_zero<DT>(v.at(5)), s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, towards_zero<DT>(v.at(6)), towards_zero<DT>(v.at(7)), s, 3);
  return byte == 255u ? 0u : positive_zeros(w);
}
// The largest of four neighbouring lanes, which share a block.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  const uint32_t a = (uint32_t)dpp_i<kDppXor1>((int)v);
  v = a > v ? a : v;
  const uint32_t b = (uint32_t)dpp_i<kDppXor2>((int)v);
  return b > v ? b : v;
}

// Four lanes a block, eight values a lane.  x is read once and in whole lines, from any border of its
// elements; bound by HBM.  FLAT: rows side by side in memory, taken as one.
template <int DT, bool FLAT>
__global__ __launch_bounds__(256) void k_quant_mxfp4(const char* x, int64_t x_stride, int64_t rows, int K, int per_row,
                                                     uint32_t* blocks, uint8_t* scales) {
  const int64_t wg = grid_row(), vecs = FLAT ? rows * (K / 8) : K / 8;
  const int64_t row = FLAT ? 0 : wg / per_row;
  if (row >= rows) return;
  const int64_t k = (FLAT ? wg : wg - row * per_row) * 256 + threadIdx.x;
  Vec8<DT> v;
  if (k < vecs) v.load_any(x + row * x_stride + k * Vec8<DT>::kBytes);
  else v.zero();
  const uint32_t byte = mx_scale_byte(quad_max(v.max_bits()));
  const uint32_t w = mx_codes<DT>(v, byte);
  if (k >= vecs) return;
  const int64_t at = row * (K / 8) + k;
  blocks[at] = w;
  if ((threadIdx.x & 3) == 0) scales[at >> 2] = (uint8_t)byte;
}

template <int DT>
hipError_t quant(const char* x, int64_t x_stride, int64_t rows, int K, uint32_t* blocks, uint8_t* scales, hipStream_t st) {
  const bool flat = x_stride == (int64_t)K / 8 * Vec8<DT>::kBytes || rows == 1;
  const int per_row = (K / 8 + 255) / 256;
  const dim3 grid = row_grid(flat ? (rows * (K / 8) + 255) / 256 : rows * per_row), wg(256);
  if (flat) k_quant_mxfp4<DT, true><<<grid, wg, 0, st>>>(x, x_stride, rows, K, per_row, blocks, scales);
  else k_quant_mxfp4<DT, false><<<grid, wg, 0, st>>>(x, x_stride, rows, K, per_row, blocks, scales);
  return hipGetLastError();
}

hipError_t launch_quant_mxfp4(const void* x, int dt, int64_t rows, int K, int64_t x_stride, uint8_t* blocks,
                              uint8_t* scales, hipStream_t st) {
  const char* p = (const char*)x;
  uint32_t* b = (uint32_t*)blocks;
  if (dt == FTM_DT_F32) return quant<FTM_DT_F32>(p, x_stride, rows, K, b, scales, st);
  if (dt == FTM_DT_F16) return quant<FTM_DT_F16>(p, x_stride, rows, K, b, scales, st);
  return quant<FTM_DT_BF16>(p, x_stride, rows, K, b, scales, st);
}

// ------------------------------------------------------------------ activation
// 1 / (1 + e^-z) from the hardware's 2^t and 1 / t, one step of fp32 off each.  Rounding
// t = -z log2(e) moves e^-z by |z| 2^-24 at most, as much as half a step of z does.  In
// fp32's own division and exponential the epilogue of a tile took half as long as its
// products (clamped gate, 8192 rows of 2880 x 5760: 231 us, so 213).
__device__ __forceinline__ float sigmoid_of(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}
// act(gate) up, the same in every kernel here; NaN where either is.
template <int A, class C>
__device__ __forceinline__ float act_gated(float g, float u, const C& c) {
  if constexpr (A == FTM_ACT_SILU) return g * sigmoid_of(g) * u;
  if constexpr (A == FTM_ACT_SWIGLU_OAI) {
    g = g > c.act_limit ? c.act_limit : g;
    u = u > c.act_limit ? c.act_limit : u < -c.act_limit ? -c.act_limit : u;
    return (u + 1.0f) * (g * sigmoid_of(c.act_alpha * g));
  }
  return gated(A, g, u, c);
}

// ------------------------------------------------------------------ any size
// 16 tokens x 16 output channels a wave, operands straight from memory with 64-bit
// addresses.  Weights are A and tokens B, so a lane has four neighbouring channels of
// one token.  Blocks past K have the scale byte 0 on both sides: 2^-254 of anything is
// nothing in fp32.
template <bool ACT>
__global__ __launch_bounds__(256) void k_w4a4_any(ftm_w4a4 c, int mtiles, int ntiles) {
  const int64_t items = (int64_t)mtiles * ntiles;
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int NO = out_cols(c), nb = c.K / 32;
  for (int64_t it = (int64_t)blockIdx.x * 4 + wave; it < items; it += (int64_t)gridDim.x * 4) {
    const RowTile rt = row_tile<16>(c, (int)(it / ntiles));
    if (rt.cnt <= 0) continue;
    const int n0 = (int)(it % ntiles) * 16;
    const int64_t src = rt.e >= 0 && m < rt.cnt ? source_row(c, rt.row0 + m) : -1;
    f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (rt.e >= 0) {
      const char* w = (const char*)c.w + rt.e * c.w_stride;
      const uint8_t* ws = c.w_scale + rt.e * c.w_scale_stride;
      const int n = n0 + m < NO ? n0 + m : NO - 1;
      const int64_t xr = src < 0 ? 0 : src;
      for (int b0 = 0; b0 < nb; b0 += 4) {
        const int b = b0 + g, bc = b < nb ? b : nb - 1;
        const u32x4 xv = *(const u32x4*)((const char*)c.x + (xr * nb + bc) * 16);
        const uint32_t xs = b < nb ? c.x_scale[xr * nb + bc] : 0u;
#pragma unroll
        for (int p = 0; p < (ACT ? 2 : 1); ++p) {
          const int64_t row = n + (int64_t)p * NO;
          const u32x4 wv = *(const u32x4*)(w + (row * nb + bc) * 16);
          const uint32_t s = b < nb ? ws[row * nb + bc] : 0u;
          acc[p] = mfma_fp4(wv, xv, acc[p], s, xs);
        }
      }
    }
    if (m >= rt.cnt) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = n0 + 4 * g + r;
      if (n >= NO) continue;
      float y = 0.0f;
      if (src >= 0) {
        const int64_t at = (int64_t)rt.e * c.N + n;
        y = acc[0][r] + (c.bias != nullptr ? load_scalar(c.bias, at, c.bias_dtype) : 0.0f);
        if constexpr (ACT) {
          const float u = acc[1][r] + (c.bias != nullptr ? load_scalar(c.bias, at + NO, c.bias_dtype) : 0.0f), g = y;
          with_act(c.act, [&](auto a) { y = act_gated<decltype(a)::value>(g, u, c); });
        }
      }
      store_scalar(c.out, (rt.row0 + m) * NO + n, c.out_dtype, y);
    }
  }
}

// ------------------------------------------------------------------ operands
// The eight scale bytes of one row and step of 256 K, nb >= 8 of them in the row, as
// loaded (no alignment asked for; the last eight of the row where fewer are left) and as
// the step's: bytes past K are 0.  Apart, because fitting would wait for the load.
__device__ __forceinline__ u32x2 load_scales(const uint8_t* row, int step, int nb) {
  u32x2 v;
  __builtin_memcpy(&v, row + (8 * step + 8 <= nb ? 8 * step : nb - 8), 8);
  return v;
}
__device__ __forceinline__ u32x2 fit_scales(u32x2 v, int step, int nb) {
  const int past = 8 * step + 8 - nb;  // blocks of the step that are not there
  const uint64_t b = past < 8 ? (((uint64_t)v.y << 32) | v.x) >> (past > 0 ? 8 * past : 0) : 0;
  return (u32x2){(uint32_t)b, (uint32_t)(b >> 32)};
}
// Bytes g and 4 + g of eight: the scale operand of a lane of group g, byte q for the
// step's q-th 128 K.
__device__ __forceinline__ uint32_t scale_operand(u32x2 v, int g) {
  return __builtin_amdgcn_perm(v.y, v.x, 0x0c0c0000u | (uint32_t)(0x0400 + 0x101 * g));
}

// Weight rows of a tile of NT blocks of 16: with an activation 8 gate rows and their 8
// up rows a block.  Copies of 8 rows, a 16-byte piece a lane; rows past the last copy
// it, what lies past the end of the last row is zeros.
template <int NT>
struct SplitWeights {
  Rsrc res;
  uint32_t off[2 * NT];
  __device__ __forceinline__ SplitWeights(const char* w, int NO, int K, bool act, int n0, int ncol) {
    const int lane = threadIdx.x & 63, Kb = K / 2;
    res = make_rsrc(w + (int64_t)n0 * Kb, (uint32_t)((act ? NO : 0) + ncol) * (uint32_t)Kb);
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      const int r = 8 * i + (lane >> 3);
      int n = act ? 8 * (i >> 1) + (r & 7) : r;
      n = n < ncol ? n : ncol - 1;
      off[i] = (uint32_t)(n + (act && (i & 1) ? NO : 0)) * (uint32_t)Kb + 16u * (uint32_t)((lane & 7) ^ swz(r));
    }
  }
  // The weight row of row r of the tile's, from the tile's first on.
  __device__ __forceinline__ static int64_t row(int NO, bool act, int ncol, int r) {
    int n = act ? 8 * (r >> 4) + (r & 7) : r;
    n = n < ncol ? n : ncol - 1;
    return n + (act && (r & 8) != 0 ? NO : 0);
  }
  // k0 past the rows: nothing is read
  __device__ __forceinline__ void issue(char* at, uint32_t k0) const {
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(res, (LPtr)(at + 1024 * i), 16, (int)(off[i] + k0), 0, 0, 0);
  }
};
constexpr int kMinK = 256;  // of the kernels that take the scales eight at a time

// A wave's scales of R rows and its `per` steps from `lo` on, kept in LDS with scale_pitch
// bytes between rows (an odd number of eights: 16 rows hit distinct banks).  A lane
// has a row of each 64 (of 32 or 16 rows two or four lanes one, in turn); `p` says where they begin.  The
// first kFlight loads of each are under way when the copies of the operands are
// requested (`then`), before any of them is waited for.  As compiled a fill ends with a
// wait for all that is under way, these copies too, whether the loop over the rest of the
// scales runs or not: all stages of a ring have landed when its first is used.
__host__ __device__ constexpr int scale_pitch(int per) { return 8 * (per | 1); }
template <int R>
struct FillScales {
  static constexpr int kRows = (R + 63) / 64, kTurns = R <= 16 ? 4 : R <= 32 ? 2 : 1, kFlight = kTurns > 1 ? 2 : 4;
  static constexpr int kWidth = 64 / kTurns;
  const uint8_t* p[kRows];
  __device__ __forceinline__ static int row(int i) {  // the lane's i-th
    const int r = (threadIdx.x & (kWidth - 1)) + 64 * i;
    return r < R ? r : R - 1;
  }
  template <class Then>
  __device__ __forceinline__ void operator()(char* at, int lo, int per, int nb, Then&& then) const {
    const int lane = threadIdx.x & 63, pitch = scale_pitch(per);
    const int turn = lane / kWidth, first = lane & (kWidth - 1);
    const int last = (nb - 1) / 8, n = lo + per <= last + 1 ? per : last + 1 - lo;
    for (int s0 = 0; s0 < n; s0 += kTurns * kFlight) {
      u32x2 v[kRows][kFlight];
#pragma unroll
      for (int f = 0; f < kFlight; ++f)
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int s = s0 + kTurns * f + turn;
          v[i][f] = load_scales(p[i], lo + (s < n ? s : n - 1), nb);
        }
      __builtin_amdgcn_sched_barrier(0);
      if (s0 == 0) then();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int f = 0; f < kFlight; ++f)
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int s = s0 + kTurns * f + turn, r = first + 64 * i;
          if (s < n && r < R) *(u32x2*)(at + r * pitch + 8 * s) = fit_scales(v[i][f], lo + s, nb);
        }
    }
  }
};

constexpr uint32_t kNowhere = 0x40000000u;  // added to an offset below 2^30: past every buffer

// Piece q (128 K each) of row r of an LDS stage, for a lane of group g.
__device__ __forceinline__ u32x4 stage_piece(const char* st, int r, int q, int g) {
  return *(const u32x4*)(st + r * kRow + 16 * ((4 * q + g) ^ swz(r)));
}

// ------------------------------------------------------------------ K split over the waves
// Biases of one 16 x 16 block's results of a lane: weight rows 4 g .. 4 g + 3 (with an
// activation rows 0..7 of a block are gate channels, 8..15 their up rows, and only
// lanes of the first eight have results).
struct SplitBias {
  uint32_t b[8];
  __device__ __forceinline__ void request(const void* bias, int dt, int64_t at, bool act, int NO, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = 0;
    if (bias == nullptr) return;
    load_run<4>(bias, at, n, NO - 1, dt, b);
    if (act) load_run<4>(bias, at + NO, n, NO - 1, dt, b + 4);
  }
  __device__ __forceinline__ float at(int i, int dt) const { return bits_to_f32(opaque_bits(b[i]), dt); }
};

template <int NT>
__device__ __forceinline__ int split_channel(bool act, int n0, int block, int g) {
  return n0 + (act ? 8 * (block % NT) + 4 * (g & 1) : 16 * (block % NT) + 4 * g);
}

// The waves' sums of the tile's MT x NT blocks, through LDS (which they may
// overwrite): f(part, block, sums, sums of the up rows) for the blocks of this wave; a
// lane's four sums are rows 4 g .. 4 g + 3 of token lane % 16.
template <int MT, int NT, int NW, class F>
__device__ __forceinline__ void split_sums(char* lds, const f32x4 (&acc)[MT][NT], bool act, F&& f) {
  constexpr int kParts = (MT * NT + NW - 1) / NW;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x4* red = (f32x4*)lds;  // [NW][MT * NT][64]
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) red[(wave * MT * NT + i * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    const int b = p * NW + wave;
    if (MT * NT % NW != 0 && b >= MT * NT) continue;
    f32x4 u = {0, 0, 0, 0}, v = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      u += red[(w * MT * NT + b) * 64 + lane];
      if (act) v += red[(w * MT * NT + b) * 64 + (lane | 32)];
    }
    f(p, b, u, v);
  }
}

// A workgroup's tile of 16 MT tokens x 16 NT weight rows; each of the NW waves takes a
// run of K over the whole tile through an LDS ring of its own (S stages of 256 K), and the
// waves' sums meet in LDS.  No barrier in the K loop; a stage's slot is filled again as
// soon as its operands are in registers.  For few rows, where the weights' stream is
// all the time, and for grids too small for the tiles that share a ring.  Bound by the
// chain of a launch, a ring's first round trip and the sums: 16 x 4096 x 4096 4.1 us, 32 x 4096 x
// 11008 7.9 us (3.0 TB/s of weights).
template <int MT, int NT, int NW, int S>
__global__ __launch_bounds__(64 * NW) void k_w4a4_split(ftm_w4a4 c, int mtiles, int ntiles) {
  constexpr int BM = 16 * MT, kStage = (MT + NT) * 16 * kRow;
  constexpr int kParts = (MT * NT + NW - 1) / NW;
  extern __shared__ __attribute__((aligned(kRow))) char lds[];  // [NW][S][kStage], then the sums
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const RowTile rt = row_tile<BM>(c, item / ntiles);
  if (rt.cnt <= 0) return;
  const int NO = out_cols(c), nb = c.K / 32;
  const bool act = c.act >= 0;
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cols = act ? 8 * NT : 16 * NT;  // output channels of the tile
  const int n0 = (item % ntiles) * cols;
  const int ncol = NO - n0 < cols ? NO - n0 : cols;
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};
  using Fill = FillScales<16 * (MT + NT)>;
  SplitBias bias[kParts];
  auto request = [&] {
#pragma unroll
    for (int p = 0; p < kParts; ++p)
      bias[p].request(c.bias, c.bias_dtype, 0, act, NO, split_channel<NT>(act, n0, p * NW + wave, g));
  };
  const int nsteps = (nb + 7) / 8, per = (nsteps + NW - 1) / NW;
  const int lo = wave * per, hi = lo + per < nsteps ? lo + per : nsteps;
  if (lo < hi) {
    // rows past the tile are not copied; offsets from its first token
    const uint32_t Kb = (uint32_t)c.K / 2;
    const Rsrc xres = make_rsrc((const char*)c.x + rt.row0 * Kb, (uint32_t)rt.cnt * Kb);
    const SplitWeights<NT> weights((const char*)c.w, NO, c.K, act, n0, ncol);
    uint32_t xoff[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
      const int r = 8 * i + (lane >> 3);
      xoff[i] = r < rt.cnt ? (uint32_t)r * Kb + 16u * (uint32_t)((lane & 7) ^ swz(r)) : kNowhere;
    }
    Fill fill;
#pragma unroll
    for (int i = 0; i < Fill::kRows; ++i) {
      const int r = Fill::row(i);
      const int64_t n = n0 + SplitWeights<NT>::row(NO, act, ncol, r < 16 * MT ? 0 : r - 16 * MT);
      fill.p[i] = r < 16 * MT ? c.x_scale + (rt.row0 + (r < rt.cnt ? r : 0)) * nb : c.w_scale + n * nb;
    }
    char* ring = lds + wave * (S * kStage);
    char* scales = lds + NW * S * kStage + wave * (MT + NT) * 16 * scale_pitch(per);
    auto issue = [&](int step, int slot) __attribute__((always_inline)) {
      const uint32_t k0 = step < hi ? (uint32_t)step * 128u : kNowhere;
      char* st = ring + slot * kStage;
      weights.issue(st + 2048 * MT, k0);
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xres, (LPtr)(st + 1024 * i), 16, (int)(xoff[i] + k0), 0, 0, 0);
    };
    fill(scales, lo, per, nb, [&] {
      request();
#pragma unroll
      for (int u = 0; u < S; ++u) issue(lo + u, u);
    });
    const int pitch = scale_pitch(per);
    int slot = 0;
    for (int step = lo; step < hi; ++step) {
      wait_vm<(S - 1) * 2 * (MT + NT)>();  // this step's copies have landed
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      const char* st = ring + slot * kStage;
      u32x4 w[2][NT], x[2][MT];
      uint32_t sw[NT], sx[MT];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int j = 0; j < NT; ++j) w[q][j] = stage_piece(st, 16 * (MT + j) + m, q, g);
#pragma unroll
        for (int i = 0; i < MT; ++i) x[q][i] = stage_piece(st, 16 * i + m, q, g);
      }
      auto scale = [&](int r) { return scale_operand(*(const u32x2*)(scales + r * pitch + 8 * (step - lo)), g); };
#pragma unroll
      for (int j = 0; j < NT; ++j) sw[j] = scale(16 * (MT + j) + m);
#pragma unroll
      for (int i = 0; i < MT; ++i) sx[i] = scale(16 * i + m);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the operands are here: the slot is free
      __builtin_amdgcn_sched_barrier(0);
      issue(step + S, slot);
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          acc[i][j] = mfma_fp4<0, 0>(w[0][j], x[0][i], acc[i][j], sw[j], sx[i]);
          acc[i][j] = mfma_fp4<1, 1>(w[1][j], x[1][i], acc[i][j], sw[j], sx[i]);
        }
      slot = slot == S - 1 ? 0 : slot + 1;
    }
    wait_vm<0>();  // the copies past the last step, before the sums take their place
  } else {
    request();
  }
  with_act(c.act, [&](auto a) {
    constexpr int A = decltype(a)::value;
    split_sums<MT, NT, NW>(lds, acc, A >= 0, [&](int p, int b, f32x4 u, f32x4 v) {
      if (A >= 0 && g >= 2) return;
      float y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        y[r] = u[r] + bias[p].at(r, c.bias_dtype);
        if constexpr (A >= 0) y[r] = act_gated<A>(y[r], v[r] + bias[p].at(4 + r, c.bias_dtype), c);
      }
      RowOut<4>(c, rt, NO, split_channel<NT>(act, n0, b, g)).store(16 * (b / NT) + m, y);
    });
  });
}

// ------------------------------------------------------------------ few tokens
constexpr int kFewRows = 16;    // of one workgroup: the columns of a 16 x 16 product
constexpr int kFewPairs = 256;  // (token, expert) pairs of a layer: four a lane

// The pairs of one expert, found by every wave for itself.  Workgroups come by pair: the
// one of the expert's pair number 0, cap, 2 cap .. takes that pair and the next cap - 1
// of the same expert, the others leave.  list[0 .. cnt) are the pairs; cnt 0: nothing to do.
struct FewPairs {
  int e, cnt;
  __device__ __forceinline__ FewPairs(const void* ids, bool ids64, int P, int E, int p, int cap, int* list) {
    const int lane = threadIdx.x & 63;
    int id[kFewPairs / 64];
#pragma unroll
    for (int i = 0; i < kFewPairs / 64; ++i) {
      const int at = lane + 64 * i;
      id[i] = -1;
      if (at < P) {
        const int64_t v = ids64 ? ((const int64_t*)ids)[at] : (int64_t)((const int32_t*)ids)[at];
        id[i] = v >= 0 && v < E ? (int)v : -1;
      }
    }
    e = -1;
#pragma unroll
    for (int i = 0; i < kFewPairs / 64; ++i)
      if ((p >> 6) == i) e = __builtin_amdgcn_readlane(id[i], p & 63);
    cnt = 0;
    if (e < 0) return;
    uint64_t mine[kFewPairs / 64];
    int before = 0, all = 0;  // matches before p, and of all pairs
#pragma unroll
    for (int i = 0; i < kFewPairs / 64; ++i) {
      mine[i] = __ballot(id[i] == e);
      all += __popcll(mine[i]);
      if ((p >> 6) > i) before += __popcll(mine[i]);
      if ((p >> 6) == i) before += __popcll(mine[i] & ((1ull << (p & 63)) - 1));
    }
    if (before % cap != 0) return;
    cnt = all - before < cap ? all - before : cap;
    int base = -before;
#pragma unroll
    for (int i = 0; i < kFewPairs / 64; ++i) {
      const int r = base + __popcll(mine[i] & ((1ull << lane) - 1));
      if (id[i] == e && r >= 0 && r < cap) list[r] = lane + 64 * i;
      base += __popcll(mine[i]);
    }
  }
};

struct FewCall {
  const char* x;          // wide rows
  int64_t x_stride;
  const char* w;          // of expert 0
  const uint8_t* w_scale;
  const void* bias;
  int64_t w_stride, w_scale_stride;
  int N, K, bias_dtype, act;
  float act_alpha, act_limit;
  int cap;                // rows of a workgroup, at most
  // dense: the product's result
  void* out;
  int out_dtype;
  // a layer's first product: its pairs, and h quantised, a row a pair
  const void* ids;
  int ids64, P, E, k;
  uint8_t *hq, *hs;
};

// LDS of one wave of k_w4a4_few: its ring, the codes of `rows` tokens over its `per` steps, the
// scales of its weights and of the tokens.  Whole stage rows: the scales of an odd number of rows end in the
// middle of 16 bytes, and the next wave's ring takes 16-byte copies and reads.
template <int NT, int S>
__host__ __device__ constexpr int few_wave_lds(int per, int rows) {
  return (S * NT * 16 * kRow + per * rows * kRow + (16 * NT + rows) * scale_pitch(per) + kRow - 1) / kRow * kRow;
}

// Up to 16 tokens whose values are still wide, one weight: a workgroup quantises them
// itself, each wave the K that it multiplies, requested together with its scales and the first S stages of
// its weights (and quantised when these have landed: FillScales), and
// multiplies them by a tile of 16 NT weight rows, K split over the waves as in k_w4a4_split.
// Bound by two round trips one behind the other: 1 x 1536 x 2048 5.1 us.
template <int XDT, int NT, int NW, int S>
__global__ __launch_bounds__(64 * NW) void k_w4a4_few(FewCall c) {
  using V = Vec8<XDT>;
  constexpr int kStage = NT * 16 * kRow, kParts = (NT + NW - 1) / NW, kBatch = 4;
  extern __shared__ __attribute__((aligned(kRow))) char lds[];  // [NW] of: ring [S][kStage], codes [per][cnt][kRow], scales of weights and tokens; then the sums
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool act = c.act >= 0;
  const int NO = act ? c.N / 2 : c.N, K = c.K, nb = K / 32, cnt = c.cap;
  const int cols = act ? 8 * NT : 16 * NT, n0 = blockIdx.x * cols, ncol = NO - n0 < cols ? NO - n0 : cols;
  f32x4 acc[1][NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[0][j] = (f32x4){0, 0, 0, 0};
  SplitBias bias[kParts];
  auto request = [&] {
#pragma unroll
    for (int p = 0; p < kParts; ++p)
      bias[p].request(c.bias, c.bias_dtype, 0, act, NO, split_channel<NT>(act, n0, p * NW + wave, g));
  };
  const int nsteps = (nb + 7) / 8, per = (nsteps + NW - 1) / NW, pitch = scale_pitch(per);
  const int lo = wave * per, hi = lo + per < nsteps ? lo + per : nsteps;
  if (lo < hi) {
    const SplitWeights<NT> weights(c.w, NO, K, act, n0, ncol);
    char* ring = lds + wave * few_wave_lds<NT, S>(per, cnt);
    char* codes = ring + S * kStage;
    char* scales = codes + per * cnt * kRow;  // of the weights, then of the tokens
    char* xscales = scales + 16 * NT * pitch;
    auto issue = [&](int step, int slot) __attribute__((always_inline)) {
      weights.issue(ring + slot * kStage, step < hi ? (uint32_t)step * 128u : kNowhere);
    };
    FillScales<16 * NT> fill;
#pragma unroll
    for (int i = 0; i < fill.kRows; ++i)
      fill.p[i] = c.w_scale + (n0 + SplitWeights<NT>::row(NO, act, ncol, fill.row(i))) * nb;
    // half a wave takes 256 values of one row: of this wave's one step two rows at a time,
    // else two steps of one
    const int half = lane >> 5, l32 = lane & 31, n = hi - lo, hp = (n + 1) / 2;
    const int turns = n == 1 ? (cnt + 1) / 2 : cnt * hp;
    auto row_of = [&](int t) { return n == 1 ? 2 * t + half : t / hp; };
    auto step_of = [&](int t) { return n == 1 ? 0 : 2 * (t % hp) + half; };
    V v[kBatch];
    auto load = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int t = t0 + i, r = row_of(t), s = step_of(t), k = 256 * (lo + s) + 8 * l32;
        if (t < turns && r < cnt && s < n && k < K) {
          v[i].load(c.x + r * c.x_stride + (int64_t)(k / 8) * V::kBytes);
        } else {
          v[i].zero();
        }
      }
    };
    auto quantise = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int t = t0 + i, r = row_of(t), s = step_of(t);
        const uint32_t byte = mx_scale_byte(quad_max(v[i].max_bits()));
        const uint32_t w = mx_codes<XDT>(v[i], byte);
        if (t < turns && r < cnt && s < n) {
          *(uint32_t*)(codes + (s * cnt + r) * kRow + 16 * ((l32 >> 2) ^ swz(r)) + 4 * (l32 & 3)) = w;
          if ((l32 & 3) == 0) *(uint8_t*)(xscales + r * pitch + 8 * s + (l32 >> 2)) = (uint8_t)byte;
        }
      }
    };
    fill(scales, lo, per, nb, [&] {
      request();
      load(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < S; ++u) issue(lo + u, u);
    });
    quantise(0);
    for (int t = kBatch; t < turns; t += kBatch) {
      load(t);
      quantise(t);
    }
    __builtin_amdgcn_wave_barrier();
    const int xr = m < cnt ? m : 0;
    int slot = 0;
    for (int step = lo; step < hi; ++step) {
      wait_vm<(S - 1) * 2 * NT>();  // this step's copies have landed
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      const char* st = ring + slot * kStage;
      u32x4 w[2][NT], x[2];
      uint32_t sw[NT];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int j = 0; j < NT; ++j) w[q][j] = stage_piece(st, 16 * j + m, q, g);
        x[q] = stage_piece(codes + (step - lo) * cnt * kRow, xr, q, g);
      }
      auto scale = [&](const char* at, int r) { return scale_operand(*(const u32x2*)(at + r * pitch + 8 * (step - lo)), g); };
#pragma unroll
      for (int j = 0; j < NT; ++j) sw[j] = scale(scales, 16 * j + m);
      const uint32_t sx = scale(xscales, xr);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the operands are here: the slot is free
      __builtin_amdgcn_sched_barrier(0);
      issue(step + S, slot);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        acc[0][j] = mfma_fp4<0, 0>(w[0][j], x[0], acc[0][j], sw[j], sx);
        acc[0][j] = mfma_fp4<1, 1>(w[1][j], x[1], acc[0][j], sw[j], sx);
      }
      slot = slot == S - 1 ? 0 : slot + 1;
    }
    wait_vm<0>();  // the copies past the last step, before the sums take their place
  } else {
    request();
  }
  with_act(c.act, [&](auto a) {
    constexpr int A = decltype(a)::value;
    split_sums<1, NT, NW>(lds, acc, A >= 0, [&](int p, int b, f32x4 u, f32x4 v) {
      if (A >= 0 && g >= 2) return;
      float y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        y[r] = u[r] + bias[p].at(r, c.bias_dtype);
        if constexpr (A >= 0) y[r] = act_gated<A>(y[r], v[r] + bias[p].at(4 + r, c.bias_dtype), c);
      }
      RowOut<4>(c, RowTile{0, cnt, 0}, NO, split_channel<NT>(act, n0, b, g)).store(m, y);
    });
  });
}

// ------------------------------------------------------------------ columns over the waves
// Up to RW rows of one expert x 64 weight rows: the rows' codes and scales over the whole K
// in LDS, for all four waves; each wave streams 16 weight rows through a ring of its
// own (S stages of 256 K) and finishes its results alone.  Where an expert has few rows and
// there are blocks for every CU: against K split over the waves there are no sums to
// exchange, the rows are held once, and a workgroup's ring holds most of its weights.
// Call is a product (codes in hand) or a layer's first (FewCall: wide tokens, which the
// workgroup quantises, its 32 channels of h quantised in the epilogue).  Bound by the
// weights' stream with the chain before it (offsets, index, rows): 16 tokens of 8 of 128 experts,
// gate_up, 26.7 us, 110 MB of weights at 4.1 TB/s; a layer's 8 tokens of 4 of 32 of 2880 41 us, 184 MB at
// 4.5 TB/s.  K split over two groups of four waves lost (38.4 to 48.7 us, on the
// item order of that time), for the chain is then paid for half the weights.
template <int XDT, int RW, int S, class Call>
__global__ __launch_bounds__(256) void k_w4a4_cols(Call c, int ntiles) {
  constexpr bool MOE = std::is_same_v<Call, FewCall>;
  constexpr int MT = (RW + 15) / 16, NC = RW / 8, kStage = 16 * kRow, kTurns = 64 / RW;
  static_assert(RW == 8 || RW % 16 == 0, "copies of 8 rows");
  extern __shared__ __attribute__((aligned(kRow))) char lds[];  // [4][S][kStage], codes [nsteps][rows][kRow], scales of the rows, and of each wave's weights
  __shared__ int lists[MOE ? 4 : 1][kFewRows];
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int K = c.K, nb = K / 32, nsteps = (nb + 7) / 8, pitch = scale_pitch(nsteps);
  int e, cnt, nt;
  RowTile rt = {0, 0, 0};
  int R = RW;  // rows of the codes in LDS
  if constexpr (MOE) {
    nt = blockIdx.x % ntiles;
    const FewPairs pairs(c.ids, c.ids64 != 0, c.P, c.E, blockIdx.x / ntiles, c.cap, lists[wave]);
    e = pairs.e;
    cnt = pairs.cnt;
    R = c.cap;
  } else {
    // Neighbours on other XCDs: the tiles that have rows come first, and a run of items for each XCD would leave those
    // of the last runs idle (16 tokens of 8 of 128 experts, gate_up, 38.4 us, so 26.7).  No weight is read twice.
    nt = blockIdx.x % ntiles;
    rt = row_tile<RW>(c, blockIdx.x / ntiles);
    e = rt.e;
    cnt = rt.cnt;
  }
  if (cnt <= 0) return;
  const bool act = MOE || c.act >= 0;
  const int NO = act ? c.N / 2 : c.N;
  const int cols = act ? 8 : 16, n0 = nt * 4 * cols + wave * cols, ncol = NO - n0 < cols ? NO - n0 : cols;
  if constexpr (!MOE) {
    if (e < 0) {  // rows of no expert
      const float zero[4] = {};
      const RowOut<4> out(c, rt, NO, n0 + 4 * (act ? g & 1 : g));
      if (ncol > 0 && (!act || g < 2)) {
#pragma unroll
        for (int i = 0; i < MT; ++i) out.store(16 * i + m, zero);
      }
      return;
    }
  }
  char* ring = lds + wave * (S * kStage);
  char* codes = lds + 4 * S * kStage;
  char* xscales = codes + nsteps * R * kRow;
  char* scales = xscales + (R + 16 * wave) * pitch;
  bool live[MT];  // of this lane's results
#pragma unroll
  for (int i = 0; i < MT; ++i) live[i] = true;
  const SplitWeights<1> weights((const char*)c.w + (int64_t)e * c.w_stride, NO, K, act, n0 < NO ? n0 : 0, ncol > 0 ? ncol : 1);
  auto issue = [&](int step, int slot) __attribute__((always_inline)) {
    weights.issue(ring + slot * kStage, step < nsteps && ncol > 0 ? (uint32_t)step * 128u : kNowhere);
  };
  FillScales<16> fill;
  fill.p[0] = c.w_scale + (int64_t)e * c.w_scale_stride +
              ((n0 < NO ? n0 : 0) + SplitWeights<1>::row(NO, act, ncol > 0 ? ncol : 1, fill.row(0))) * nb;
  SplitBias bias;
  auto request = [&] {
    bias.request(c.bias, c.bias_dtype, (int64_t)e * c.N, act, NO, n0 + 4 * (act ? g & 1 : g));
  };
  if constexpr (MOE) {
    using V = Vec8<XDT>;
    constexpr int kBatch = 4;
    // half a wave takes 256 values of one row; the (row, step) pairs in turn over the half waves
    const int l32 = lane & 31, turns = cnt * nsteps;
    V v[kBatch];
    auto load = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int t = t0 + 8 * i, r = t / nsteps, k = 256 * (t % nsteps) + 8 * l32;
        if (t < turns && k < K) v[i].load(c.x + (int64_t)(lists[wave][r] / c.k) * c.x_stride + (int64_t)(k / 8) * V::kBytes);
        else v[i].zero();
      }
    };
    auto quantise = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int t = t0 + 8 * i, r = t / nsteps, s = t % nsteps;
        const uint32_t byte = mx_scale_byte(quad_max(v[i].max_bits()));
        const uint32_t w = mx_codes<XDT>(v[i], byte);
        if (t < turns) {
          *(uint32_t*)(codes + (s * R + r) * kRow + 16 * ((l32 >> 2) ^ swz(r)) + 4 * (l32 & 3)) = w;
          if ((l32 & 3) == 0) *(uint8_t*)(xscales + r * pitch + 8 * s + (l32 >> 2)) = (uint8_t)byte;
        }
      }
    };
    const int first = 2 * wave + (lane >> 5);
    fill(scales, 0, nsteps, nb, [&] {
      request();
      load(first);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < S; ++u) issue(u, u);
    });
    quantise(first);
    for (int t = first + 8 * kBatch; t - (lane >> 5) < turns; t += 8 * kBatch) {
      load(t);
      quantise(t);
    }
    __syncthreads();
  } else {
    // The rows of x: of the copies, of the scales, of the results
    const bool indexed = c.row_index != nullptr;
    const int64_t x_rows = indexed ? c.x_rows : c.rows;
    const uint32_t Kb = (uint32_t)K / 2;
    const int rs = lane & (RW - 1), turn = kTurns * wave + lane / RW;
    auto in_tile = [&](int r) { return r < cnt ? r : 0; };
    int ic[NC], ir[MT], is = in_tile(rs);
#pragma unroll
    for (int i = 0; i < NC; ++i) ic[i] = in_tile(8 * i + (lane >> 3));
#pragma unroll
    for (int i = 0; i < MT; ++i) ir[i] = in_tile(16 * i + m);
    if (indexed) {
#pragma unroll
      for (int i = 0; i < NC; ++i) ic[i] = c.row_index[rt.row0 + ic[i]];
#pragma unroll
      for (int i = 0; i < MT; ++i) ir[i] = c.row_index[rt.row0 + ir[i]];
      is = c.row_index[rt.row0 + is];
    } else {
      is += (int)rt.row0;
    }
    // rows past the tile and rows that are none are not copied
    const Rsrc xres = make_rsrc((const char*)c.x + (indexed ? 0 : rt.row0 * Kb), (uint32_t)(indexed ? c.x_rows : rt.cnt) * Kb);
    uint32_t xoff[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int r = 8 * i + (lane >> 3);
      const bool in = r < cnt && ic[i] >= 0 && ic[i] < (indexed ? x_rows : (int64_t)cnt);
      xoff[i] = in ? (uint32_t)ic[i] * Kb + 16u * (uint32_t)((lane & 7) ^ swz(r)) : kNowhere;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) live[i] = !indexed || (ir[i] >= 0 && ir[i] < x_rows);
    const uint8_t* xs = c.x_scale + (int64_t)(is >= 0 && is < x_rows ? is : 0) * nb;
    u32x2 own[2];  // the lane's row at steps turn and turn + 4 kTurns
    fill(scales, 0, nsteps, nb, [&] {
      request();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int s = turn + 4 * kTurns * i;
        own[i] = load_scales(xs, s < nsteps ? s : nsteps - 1, nb);
      }
      __builtin_amdgcn_sched_barrier(0);
      for (int s = wave; s < nsteps; s += 4)
#pragma unroll
        for (int i = 0; i < NC; ++i)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(xres, (LPtr)(codes + (s * R + 8 * i) * kRow), 16, (int)(xoff[i] + 128u * s), 0, 0, 0);
#pragma unroll
      for (int u = 0; u < S; ++u) issue(u, u);
    });
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int s = turn + 4 * kTurns * i;
      if (s < nsteps) *(u32x2*)(xscales + rs * pitch + 8 * s) = fit_scales(own[i], s, nb);
    }
    for (int s = turn + 8 * kTurns; s < nsteps; s += 4 * kTurns) *(u32x2*)(xscales + rs * pitch + 8 * s) = fit_scales(load_scales(xs, s, nb), s, nb);
    wait_vm<2 * S>();  // the rows' copies have landed
    __syncthreads();   // (compiled with a wait for the ring's as well)
  }
  f32x4 acc[MT];
  int xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    acc[i] = (f32x4){0, 0, 0, 0};
    xr[i] = 16 * i + m < cnt ? 16 * i + m : 0;
  }
  int slot = 0;
  for (int step = 0; step < nsteps; ++step) {
    wait_vm<(S - 1) * 2>();  // this step's copies have landed
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const char* st = ring + slot * kStage;
    u32x4 w[2], x[MT][2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      w[q] = stage_piece(st, m, q, g);
#pragma unroll
      for (int i = 0; i < MT; ++i) x[i][q] = stage_piece(codes + step * R * kRow, xr[i], q, g);
    }
    auto scale = [&](const char* at, int r) { return scale_operand(*(const u32x2*)(at + r * pitch + 8 * step), g); };
    const uint32_t sw = scale(scales, m);
    uint32_t sx[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) sx[i] = scale(xscales, xr[i]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the operands are here: the slot is free
    __builtin_amdgcn_sched_barrier(0);
    issue(step + S, slot);
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = mfma_fp4<0, 0>(w[0], x[i][0], acc[i], sw, sx[i]);
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = mfma_fp4<1, 1>(w[1], x[i][1], acc[i], sw, sx[i]);
    slot = slot == S - 1 ? 0 : slot + 1;
  }
  wait_vm<0>();  // the copies past the last step, before the LDS is given back
  if constexpr (MOE) __syncthreads();  // the rows' codes make place for h
  float* h = (float*)codes;  // [16][36]
  with_act(c.act, [&](auto a) {
    constexpr int A = decltype(a)::value;
    if constexpr (!MOE || A >= 0) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          y[r] = acc[i][r] + bias.at(r, c.bias_dtype);
          if constexpr (A >= 0) {  // the up rows are the lanes 32 on
            const float u = __shfl_xor(acc[i][r], 32) + bias.at(4 + r, c.bias_dtype);
            y[r] = act_gated<A>(y[r], u, c);
          }
          y[r] = live[i] ? y[r] : 0.0f;
        }
        if (A >= 0 && g >= 2) continue;
        if constexpr (MOE) {
#pragma unroll
          for (int r = 0; r < 4; ++r) h[m * 36 + 8 * wave + 4 * g + r] = y[r];
        } else if (ncol > 0) {
          RowOut<4>(c, rt, NO, n0 + 4 * (act ? g & 1 : g)).store(16 * i + m, y);
        }
      }
    }
  });
  if constexpr (MOE) {
    __syncthreads();
    const int row = lane >> 2, part = lane & 3;
    if (wave != 0) return;
    Vec8<FTM_DT_F32> v;
    v.load((const char*)(h + row * 36 + 8 * part));
    const uint32_t byte = mx_scale_byte(quad_max(v.max_bits()));
    const uint32_t q = mx_codes<FTM_DT_F32>(v, byte);
    if (row >= cnt) return;
    const int64_t at = (int64_t)lists[0][row] * (NO / 32) + nt;
    *(uint32_t*)(c.hq + at * 16 + 4 * part) = q;
    if (part == 0) c.hs[at] = (uint8_t)byte;
  }
}

// A layer's second product and sum for few tokens: one token x 16 output channels a
// workgroup.  The steps of 256 K of the token's experts, one expert behind the other, are
// split over the waves; a step's results are weighted by its expert's weight and added
// up in fp32, the waves' sums in order, so the order is the same in each call.  h comes
// from memory (every lane of a group the same block), the weights through LDS.  Bound by
// the workgroups' chains, of which two rounds are resident: 128 experts at 1 token 4.4 us, 32 of 2880 at
// 8 tokens 31 us (82 MB from memory, 141 MB into LDS).  One workgroup for all tokens of its
// channels, so that weights are read once, lost: 34 us there, 128 experts at 16 tokens 19.0 to
// 25.9.
template <int NW, int S>
__global__ __launch_bounds__(64 * NW) void k_w4a4_few_down(ftm_w4a4_moe c, const uint8_t* hq, const uint8_t* hs, int ntiles) {
  __shared__ __attribute__((aligned(1024))) char ring[NW][S][16 * kRow];
  __shared__ float sums[NW][16];
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = xcd_item(blockIdx.x, gridDim.x);  // the tokens of a column side by side: they share weights
  const int t = item % c.T, n0 = item / c.T * 16, H = c.hidden, nb = c.inter / 32, Kb = c.inter / 2;
  const int ns = (nb + 7) / 8;
  // lane j: the token's j-th expert and its weight
  int e = -1;
  float wt = 0.0f;
  if (lane < c.k) {
    const int64_t at = (int64_t)t * c.k + lane;
    const int64_t v = c.ids_dtype == FTM_ID_I64 ? ((const int64_t*)c.topk_ids)[at] : (int64_t)((const int32_t*)c.topk_ids)[at];
    e = v >= 0 && v < c.num_experts ? (int)v : -1;
    wt = load_scalar(c.topk_w, at, c.topk_w_dtype);
  }
  const uint64_t valid = __ballot(e >= 0);
  const int total = __popcll(valid) * ns, per = (total + NW - 1) / NW;
  const int lo = wave * per, hi = lo + per < total ? lo + per : total;
  const int ncol = H - n0 < 16 ? H - n0 : 16, row = m < ncol ? m : ncol - 1;
  f32x4 sum = {0, 0, 0, 0};
  uint64_t left = valid;  // the experts from this wave's first on
  int s = lo;             // its step within the first of them
  for (; s >= ns && left != 0; s -= ns) left &= left - 1;
  for (int u0 = lo; u0 < hi; u0 += S) {
    u32x4 h[S][2];
    u32x2 sh[S], sw[S];
    float wj[S];
    int at[S];
#pragma unroll
    for (int u = 0; u < S; ++u) {
      if (u0 + u >= hi) break;
      const int j = __builtin_ctzll(left), ej = __builtin_amdgcn_readlane(e, j);
      wj[u] = readlane_f(wt, j);
      at[u] = s;
      const Rsrc res = make_rsrc((const char*)c.w2 + ((int64_t)ej * H + n0) * Kb, (uint32_t)(ncol * Kb));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 8 * i + (lane >> 3), in = r < ncol ? r : ncol - 1;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(res, (LPtr)(ring[wave][u] + 1024 * i), 16,
                                                 in * Kb + 128 * s + 16 * ((lane & 7) ^ swz(r)), 0, 0, 0);
      }
      const int64_t pair = (int64_t)t * c.k + j;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int b = 8 * s + 4 * q + g;
        h[u][q] = *(const u32x4*)(hq + (pair * nb + (b < nb ? b : nb - 1)) * 16);
      }
      sh[u] = load_scales(hs + pair * nb, s, nb);
      sw[u] = load_scales(c.w2_scale + ((int64_t)ej * H + n0 + row) * nb, s, nb);
      if (++s == ns) {
        s = 0;
        left &= left - 1;
      }
    }
    wait_vm<0>();  // the steps' copies have landed
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < S; ++u) {
      if (u0 + u >= hi) break;
      const uint32_t a = scale_operand(fit_scales(sw[u], at[u], nb), g), b = scale_operand(fit_scales(sh[u], at[u], nb), g);
      f32x4 d = mfma_fp4<0, 0>(stage_piece(ring[wave][u], m, 0, g), h[u][0], (f32x4){0, 0, 0, 0}, a, b);
      d = mfma_fp4<1, 1>(stage_piece(ring[wave][u], m, 1, g), h[u][1], d, a, b);
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[r] = fmaf(wj[u], d[r], sum[r]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slots are free
  }
  if (m == 0) {
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[wave][4 * g + r] = sum[r];
  }
  __syncthreads();
  if (threadIdx.x >= 16 || n0 + (int)threadIdx.x >= H) return;
  const int n = n0 + threadIdx.x;
  float y = 0.0f;
#pragma unroll
  for (int w = 0; w < NW; ++w) y += sums[w][threadIdx.x];
  if (c.w2_bias != nullptr)
    for (uint64_t b = valid; b != 0; b &= b - 1) {
      const int j = __builtin_ctzll(b);
      y = fmaf(readlane_f(wt, j), load_scalar(c.w2_bias, (int64_t)__builtin_amdgcn_readlane(e, j) * H + n, c.w2_bias_dtype), y);
    }
  store_scalar(c.out, (int64_t)t * H + n, c.dtype, y);
}

// ------------------------------------------------------------------ LDS tiles
// A tile is BM = 16 MI WM tokens x BN = 16 NJ WN weight rows (with an activation BN / 2 gate
// rows and their up rows): WM WN waves of 16 MI tokens x 16 NJ weight rows each over the
// whole K.  Codes go through a ring of S LDS stages of 256 K, filled by direct copies,
// one barrier a step; scale bytes through registers into two slots of LDS, one step
// ahead.  Few large waves: a step reads (16 MI + 16 NJ) rows of LDS a wave for 16 MI x 16 NJ
// results, and with one wave a SIMD every other instruction is written into the
// shadow of an MFMA (16 cycles), in the order in which it is to be issued.  So it is compiled for
// 256 x 256; of the others the compiler takes some steps of a tile apart and puts their copies in one burst
// before their products: the first of 64 x 256, the last of 128 x 256, the last two of 128 x 128.  A workgroup
// takes one tile after another, and the copies run on from tile to tile.  Bound by power and
// MFMA issue where a tile is large (4096 x 12288 x 4096 105 to 109 us, 3.9 POP/s; MFMA busy 44 % of the
// cycles), by the copies of a step where it is small.
template <int WM, int WN, int MI, int NJ, int S, bool ACT, bool GROUPED, bool QOUT>
__global__ __launch_bounds__(64 * WM * WN, 1) void k_w4a4_tile(ftm_w4a4 c, uint8_t* out_scale, int mtiles, int ntiles) {
  constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  constexpr int BM = 16 * MI * WM, BN = 16 * NJ * WN, kRows = BM + BN;
  constexpr int kX = BM * kRow, kStage = kRows * kRow, kSlot = 8 * kRows;  // of codes, of scales
  constexpr int NX = BM / 8 / kWaves, NB = BN / 8 / kWaves, ND = NX + NB;  // 1 KiB copies a wave and step
  constexpr int NR = 2;                                  // rows whose scales a thread carries: of x, of the weights
  static_assert(NX <= 8 && BN <= kThreads, "rows of scales");
  constexpr int kCols = ACT ? BN / 2 : BN;               // output channels of the tile
  constexpr int CN = ACT ? NJ / 2 : NJ;                  // neighbouring ones of a lane
  constexpr int kAhead = MI >= 4 ? 7 : 2 * MI - 1;       // row blocks read ahead of their products
  constexpr int kLast = 2 * MI - kAhead;                 // from this one on they are the next step's
  constexpr int kNextX = MI < kAhead ? MI : kAhead;      // row blocks whose scales are read a step ahead
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0, "copies of 8 rows, as many for each wave");
  constexpr int kSecond = MI < kLast ? MI : kLast;       // row blocks that read the second half's weights
  static_assert(2 * MI % (kAhead + 1) == 0 && NJ % 4 == 0 && NJ % kSecond == 0, "the order of the reads");
  static_assert(MI <= 8, "a bit for each of a lane's rows");
  constexpr uint32_t kAllRows = ~0u >> (32 - 4 * MI);
  extern __shared__ __attribute__((aligned(kRow))) char lds[];  // [S][kStage], [2][kSlot], the rows of x [BM]
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int NO = out_cols(c), nb = c.K / 32;
  const uint32_t Kb = (uint32_t)c.K / 2;
  const int nsteps = (nb + 7) / 8, nrun = nsteps > S ? nsteps : S;  // steps past K multiply zeros
  const bool indexed = GROUPED && c.row_index != nullptr;
  int32_t* const index = (int32_t*)(lds + S * kStage + 2 * kSlot);

  // this workgroup's items: every (workgroups per XCD)-th of its XCD's run
  using Scan = std::conditional_t<GROUPED, RowScan<BM>, int>;
  const Scan scan = [&] {
    if constexpr (GROUPED) return RowScan<BM>(c);
    else return 0;
  }();
  int row_tiles = mtiles;
  if constexpr (GROUPED) row_tiles = scan.total;
  const int items = row_tiles * ntiles, xcd = blockIdx.x & 7, rem = items & 7;
  const int begin = xcd * (items >> 3) + (xcd < rem ? xcd : rem), end = begin + (items >> 3) + (xcd < rem ? 1 : 0);
  struct Tile {
    RowTile rt;
    int n;  // first output channel
  };
  auto tile_at = [&](int item) __attribute__((always_inline)) {
    if constexpr (GROUPED) {
      const auto x = scan.expert(item / ntiles);
      const ItemOrder o(item - x.before * ntiles, x.tiles, ntiles);
      return Tile{scan.tile(x, o.m), o.nt * kCols};
    } else {
      const ItemOrder o(item, mtiles, ntiles);
      return Tile{dense_tile<BM>(c, o.m), o.nt * kCols};
    }
  };
  // Weight row of the tile's LDS row r: wave r / (16 NJ) of the columns; its operand block
  // j, operand row o is channel NJ o + j, so that a lane's results are neighbours
  // (with an activation: NJ / 2 o + j of gate, j < NJ / 2, and of up); rows past the last copy it
  auto weight_row = [&](int r, int cols) __attribute__((always_inline)) {
    const int j = (r >> 4) % NJ, o = r & 15;
    int n = r / (16 * NJ) * (kCols / WN) + CN * o + j % CN;
    n = n < cols ? n : cols - 1;
    return n + (ACT && j >= CN ? NO : 0);
  };
  int item = begin + (blockIdx.x >> 3);
  if (item < end) {
    Tile cur = tile_at(item);
    // The next tile's rows of x, where they are read through an index, are copied to LDS a
    // tile ahead: a load of them into registers would be waited for with every copy
    // before it.  They are there from step S on; a shorter tile waits for them.
    auto copy_index = [&](const Tile& t) __attribute__((always_inline)) {
      if (!indexed || wave != 0) return;
      const Rsrc res = make_rsrc(c.row_index + t.rt.row0, 4u * (uint32_t)t.rt.cnt);
#pragma unroll
      for (int i = 0; i < BM / 64; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(res, (LPtr)(index + 64 * i), 4, 4 * lane + 256 * i, 0, 0, 0);
    };
    auto index_here = [&] {
      wait_vm<0>();
      asm volatile("s_barrier" ::: "memory");
    };
    const bool index_late = indexed && nrun < 2 * S;
    // Offsets of a wave's copies: 8 rows each, a 16-byte piece a lane, swizzled; tokens
    // from the tile's first row, or, read through an index, from x's; weights from the tile's
    // first gate row.  Rows past the tile are not copied.
    Rsrc xres, wres;
    uint32_t xoff[NX], woff[NB];
    auto aim = [&](const Tile& t) __attribute__((always_inline)) {
      const int lane = opaque_lane();
      xres = make_rsrc((const char*)c.x + (indexed ? 0 : t.rt.row0 * Kb), (uint32_t)(indexed ? c.x_rows : t.rt.cnt) * Kb);
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const int r = 8 * (wave * NX + i) + (lane >> 3);
        const int ix = indexed ? index[r] : r;
        const bool in = r < t.rt.cnt && ix >= 0 && (!indexed || ix < c.x_rows);
        xoff[i] = in ? (uint32_t)ix * Kb + 16u * (uint32_t)((lane & 7) ^ swz(r)) : kNowhere;
      }
      const int cols = NO - t.n < kCols ? NO - t.n : kCols;
      wres = make_rsrc((const char*)c.w + (int64_t)t.rt.e * c.w_stride + (int64_t)t.n * Kb, (uint32_t)((ACT ? NO : 0) + cols) * Kb);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int r = 8 * (wave * NB + i) + (lane >> 3);
        woff[i] = (uint32_t)weight_row(r, cols) * Kb + 16u * (uint32_t)((lane & 7) ^ swz(r));
      }
    };
    // copy d of the wave's: tokens, then weights.  The sum is kept at its place: all of
    // them ahead would stand between two products.
    auto copy = [&](int d, uint32_t k0, char* st) __attribute__((always_inline)) {
      uint32_t at;
      asm volatile("v_add_u32 %0, %1, %2" : "=v"(at) : "v"(d < NX ? xoff[d < NX ? d : 0] : woff[d < NX ? 0 : d - NX]), "s"(k0));
      if (d < NX) __builtin_amdgcn_raw_ptr_buffer_load_lds(xres, (LPtr)(st + 1024 * (wave * NX + d)), 16, (int)at, 0, 0, 0);
      else __builtin_amdgcn_raw_ptr_buffer_load_lds(wres, (LPtr)(st + kX + 1024 * (wave * NB + d - NX)), 16, (int)at, 0, 0, 0);
    };
    auto k_of = [&](int kb) { return (uint32_t)(kb < nsteps ? kb : nsteps - 1) * 128u; };
    // Scales: a thread's rows, one of x (of those that its wave copies) and one of the
    // weights, the eight bytes of the step after next under way
    const uint8_t* srow[NR];
    u32x2 sraw[NR];
    auto saim = [&](const Tile& t) __attribute__((always_inline)) {
      const int cols = NO - t.n < kCols ? NO - t.n : kCols, l = opaque_lane();
      int r = 8 * NX * wave + (l < 8 * NX ? l : 0);
      r = r < t.rt.cnt ? r : 0;
      int64_t x = t.rt.row0 + r;
      if (indexed) {
        const int ix = index[r];
        x = ix >= 0 && ix < c.x_rows ? ix : 0;
      }
      srow[0] = c.x_scale + x * nb;
      const int wr = (64 * wave + l) & (BN - 1);
      srow[1] = c.w_scale + (int64_t)t.rt.e * c.w_scale_stride + (int64_t)(t.n + weight_row(wr, cols)) * nb;
    };
    auto load_s = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NR; ++i) sraw[i] = load_scales(srow[i], kb < nsteps ? kb : nsteps - 1, nb);
    };
    // bytes b0 b4 b1 b5 b2 b6 b3 b7: group g's two are neighbours
    auto store_s = [&](int kb, int slot) __attribute__((always_inline)) {
      char* at = lds + S * kStage + slot * kSlot;
      if (8 * kb + 8 > nb) {  // not all of the step's blocks are there
#pragma unroll
        for (int i = 0; i < NR; ++i) sraw[i] = fit_scales(sraw[i], kb, nb);
      }
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const u32x2 v = sraw[i];
        const int r = i == 0 ? 8 * NX * wave + lane : BM + ((64 * wave + lane) & (BN - 1));
        if (i == 1 || NX == 8 || lane < 8 * NX)
          *(u32x2*)(at + 8 * r) = (u32x2){__builtin_amdgcn_perm(v.y, v.x, 0x05010400u), __builtin_amdgcn_perm(v.y, v.x, 0x07030602u)};
      }
    };
    f32x4 acc[MI][NJ];
    u32x4 b[2][NJ], x[kAhead + 1];
    uint32_t sx[MI], sb[NJ], nx[kNextX], sn[NJ];
    // The swizzle of row 16 i + m is that of row m: a base for each half of a stage and
    // operand, the row block as an immediate
    const uint32_t piece[2] = {16u * (uint32_t)(g ^ swz(m)), 16u * (uint32_t)((4 + g) ^ swz(m))};
    const uint32_t xbase = (uint32_t)((16 * wm * MI + m) * kRow), wbase = (uint32_t)((BM + 16 * wn * NJ + m) * kRow);
    const uint32_t sxbase = (uint32_t)(S * kStage + 8 * (16 * wm * MI + m) + 2 * g);
    const uint32_t swbase = (uint32_t)(S * kStage + 8 * (BM + 16 * wn * NJ + m) + 2 * g);
    auto xfrag = [&](int slot, int at) __attribute__((always_inline)) {
      return *(const u32x4*)(lds + (xbase + piece[at / MI] + (uint32_t)(slot * kStage)) + at % MI * 16 * kRow);
    };
    auto wfrag = [&](int slot, int j, int q) __attribute__((always_inline)) {
      return *(const u32x4*)(lds + (wbase + piece[q] + (uint32_t)(slot * kStage)) + j * 16 * kRow);
    };
    auto xscale = [&](int slot, int i) __attribute__((always_inline)) {
      return (uint32_t)*(const uint16_t*)(lds + (sxbase + (uint32_t)(slot * kSlot)) + 128 * i);
    };
    auto wscale = [&](int slot, int j) __attribute__((always_inline)) {
      return (uint32_t)*(const uint16_t*)(lds + (swbase + (uint32_t)(slot * kSlot)) + 128 * j);
    };
    // Products of step kb, whose first operands are in registers; the rest is read
    // kAhead row blocks ahead.  Once every wave has read the last of them, the stage's slot
    // takes the copies of the step S later (`k0`: its place in the tile that the copies
    // are at), and the first operands of the next step, whose copies have landed, are
    // read under the products left.
    auto step = [&](int kb, int snext, int sload, uint32_t k0, int slot, int par) __attribute__((always_inline)) {
      const int next = slot == S - 1 ? 0 : slot + 1;
      constexpr int kSlots = kAhead * NJ;
      // the next step's first weights take registers that are free from the second half on
      constexpr int kFirstB = MI > kLast ? (MI - kLast) * NJ : 0;
#pragma unroll
      for (int at = 0; at < 2 * MI; ++at) {
        const int q = at / MI, i = at % MI;
        if (at == kLast) {
          // the next step's copies have landed (a tile's first S stages are here already)
          if (kb >= S - 1) wait_vm<(S - 2) * ND + NR>();
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          __builtin_amdgcn_sched_barrier(0);
          if (q == 0) acc[i][j] = mfma_fp4<0, 0>(x[at % (kAhead + 1)], b[0][j], acc[i][j], sx[i], sb[j]);
          else acc[i][j] = mfma_fp4<1, 1>(x[at % (kAhead + 1)], b[1][j], acc[i][j], sx[i], sb[j]);
          __builtin_amdgcn_sched_barrier(0);
          const int a = at + kAhead;
          if (j == 0 && a < 2 * MI) x[a % (kAhead + 1)] = xfrag(slot, a);
          if (j == 1 && a < MI) sx[a] = xscale(par, a);
          if (at < kSecond) {  // the second half's weights, before the slot is given away
            constexpr int kPer = NJ / kSecond;
#pragma unroll
            for (int n = 0; n < kPer; ++n)
              if (j == (2 + n) % NJ) b[1][at * kPer + n] = wfrag(slot, at * kPer + n, 1);
          }
          if (at >= kLast) {
            const int t = (at - kLast) * NJ + j;
            if (j == 0) x[a % (kAhead + 1)] = xfrag(next, a - 2 * MI);
            if (j == 1 && at - kLast < kNextX) nx[at - kLast] = xscale(1 - par, at - kLast);
#pragma unroll
            for (int n = 0; n < NJ; ++n) {
              if (kFirstB + n * (kSlots - kFirstB) / NJ == t) b[0][n] = wfrag(next, n, 0);
              if (n * kSlots / NJ == t) sn[n] = wscale(1 - par, n);
            }
#pragma unroll
            for (int d = 0; d < ND; ++d)
              if (d * kSlots / ND == t) copy(d, k0, lds + slot * kStage);
          }
        }
        if (at == 0) store_s(snext, 1 - par);
        if (at == 0) load_s(sload);
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) sb[j] = sn[j];
#pragma unroll
      for (int i = 0; i < kNextX; ++i) sx[i] = nx[i];
      __builtin_amdgcn_sched_barrier(0);
    };
    if (indexed) {
      copy_index(cur);
      index_here();
    }
    aim(cur);
    saim(cur);
    load_s(0);
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int d = 0; d < ND; ++d) copy(d, k_of(s), lds + s * kStage);
    store_s(0, 0);
    load_s(1);
    wait_vm<0>();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      b[0][j] = wfrag(0, j, 0);
      sb[j] = wscale(0, j);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) x[i] = xfrag(0, i);
#pragma unroll
    for (int i = 0; i < kNextX; ++i) sx[i] = xscale(0, i);
    int slot = 0, par = 0;
    for (;;) {
      const int after = item + (int)(gridDim.x >> 3);
      const Tile next = after < end ? tile_at(after) : cur;  // (the last tile's copies go on over it: nothing reads them)
      copy_index(next);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};
      for (int kb = 0; kb < nrun; ++kb) {
        if (kb == nrun - S) {
          if (index_late) index_here();
          aim(next);  // from here on the copies are the next tile's
        }
        if (kb == nrun - 2) saim(next);
        const int ahead = kb + S < nrun ? kb + S : kb + S - nrun;
        step(kb, kb + 1 < nrun ? kb + 1 : 0, kb + 2 < nrun ? kb + 2 : kb + 2 - nrun, k_of(ahead), slot, par);
        slot = slot == S - 1 ? 0 : slot + 1;
        par = 1 - par;
      }
      // A lane has tokens 16 i + 4 g + r (r 0..3) and CN neighbouring channels from n0 on
      // (with an activation, and their up rows)
      const int el = opaque_lane(), em = el & 15, eg = el >> 4;
      const int n0 = cur.n + wn * (kCols / WN) + CN * em;
      const int t0 = 16 * wm * MI + 4 * eg;
      uint32_t live = kAllRows;  // bit 4 i + r: the row is one of x
      if (indexed) {
        int er[MI][4];
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) er[i][r] = c.row_index[cur.rt.row0 + (t0 + 16 * i + r < cur.rt.cnt ? t0 + 16 * i + r : 0)];
        live = 0;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) live |= er[i][r] >= 0 && er[i][r] < c.x_rows ? 1u << (4 * i + r) : 0u;
      }
      uint32_t bb[NJ];
#pragma unroll
      for (int n = 0; n < NJ; ++n) bb[n] = 0;
      if (c.bias != nullptr) {
        const int64_t at = (int64_t)cur.rt.e * c.N;
        load_run<CN>(c.bias, at, n0, NO - 1, c.bias_dtype, bb);
        if constexpr (ACT) load_run<CN>(c.bias, at + NO, n0, NO - 1, c.bias_dtype, bb + CN);
      }
      // With the biases, the next tile's first S stages are here: the steps that would
      // wait for them need not wait for the stores below
      wait_vm<0>();
      float bias[NJ];
#pragma unroll
      for (int n = 0; n < NJ; ++n) bias[n] = bits_to_f32(opaque_bits(bb[n]), c.bias_dtype);
      // A path for each activation and type, as long as its work: instructions that a tile
      // runs once are fetched anew, and a path that jumped over the other types' stores
      // took 3.9 us for 128 x 256 results, so 1.3
      const RowOut<CN> out(c, cur.rt, NO, n0);
      with_act(ACT ? c.act : -1, [&](auto a) __attribute__((always_inline)) {
        constexpr int A = decltype(a)::value;
        if constexpr (ACT == (A >= 0)) {
          auto each_row = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < MI; ++i) {
              // one row block after the other, so that their results do not all sit in
              // registers at once
              f32x4 v[NJ];
#pragma unroll
              for (int j = 0; j < NJ; ++j) {
                v[j] = acc[i][j];
                asm volatile("" : "+v"(v[j]) : : "memory");
              }
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                float y[CN];
#pragma unroll
                for (int n = 0; n < CN; ++n) {
                  y[n] = v[n][r] + bias[n];
                  if constexpr (ACT) y[n] = act_gated<A>(y[n], v[CN + n][r] + bias[CN + n], c);
                }
                f(t0 + 16 * i + r, y);
              }
            }
          };
          if constexpr (QOUT) {  // a block of 32 is 32 / CN neighbouring lanes
            each_row([&](int t, const float(&y)[CN]) __attribute__((always_inline)) {
              uint32_t top = 0;
#pragma unroll
              for (int n = 0; n < CN; ++n) {
                const uint32_t b = __float_as_uint(y[n]) & 0x7fffffffu;
                top = b > top ? b : top;
              }
              top = quad_max(top);
              auto with = [&](uint32_t o) { top = o > top ? o : top; };
              with((uint32_t)dpp_i<kDppHalfMirror>((int)top));
              if constexpr (CN == 2) with((uint32_t)dpp_i<kDppMirror>((int)top));
              const uint32_t byte = mx_scale_byte(top);
              const float s = __uint_as_float(byte << 23);
              uint32_t w =
                  __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, towards_zero<FTM_DT_F32>(y[0]), towards_zero<FTM_DT_F32>(y[1]), s, 0);
              if constexpr (CN == 4)
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, towards_zero<FTM_DT_F32>(y[2]), towards_zero<FTM_DT_F32>(y[3]), s, 1);
              w = byte == 255u ? 0u : positive_zeros(w);
              if (t < cur.rt.cnt && n0 < NO) {
                const int64_t row = cur.rt.row0 + t;
                if constexpr (CN == 4) *(uint16_t*)((char*)c.out + (row * NO + n0) / 2) = (uint16_t)w;
                else *((uint8_t*)c.out + (row * NO + n0) / 2) = (uint8_t)w;
                if ((em & (32 / CN - 1)) == 0) out_scale[(row * NO + n0) / 32] = (uint8_t)byte;
              }
            });
          } else if (out.vec && c.out_dtype == FTM_DT_BF16) {
            each_row([&](int t, const float(&y)[CN]) __attribute__((always_inline)) { out.template store_vec<FTM_DT_BF16>(t, y); });
          } else if (out.vec && c.out_dtype == FTM_DT_F32) {
            each_row([&](int t, const float(&y)[CN]) __attribute__((always_inline)) { out.template store_vec<FTM_DT_F32>(t, y); });
          } else if (out.vec) {
            each_row([&](int t, const float(&y)[CN]) __attribute__((always_inline)) { out.template store_vec<FTM_DT_F16>(t, y); });
          } else {
            constexpr int ON = CN == 8 ? 4 : CN;  // of a store of any alignment
            each_row([&](int t, const float(&y)[CN]) __attribute__((always_inline)) {
#pragma unroll
              for (int o = 0; o < CN; o += ON) {
                float z[ON];
#pragma unroll
                for (int n = 0; n < ON; ++n) z[n] = y[o + n];
                RowOut<ON>(c, cur.rt, NO, n0 + o).store(t, z);
              }
            });
          }
        }
      });
      if constexpr (GROUPED && !QOUT) {  // rows whose index names none: zeros over them
        if (live != kAllRows) {
          wait_vm<0>();  // behind the results
          for (int o = 0; o < CN; ++o)
            for (int t = 0; t < 4 * MI; ++t) {
              const int row = t0 + 16 * (t >> 2) + (t & 3);
              if (!((live >> t) & 1u) && row < cur.rt.cnt && n0 + o < NO)
                store_scalar(c.out, (cur.rt.row0 + row) * NO + n0 + o, c.out_dtype, 0.0f);
            }
        }
      }
      if (after >= end) break;
      cur = next;
      item = after;
    }
    wait_vm<0>();  // the copies past the last step, before the LDS is given back
  }
  if constexpr (GROUPED && !QOUT) {  // rows of no expert
    const int head = scan.head(), tail = scan.tail(), none = head + ((int)c.rows - tail);
    for (int z = blockIdx.x; z < none; z += gridDim.x) {
      const int64_t row = z < head ? z : tail + (z - head);
      for (int n = threadIdx.x; n < NO; n += kThreads) store_scalar(c.out, row * NO + n, c.out_dtype, 0.0f);
    }
  }
}

namespace {

hipError_t any(const ftm_w4a4& c, hipStream_t st) {
  const int64_t mt = row_tiles(c, 16), nt = (out_cols(c) + 15) / 16;
  const int64_t wgs = (mt * nt + 3) / 4, grid = wgs < kMaxGroups ? wgs : kMaxGroups;
  if (mt > INT32_MAX) return hipErrorInvalidValue;
  if (c.act >= 0) k_w4a4_any<true><<<dim3((unsigned)grid), dim3(256), 0, st>>>(c, (int)mt, (int)nt);
  else k_w4a4_any<false><<<dim3((unsigned)grid), dim3(256), 0, st>>>(c, (int)mt, (int)nt);
  return hipGetLastError();
}

constexpr int kMaxLds = 160 * 1024, kListLds = 1024;  // of which k_w4a4_cols has its lists

template <int MT, int NT, int NW, int S>
int split_lds(const ftm_w4a4& c) {
  constexpr int ring = NW * S * (MT + NT) * 16 * kRow, sums = NW * MT * NT * 1024;
  const int nsteps = (c.K + 255) / 256, lds = ring + NW * (MT + NT) * 16 * scale_pitch((nsteps + NW - 1) / NW);
  return lds > sums ? lds : sums;
}
template <int MT, int NT, int NW, int S>
bool split_fits(const ftm_w4a4& c) {
  const int cols = c.act >= 0 ? 8 * NT : 16 * NT;
  return split_lds<MT, NT, NW, S>(c) <= kMaxLds && row_tiles(c, 16 * MT) * ((out_cols(c) + cols - 1) / cols) <= kMaxGroups;
}
template <int MT, int NT, int NW, int S>
hipError_t split(const ftm_w4a4& c, hipStream_t st) {
  const int cols = c.act >= 0 ? 8 * NT : 16 * NT;
  const int64_t mt = row_tiles(c, 16 * MT), nt = (out_cols(c) + cols - 1) / cols;
  static DeviceBits lds_set{0};
  const hipError_t e = allow_lds(lds_set, (const void*)k_w4a4_split<MT, NT, NW, S>, kMaxLds);
  if (e != hipSuccess) return e;
  k_w4a4_split<MT, NT, NW, S><<<dim3((unsigned)(mt * nt)), dim3(64 * NW), split_lds<MT, NT, NW, S>(c), st>>>(c, (int)mt, (int)nt);
  return hipGetLastError();
}

template <int S>
int cols_lds(int K, int rows) {
  const int nsteps = (K + 255) / 256, codes = nsteps * rows * kRow, pitch = scale_pitch(nsteps);
  return 4 * S * 16 * kRow + (codes > 16 * 36 * 4 ? codes : 16 * 36 * 4) + (rows + 64) * pitch;
}
template <int RW, int S>
bool cols_fits(const ftm_w4a4& c) {
  const int per = c.act >= 0 ? 32 : 64;
  return cols_lds<S>(c.K, RW) <= kMaxLds - kListLds && row_tiles(c, RW) * ((out_cols(c) + per - 1) / per) <= kMaxGroups;
}
template <int RW, int S>
hipError_t cols(const ftm_w4a4& c, hipStream_t st) {
  const int per = c.act >= 0 ? 32 : 64;
  const int64_t mt = row_tiles(c, RW), nt = (out_cols(c) + per - 1) / per;
  static DeviceBits lds_set{0};
  const auto kernel = k_w4a4_cols<-1, RW, S, ftm_w4a4>;
  const hipError_t e = allow_lds(lds_set, (const void*)kernel, kMaxLds - kListLds);
  if (e != hipSuccess) return e;
  kernel<<<dim3((unsigned)(mt * nt)), dim3(256), cols_lds<S>(c.K, RW), st>>>(c, (int)nt);
  return hipGetLastError();
}

template <int WM, int WN, int MI, int NJ, int S, bool ACT, bool GROUPED, bool QOUT>
hipError_t tile(const ftm_w4a4& c, uint8_t* out_scale, hipStream_t st) {
  constexpr int BM = 16 * MI * WM, BN = 16 * NJ * WN, lds = S * (BM + BN) * kRow + 16 * (BM + BN) + 4 * BM;
  static_assert(lds <= kMaxLds, "fits a CU");
  constexpr int resident = kCUs * (2 * lds <= kMaxLds ? 2 : 1);  // workgroups the chip holds at once
  const int cols = ACT ? BN / 2 : BN;
  const int64_t mt = row_tiles(c, BM), nt = (out_cols(c) + cols - 1) / cols;
  if (mt * nt > INT32_MAX) return hipErrorInvalidValue;
  static DeviceBits lds_set{0};
  const auto kernel = k_w4a4_tile<WM, WN, MI, NJ, S, ACT, GROUPED, QOUT>;
  const hipError_t e = allow_lds(lds_set, (const void*)kernel, lds);
  if (e != hipSuccess) return e;
  const int64_t grid = mt * nt < resident ? (mt * nt + 7) / 8 * 8 : resident;  // the same for every XCD
  kernel<<<dim3((unsigned)grid), dim3(64 * WM * WN), lds, st>>>(c, out_scale, (int)mt, (int)nt);
  return hipGetLastError();
}
template <int WM, int WN, int MI, int NJ, int S, bool GROUPED>
hipError_t tile(const ftm_w4a4& c, hipStream_t st) {
  return c.act >= 0 ? tile<WM, WN, MI, NJ, S, true, GROUPED, false>(c, nullptr, st)
                    : tile<WM, WN, MI, NJ, S, false, GROUPED, false>(c, nullptr, st);
}

// Whether a tile's 32-bit offsets (below 2^30) reach its tokens (256 rows from its
// first, or all of x where they are read through an index), its weight rows and its results.
bool offsets_ok(const ftm_w4a4& c) {
  const int64_t rows = c.row_index != nullptr ? c.x_rows : c.x_rows < 256 ? c.x_rows : 256;
  const int64_t wrows = 256 + (c.act >= 0 ? c.N / 2 : 0), Kb = c.K / 2 + 256;
  return rows * Kb < (int64_t)kNowhere && wrows * Kb < (int64_t)kNowhere && 4 * 256 * (int64_t)c.N < (int64_t)kNowhere;
}

}  // namespace

// The mean rows of the experts that can have any.
static int64_t rows_an_expert(const ftm_w4a4& c) {
  const int64_t hit = c.rows < c.num_experts ? c.rows : c.num_experts;
  return (c.rows + hit - 1) / hit;
}
constexpr int kTileRows = 16, kLargeRows = 96;  // an expert: from these on tiles of 64 x 256, of 256 x 256

// By the rows an expert has.  In us, for 128 experts of [2 x 768, 2048] through an index, of [2048, 768], and 32
// of [2 x 2880, 2880] through an index, by the mean rows of an expert; their popularity is uneven (at a mean of
// 256 rows 25 to 1000), so that of few rows not all are hit, and of many most tiles of 256 are partly filled:
//                     1 row              4 rows             8 rows             12 rows
//   cols of 8         25.0  15.3  41.2   40.7  23.4  61.4   49.8  33.4  79.2   58.2  42.3  97.8
//   cols of 16        24.4  14.9  44.7   41.7  21.5  61.7   48.2  27.6  71.4   51.6  33.3  77.7
//   tiles 64 x 256                       50.0  28.4  79.8   51.8  30.4  82.7   53.4  31.8  82.4
//                     16 rows            64 rows            96 rows            128 rows
//   cols of 16        56.8  36.8  88.7
//   tiles 64 x 256    56.7  34.1  84.2   68.8  48.8 117.1   84.5  57.8 136.6   94.3  66.8
//   tiles 256 x 256                      90.4  57.0 109.8   90.5  58.4 128.9   92.3  59.7
// The same rows for every expert, gate_up, 128 experts and 32: tiles of 64 at 64 rows 52.0 and 78.0, of 256 70.0 and
// 96.0; at 96 rows 75.0 and 123.0, 71.5 and 98.0; at 128 rows 77.0 and 125.4, 73.3 and 99.5.  At 16 rows cols of
// 16 would be the faster there, 48.0 and 69.5, tiles of 64 50.1 and 74.3.
// Tiles of 128 x 256 (94.2, 53.6, 133.0 at 96 rows) gain less than 7% and only there.  Where
// the codes of few rows do not fit the LDS (K above 13 thousand) it is tiles too.
static hipError_t grouped(const ftm_w4a4& c, hipStream_t st) {
  const int64_t seg = rows_an_expert(c);
  if (seg >= kLargeRows) return tile<2, 2, 8, 8, 2, true>(c, st);
  if (seg <= 2 && cols_fits<8, 2>(c)) return cols<8, 2>(c, st);
  if (seg < kTileRows && cols_fits<16, 2>(c)) return cols<16, 2>(c, st);
  return tile<2, 2, 2, 8, 3, true>(c, st);
}

// Blocks that the chip holds at once take one another's time; of the tiles, the least time of
// all rounds is taken, a round of 256 workgroups being 4, 7 and 9 (13, 23.5 and 30 us at K = 4096).
// In us, M x N x K:
//   16 x 16 (K over four waves) against 32 x 16:  16 x 4096 x 4096 4.1, 4.9; 16 x 12288 x 4096 9.0, 11.9
//   32 x 16 against 32 x 32:  32 x 4096 x 4096 5.1, 5.5; x 12288 11.3, 8.9; x 5760 x 2880 6.9, 5.8
//   32 x 32 against 64 x 64 (eight waves):  512 blocks 9.4, 11.5; 528 9.6, 8.1; 540 12.7, 10.3; 768 13.9, 11.5
//   32 x 32 against tiles, K = 11008 where 64 x 64 does not fit:  640 blocks 28.3, 32.0; 1024 39.8, 32.9
//   64 x 64 against tiles of 128 x 128:  256 blocks 12.3, 15.5; 270 18.1, 13.4; 384 21.1, 15.7
//   tiles of 128 x 128, 128 x 256 and 256 x 256:  1024 x 4096 x 4096 18.5, 25.0, 29.7; 2048 x 4096 x 4096
//   31.2, 29.0, 31.5; 1024 x 12288 x 4096 42.3, 46.2, 33.0; 2048 x 12288 x 4096 78.4, 71.6, 64.1
static hipError_t dense(const ftm_w4a4& c, hipStream_t st) {
  const int64_t M = c.rows;
  const auto blocks = [&](int rows, int cols) { return ((M + rows - 1) / rows) * ((c.N + cols - 1) / cols); };
  if (M <= 16 && split_fits<1, 1, 4, 4>(c)) return split<1, 1, 4, 4>(c, st);
  if (M <= 32 && blocks(32, 16) <= kCUs && split_fits<2, 1, 4, 3>(c)) return split<2, 1, 4, 3>(c, st);
  const bool few64 = blocks(64, 64) <= kCUs && split_fits<4, 4, 8, 1>(c);
  if ((blocks(32, 32) <= 2 * kCUs || (blocks(32, 32) <= 3 * kCUs && !few64)) && split_fits<2, 2, 4, 2>(c))
    return split<2, 2, 4, 2>(c, st);
  if (few64) return split<4, 4, 8, 1>(c, st);
  const auto time = [&](int rows, int cols, int each) { return (blocks(rows, cols) + kCUs - 1) / kCUs * each; };
  const int64_t t128 = time(128, 128, 4), t256 = time(128, 256, 7), t512 = time(256, 256, 9);
  if (t128 <= t256 && t128 <= t512) return tile<2, 2, 4, 4, 4, false>(c, st);
  return t256 <= t512 ? tile<2, 2, 4, 8, 3, false>(c, st) : tile<2, 2, 8, 8, 2, false>(c, st);
}

hipError_t launch_w4a4(const ftm_w4a4& c, hipStream_t st) {
  if (c.K < kMinK || !offsets_ok(c)) return any(c, st);
  return c.offsets != nullptr ? grouped(c, st) : dense(c, st);
}

namespace {

constexpr bool few_rings_aligned() {
  for (int rows = 1; rows <= kFewRows; ++rows)
    for (int per = 1; per <= 16; ++per)
      if (few_wave_lds<1, 4>(per, rows) % kRow != 0) return false;
  return true;
}
static_assert(few_rings_aligned(), "each wave's ring begins on a stage row's border");

template <int NT, int NW, int S>
int few_lds(int K, int rows) {
  const int per = ((K + 255) / 256 + NW - 1) / NW;
  const int lds = NW * few_wave_lds<NT, S>(per, rows);
  constexpr int sums = NW * NT * 1024;
  return lds > sums ? lds : sums;
}
template <int XDT, int NT, int NW, int S>
hipError_t few(const FewCall& c, hipStream_t st) {
  const int cols = c.act >= 0 ? 8 * NT : 16 * NT, NO = c.act >= 0 ? c.N / 2 : c.N;
  static DeviceBits lds_set{0};
  const auto kernel = k_w4a4_few<XDT, NT, NW, S>;
  const hipError_t e = allow_lds(lds_set, (const void*)kernel, kMaxLds);
  if (e != hipSuccess) return e;
  kernel<<<dim3((unsigned)((NO + cols - 1) / cols)), dim3(64 * NW), few_lds<NT, NW, S>(c.K, c.cap), st>>>(c);
  return hipGetLastError();
}
template <int NT, int NW, int S>
hipError_t few(const FewCall& c, int dt, hipStream_t st) {
  if (dt == FTM_DT_F32) return few<FTM_DT_F32, NT, NW, S>(c, st);
  if (dt == FTM_DT_F16) return few<FTM_DT_F16, NT, NW, S>(c, st);
  return few<FTM_DT_BF16, NT, NW, S>(c, st);
}

template <int XDT, int S>
hipError_t cols_moe(const FewCall& c, hipStream_t st) {
  const int ntiles = c.N / 64;
  static DeviceBits lds_set{0};
  const auto kernel = k_w4a4_cols<XDT, 16, S, FewCall>;
  const hipError_t e = allow_lds(lds_set, (const void*)kernel, kMaxLds - kListLds);
  if (e != hipSuccess) return e;
  kernel<<<dim3((unsigned)(c.P * ntiles)), dim3(256), cols_lds<S>(c.K, c.cap), st>>>(c, ntiles);
  return hipGetLastError();
}
template <int S>
hipError_t cols_moe(const FewCall& c, int dt, hipStream_t st) {
  if (dt == FTM_DT_F32) return cols_moe<FTM_DT_F32, S>(c, st);
  if (dt == FTM_DT_F16) return cols_moe<FTM_DT_F16, S>(c, st);
  return cols_moe<FTM_DT_BF16, S>(c, st);
}

}  // namespace

// A layer of few tokens in two kernels, if it is one: hq and hs hold h, a row a pair.  Against
// the kernels of any layer (sort, quantise, product, quantise, product, sum; without the gaps
// between six launches), in us: 16 experts of 512 at 16 tokens 11.9, 25.8; 128 of 768 at 1 token 11.9, 27.6,
// at 16 49.1, 62.0; 32 of 2880 at 1 token 18.9, 34.4, at 8 75.1, 78.9, at 16 108.5, 92.9.  The
// limits are the 16 columns of a product, for an expert's tokens are one workgroup's, and what the
// second product reads again, an expert's weights once for each of its tokens: at least 64 MB of it (32
// of 2880 from 13 tokens on) and the kernels of any layer are faster.
bool launch_w4a4_moe_few(const ftm_w4a4_moe& c, uint8_t* hq, uint8_t* hs, hipStream_t st, hipError_t& e) {
  const int P = c.T * c.k, H = c.hidden, I = c.inter, cap = c.T < kFewRows ? c.T : kFewRows;
  if (c.T > kFewRows || P > kFewPairs || c.k > 64 || H < kMinK || I < kMinK) return false;
  if ((((uintptr_t)c.x | (uint64_t)c.x_stride) & 15u) != 0) return false;
  if ((int64_t)(P - (P < c.num_experts ? P : c.num_experts)) * H * (I / 2) > (64 << 20)) return false;
  if ((int64_t)2 * I * (H / 2) + 256 >= (int64_t)kNowhere) return false;
  const FewCall f = {(const char*)c.x, c.x_stride, (const char*)c.w13, c.w13_scale, c.w13_bias, (int64_t)2 * I * (H / 2),
                     (int64_t)2 * I * (H / 32), 2 * I, H, c.w13_bias_dtype, c.act, c.act_alpha, c.act_limit, cap, nullptr, 0,
                     c.topk_ids, c.ids_dtype == FTM_ID_I64, P, c.num_experts, c.k, hq, hs};
  if (cols_lds<2>(H, cap) > kMaxLds - kListLds) return false;
  e = cols_moe<2>(f, c.dtype, st);
  if (e != hipSuccess) return true;
  const int ntiles = (H + 15) / 16;
  k_w4a4_few_down<8, 3><<<dim3((unsigned)(ntiles * c.T)), dim3(512), 0, st>>>(c, hq, hs, ntiles);
  e = hipGetLastError();
  return true;
}

// Rows sorted by expert through a gated activation, the result quantised: out holds its
// blocks [rows, N / 64, 16] and out_scale their scales.  On tiles the epilogue does it,
// else (h: scratch, fp32 [rows, N / 2]) a kernel of its own; rows of no expert are then
// those of zeros, on tiles left as they were.
hipError_t launch_w4a4_quantised(const ftm_w4a4& c, float* h, uint8_t* out_scale, hipStream_t st) {
  const int64_t seg = rows_an_expert(c);
  // In us, on uneven popularity as above, tiles of 64 x 256, 128 x 256 and 256 x 256, with the quantisation in the
  // epilogue, for 128 experts of [2 x 768, 2048] and 32 of [2 x 2880, 2880]: 64 rows an expert 72.9, 79.7, 110.8 and
  // 119.3, 122.1, 124.8; 96 rows 91.5, 91.8, 113.5 and 139.8, 129.9, 149.3; 128 rows 102.3, 96.9, 114.6
  // and 172.2, 144.8, 159.6; 200 rows 134.2, 134.8, 140.6 and 227.0, 176.9, 171.2; 256 rows 166.6, 145.5,
  // 142.4 and 267.5, 207.1, 197.8.
  // Below 12, the columns' kernel and the quantiser: at 8 rows 48.3 + 4.2 against 55.1 on tiles, 71.4 + 4.2 against
  // 82.6; at 12 rows 51.0 + 4.2 against 55.4, 79.2 + 4.2 against 83.6, and one launch more.
  if (c.K >= kMinK && offsets_ok(c) && seg >= 12) {
    if (seg >= 200) return tile<2, 2, 8, 8, 2, true, true, true>(c, out_scale, st);
    if (seg >= 96) return tile<2, 2, 4, 8, 3, true, true, true>(c, out_scale, st);
    return tile<2, 2, 2, 8, 3, true, true, true>(c, out_scale, st);
  }
  ftm_w4a4 wide = c;
  wide.out = h;
  wide.out_dtype = FTM_DT_F32;
  const hipError_t e = launch_w4a4(wide, st);
  const int I = out_cols(c);
  return e != hipSuccess ? e : launch_quant_mxfp4(h, FTM_DT_F32, c.rows, I, (int64_t)I * 4, (uint8_t*)c.out, out_scale, st);
}

// Few values: each workgroup of the product quantises them all, and one launch does.  In us,
// against the quantiser and the product (and the gap between them, which is not in these
// figures): 2 x 1536 x 2048 4.9, 5.7; 8 x 1536 x 2048 7.1, 7.5; 4 x 4096 x 4096 7.5, 8.0;
// 8 x 4096 x 4096 11.9, 7.8; 1 x 4096 x 11008 10.5, 10.6; 2 x 4096 x 11008 12.2, 10.9.
hipError_t launch_w4a4_dynamic(const ftm_w4a4& c, const void* x, int dt, int64_t x_stride, hipStream_t st) {
  if (c.offsets == nullptr && c.rows <= 8 && c.rows * c.K <= 16384 && c.K >= kMinK && offsets_ok(c) &&
      (((uintptr_t)x | (uint64_t)x_stride) & 15u) == 0) {
    const FewCall f = {(const char*)x, x_stride, (const char*)c.w, c.w_scale, c.bias, 0, 0, c.N, c.K, c.bias_dtype, c.act, c.act_alpha,
                       c.act_limit, (int)c.rows, c.out, c.out_dtype, nullptr, 0, 0, 1, 1, nullptr, nullptr};
    return few<1, 4, 4>(f, dt, st);
  }
  const hipError_t e = launch_quant_mxfp4(x, dt, c.x_rows, c.K, x_stride, (uint8_t*)const_cast<void*>(c.x),
                                          const_cast<uint8_t*>(c.x_scale), st);
  return e != hipSuccess ? e : launch_w4a4(c, st);
}

}  // namespace ftm
