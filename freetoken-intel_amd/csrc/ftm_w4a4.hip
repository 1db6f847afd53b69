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

// Four lanes a block, NV blocks' parts a lane, 256 lanes apart.  x is read once and in
// whole lines; bound by HBM.  FLAT: rows side by side in memory, taken as one.
template <int DT, int NV, bool FLAT, bool ALIGNED>
__global__ __launch_bounds__(256) void k_quant_mxfp4(const char* x, int64_t x_stride, int64_t rows, int K, int per_row,
                                                     uint32_t* blocks, uint8_t* scales) {
  const int64_t wg = grid_row(), vecs = FLAT ? rows * (K / 8) : K / 8;
  const int64_t row = FLAT ? 0 : wg / per_row;
  if (row >= rows) return;
  const int64_t first = (FLAT ? wg : wg - row * per_row) * (256 * NV) + threadIdx.x;
  const char* src = x + row * x_stride;
  const int64_t at = row * (K / 8);
  Vec8<DT> v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t k = first + 256 * i;
    if (k >= vecs) v[i].zero();
    else if constexpr (ALIGNED) v[i].load(src + k * Vec8<DT>::kBytes);
    else v[i].load_any(src + k * Vec8<DT>::kBytes);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t k = first + 256 * i;
    const uint32_t byte = mx_scale_byte(quad_max(v[i].max_bits()));
    const uint32_t w = mx_codes<DT>(v[i], byte);
    if (k >= vecs) continue;
    blocks[at + k] = w;
    if ((threadIdx.x & 3) == 0) scales[(at + k) >> 2] = (uint8_t)byte;
  }
}

template <int DT, int NV>
hipError_t quant(const char* x, int64_t x_stride, int64_t rows, int K, uint32_t* blocks, uint8_t* scales, hipStream_t st) {
  const int64_t row_bytes = (int64_t)K / 8 * Vec8<DT>::kBytes;
  const bool flat = x_stride == row_bytes || rows == 1, aligned = (((uintptr_t)x | (uint64_t)(rows > 1 ? x_stride : 0)) & 15u) == 0;
  const int per_row = (K / 8 + 256 * NV - 1) / (256 * NV);
  const dim3 grid = row_grid(flat ? (rows * (K / 8) + 256 * NV - 1) / (256 * NV) : rows * per_row), wg(256);
  if (flat && aligned) k_quant_mxfp4<DT, NV, true, true><<<grid, wg, 0, st>>>(x, x_stride, rows, K, per_row, blocks, scales);
  else if (flat) k_quant_mxfp4<DT, NV, true, false><<<grid, wg, 0, st>>>(x, x_stride, rows, K, per_row, blocks, scales);
  else if (aligned) k_quant_mxfp4<DT, NV, false, true><<<grid, wg, 0, st>>>(x, x_stride, rows, K, per_row, blocks, scales);
  else k_quant_mxfp4<DT, NV, false, false><<<grid, wg, 0, st>>>(x, x_stride, rows, K, per_row, blocks, scales);
  return hipGetLastError();
}

hipError_t launch_quant_mxfp4(const void* x, int dt, int64_t rows, int K, int64_t x_stride, uint8_t* blocks,
                              uint8_t* scales, hipStream_t st) {
  const char* p = (const char*)x;
  uint32_t* b = (uint32_t*)blocks;
  if (dt == FTM_DT_F32) return quant<FTM_DT_F32, 1>(p, x_stride, rows, K, b, scales, st);
  if (dt == FTM_DT_F16) return quant<FTM_DT_F16, 1>(p, x_stride, rows, K, b, scales, st);
  return quant<FTM_DT_BF16, 1>(p, x_stride, rows, K, b, scales, st);
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
        if constexpr (ACT)
          y = gated(c.act, y, acc[1][r] + (c.bias != nullptr ? load_scalar(c.bias, at + NO, c.bias_dtype) : 0.0f), c);
      }
      store_scalar(c.out, (rt.row0 + m) * NO + n, c.out_dtype, y);
    }
  }
}

hipError_t launch_w4a4(const ftm_w4a4& c, hipStream_t st) {
  const int64_t mt = row_tiles(c, 16), nt = (out_cols(c) + 15) / 16;
  const int64_t wgs = (mt * nt + 3) / 4, grid = wgs < kMaxGroups ? wgs : kMaxGroups;
  if (mt > INT32_MAX) return hipErrorInvalidValue;
  if (c.act >= 0) k_w4a4_any<true><<<dim3((unsigned)grid), dim3(256), 0, st>>>(c, (int)mt, (int)nt);
  else k_w4a4_any<false><<<dim3((unsigned)grid), dim3(256), 0, st>>>(c, (int)mt, (int)nt);
  return hipGetLastError();
}

hipError_t launch_w4a4_dynamic(const ftm_w4a4& c, const void* x, int dt, int64_t x_stride, hipStream_t st) {
  const hipError_t e = launch_quant_mxfp4(x, dt, c.x_rows, c.K, x_stride, (uint8_t*)const_cast<void*>(c.x),
                                          const_cast<uint8_t*>(c.x_scale), st);
  return e != hipSuccess ? e : launch_w4a4(c, st);
}

}  // namespace ftm
