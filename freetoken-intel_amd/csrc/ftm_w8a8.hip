// ftm_w8a8.hip -- int8 activations x int8 weights: the per-token quantiser and
// the integer product with one scale per token and one per output channel,
// dense or grouped by expert (rows sorted by expert, one weight per expert).
//
//   s_m = max_k |x_mk| * (1 / 127), both fp32, q_mk = the whole number nearest x_mk / s_m
//   y_mn = (sum_k q_mk w_nk) s_m t_n (+ b_n), optionally h = act(gate) * up
//
// The sum is exact in int32 (K <= 131071, checked by the callers), so its order
// is free: every kernel here returns the same bits whatever its tile and
// however it splits K.  One rounding of the sum to fp32, one for each scale and
// for the bias, one to the output dtype.
//
// Operands of v_mfma_i32_16x16x64_i8 (lane l): A[i][k] i = l % 16, B[k][j] j =
// l % 16, both k = 16 (l / 16) + 0..15; D[i][j] j = l % 16, i = 4 (l / 16) +
// 0..3.  Where K is split over the waves the weights are A and the tokens B, so a
// lane's results are neighbouring output channels of one token; in the LDS tiles
// the tokens are A and the weights B, so a lane has four tokens of one channel a
// block, and the order in which the weight rows are laid into LDS makes the
// channels of its blocks neighbours.
#include "ftm_rows.h"

namespace ftm {

typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ i32x4 mfma_i8(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// A weight operand for the product: packed bytes are offset by 128, and past K (keep
// 0, else all ones) it has to be zero.  Bit operations: a choice would be a branch
// between the MFMA and what it reads.
template <bool PACKED>
__device__ __forceinline__ u32x4 weight_operand(u32x4 v, uint32_t keep) {
  return PACKED ? (v ^ 0x80808080u) & keep : v & keep;
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

// A row's scale and the factor of its first guess.  The product with the fp32
// nearest 1 / 127, not a division: what torch makes of `amax / 127` on the GPU, so
// the codes are those of a torch quantiser there (where the scales are an ulp
// apart, quotients of bf16 values that end in .5 round to other codes).  A row with a value that is
// not finite gets the scale NaN and codes 0, so its outputs are NaN and no
// other row's change.
struct QuantScale {
  float s, inv;
};
__device__ __forceinline__ QuantScale quant_scale(uint32_t max_bits) {
  if (max_bits >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.0f};
  const float s = fmaxf(__uint_as_float(max_bits), 1e-12f) * (1.0f / 127.0f);
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
  const int64_t row = grid_row() * kRows + wave / WPR;
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
__global__ __launch_bounds__(256) void k_quant_int8_any(const char* x, int64_t x_stride, int64_t rows, int K, int8_t* q,
                                                        int64_t q_stride, float* scale) {
  __shared__ uint32_t wmax[4];
  const int64_t row = grid_row();
  if (row >= rows) return;
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
    k_quant_int8_any<DT><<<row_grid(rows), dim3(256), 0, st>>>(x, x_stride, rows, K, q, q_stride, scale);
    return hipGetLastError();
  }
  const dim3 by4 = row_grid((rows + 3) / 4), by1 = row_grid(rows), wg(256);
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

// One result: the sum(s) of channel `col` with the token's scale.
struct Channel {
  float t, b;
};
__device__ __forceinline__ Channel channel(const ftm_w8a8& c, int e, int n) {
  const int64_t i = (int64_t)e * c.N + n;
  return {load_scalar(c.w_scale, i, c.w_scale_dtype), c.bias != nullptr ? load_scalar(c.bias, i, c.bias_dtype) : 0.0f};
}
// The same as raw bits, requested ahead of their use (converting would wait for
// the load).
struct ChannelBits {
  uint32_t t, b;
};
__device__ __forceinline__ Channel channel(const ftm_w8a8& c, ChannelBits r) {
  return {bits_to_f32(opaque_bits(r.t), c.w_scale_dtype), bits_to_f32(opaque_bits(r.b), c.bias_dtype)};
}
__device__ __forceinline__ float scaled(int sum, float s, Channel ch) {
  return fmaf((float)sum * s, ch.t, ch.b);
}

// ------------------------------------------------------------------ K split over the waves
// One 16 x 16 block of results that a wave finishes from the waves' sums: a lane
// has weight rows 4 g .. 4 g + 3 of token m (with an activation rows 0..7 of a block
// are gate channels, 8..15 their up rows, and only lanes of the first eight have
// results).
struct SplitBlock {
  uint32_t t[8], b[8];  // scales and biases of its four channels, and of their up rows
  float xscale;         // the token's
  bool live;            // it names a row of x

  __device__ __forceinline__ void request(const ftm_w8a8& c, const RowTile& rt, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = b[i] = 0;
    if (rt.e < 0) return;
    const int last = out_cols(c) - 1;
    const int64_t at = (int64_t)rt.e * c.N;
    load_run<4>(c.w_scale, at, n, last, c.w_scale_dtype, t);
    if (c.act >= 0) load_run<4>(c.w_scale, at + last + 1, n, last, c.w_scale_dtype, t + 4);
    if (c.bias == nullptr) return;
    load_run<4>(c.bias, at, n, last, c.bias_dtype, b);
    if (c.act >= 0) load_run<4>(c.bias, at + last + 1, n, last, c.bias_dtype, b + 4);
  }
};

template <int NT>
__device__ __forceinline__ int split_channel(const ftm_w8a8& c, int n0, int block, int g) {
  return n0 + (c.act >= 0 ? 8 * (block % NT) + 4 * (g & 1) : 16 * (block % NT) + 4 * g);
}

// The waves' sums of the tile's MT x NT blocks, through LDS (which they may
// overwrite), and the results.
template <int MT, int NT, int NW, int PARTS>
__device__ __forceinline__ void split_finish(const ftm_w8a8& c, const RowTile& rt, char* lds, int n0,
                                             const i32x4 (&acc)[MT][NT], const SplitBlock (&blocks)[PARTS]) {
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  i32x4* red = (i32x4*)lds;  // [NW][MT * NT][64]
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) red[(wave * MT * NT + i * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  if (c.act >= 0 && g >= 2) return;
  with_act(c.act, [&](auto a) {
    constexpr int A = decltype(a)::value;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      const int f = p * NW + wave;
      if (MT * NT % NW != 0 && f >= MT * NT) continue;
      i32x4 u = {0, 0, 0, 0}, v = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        u += red[(w * MT * NT + f) * 64 + lane];
        if constexpr (A >= 0) v += red[(w * MT * NT + f) * 64 + lane + 32];
      }
      const SplitBlock& k = blocks[p];
      float y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        y[r] = scaled(u[r], k.xscale, channel(c, {k.t[r], k.b[r]}));
        if constexpr (A >= 0)
          y[r] = gated(A, y[r], scaled(v[r], k.xscale, channel(c, {k.t[4 + r], k.b[4 + r]})), c);
        y[r] = k.live ? y[r] : 0.0f;
      }
      RowOut<4>(c, rt, out_cols(c), split_channel<NT>(c, n0, f, g)).store(16 * (f / NT) + m, y);
    }
  });
}

// The weight rows of a split tile: copies of 8 rows, a 16-byte piece a lane, from
// the tile's first row (and the up rows N / 2 on); rows past the last copy it.
template <int NT>
struct SplitWeights {
  Rsrc res;
  uint32_t off[2 * NT];
  __device__ __forceinline__ SplitWeights(const ftm_w8a8& c, const RowTile& rt, int n0, int ncol) {
    const bool act = c.act >= 0;
    const int lane = threadIdx.x & 63, NO = out_cols(c);
    res = make_rsrc((const char*)c.w + (int64_t)rt.e * c.w_stride + (int64_t)n0 * c.K,
                    (uint32_t)((act ? NO : 0) + ncol) * (uint32_t)c.K);
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      const int r = 8 * i + (lane >> 3);
      int n = act ? 8 * (i >> 1) + (r & 7) : r;
      n = n < ncol ? n : ncol - 1;
      off[i] = (uint32_t)(n + (act && (i & 1) ? NO : 0)) * (uint32_t)c.K + 16u * (uint32_t)((lane & 7) ^ swz(r));
    }
  }
  __device__ __forceinline__ void issue(char* at, uint32_t k0) const {
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(res, (LPtr)(at + 1024 * i), 16, (int)(off[i] + k0), 0, 0, 0);
  }
};

// A workgroup's tile of 16 MT tokens x 16 NT weight rows (with an activation 8
// gate rows and their 8 up rows a block); each of the NW waves takes a run of
// K over the whole tile through an LDS ring of its own (S stages of 128 K), and
// the waves' sums meet in LDS.  No barrier in the K loop.  For few rows, and
// for grids too small for the tiles that share a ring.  The copies go to LDS
// because eight neighbouring lanes then read 128 bytes of one row: loads in
// operand layout touch another row with every lane, and a CU looks up four
// times as many cache lines for them.
template <int MT, int NT, int NW, int S, bool PACKED>
__global__ __launch_bounds__(64 * NW) void k_w8a8_split(ftm_w8a8 c, int mtiles, int ntiles) {
  constexpr int BM = 16 * MT, kStage = (MT + NT) * 16 * kRow, NC = 2 * (MT + NT);
  constexpr int kParts = (MT * NT + NW - 1) / NW;
  extern __shared__ char lds[];  // [NW][S][kStage], then the sums
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const RowTile rt = row_tile<BM>(c, item / ntiles);
  if (rt.cnt <= 0) return;
  const int NO = out_cols(c), K = c.K;
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cols = c.act >= 0 ? 8 * NT : 16 * NT;  // output channels of the tile
  const int n0 = (item % ntiles) * cols;
  const int ncol = NO - n0 < cols ? NO - n0 : cols;
  i32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};
  SplitBlock blocks[kParts];
  auto request_scales = [&] {
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const int f = p * NW + wave, r = 16 * (f / NT) + m;
      const int64_t src = f < MT * NT && r < rt.cnt && rt.e >= 0 ? source_row(c, rt.row0 + r) : -1;
      blocks[p].live = src >= 0;
      blocks[p].xscale = src >= 0 ? c.x_scale[src] : 0.0f;
      blocks[p].request(c, rt, split_channel<NT>(c, n0, f, g));
    }
  };
  const int nsteps = (K + 127) / 128, per = (nsteps + NW - 1) / NW;
  const int lo = wave * per, hi = lo + per < nsteps ? lo + per : nsteps;
  if (rt.e >= 0 && lo < hi) {
    // rows past the tile copy one inside it, pieces past K what follows the row
    // (their weights are made zero); offsets from the tile's first token, or, read
    // through an index, from x's
    const bool indexed = c.row_index != nullptr;
    const char* xbase = (const char*)c.x + (indexed ? 0 : rt.row0 * c.x_stride);
    const Rsrc xres = make_rsrc(xbase, (uint32_t)((indexed ? c.x_rows - 1 : (int64_t)rt.cnt - 1) * c.x_stride + K));
    const SplitWeights<NT> weights(c, rt, n0, ncol);
    uint32_t xoff[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
      const int r = 8 * i + (lane >> 3);
      int64_t s = r < rt.cnt ? r : 0;
      if (indexed) {
        s = source_row(c, rt.row0 + s);
        s = s < 0 ? 0 : s;
      }
      xoff[i] = (uint32_t)(s * c.x_stride) + 16u * (uint32_t)((lane & 7) ^ swz(r));
    }
    char* ring = lds + wave * (S * kStage);
    auto issue = [&](int step, int slot) {
      const uint32_t k0 = (uint32_t)(step < hi ? step : hi - 1) * 128u;
      char* st = ring + slot * kStage;
      weights.issue(st + 2048 * MT, k0);
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xres, (LPtr)(st + 1024 * i), 16, (int)(xoff[i] + k0), 0, 0, 0);
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue(lo + i, i);
    request_scales();  // behind the first copies and ahead of the K loop
    int slot = 0;
    for (int step = lo; step < hi; ++step) {
      issue(step + S - 1, slot == 0 ? S - 1 : slot - 1);
      wait_vm<(S - 1) * NC>();  // this step's copies have landed
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      const char* st = ring + slot * kStage;
      auto piece = [&](int r, int q) { return *(const u32x4*)(st + r * kRow + 16 * ((4 * q + g) ^ swz(r))); };
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t keep = step * 128 + 64 * q + 16 * g < K ? ~0u : 0u;
        u32x4 w[NT], x[MT];
#pragma unroll
        for (int j = 0; j < NT; ++j) w[j] = weight_operand<PACKED>(piece(16 * (MT + j) + m, q), keep);
#pragma unroll
        for (int i = 0; i < MT; ++i) x[i] = piece(16 * i + m, q);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i][j] = mfma_i8(w[j], x[i], acc[i][j]);
      }
      __builtin_amdgcn_sched_barrier(0);  // the next copies overwrite what these products have read
      slot = slot == S - 1 ? 0 : slot + 1;
    }
    wait_vm<0>();  // the copies past the last step, before the sums take their place
  } else {
    request_scales();
  }
  split_finish<MT, NT, NW>(c, rt, lds, n0, acc, blocks);
}

constexpr int kWideRows = 4;
constexpr int kWideK = 8192;  // their codes are kept in LDS

// The same for at most kWideRows tokens a tile whose values are still wide (XDT; x_stride
// bytes between rows): every workgroup quantises its tokens itself, each wave the
// K that it multiplies, into LDS, while its first weights are under way.  The
// codes and scales are the quantiser's; the launch that would write them is
// saved (the figures are at launch_w8a8_dynamic).
template <int XDT, int NT, int S, bool PACKED>
__global__ __launch_bounds__(256) void k_w8a8_wide(ftm_w8a8 c, const char* x, int64_t x_stride, int ntiles) {
  using V = QuantVec<XDT>;
  constexpr int kStage = NT * 16 * kRow, NC = 2 * NT;
  extern __shared__ char lds[];  // [4][S][kStage], then [step][kWideRows][kRow] codes
  __shared__ uint32_t maxima[4][16];
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const RowTile rt = row_tile<kWideRows>(c, item / ntiles);
  if (rt.cnt <= 0) return;
  const int NO = out_cols(c), K = c.K;
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cols = c.act >= 0 ? 8 * NT : 16 * NT;
  const int n0 = (item % ntiles) * cols;
  const int ncol = NO - n0 < cols ? NO - n0 : cols;
  i32x4 acc[1][NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[0][j] = (i32x4){0, 0, 0, 0};
  SplitBlock blocks[1];
  const int nsteps = (K + 127) / 128, per = (nsteps + 3) / 4;
  const int lo = wave * per < nsteps ? wave * per : nsteps, hi = lo + per < nsteps ? lo + per : nsteps;
  const int64_t src = m < rt.cnt && rt.e >= 0 ? source_row(c, rt.row0 + m) : -1;  // of row m
  blocks[0].live = src >= 0;
  blocks[0].xscale = 0.0f;
  if (rt.e >= 0) {
    const SplitWeights<NT> weights(c, rt, n0, ncol);
    char* ring = lds + wave * (S * kStage);
    char* codes = lds + 4 * S * kStage;
    auto issue = [&](int step, int slot) {
      weights.issue(ring + slot * kStage, (uint32_t)(step < hi ? step : nsteps - 1) * 128u);
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue(lo + i, i);
    blocks[0].request(c, rt, split_channel<NT>(c, n0, wave, g));
    // the largest of each row: this wave's K, then all waves'
    const int k_hi = hi * 128 < K ? hi * 128 : K;
    auto row_at = [&](int r) {
      const int s = __builtin_amdgcn_readlane((int)src, r);
      return x + (int64_t)(s < 0 ? 0 : s) * x_stride;
    };
    const char* p[kWideRows];
#pragma unroll
    for (int r = 0; r < kWideRows; ++r) p[r] = row_at(r);
    uint32_t v[kWideRows] = {};
    for (int k = lo * 128 + lane * V::kN; k < k_hi; k += 64 * V::kN)
#pragma unroll
      for (int r = 0; r < kWideRows; ++r)
        if (r < rt.cnt) {
          const uint32_t b = V::max_bits(*(const u32x4*)(p[r] + (int64_t)k * (16 / V::kN)));
          v[r] = b > v[r] ? b : v[r];
        }
    uint32_t mine = 0;
#pragma unroll
    for (int r = 0; r < kWideRows; ++r) {
      const uint32_t top = r < rt.cnt ? wave_max_bits(v[r]) : 0;
      mine = m == r ? top : mine;
    }
    if (lane < 16) maxima[wave][lane] = mine;
    __syncthreads();
    uint32_t top = maxima[0][m];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = maxima[w][m] > top ? maxima[w][m] : top;
    const QuantScale own = quant_scale(top);  // of row m
    blocks[0].xscale = own.s;
    for (int k = lo * 128 + lane * V::kN; k < k_hi; k += 64 * V::kN)
#pragma unroll
      for (int r = 0; r < kWideRows; ++r)
        if (r < rt.cnt) {
          const QuantScale qs = {readlane_f(own.s, r), readlane_f(own.inv, r)};
          V::store((int8_t*)codes + ((k >> 7) * kWideRows + r) * kRow + 16 * (((k >> 4) & 7) ^ swz(r)) + (k & 15),
                   *(const u32x4*)(p[r] + (int64_t)k * (16 / V::kN)), qs);
        }
    __builtin_amdgcn_wave_barrier();
    const int xr = m < rt.cnt ? m : 0;
    int slot = 0;
    for (int step = lo; step < hi; ++step) {
      issue(step + S - 1, slot == 0 ? S - 1 : slot - 1);
      wait_vm<(S - 1) * NC>();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      const char* st = ring + slot * kStage;
      const char* xt = codes + step * kWideRows * kRow;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t keep = step * 128 + 64 * q + 16 * g < K ? ~0u : 0u;
        const u32x4 xv = *(const u32x4*)(xt + xr * kRow + 16 * ((4 * q + g) ^ swz(xr)));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int r = 16 * j + m;
          const u32x4 v = *(const u32x4*)(st + r * kRow + 16 * ((4 * q + g) ^ swz(r)));
          acc[0][j] = mfma_i8(weight_operand<PACKED>(v, keep), xv, acc[0][j]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      slot = slot == S - 1 ? 0 : slot + 1;
    }
    wait_vm<0>();
  }
  split_finish<1, NT, 4>(c, rt, lds, n0, acc, blocks);
}

// ------------------------------------------------------------------ LDS tiles
// A tile is BM = 16 MI WM tokens x 256 weight rows (with an activation 128 gate
// rows and their up rows): 4 WM waves of 16 MI tokens x 64 weight rows each over
// the whole K.  Tokens and weights go through a ring of S LDS stages of 128 K,
// filled by direct copies S steps ahead, one barrier a step.  A workgroup takes
// one tile after another, and the copies run on from tile to tile: the first
// stages of the next are under way during the last products and the epilogue
// of this one.

template <int WM, int MI, int S, bool PACKED, bool ACT, bool TAIL, bool GROUPED, bool ONCE>
__global__ __launch_bounds__(256 * WM, 2) void k_w8a8_tile(ftm_w8a8 c, int mtiles, int ntiles) {
  constexpr int BM = 16 * MI * WM;
  constexpr int kX = BM * kRow, kStage = kX + 256 * kRow;
  constexpr int NX = (BM / 8 + 4 * WM - 1) / (4 * WM), NB = 32 / (4 * WM);  // 1 KiB copies a wave and step: tokens, weights
  constexpr int kCols = ACT ? 128 : 256;                     // output channels of the tile
  constexpr int kAhead = MI % 5 == 0 ? 4 : 3;                // row blocks read ahead of their products
  static_assert(2 * MI % (kAhead + 1) == 0, "a step leaves its row blocks where it found them");
  static_assert(kAhead <= MI && MI >= 4, "the next step's first weights take registers that are done");
  extern __shared__ char lds[];
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / 4, wn = wave % 4;
  const int NO = out_cols(c), K = c.K;
  const int nsteps = (K + 127) / 128, nrun = nsteps > S ? nsteps : S;  // steps past K multiply zeros
  const bool indexed = GROUPED && c.row_index != nullptr;

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
  int item = begin + (blockIdx.x >> 3);
  if (item < end) {
    Tile cur = tile_at(item);
    // A wave's copies: 8 rows each, a 16-byte piece a lane; rows past the tile
    // copy one inside it, pieces past K what follows the row (their weights are
    // made zero).  Tokens: offsets from the tile's first row, or, read through an
    // index, from x's; weights from the tile's first gate row, so that 32 bits
    // reach them (the launch sees to it).
    Rsrc xres, wres;
    uint32_t xoff[NX], woff[NB];
    int ix[NX];  // rows of x that the copies read
    auto xblock = [&](int i) __attribute__((always_inline)) {  // the waves' last may copy the last again
      const int b = wave * NX + i;
      return b < BM / 8 ? b : BM / 8 - 1;
    };
    auto copy_rows = [&](const Tile& t) __attribute__((always_inline)) {
      const int lane = opaque_lane();
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const int r = 8 * xblock(i) + (lane >> 3), in = r < t.rt.cnt ? r : 0;
        ix[i] = indexed ? c.row_index[t.rt.row0 + in] : in;
      }
    };
    auto aim = [&](const Tile& t) __attribute__((always_inline)) {
      const int lane = opaque_lane();
      xres = make_rsrc((const char*)c.x + (indexed ? 0 : t.rt.row0 * c.x_stride),
                       (uint32_t)((indexed ? c.x_rows - 1 : (int64_t)t.rt.cnt - 1) * c.x_stride + K));
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const int r = 8 * xblock(i) + (lane >> 3);
        const bool ok = !indexed || (ix[i] >= 0 && ix[i] < c.x_rows);
        xoff[i] = (uint32_t)((ok ? ix[i] : 0) * c.x_stride) + 16u * (uint32_t)((lane & 7) ^ swz(r));
      }
      const int cols = NO - t.n < kCols ? NO - t.n : kCols;
      wres = make_rsrc((const char*)c.w + (int64_t)t.rt.e * c.w_stride + (int64_t)t.n * K,
                       (uint32_t)((ACT ? NO : 0) + cols) * (uint32_t)K);
      // Weight row of LDS row r: wave r / 64 of the columns; its operand block j = r
      // % 64 / 16, operand row o = r % 16 is channel 4 o + j, so that a lane's
      // results are four neighbours, its neighbour's the next (with an activation: 2 o
      // + j % 2 of gate, j < 2, and of up); rows past the last copy it
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int r = 8 * (wave * NB + i) + (lane >> 3), j = (r >> 4) & 3, o = r & 15;
        int n = (r >> 6) * (kCols / 4) + (ACT ? 2 * o + (j & 1) : 4 * o + j);
        n = n < cols ? n : cols - 1;
        woff[i] = (uint32_t)(n + (ACT && j >= 2 ? NO : 0)) * (uint32_t)K + 16u * (uint32_t)((lane & 7) ^ swz(r));
      }
    };
    auto issue = [&](int kb, int slot) __attribute__((always_inline)) {
      const uint32_t k0 = (uint32_t)(kb < nsteps ? kb : nsteps - 1) * 128u;
      char* st = lds + slot * kStage;
#pragma unroll
      for (int i = 0; i < NX; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xres, (LPtr)(st + 1024 * xblock(i)), 16, (int)(xoff[i] + k0), 0, 0, 0);
#pragma unroll
      for (int i = 0; i < NB; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wres, (LPtr)(st + kX + 1024 * (wave * NB + i)), 16, (int)(woff[i] + k0), 0, 0,
                                                 ONCE ? kNT : 0);
    };
    i32x4 acc[MI][4];
    u32x4 b[2][4], x[kAhead + 1];
    auto piece = [&](int slot, int r, int q) __attribute__((always_inline)) {
      return *(const u32x4*)(lds + slot * kStage + r * kRow + 16 * ((4 * q + g) ^ swz(r)));
    };
    auto xfrag = [&](int slot, int at) __attribute__((always_inline)) { return piece(slot, 16 * (wm * MI + at % MI) + m, at / MI); };
    auto wfrag = [&](int slot, int j, int q) __attribute__((always_inline)) { return piece(slot, BM + 64 * wn + 16 * j + m, q); };
    // Products of step kb, whose first operands are in registers; the rest is
    // read kAhead row blocks ahead.  Once every wave has read the last of them,
    // the stage's slot takes the copies of step kb + S (`ahead`: its number in the
    // tile that the copies are at) and the first operands of step kb + 1, whose
    // copies have landed, are read under the products left.
    auto step = [&](int kb, int ahead, int slot) __attribute__((always_inline)) {
      const int next = slot == S - 1 ? 0 : slot + 1;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if constexpr (PACKED || TAIL) {
          const uint32_t keep = !TAIL || kb * 128 + 64 * q + 16 * g < K ? ~0u : 0u;
#pragma unroll
          for (int j = 0; j < 4; ++j) b[q][j] = weight_operand<PACKED>(b[q][j], keep);
        }
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          const int at = MI * q + i;
          if (at == 2 * MI - kAhead) {
            if (kb >= S - 1) wait_vm<(S - 2) * (NX + NB)>();  // a tile's first S stages are here already
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            issue(ahead, slot);
#pragma unroll
            for (int j = 0; j < 4; ++j) b[0][j] = wfrag(next, j, 0);
          }
          const int a = at + kAhead;
          x[a % (kAhead + 1)] = a < 2 * MI ? xfrag(slot, a) : xfrag(next, a - 2 * MI);
          if (q == 0 && i >= MI - 4) b[1][i - (MI - 4)] = wfrag(slot, i - (MI - 4), 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = mfma_i8(x[at % (kAhead + 1)], b[q][j], acc[i][j]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    copy_rows(cur);
    aim(cur);
#pragma unroll
    for (int i = 0; i < S; ++i) issue(i, i);
    wait_vm<0>();
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int j = 0; j < 4; ++j) b[0][j] = wfrag(0, j, 0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) x[i] = xfrag(0, i);
    int slot = 0;
    for (;;) {
      const int after = item + (int)(gridDim.x >> 3);
      const Tile next = after < end ? tile_at(after) : cur;  // (the last tile's copies go on over it: nothing reads them)
      copy_rows(next);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};
      for (int kb = 0; kb < nrun; ++kb) {
        if (kb == nrun - S) aim(next);  // from here on the copies are the next tile's
        step(kb, kb + S < nrun ? kb + S : kb + S - nrun, slot);
        slot = slot == S - 1 ? 0 : slot + 1;
      }
      // A lane has tokens 16 i + 4 g + r (r 0..3) and CN neighbouring channels from
      // n0 on (with an activation two, and their up rows)
      constexpr int CN = ACT ? 2 : 4;
      const int el = opaque_lane(), eg = el >> 4;
      const int n0 = cur.n + wn * (kCols / 4) + CN * (el & 15);
      const int t0 = 16 * wm * MI + 4 * eg;
      int er[MI][4];
      float xs[MI][4];
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = t0 + 16 * i + r, in = t < cur.rt.cnt ? t : 0;
          er[i][r] = indexed ? c.row_index[cur.rt.row0 + in] : (int)cur.rt.row0 + in;
        }
      uint32_t tb[4], bb[4] = {0, 0, 0, 0};
      const int64_t at = (int64_t)cur.rt.e * c.N;
      load_run<CN>(c.w_scale, at, n0, NO - 1, c.w_scale_dtype, tb);
      if constexpr (ACT) load_run<CN>(c.w_scale, at + NO, n0, NO - 1, c.w_scale_dtype, tb + 2);
      if (c.bias != nullptr) {
        load_run<CN>(c.bias, at, n0, NO - 1, c.bias_dtype, bb);
        if constexpr (ACT) load_run<CN>(c.bias, at + NO, n0, NO - 1, c.bias_dtype, bb + 2);
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) xs[i][r] = c.x_scale[er[i][r] >= 0 && er[i][r] < c.x_rows ? er[i][r] : 0];
      // With the scales, the next tile's first S stages are here: the steps that would
      // wait for them need not wait for the stores below
      wait_vm<0>();
      Channel ch[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) ch[n] = channel(c, ChannelBits{tb[n], bb[n]});
      const RowOut<CN> out(c, cur.rt, NO, n0);
      with_act(ACT ? c.act : -1, [&](auto a) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          // one row block after the other, so that their results do not all sit in
          // registers at once
          asm volatile("" : "+v"(acc[i][0]), "+v"(acc[i][1]), "+v"(acc[i][2]), "+v"(acc[i][3]) : : "memory");
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool live = !GROUPED || (er[i][r] >= 0 && er[i][r] < c.x_rows);
            float y[CN];
#pragma unroll
            for (int n = 0; n < CN; ++n) {
              y[n] = scaled(acc[i][n][r], xs[i][r], ch[n]);
              if constexpr (ACT)
                y[n] = gated(decltype(a)::value, y[n], scaled(acc[i][2 + n][r], xs[i][r], ch[2 + n]), c);
              y[n] = live ? y[n] : 0.0f;
            }
            out.store(t0 + 16 * i + r, y);
          }
        }
      });
      if (after >= end) break;
      cur = next;
      item = after;
    }
    wait_vm<0>();  // the copies past the last step, before the LDS is given back
  }
  if constexpr (GROUPED) {  // rows of no expert
    const int head = scan.head(), tail = scan.tail(), none = head + ((int)c.rows - tail);
    for (int z = blockIdx.x; z < none; z += gridDim.x) {
      const int64_t row = z < head ? z : tail + (z - head);
      for (int n = threadIdx.x; n < NO; n += 256 * WM) store_scalar(c.out, row * NO + n, c.out_dtype, 0.0f);
    }
  }
}

// ------------------------------------------------------------------ any K and alignment
// 16 tokens x 16 output channels a workgroup, bytes through LDS: for K not a
// multiple of 16 and rows that are not 16-byte aligned.
__device__ __forceinline__ void any_item(const ftm_w8a8& c, int mt, int nt) {
  constexpr int KC = 64;
  __shared__ int8_t xs[16][KC + 4], ws[2][16][KC + 4];
  const RowTile rt = row_tile<16>(c, mt);
  if (rt.cnt <= 0) return;
  const bool act = c.act >= 0;
  const int NO = out_cols(c), n0 = nt * 16;
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
    if (act) y = gated(c.act, y, scaled(b, s, channel(c, rt.e, NO + n0 + col)), c);
  }
  store_scalar(c.out, orow * NO + n0 + col, c.out_dtype, y);
}

__global__ __launch_bounds__(256) void k_w8a8_any(ftm_w8a8 c, int mtiles, int ntiles) {
  const int64_t items = (int64_t)mtiles * ntiles;
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) any_item(c, (int)(i / ntiles), (int)(i % ntiles));
}

namespace {

template <int MT, int NT, int NW, int S, bool PACKED>
hipError_t split(const ftm_w8a8& c, hipStream_t st) {
  constexpr int ring = NW * S * (MT + NT) * 16 * kRow, sums = NW * MT * NT * 1024;
  constexpr int lds = ring > sums ? ring : sums;
  const int cols = c.act >= 0 ? 8 * NT : 16 * NT;
  const int64_t mt = row_tiles(c, 16 * MT), nt = (out_cols(c) + cols - 1) / cols;
  if (mt * nt > kMaxGroups) return hipErrorInvalidValue;
  static DeviceBits lds_set{0};
  const hipError_t e = allow_lds(lds_set, (const void*)k_w8a8_split<MT, NT, NW, S, PACKED>, lds);
  if (e != hipSuccess) return e;
  k_w8a8_split<MT, NT, NW, S, PACKED><<<dim3((unsigned)(mt * nt)), dim3(64 * NW), lds, st>>>(c, (int)mt, (int)nt);
  return hipGetLastError();
}
template <int MT, int NT, int NW, int S>
hipError_t split(const ftm_w8a8& c, hipStream_t st) {
  return c.w_packed ? split<MT, NT, NW, S, true>(c, st) : split<MT, NT, NW, S, false>(c, st);
}

// k_w8a8_wide with one block of 16 weight rows (with an activation, grouped: two) a
// tile.
template <int XDT, int NT, bool PACKED>
hipError_t wide(const ftm_w8a8& c, const void* x, int64_t x_stride, hipStream_t st) {
  constexpr int S = NT == 1 ? 4 : 2, ring = 4 * S * NT * 16 * kRow;
  const int cols = c.act >= 0 ? 8 * NT : 16 * NT, lds = ring + kWideRows * ((c.K + 127) / 128) * kRow;
  const int64_t mt = row_tiles(c, kWideRows), nt = (out_cols(c) + cols - 1) / cols;
  if (mt * nt > kMaxGroups) return hipErrorInvalidValue;
  static DeviceBits lds_set{0};
  const auto kernel = k_w8a8_wide<XDT, NT, S, PACKED>;
  const hipError_t e = allow_lds(lds_set, (const void*)kernel, ring + kWideRows * kWideK);
  if (e != hipSuccess) return e;
  kernel<<<dim3((unsigned)(mt * nt)), dim3(256), lds, st>>>(c, (const char*)x, x_stride, (int)nt);
  return hipGetLastError();
}
template <int XDT>
hipError_t wide(const ftm_w8a8& c, const void* x, int64_t x_stride, hipStream_t st) {
  if (c.offsets == nullptr) return c.w_packed ? wide<XDT, 1, true>(c, x, x_stride, st) : wide<XDT, 1, false>(c, x, x_stride, st);
  return c.w_packed ? wide<XDT, 2, true>(c, x, x_stride, st) : wide<XDT, 2, false>(c, x, x_stride, st);
}

template <int WM, int MI, int S, bool PACKED, bool ACT, bool TAIL, bool GROUPED, bool ONCE>
hipError_t tile(const ftm_w8a8& c, hipStream_t st) {
  constexpr int BM = 16 * MI * WM, lds = S * (BM + 256) * kRow;
  constexpr int resident = kCUs * (2 * lds <= 160 * 1024 ? 2 : 1);  // workgroups the chip holds at once
  const int cols = ACT ? 128 : 256;
  const int64_t mt = row_tiles(c, BM), nt = (out_cols(c) + cols - 1) / cols;
  if (mt * nt > 0x7fffffff) return hipErrorInvalidValue;
  static DeviceBits lds_set{0};
  const auto kernel = k_w8a8_tile<WM, MI, S, PACKED, ACT, TAIL, GROUPED, ONCE>;
  const hipError_t e = allow_lds(lds_set, (const void*)kernel, lds);
  if (e != hipSuccess) return e;
  const int64_t grid = mt * nt < resident ? (mt * nt + 7) / 8 * 8 : resident;  // the same for every XCD
  kernel<<<dim3((unsigned)grid), dim3(256 * WM), lds, st>>>(c, (int)mt, (int)nt);
  return hipGetLastError();
}
template <int WM, int MI, int S, bool ACT, bool GROUPED, bool ONCE>
hipError_t tile(const ftm_w8a8& c, hipStream_t st) {
  if (c.K % 128 != 0 || c.K < 128 * S)
    return c.w_packed ? tile<WM, MI, S, true, ACT, true, GROUPED, ONCE>(c, st)
                      : tile<WM, MI, S, false, ACT, true, GROUPED, ONCE>(c, st);
  return c.w_packed ? tile<WM, MI, S, true, ACT, false, GROUPED, ONCE>(c, st)
                    : tile<WM, MI, S, false, ACT, false, GROUPED, ONCE>(c, st);
}
template <int WM, int MI, int S, bool GROUPED, bool ONCE = false>
hipError_t tile(const ftm_w8a8& c, hipStream_t st) {
  return c.act >= 0 ? tile<WM, MI, S, true, GROUPED, ONCE>(c, st) : tile<WM, MI, S, false, GROUPED, ONCE>(c, st);
}

// us on MI355X beside each rule: 'split' 64 x 64 is k_w8a8_split's tile of 64
// tokens and 64 weight rows, 'tile' 64 k_w8a8_tile's of 64 tokens.

// The split tile of up to 64 tokens whose columns give every CU one workgroup at
// most (wider tiles read the tokens less often, but their CUs stay idle), or
// none: 64 x 16 / 64 x 32 / 64 x 64 / tile 64: 64 rows of 4096 x 4096 8.0 / 8.7 / 14.4 /
// 25.5, 100 14.0 / 9.4 / 14.4 / 25.4, 160 20.2 / 16.5 / 15.3 / 25.5, 512 50.6 / 32.6 /
// 31.9 / 27.0; 512 of 1408 x 2048 (1024 blocks) 18.2 / 12.0 / 11.8 / 13.7, 333 of 2048
// x 4096 (1536) 28.9 / 18.5 / 22.0 / 16.6
bool split64(const ftm_w8a8& c, int64_t row_tiles, hipStream_t st, hipError_t& e) {
  const int64_t blocks = row_tiles * ((c.N + 15) / 16);  // of 16 weight rows
  if (blocks <= kCUs) e = split<4, 1, 4, 3>(c, st);
  else if (blocks <= 2 * kCUs) e = split<4, 2, 4, 2>(c, st);
  else if (blocks <= 4 * kCUs) e = split<4, 4, 4, 2>(c, st);
  else return false;
  return true;
}

hipError_t dense(const ftm_w8a8& c, hipStream_t st) {
  const int64_t M = c.rows, blocks = (c.N + 15) / 16;
  // Few rows: the weights' stream.  16 x 16 with four or two stages, 16 rows of
  // 11008 x 4096 11.7 / 12.4, of 4096 x 12288 13.7 / 12.5; 32 x 16 / 32 x 32, 32
  // rows of 4096 x 4096 5.8 / 7.2, of 4096 x 12288 16.3 / 14.8
  if (M <= 16) return blocks <= 2 * kCUs ? split<1, 1, 4, 4>(c, st) : split<1, 1, 4, 2>(c, st);
  if (M <= 32) return blocks <= 2 * kCUs ? split<2, 1, 4, 3>(c, st) : split<2, 2, 4, 2>(c, st);
  hipError_t e = hipSuccess;
  if (c.row_index != nullptr) {
    // Through an index (a C call only; the tiles of a dense product take rows in order):
    // 64 x 64 split tiles, as many rows a launch as one grid dimension counts
    const int cols = out_cols(c), esz = c.out_dtype == FTM_DT_F32 ? 4 : 2, wide = c.act >= 0 ? 32 : 64;
    const int64_t at_once = (int64_t)(kMaxGroups / ((cols + wide - 1) / wide)) * 64;
    for (int64_t row = 0; row < M && e == hipSuccess; row += at_once) {
      ftm_w8a8 part = c;
      part.rows = M - row < at_once ? M - row : at_once;
      part.row_index = c.row_index + row;
      part.out = (char*)c.out + row * cols * esz;
      e = split<4, 4, 4, 2>(part, st);
    }
    return e;
  }
  if (split64(c, (M + 63) / 64, st, e)) return e;
  // The largest tile reads its operands least often, but a launch takes whole
  // rounds of them: rounds x the time of one, in that of a 256-token tile (1;
  // 128 tokens 0.6; two of 64 on a CU 0.68, one 0.58; 8192 rows of 8192 x 8192
  // 460 / 558 / 625, 1024 of 4096 x 4096 50 / 33 / 30)
  const int64_t nt = (c.N + 255) / 256;
  auto rounds = [&](int rows, int at_once) { return (double)(((M + rows - 1) / rows * nt + at_once - 1) / at_once); };
  const double t256 = rounds(256, kCUs), t128 = 0.6 * rounds(128, kCUs);
  const double t64 = rounds(64, kCUs) <= 1 ? 0.58 : 0.68 * rounds(64, 2 * kCUs);
  if (t256 <= t128 && t256 <= t64) return tile<2, 8, 2, false>(c, st);
  return t128 <= t64 ? tile<2, 4, 3, false>(c, st) : tile<1, 4, 2, false>(c, st);
}

hipError_t grouped(const ftm_w8a8& c, hipStream_t st) {
  // experts with rows, at most, and the rows of each if all have as many
  const int64_t hit = c.rows < c.num_experts ? c.rows : c.num_experts, seg = (c.rows + hit - 1) / hit;
  const int64_t blocks = (hit + c.rows / 16) * ((c.N + 31) / 32);  // 16 x 32, the last of an expert partly filled
  // Too few tiles to keep the memory busy: K split.  16 x 32 / tile 64, with the
  // blocks of the first: 1 token over 8 of 256 experts of 2048 x 1024 (256) 7.5 /
  // 18.6; 2 of 16 of 1024 x 1024, 128 tokens (1024) 12.2 / 15.4, 256 (1536) 15.3 /
  // 15.5, 512 (2560) 23 / 15.6; 4 of 32 of 2048 x 1536, 8 tokens (1632) 21.8 / 23.9,
  // 32 (1920) 28.9 / 28.9, 64 (2304) 32.3 / 29.3, 256 (4608) 48.5 / 29.4
  if (blocks < 8 * kCUs) return split<1, 2, 4, 2>(c, st);
  // Mostly one tile an expert: its weights are not kept for another, where a row's 128
  // bytes are one line and no neighbour's copy needs the rest.  The layer of 8 of 128
  // experts of 2048 x 768, 512 / 768 / 1024 tokens (32, 48, 64 rows an expert) 159 / 182 /
  // 213, kept 169 / 192 / 208; of 4 of 32 of 2880 x 2880, 384 tokens 253 / 230
  if (seg <= 48 && c.K % 128 == 0 && ((uintptr_t)c.w & 127u) == 0) return tile<1, 4, 2, true, true>(c, st);
  // 64, 128 or 160 tokens a tile, the layers above: 64 rows an expert 212 / 200 / 209, 96
  // 239 / 220 / 227 and 305 / 262 / 269, 188 346 / 342 / 363, 256 451 / 420 / 404 and 524 /
  // 495 / 439, 1024 1467 / 1337 / 1306; 48 230 / 236; with fewer tiles than CUs, 2 of
  // 16 of 1024 x 512, 64 rows 41 / 45.  Five tiles of 64 take the time of three of 128,
  // for an expert with an eighth more rows than the mean; around 128 rows evenly routed
  // 281 / 283 / 272, but 278 / 280 / 292 where the experts' rows differ more
  const int64_t n = seg + seg / 8, n64 = (n + 63) / 64, n128 = (n + 127) / 128, nt = (c.N + 255) / 256;
  if (seg >= 200 && hit * ((seg + 159) / 160) * nt >= kCUs) return tile<2, 5, 3, true>(c, st);
  if (5 * n128 <= 3 * n64 && hit * n128 * nt >= kCUs) return tile<2, 4, 3, true>(c, st);
  return tile<1, 4, 2, true>(c, st);
}

}  // namespace

// Whether a tile's 32-bit offsets reach its tokens (256 rows from its first, or
// all of x where they are read through an index), its weight rows and its results.
static bool offsets_ok(const ftm_w8a8& c) {
  const int64_t rows = c.row_index != nullptr ? c.x_rows : c.x_rows < 256 ? c.x_rows : 256;
  const int64_t wrows = 256 + (c.act >= 0 ? c.N / 2 : 0);
  return (rows - 1) * c.x_stride + c.K + 256 < INT32_MAX && wrows * c.K + 256 < INT32_MAX &&
         4 * 256 * (int64_t)c.N < INT32_MAX;
}

// What the fast kernels need of a call's layout.
static bool aligned_call(const ftm_w8a8& c) {
  return c.K % 16 == 0 && (((uintptr_t)c.x | (uintptr_t)c.w) & 15u) == 0 && (c.x_stride & 15) == 0 &&
         (c.offsets == nullptr || (c.w_stride & 15) == 0) && offsets_ok(c);
}

hipError_t launch_w8a8(const ftm_w8a8& c, hipStream_t st) {
  if (!aligned_call(c)) {
    const int64_t mt = row_tiles(c, 16), nt = (out_cols(c) + 15) / 16;
    const int64_t grid = mt * nt < kMaxGroups ? mt * nt : kMaxGroups;
    k_w8a8_any<<<dim3((unsigned)grid), dim3(256), 0, st>>>(c, (int)mt, (int)nt);
    return hipGetLastError();
  }
  return c.offsets != nullptr ? grouped(c, st) : dense(c, st);
}

hipError_t launch_w8a8_dynamic(const ftm_w8a8& c, const void* x, int dt, int64_t x_stride, hipStream_t st) {
  const bool in = aligned_call(c) && ((uintptr_t)x & 15u) == 0 && (x_stride & 15) == 0;
  bool few;
  if (c.offsets == nullptr) {
    // every workgroup quantises all tokens, which pays while they are few: 1 / 2 / 4
    // tokens of 2048 x 1536 4.9 / 5.7 / 7.3 us, in two launches 7.7 / 7.8 / 7.9 and
    // about 3 more of the host's; 1 / 2 / 4 of 4096 x 4096 6.3 / 7.9 / 11.2, two 7.6
    few = c.rows <= kWideRows && c.rows * c.K <= 8192;
  } else {
    // up to one row an expert on average and three rounds of workgroups: both
    // products with all else of the expert layer, here / in two launches each, 1 / 2
    // tokens through 8 of 128 experts of 2048 x 768 25.3 / 29.1, 37.3 / 38.5, 4 through
    // 2 of 16 of 1024 x 512 19.0 / 21.0, but 2 through 4 of 32 of 2880 x 2880 69 / 62
    const int64_t hit = c.rows < c.num_experts ? c.rows : c.num_experts;
    few = c.rows <= c.num_experts && hit * ((c.N + 31) / 32) <= 3 * kCUs;
  }
  if (in && few && c.K <= kWideK && c.x_rows > 0) {
    if (dt == FTM_DT_F32) return wide<FTM_DT_F32>(c, x, x_stride, st);
    if (dt == FTM_DT_F16) return wide<FTM_DT_F16>(c, x, x_stride, st);
    return wide<FTM_DT_BF16>(c, x, x_stride, st);
  }
  const hipError_t e = launch_quant_int8(x, dt, c.x_rows, c.K, x_stride, const_cast<int8_t*>(c.x), c.K,
                                         const_cast<float*>(c.x_scale), st);
  return e != hipSuccess ? e : launch_w8a8(c, st);
}

}  // namespace ftm
