// ftm_rows.h -- what the products of quantised rows share (ftm_w8a8.hip,
// ftm_w4a4.hip): the cut of dense or expert-sorted rows into tiles, the order of the
// tiles, the layout of their LDS stages, the gated activation and the stores of a
// tile's results.  C is the call: rows, x_rows, offsets, row_index, num_experts, N,
// act, act_alpha, act_limit, out, out_dtype.
#pragma once

#include <type_traits>

#include "ftm_layer.h"

namespace ftm {

// ------------------------------------------------------------------ tiles
// Rows of one tile: `cnt` (up to the tile's height) from output row `row0` on,
// of expert `e`; e < 0: rows behind (or before) every expert's, written as
// zeros; cnt 0: nothing to do.
struct RowTile {
  int64_t row0;
  int cnt, e;
};

// The experts' rows cut into tiles of height BM, in order of the experts, found by
// every wave for itself: eight experts a lane, one prefix sum over the wave.
// The offsets are clamped to [0, rows], so a bad table reads and writes no
// other memory.
template <int BM>
struct RowScan {
  int lo[9];  // first rows of the lane's eight experts, and the end of the last
  int first;  // tiles of the experts before them
  int total;  // tiles of all experts

  __device__ __forceinline__ static int tiles(int begin, int end) { return end > begin ? (end - begin + BM - 1) / BM : 0; }

  template <class C>
  __device__ __forceinline__ explicit RowScan(const C& c) {
    const int lane = threadIdx.x & 63, E = c.num_experts, P = (int)c.rows;
#pragma unroll
    for (int i = 0; i < 9; ++i) {
      const int e = 8 * lane + i;
      const int o = c.offsets[e < E ? e : E];
      lo[i] = o < 0 ? 0 : o > P ? P : o;
    }
    int sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += tiles(lo[i], lo[i + 1]);
    const int upto = wave_prefix_sum(sum);
    first = upto - sum;
    total = __builtin_amdgcn_readlane(upto, 63);
  }

  // The expert of tile t < total: its rows, its tiles and the tiles before them.
  struct Expert {
    int e, begin, end, tiles, before;
  };
  __device__ __forceinline__ Expert expert(int t) const {
    int before = first, e = -1, start = 0, begin = 0, end = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = tiles(lo[i], lo[i + 1]);
      const bool here = t >= before && t < before + n;
      e = here ? 8 * (int)(threadIdx.x & 63) + i : e;
      start = here ? before : start;
      begin = here ? lo[i] : begin;
      end = here ? lo[i + 1] : end;
      before += n;
    }
    const int src = __builtin_ctzll(__ballot(e >= 0));
    begin = __builtin_amdgcn_readlane(begin, src);
    end = __builtin_amdgcn_readlane(end, src);
    return {__builtin_amdgcn_readlane(e, src), begin, end, tiles(begin, end), __builtin_amdgcn_readlane(start, src)};
  }
  // Its m-th tile.
  __device__ __forceinline__ static RowTile tile(const Expert& x, int m) {
    const int begin = x.begin + BM * m;
    return {begin, x.end - begin < BM ? x.end - begin : BM, x.e};
  }

  // The rows of no expert: before the first offset and from the last on.
  __device__ __forceinline__ int head() const { return __builtin_amdgcn_readlane(lo[0], 0); }
  __device__ __forceinline__ int tail() const { return __builtin_amdgcn_readlane(lo[8], 63); }
};

// Tile t of a dense product.
template <int BM, class C>
__device__ __forceinline__ RowTile dense_tile(const C& c, int t) {
  const int64_t row0 = (int64_t)t * BM, left = c.rows - row0;
  return {row0, left < BM ? (int)left : BM, 0};
}

// Row tile t: dense, or of a grouped product the experts' and behind them those
// over the rows of no expert.
template <int BM, class C>
__device__ __forceinline__ RowTile row_tile(const C& c, int t) {
  if (c.offsets == nullptr) return dense_tile<BM>(c, t);
  const RowScan<BM> scan(c);
  if (t < scan.total) {
    const auto x = scan.expert(t);
    return scan.tile(x, t - x.before);
  }
  const int head = scan.head(), head_tiles = (head + BM - 1) / BM, u = t - scan.total;
  const int begin = u < head_tiles ? u * BM : scan.tail() + (u - head_tiles) * BM;
  const int end = u < head_tiles ? head : (int)c.rows;
  return {begin, end - begin < BM ? (end > begin ? end - begin : 0) : BM, -1};
}

// Row tiles that row_tile<BM> can name: each expert ends in one partly filled
// tile at most, and so do the rows before and behind them.
template <class C>
inline int64_t row_tiles(const C& c, int BM) {
  if (c.offsets == nullptr) return (c.rows + BM - 1) / BM;
  const int64_t e = c.rows < c.num_experts ? c.rows : c.num_experts;
  return c.rows / BM + e + 2;
}

// Source row of output row `row` (inside an expert's rows), or -1 where the
// index names none.
template <class C>
__device__ __forceinline__ int64_t source_row(const C& c, int64_t row) {
  if (c.row_index == nullptr) return row;
  const int i = c.row_index[row];
  return i >= 0 && i < c.x_rows ? i : -1;
}

// Output channels: with an activation the weight rows [0, N/2) are gate and
// [N/2, N) up.
template <class C>
__host__ __device__ inline int out_cols(const C& c) { return c.act >= 0 ? c.N / 2 : c.N; }

// Raw bits of N neighbouring entries (index capped at `last`).
template <int N>
__device__ __forceinline__ void load_run(const void* p, int64_t base, int first, int last, int dt, uint32_t* bits) {
  if (dt == FTM_DT_F32) {
#pragma unroll
    for (int i = 0; i < N; ++i) bits[i] = ((const uint32_t*)p)[base + (first + i < last ? first + i : last)];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) bits[i] = ((const uint16_t*)p)[base + (first + i < last ? first + i : last)];
  }
}

// Slot s of row r of a 128-byte wide LDS stage holds 16-byte piece s ^ swz(r): the
// 16 rows of one operand read (128 bytes apart, 256 bytes of banks) hit distinct
// banks.
constexpr int kRow = 128;
__device__ __forceinline__ int swz(int r) { return (r >> 1) & 7; }
typedef __attribute__((address_space(3))) void* LPtr;

// Cache policy of what a kernel does not read again: nothing keeps it.  Results stored
// so leave their place in the last cache to the weights.  Past / kept, four sets of
// inputs in turn (none is in a cache): 4096 x 4096 x 12288 190 / 193 us, grouped down of
// 2048 tokens of 8 of 128 experts of 768 x 2048 87 / 88, gate_up to fp32 129 / 133; one set
// again and again: down 66 / 77.  In the expert layer the next kernel reads the results:
// 512 tokens 172 / 175, but 2048 277 / 274, and of 4 of 32 of 2880 x 2880 467 / 460.
constexpr int kNT = 2;

// The results of a row tile: N = 8, 4 or 2 neighbouring channels from n0 on of one row
// at a time, through a buffer that drops rows past the tile; channels past the
// last take an offset past its end, so there is no branch around a store.
template <int N>
struct RowOut {
  Rsrc res;
  int NO, n0, dt;
  bool vec;  // all N in one store
  template <class C>
  __device__ __forceinline__ RowOut(const C& c, const RowTile& t, int NO_, int n0_) : NO(NO_), n0(n0_), dt(c.out_dtype) {
    const int esz = dt == FTM_DT_F32 ? 4 : 2;
    res = make_rsrc((char*)c.out + t.row0 * NO * esz, (uint32_t)(t.cnt * NO) * (uint32_t)esz);
    vec = NO % N == 0 && ((uintptr_t)c.out & 15u) == 0;
  }
  __device__ __forceinline__ uint32_t half2(float a, float b) const {
    return dt == FTM_DT_BF16 ? pack_bf16x2(a, b) : (uint32_t)f32_to_f16(a) | ((uint32_t)f32_to_f16(b) << 16);
  }
  // All N in one store (where vec says so) of a type known beforehand.
  template <int DT>
  __device__ __forceinline__ void store_vec(int row, const float (&y)[N]) const {
    const uint32_t at = (uint32_t)(row * NO + n0);
    if constexpr (DT == FTM_DT_F32) {
      const uint32_t off = n0 < NO ? 4u * at : kOOB;
      if constexpr (N == 2) {
        __builtin_amdgcn_raw_buffer_store_b64((u32x2){__float_as_uint(y[0]), __float_as_uint(y[1])}, res, off, 0, kNT);
      } else {
#pragma unroll
        for (int h = 0; h < N; h += 4)
          __builtin_amdgcn_raw_buffer_store_b128(
              (u32x4){__float_as_uint(y[h]), __float_as_uint(y[h + 1]), __float_as_uint(y[h + 2]), __float_as_uint(y[h + 3])}, res,
              n0 < NO ? off + 4u * h : kOOB, 0, kNT);
      }
    } else {
      const uint32_t off = n0 < NO ? 2u * at : kOOB;
      auto half2 = [](float a, float b) {
        return DT == FTM_DT_BF16 ? pack_bf16x2(a, b) : (uint32_t)f32_to_f16(a) | ((uint32_t)f32_to_f16(b) << 16);
      };
      if constexpr (N == 8)
        __builtin_amdgcn_raw_buffer_store_b128((u32x4){half2(y[0], y[1]), half2(y[2], y[3]), half2(y[4], y[5]), half2(y[6], y[7])},
                                               res, off, 0, kNT);
      else if constexpr (N == 4)
        __builtin_amdgcn_raw_buffer_store_b64((u32x2){half2(y[0], y[1]), half2(y[2], y[3])}, res, off, 0, kNT);
      else
        __builtin_amdgcn_raw_buffer_store_b32(half2(y[0], y[1]), res, off, 0, kNT);
    }
  }
  __device__ __forceinline__ void store(int row, const float (&y)[N]) const {
    const uint32_t at = (uint32_t)(row * NO + n0);
    if (dt == FTM_DT_F32) {
      const uint32_t off = n0 < NO ? 4u * at : kOOB;
      if (vec) {
        if constexpr (N == 4)
          __builtin_amdgcn_raw_buffer_store_b128(
              (u32x4){__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])}, res, off, 0,
              kNT);
        else
          __builtin_amdgcn_raw_buffer_store_b64((u32x2){__float_as_uint(y[0]), __float_as_uint(y[1])}, res, off, 0, kNT);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y[i]), res, n0 + i < NO ? 4u * (at + i) : kOOB, 0, kNT);
      }
      return;
    }
    const uint32_t off = n0 < NO ? 2u * at : kOOB;
    if (vec) {
      if constexpr (N == 4)
        __builtin_amdgcn_raw_buffer_store_b64((u32x2){half2(y[0], y[1]), half2(y[2], y[3])}, res, off, 0, kNT);
      else
        __builtin_amdgcn_raw_buffer_store_b32(half2(y[0], y[1]), res, off, 0, kNT);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        __builtin_amdgcn_raw_buffer_store_b16((uint16_t)half2(y[i], 0.0f), res, n0 + i < NO ? 2u * (at + i) : kOOB, 0, kNT);
    }
  }
};

// act(gate) up.  A NaN in either (the scale of its token or channel is one) is the
// result; the clamps of act_fn would replace it by their limit.
template <class C>
__device__ __forceinline__ float gated(int act, float g, float u, const C& c) {
  const float y = act_fn(act, g, u, c.act_alpha, c.act_limit);
  if (act != FTM_ACT_RELU && act != FTM_ACT_SWIGLU_OAI) return y;
  return __builtin_isunordered(g, u) ? __uint_as_float(0x7fc00000u) : y;
}

// f(activation) with the selection outside the loops (-1: none).
template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  if (act < 0) f(std::integral_constant<int, -1>{});
  else if (act == FTM_ACT_SILU) f(std::integral_constant<int, FTM_ACT_SILU>{});
  else if (act == FTM_ACT_GELU) f(std::integral_constant<int, FTM_ACT_GELU>{});
  else if (act == FTM_ACT_RELU) f(std::integral_constant<int, FTM_ACT_RELU>{});
  else f(std::integral_constant<int, FTM_ACT_SWIGLU_OAI>{});
}

// The order of a product's tiles (an expert's, grouped): groups of eight row tiles,
// their columns one after another, so that the tiles in flight on one XCD share
// both operands, and where a round of them ends inside an expert only the weights
// of one column are read a second time.
struct ItemOrder {
  int m, nt;  // row tile, column
  __device__ __forceinline__ ItemOrder(int item, int mtiles, int ntiles) {
    const int per = 8 * ntiles, first = item / per * 8;
    const int rows = mtiles - first < 8 ? mtiles - first : 8;
    nt = item % per / rows;
    m = first + item % per % rows;
  }
};

// The lane's number, anew: what is computed from it inside a loop is not kept in
// registers over the loop.
__device__ __forceinline__ int opaque_lane() {
  int l = threadIdx.x & 63;
  asm volatile("" : "+v"(l));
  return l;
}

constexpr int kMaxGroups = (1 << 24) - 1;  // workgroups of 256 threads that one grid dimension counts

constexpr int kCUs = 256;

}  // namespace ftm
