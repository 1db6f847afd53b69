// ftm_sort.hip -- (token, expert) pairs sorted by expert, tokens copied into
// that order, and rows back in token order with weights, with the gradients.
//
// Pair p = t k + j is entry j of token t.  Rows [offsets[e], offsets[e+1]) are
// the pairs of expert e in order of p; rows from offsets[E] on are the pairs
// without an expert (an id outside [0, E)), which every kernel writes as zeros
// and none reads.  row_of_pair[p] is the row r of pair p, pair_of_row[r] its
// inverse, token_of_row[r] = p / k; for a pair without an expert the first two
// hold the complements ~r and ~p, the third -1.
#include <type_traits>

#include "ftm_layer.h"

namespace ftm {

namespace {

constexpr int kSortWaves = 16;
constexpr int kSortKeys = kMaxExperts + 1;  // the last: no expert
constexpr int kSortOne = 8192;              // pairs that one workgroup sorts
constexpr int kSortBlocks = 128;            // workgroups above that, at most
constexpr int kSortPer = 4096;              // pairs a workgroup, at least

inline int64_t sort_per(int64_t P) {
  const int64_t per = (P + kSortBlocks - 1) / kSortBlocks;
  return per < kSortPer ? kSortPer : (per + 1023) / 1024 * 1024;
}

}  // namespace

template <class ID>
__device__ __forceinline__ int sort_key(const ID* ids, int64_t p, int64_t end, int E) {
  const ID v = p < end ? ids[p] : (ID)-1;
  return v >= 0 && v < (ID)E ? (int)v : E;
}

// Lanes of the wave with this lane's key (`bits` bits), among `live`.
__device__ __forceinline__ uint64_t same_key(int key, int bits, uint64_t live) {
  uint64_t m = live;
  for (int b = 0; b < bits; ++b) {
    const uint64_t v = __ballot((key >> b) & 1);
    m &= (key >> b) & 1 ? v : ~v;
  }
  return m;
}

// Counts of a workgroup's pairs by wave and key: each wave walks a run of its
// own, one leader lane a key adds the number of lanes that share it, so the
// order of the pairs is kept and no atomics are used.
template <class ID>
__device__ __forceinline__ void sort_count(const ID* ids, int64_t lo, int64_t hi, int64_t run, int E, int bits,
                                           int (*hist)[kSortKeys]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < kSortWaves * kSortKeys; i += 64 * kSortWaves) ((int*)hist)[i] = 0;
  __syncthreads();
  const int64_t w_lo = lo + wave * run, w_hi = w_lo + run < hi ? w_lo + run : hi;
  for (int64_t p0 = w_lo; p0 < w_hi; p0 += 64) {
    const int64_t p = p0 + lane;
    const int key = sort_key(ids, p, w_hi, E);
    const uint64_t m = same_key(key, bits, __ballot(p < w_hi));
    if (p < w_hi && (m & ((1ull << lane) - 1)) == 0) hist[wave][key] += __popcll(m);
  }
  __syncthreads();
}

// counts[b][key] of workgroup b's pairs.
template <class ID>
__global__ __launch_bounds__(64 * kSortWaves) void k_sort_count(const ID* ids, int64_t P, int64_t per, int E, int bits,
                                                                int32_t* counts) {
  __shared__ int hist[kSortWaves][kSortKeys];
  const int64_t lo = blockIdx.x * per, hi = lo + per < P ? lo + per : P;
  sort_count(ids, lo, hi, per / kSortWaves, E, bits, hist);
  for (int e = threadIdx.x; e <= E; e += 64 * kSortWaves) {
    int n = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) n += hist[w][e];
    counts[(int64_t)blockIdx.x * (E + 1) + e] = n;
  }
}

// The rows of workgroup b's pairs: the keys' totals over all workgroups and
// those before b (counts; none: one workgroup sorts everything), their prefix
// sum, then a second walk in the order of the first.
template <class ID>
__global__ __launch_bounds__(64 * kSortWaves) void k_sort_place(const ID* ids, int64_t P, int64_t per, int E, int bits,
                                                                int k, const int32_t* counts, int blocks,
                                                                int32_t* offsets, int32_t* row_of_pair,
                                                                int32_t* pair_of_row, int32_t* token_of_row) {
  __shared__ int hist[kSortWaves][kSortKeys];
  __shared__ int total[64 * 9], mine[64 * 9];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t lo = blockIdx.x * per, hi = lo + per < P ? lo + per : P;
  const int64_t run = per / kSortWaves;
  sort_count(ids, lo, hi, run, E, bits, hist);
  for (int e = threadIdx.x; e < 64 * 9; e += 64 * kSortWaves) {
    int all = 0, before = 0;
    if (e <= E) {
      if (counts == nullptr) {
        for (int w = 0; w < kSortWaves; ++w) all += hist[w][e];
      } else {
        for (int b = 0; b < blocks; ++b) {
          const int n = counts[(int64_t)b * (E + 1) + e];
          all += n;
          before += b < (int)blockIdx.x ? n : 0;
        }
      }
    }
    total[e] = all;
    mine[e] = before;
  }
  __syncthreads();
  if (wave == 0) {  // exclusive prefix sum over the keys, nine a lane
    int v[9], sum = 0;
#pragma unroll
    for (int i = 0; i < 9; ++i) {
      v[i] = total[9 * lane + i];
      sum += v[i];
    }
    int upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d);
      upto += lane >= d ? o : 0;
    }
    int at = upto - sum;
#pragma unroll
    for (int i = 0; i < 9; ++i) {
      const int e = 9 * lane + i;
      if (blockIdx.x == 0 && e <= E) offsets[e] = at;
      mine[e] += at;
      at += v[i];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += 64 * kSortWaves) {  // first row of every wave's pairs of key e
    int at = mine[e];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const int n = hist[w][e];
      hist[w][e] = at;
      at += n;
    }
  }
  __syncthreads();
  const int64_t w_lo = lo + wave * run, w_hi = w_lo + run < hi ? w_lo + run : hi;
  for (int64_t p0 = w_lo; p0 < w_hi; p0 += 64) {
    const int64_t p = p0 + lane;
    const int key = sort_key(ids, p, w_hi, E);
    const uint64_t m = same_key(key, bits, __ballot(p < w_hi));
    const uint64_t lower = m & ((1ull << lane) - 1);
    if (p >= w_hi) continue;
    const int first = hist[wave][key];
    const int row = first + __popcll(lower);
    const bool here = key < E;
    row_of_pair[p] = here ? row : ~row;
    pair_of_row[row] = here ? (int)p : ~(int)p;
    token_of_row[row] = here ? (int)p / k : -1;
    // the last lane of a key moves its first row on for the next 64 pairs
    // (every lane has read it: the wave runs in step, LDS in order)
    if ((m >> lane) == 1) hist[wave][key] = row + 1;
  }
}

size_t sort_workspace_bytes(int64_t P, int E) {
  if (P <= kSortOne) return 0;
  const int64_t per = sort_per(P);
  return (size_t)((P + per - 1) / per) * (size_t)(E + 1) * 4;
}

template <class ID>
static hipError_t sort_ids(const ID* ids, int64_t P, int k, int E, int32_t* offsets, int32_t* row_of_pair,
                           int32_t* pair_of_row, int32_t* token_of_row, int32_t* counts, hipStream_t st) {
  int bits = 1;
  while ((E >> bits) != 0) ++bits;
  const dim3 wg(64 * kSortWaves);
  if (P <= kSortOne) {
    const int64_t per = (P + 64 * kSortWaves - 1) / (64 * kSortWaves) * (64 * kSortWaves);
    k_sort_place<ID><<<dim3(1), wg, 0, st>>>(ids, P, per > 0 ? per : 64 * kSortWaves, E, bits, k, nullptr, 1, offsets,
                                             row_of_pair, pair_of_row, token_of_row);
    return hipGetLastError();
  }
  const int64_t per = sort_per(P);
  const int blocks = (int)((P + per - 1) / per);
  k_sort_count<ID><<<dim3(blocks), wg, 0, st>>>(ids, P, per, E, bits, counts);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  k_sort_place<ID><<<dim3(blocks), wg, 0, st>>>(ids, P, per, E, bits, k, counts, blocks, offsets, row_of_pair,
                                                pair_of_row, token_of_row);
  return hipGetLastError();
}

hipError_t launch_sort(const void* ids, bool ids64, int64_t P, int k, int E, int32_t* offsets, int32_t* row_of_pair,
                       int32_t* pair_of_row, int32_t* token_of_row, void* ws, hipStream_t st) {
  int32_t* counts = (int32_t*)ws;
  return ids64 ? sort_ids((const int64_t*)ids, P, k, E, offsets, row_of_pair, pair_of_row, token_of_row, counts, st)
               : sort_ids((const int32_t*)ids, P, k, E, offsets, row_of_pair, pair_of_row, token_of_row, counts, st);
}

// ------------------------------------------------------------------ rows out of tokens
// A pair's row: [0, rows), its complement for a pair without an expert; an
// entry of a table that names neither is left out (~rows).
__device__ __forceinline__ int pair_row(const int32_t* row_of_pair, int64_t p, int rows) {
  const int r = row_of_pair[p];
  return (r < 0 ? ~r : r) < rows ? r : ~rows;
}

// One workgroup a token: its row is read once and written to the rows of its k
// pairs (zeros where a pair has no expert).  Bound by the writes.
template <class V>
__global__ __launch_bounds__(256) void k_gather_tokens(const char* x, int64_t x_stride, int n, const int32_t* row_of_pair,
                                                       int k, V* rows) {
  const int64_t t = blockIdx.x;
  const int P = (int)gridDim.x * k;
  const V* src = (const V*)(x + t * x_stride);
  for (int i = threadIdx.x; i < n; i += 256) {
    const V v = src[i];
    for (int j = 0; j < k; ++j) {
      const int r = pair_row(row_of_pair, t * k + j, P);
      if (r != ~P) rows[(int64_t)(r < 0 ? ~r : r) * n + i] = r < 0 ? V{} : v;
    }
  }
}

hipError_t launch_gather(const void* x, int64_t x_stride, int elem, int H, const int32_t* row_of_pair, int T, int k,
                         void* rows, hipStream_t st) {
  const int64_t bytes = (int64_t)elem * H;
  const char* p = (const char*)x;
  const dim3 grid((unsigned)T), wg(256);
  if (((uintptr_t)x | (uintptr_t)rows | (uint64_t)x_stride | (uint64_t)bytes) % 16 == 0)
    k_gather_tokens<u32x4><<<grid, wg, 0, st>>>(p, x_stride, (int)(bytes / 16), row_of_pair, k, (u32x4*)rows);
  else if (elem == 4) k_gather_tokens<uint32_t><<<grid, wg, 0, st>>>(p, x_stride, H, row_of_pair, k, (uint32_t*)rows);
  else if (elem == 2) k_gather_tokens<uint16_t><<<grid, wg, 0, st>>>(p, x_stride, H, row_of_pair, k, (uint16_t*)rows);
  else k_gather_tokens<uint8_t><<<grid, wg, 0, st>>>(p, x_stride, H, row_of_pair, k, (uint8_t*)rows);
  return hipGetLastError();
}

// ------------------------------------------------------------------ rows back into tokens
// N neighbouring values of a row as fp32: 1, or 4 or 8 in one load of up to 16 bytes.
template <int DT, int N>
struct RowVec {
  static constexpr int kBytes = N * (DT == FTM_DT_F32 ? 4 : 2);
  using Raw = std::conditional_t<kBytes == 16, u32x4, u32x2>;
  __device__ __forceinline__ static void load(const char* p, int64_t i, float (&f)[N]) {
    if constexpr (N == 1) {
      f[0] = load_scalar(p, i, DT);
    } else {
      const Raw v = ((const Raw*)p)[i];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if constexpr (DT == FTM_DT_F32) {
          f[n] = __uint_as_float(v[n]);
        } else {
          const uint32_t h = (v[n >> 1] >> (16 * (n & 1))) & 0xffffu;
          f[n] = DT == FTM_DT_F16 ? f16_to_f32((uint16_t)h) : __uint_as_float(h << 16);
        }
      }
    }
  }
  __device__ __forceinline__ static void store(char* p, int64_t i, const float (&f)[N]) {
    if constexpr (N == 1) {
      store_scalar(p, i, DT, f[0]);
    } else {
      Raw v;
#pragma unroll
      for (int n = 0; n < kBytes / 4; ++n) {
        if constexpr (DT == FTM_DT_F32) v[n] = __float_as_uint(f[n]);
        else if constexpr (DT == FTM_DT_BF16) v[n] = pack_bf16x2(f[2 * n], f[2 * n + 1]);
        else v[n] = (uint32_t)f32_to_f16(f[2 * n]) | ((uint32_t)f32_to_f16(f[2 * n + 1]) << 16);
      }
      ((Raw*)p)[i] = v;
    }
  }
};

// out[t] = sum_j w[t, j] rows[row(t, j)] in order of j, fp32 sums, one
// rounding; w null: ones.  One workgroup a token.  Bound by reading the rows.
template <int DT, int OT, int N>
__global__ __launch_bounds__(256) void k_combine_tokens(const char* rows, int64_t row_stride, const void* w, int w_dt,
                                                        const int32_t* row_of_pair, int k, int n, char* out,
                                                        int64_t out_stride) {
  const int64_t t = blockIdx.x;
  for (int i = threadIdx.x; i < n; i += 256) {
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0f;
#pragma unroll 8
    for (int j = 0; j < k; ++j) {
      const int r = pair_row(row_of_pair, t * k + j, (int)gridDim.x * k);
      if (r < 0) continue;
      const float wt = w != nullptr ? load_scalar(w, t * k + j, w_dt) : 1.0f;
      float v[N];
      RowVec<DT, N>::load(rows + (int64_t)r * row_stride, i, v);
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = fmaf(wt, v[e], acc[e]);
    }
    RowVec<OT, N>::store(out + t * out_stride, i, acc);
  }
}

// The gradients of out[t] = sum_j w[t, j] rows[row(t, j)]: grad_rows[row] = w g
// (zeros on rows of no expert), grad_w[t, j] = g[t] . rows[row] (0 without an
// expert), fp32 sums in a fixed order.  One workgroup a token; either may be
// null.
template <int DT, int OT, int N>
__global__ __launch_bounds__(256) void k_combine_grad(const char* g, int64_t g_stride, const char* rows,
                                                      int64_t row_stride, const void* w, int w_dt,
                                                      const int32_t* row_of_pair, int k, int n, char* grad_rows,
                                                      int64_t grad_stride, void* grad_w) {
  __shared__ float part[4][8];
  const int64_t t = blockIdx.x;
  const int P = (int)gridDim.x * k;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int j0 = 0; j0 < k; j0 += 8) {
    float dot[8];
    int r[8];
    float wt[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      dot[j] = 0.0f;
      const bool in = j0 + j < k;
      r[j] = in ? pair_row(row_of_pair, t * k + j0 + j, P) : ~P;
      wt[j] = in && grad_rows != nullptr && r[j] >= 0 ? load_scalar(w, t * k + j0 + j, w_dt) : 0.0f;
    }
    for (int i = threadIdx.x; i < n; i += 256) {
      float gv[N];
      RowVec<OT, N>::load(g + t * g_stride, i, gv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (r[j] == ~P) continue;
        float v[N];
        if (grad_w != nullptr && r[j] >= 0) {
          RowVec<DT, N>::load(rows + (int64_t)r[j] * row_stride, i, v);
#pragma unroll
          for (int e = 0; e < N; ++e) dot[j] = fmaf(gv[e], v[e], dot[j]);
        }
        if (grad_rows != nullptr) {
#pragma unroll
          for (int e = 0; e < N; ++e) v[e] = r[j] >= 0 ? wt[j] * gv[e] : 0.0f;
          RowVec<DT, N>::store(grad_rows + (int64_t)(r[j] < 0 ? ~r[j] : r[j]) * grad_stride, i, v);
        }
      }
    }
    if (grad_w != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float s = wave_sum_dpp(dot[j]);
        if (lane == 0) part[wave][j] = s;
      }
      __syncthreads();
      const int j = threadIdx.x;
      if (j < 8 && j0 + j < k)
        store_scalar(grad_w, t * k + j0 + j, w_dt, (part[0][j] + part[1][j]) + (part[2][j] + part[3][j]));
      __syncthreads();
    }
  }
}

// f(rows dtype, dtype of the tokens' side) for the pairs that are taken: equal
// ones, and fp32 rows with any.
template <class F>
static hipError_t row_types(int dt, int ot, F&& f) {
  using std::integral_constant;
  using F32 = integral_constant<int, FTM_DT_F32>;
  using F16 = integral_constant<int, FTM_DT_F16>;
  using BF16 = integral_constant<int, FTM_DT_BF16>;
  if (dt == FTM_DT_F32) {
    if (ot == FTM_DT_F32) return f(F32{}, F32{});
    return ot == FTM_DT_F16 ? f(F32{}, F16{}) : f(F32{}, BF16{});
  }
  if (dt != ot) return hipErrorInvalidValue;
  return dt == FTM_DT_F16 ? f(F16{}, F16{}) : f(BF16{}, BF16{});
}

hipError_t launch_combine(const void* rows, int dt, int64_t row_stride, const void* w, int w_dt,
                          const int32_t* row_of_pair, int T, int k, int H, void* out, int out_dt, hipStream_t st) {
  return row_types(dt, out_dt, [&](auto d, auto o) {
    constexpr int D = decltype(d)::value, O = decltype(o)::value, N = D == FTM_DT_F32 ? 4 : 8;
    const int64_t os = (int64_t)H * (O == FTM_DT_F32 ? 4 : 2);
    const dim3 grid((unsigned)T), wg(256);
    if (H % N == 0 && ((uintptr_t)rows | (uintptr_t)out | (uint64_t)row_stride) % 16 == 0)
      k_combine_tokens<D, O, N><<<grid, wg, 0, st>>>((const char*)rows, row_stride, w, w_dt, row_of_pair, k, H / N,
                                                     (char*)out, os);
    else
      k_combine_tokens<D, O, 1><<<grid, wg, 0, st>>>((const char*)rows, row_stride, w, w_dt, row_of_pair, k, H,
                                                     (char*)out, os);
    return hipGetLastError();
  });
}

hipError_t launch_combine_grad(const void* g, int g_dt, int64_t g_stride, const void* rows, int dt, int64_t row_stride,
                               const void* w, int w_dt, const int32_t* row_of_pair, int T, int k, int H,
                               void* grad_rows, void* grad_w, hipStream_t st) {
  return row_types(dt, g_dt, [&](auto d, auto o) {
    constexpr int D = decltype(d)::value, O = decltype(o)::value, N = D == FTM_DT_F32 ? 4 : 8;
    const int64_t rs = (int64_t)H * (D == FTM_DT_F32 ? 4 : 2);
    const dim3 grid((unsigned)T), wg(256);
    const uint64_t read = grad_w != nullptr ? (uintptr_t)rows | (uint64_t)row_stride : 0;
    if (H % N == 0 && ((uintptr_t)g | (uint64_t)g_stride | read | (uintptr_t)grad_rows) % 16 == 0)
      k_combine_grad<D, O, N><<<grid, wg, 0, st>>>((const char*)g, g_stride, (const char*)rows, row_stride, w, w_dt,
                                                   row_of_pair, k, H / N, (char*)grad_rows, rs, grad_w);
    else
      k_combine_grad<D, O, 1><<<grid, wg, 0, st>>>((const char*)g, g_stride, (const char*)rows, row_stride, w, w_dt,
                                                   row_of_pair, k, H, (char*)grad_rows, rs, grad_w);
    return hipGetLastError();
  });
}

}  // namespace ftm
