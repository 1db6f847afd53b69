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
constexpr int kSortWg = 64 * kSortWaves;  // threads and pairs of one round of a workgroup
constexpr int kSortOne = 4 * kSortWg;     // pairs that one workgroup sorts by itself

// Pairs a workgroup takes: up to four rounds by itself, one of several takes
// one round, four where there are more than 256 of them otherwise (every one reads
// all counts).
inline int sort_rounds(int64_t P) {
  const int64_t r = (P + kSortWg - 1) / kSortWg;
  if (P <= kSortOne) return r <= 1 ? 1 : r <= 2 ? 2 : 4;
  return r <= 256 ? 1 : 4;
}

// Workgroups up to which each placing one reads all their counts; beyond, a pass of
// its own sums them, so that the work stays proportional to the pairs.  us of the sort
// with / without it, 128 experts: 65 workgroups 18.7 / 17.9, 256 26 / 30, 512 (2^21
// pairs) 40 / 52, 2048 123 / 411.
constexpr int kSortDirect = 256;
inline int64_t sort_groups(int64_t P) {
  const int64_t per = (int64_t)sort_rounds(P) * kSortWg;
  return (P + per - 1) / per;
}

}  // namespace

template <class ID>
__device__ __forceinline__ int sort_key(const ID* ids, int64_t p, int64_t P, int E) {
  const ID v = p < P ? ids[p] : (ID)-1;
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

// Pairs of one workgroup: wave w's run is pairs 64 R w .. of the workgroup's, 64 a
// round.  hist[w][key] counts the wave's; a lane's rank is the number of pairs
// before it in its run with its key.  One lane a key adds for the others, so the
// order of the pairs is kept and no atomics are used.
template <class ID, int R>
struct SortRun {
  int key[R], rank[R];
  int64_t p0;  // the lane's pair of the first round

  __device__ __forceinline__ SortRun(const ID* ids, int64_t P, int E, int bits, int* hist) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    p0 = (int64_t)blockIdx.x * (R * kSortWg) + wave * (64 * R) + lane;
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = sort_key(ids, p0 + 64 * r, P, E);
    for (int i = threadIdx.x; i < kSortWaves * (E + 1); i += kSortWg) hist[i] = 0;
    __syncthreads();
    int* mine = hist + wave * (E + 1);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = p0 + 64 * r < P;
      const uint64_t m = same_key(key[r], bits, __ballot(live));
      rank[r] = live ? mine[key[r]] + __popcll(m & ((1ull << lane) - 1)) : 0;
      __builtin_amdgcn_wave_barrier();
      // the last lane of a key, once every lane has read the count (the wave runs
      // in step, its LDS accesses in order)
      if (live && (m >> lane) == 1) mine[key[r]] = rank[r] + 1;
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
  }
};

// counts[b][key] of workgroup b's pairs.
template <class ID, int R>
__global__ __launch_bounds__(kSortWg) void k_sort_count(const ID* ids, int64_t P, int E, int bits, int32_t* counts) {
  __shared__ int hist[kSortWaves * (kMaxExperts + 1)];
  const SortRun<ID, R> run(ids, P, E, bits, hist);
  for (int e = threadIdx.x; e <= E; e += kSortWg) {
    int n = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) n += hist[w * (E + 1) + e];
    counts[(int64_t)blockIdx.x * (E + 1) + e] = n;
  }
}

// counts[b][key] become the counts of the workgroups before b, counts[groups][key]
// their total: 64 keys a workgroup, a run of the workgroups a wave.
__global__ __launch_bounds__(kSortWg) void k_sort_scan(int32_t* counts, int groups, int E) {
  __shared__ int sums[kSortWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int key = 64 * (int)blockIdx.x + lane, per = (groups + kSortWaves - 1) / kSortWaves;
  const int lo = wave * per < groups ? wave * per : groups, hi = lo + per < groups ? lo + per : groups;
  int32_t* at = counts + key;
  const int64_t row = E + 1;
  int n[8], sum = 0;
  auto load = [&](int b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = key <= E && b + i < hi ? at[(b + i) * row] : 0;
  };
  for (int b = lo; b < hi; b += 8) {
    load(b);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += n[i];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < wave; ++w) before += sums[w][lane];
  for (int b = lo; b < hi; b += 8) {
    load(b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (key <= E && b + i < hi) at[(b + i) * row] = before;
      before += n[i];
    }
  }
  if (wave == kSortWaves - 1 && key <= E) at[groups * row] = before;
}

// The rows of workgroup b's pairs: the keys' totals over all workgroups and
// those before b (counts, `scanned`: k_sort_scan's sums of them; null: this one
// sorts everything) and their prefix sum give the first row of every wave's pairs
// of every key; a pair's rank is added.
template <class ID, int R>
__global__ __launch_bounds__(kSortWg) void k_sort_place(const ID* ids, int64_t P, int E, int bits, int k,
                                                        const int32_t* counts, bool scanned, int32_t* offsets,
                                                        int32_t* row_of_pair, int32_t* pair_of_row,
                                                        int32_t* token_of_row) {
  __shared__ int hist[kSortWaves * (kMaxExperts + 1)];
  __shared__ int total[64 * 9], first[64 * 9];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const SortRun<ID, R> run(ids, P, E, bits, hist);
  for (int e = threadIdx.x; e < 64 * 9; e += kSortWg) {
    int all = 0, before = 0;
    if (e <= E) {
      int own = 0;
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {  // the waves' counts become their starts
        const int n = hist[w * (E + 1) + e];
        hist[w * (E + 1) + e] = own;
        own += n;
      }
      all = own;
      if (scanned) {
        before = counts[(int64_t)blockIdx.x * (E + 1) + e];
        all = counts[(int64_t)gridDim.x * (E + 1) + e];
      } else if (counts != nullptr) {
        all = 0;
#pragma unroll 8
        for (int b = 0; b < (int)gridDim.x; ++b) {
          const int n = counts[(int64_t)b * (E + 1) + e];
          all += n;
          before += b < (int)blockIdx.x ? n : 0;
        }
      }
    }
    total[e] = all;
    first[e] = before;
  }
  __syncthreads();
  if (wave == 0) {  // exclusive prefix sum over the keys, nine a lane
    int v[9], sum = 0;
#pragma unroll
    for (int i = 0; i < 9; ++i) {
      v[i] = total[9 * lane + i];
      sum += v[i];
    }
    int at = wave_prefix_sum(sum) - sum;
#pragma unroll
    for (int i = 0; i < 9; ++i) {
      const int e = 9 * lane + i;
      if (blockIdx.x == 0 && e <= E) offsets[e] = at;
      first[e] += at;
      at += v[i];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t p = run.p0 + 64 * r;
    if (p >= P) continue;
    const int key = run.key[r], row = first[key] + hist[wave * (E + 1) + key] + run.rank[r];
    const bool here = key < E;
    row_of_pair[p] = here ? row : ~row;
    pair_of_row[row] = here ? (int)p : ~(int)p;
    token_of_row[row] = here ? (int)p / k : -1;
  }
}

size_t sort_workspace_bytes(int64_t P, int E) {
  if (P <= kSortOne) return 0;
  const int64_t groups = sort_groups(P);
  return (size_t)(groups > kSortDirect ? groups + 1 : groups) * (size_t)(E + 1) * 4;
}

template <class ID>
static hipError_t sort_ids(const ID* ids, int64_t P, int k, int E, int32_t* offsets, int32_t* row_of_pair,
                           int32_t* pair_of_row, int32_t* token_of_row, int32_t* counts, hipStream_t st) {
  int bits = 1;
  while ((E >> bits) != 0) ++bits;
  const int rounds = sort_rounds(P);
  const dim3 grid((unsigned)(P > 0 ? sort_groups(P) : 1)), wg(kSortWg);
  const bool scan = grid.x > kSortDirect;
  auto place = [&](auto r, const int32_t* n) {
    k_sort_place<ID, decltype(r)::value><<<grid, wg, 0, st>>>(ids, P, E, bits, k, n, scan, offsets, row_of_pair,
                                                              pair_of_row, token_of_row);
  };
  using std::integral_constant;
  if (P <= kSortOne) {
    if (rounds == 1) place(integral_constant<int, 1>{}, nullptr);
    else if (rounds == 2) place(integral_constant<int, 2>{}, nullptr);
    else place(integral_constant<int, 4>{}, nullptr);
    return hipGetLastError();
  }
  if (rounds == 1) k_sort_count<ID, 1><<<grid, wg, 0, st>>>(ids, P, E, bits, counts);
  else k_sort_count<ID, 4><<<grid, wg, 0, st>>>(ids, P, E, bits, counts);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (scan) {
    k_sort_scan<<<dim3((unsigned)(E / 64 + 1)), wg, 0, st>>>(counts, (int)grid.x, E);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (rounds == 1) place(integral_constant<int, 1>{}, counts);
  else place(integral_constant<int, 4>{}, counts);
  return hipGetLastError();
}

hipError_t launch_sort(const void* ids, bool ids64, int64_t P, int k, int E, int32_t* offsets, int32_t* row_of_pair,
                       int32_t* pair_of_row, int32_t* token_of_row, void* ws, hipStream_t st) {
  int32_t* counts = (int32_t*)ws;
  return ids64 ? sort_ids((const int64_t*)ids, P, k, E, offsets, row_of_pair, pair_of_row, token_of_row, counts, st)
               : sort_ids((const int32_t*)ids, P, k, E, offsets, row_of_pair, pair_of_row, token_of_row, counts, st);
}

// ------------------------------------------------------------------ rows out of tokens
// Rows and weights of up to eight pairs of a token, in scalar registers: eight
// lanes request them at once (one after another each would cost its latency).
// A row is in [0, rows) or, for a pair without an expert, its complement; an
// entry of a table that names neither, and entries past k, become ~rows.  To be
// built where every lane of the wave is active: a lane that is not has no entry.
struct TokenRows {
  int row[8];
  float w[8];
  __device__ __forceinline__ TokenRows(const int32_t* row_of_pair, const void* weights, int w_dt, int64_t p, int n, int rows) {
    const int l = threadIdx.x & 7;
    int r = ~rows;
    float wt = 1.0f;
    if (l < n) {
      r = row_of_pair[p + l];
      r = (r < 0 ? ~r : r) < rows ? r : ~rows;
      if (weights != nullptr) wt = load_scalar(weights, p + l, w_dt);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      row[j] = __builtin_amdgcn_readlane(r, j);
      w[j] = readlane_f(wt, j);
    }
  }
};

// One workgroup a token: its row is read once and written to the rows of its k
// pairs (zeros where a pair has no expert).  Bound by the writes.
template <class V>
__global__ __launch_bounds__(256) void k_gather_tokens(const char* x, int64_t x_stride, int n, const int32_t* row_of_pair,
                                                       int T, int k, V* rows) {
  const int64_t t = grid_row();
  if (t >= T) return;
  const int P = T * k;
  const V* src = (const V*)(x + t * x_stride);
  for (int j0 = 0; j0 < k; j0 += 8) {
    const TokenRows to(row_of_pair, nullptr, 0, t * k + j0, k - j0, P);
    for (int i = threadIdx.x; i < n; i += 256) {
      const V v = src[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = to.row[j];
        if (r != ~P) rows[(int64_t)(r < 0 ? ~r : r) * n + i] = r < 0 ? V{} : v;
      }
    }
  }
}

hipError_t launch_gather(const void* x, int64_t x_stride, int elem, int H, const int32_t* row_of_pair, int T, int k,
                         void* rows, hipStream_t st) {
  const int64_t bytes = (int64_t)elem * H;
  const char* p = (const char*)x;
  const dim3 grid = row_grid(T), wg(256);
  if (((uintptr_t)x | (uintptr_t)rows | (uint64_t)x_stride | (uint64_t)bytes) % 16 == 0)
    k_gather_tokens<u32x4><<<grid, wg, 0, st>>>(p, x_stride, (int)(bytes / 16), row_of_pair, T, k, (u32x4*)rows);
  else if (elem == 4) k_gather_tokens<uint32_t><<<grid, wg, 0, st>>>(p, x_stride, H, row_of_pair, T, k, (uint32_t*)rows);
  else if (elem == 2) k_gather_tokens<uint16_t><<<grid, wg, 0, st>>>(p, x_stride, H, row_of_pair, T, k, (uint16_t*)rows);
  else k_gather_tokens<uint8_t><<<grid, wg, 0, st>>>(p, x_stride, H, row_of_pair, T, k, (uint8_t*)rows);
  return hipGetLastError();
}

// ------------------------------------------------------------------ rows back into tokens
// N neighbouring values of a row: 1, or 4 or 8 in one access of up to 16 bytes.
// Loads are requested raw and converted at their use, through buffers of one
// row each (zeros past its end, and everywhere for a row that is not there), so
// that nothing stands between the requests of several rows.
template <int DT, int N>
struct RowVec {
  static constexpr int kBytes = N * (DT == FTM_DT_F32 ? 4 : 2);
  using Raw = std::conditional_t<N == 1, uint32_t, std::conditional_t<kBytes == 16, u32x4, u32x2>>;
  __device__ __forceinline__ static Rsrc row(const char* base, int64_t stride, int r, int n) {
    return make_rsrc(base + (r >= 0 ? r : 0) * stride, r >= 0 ? (uint32_t)n * kBytes : 0u);
  }
  __device__ __forceinline__ static Raw request(Rsrc res, int i) {
    const uint32_t off = (uint32_t)i * kBytes;
    if constexpr (kBytes == 16) return __builtin_amdgcn_raw_buffer_load_b128(res, off, 0, 0);
    else if constexpr (kBytes == 8) return __builtin_amdgcn_raw_buffer_load_b64(res, off, 0, 0);
    else if constexpr (kBytes == 4) return bload4(res, off);
    else return bload2(res, off);
  }
  __device__ __forceinline__ static void values(Raw v, float (&f)[N]) {
    if constexpr (N == 1) {
      f[0] = bits_to_f32(v, DT);
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if constexpr (DT == FTM_DT_F32) f[n] = __uint_as_float(v[n]);
        else f[n] = bits_to_f32((v[n >> 1] >> (16 * (n & 1))) & 0xffffu, DT);
      }
    }
  }
  // ONCE: the row is not kept in the caches.
  template <bool ONCE>
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
      if constexpr (ONCE) __builtin_nontemporal_store(v, (Raw*)p + i);
      else ((Raw*)p)[i] = v;
    }
  }
};

// out[t] = sum_j w[t, j] rows[row(t, j)] in order of j, fp32 sums, one
// rounding; w null: ones.  One workgroup a token.  Bound by reading the rows.
template <int DT, int OT, int N>
__global__ __launch_bounds__(256) void k_combine_tokens(const char* rows, int64_t row_stride, const void* w, int w_dt,
                                                        const int32_t* row_of_pair, int T, int k, int n, char* out,
                                                        int64_t out_stride) {
  const int64_t t = grid_row();
  if (t >= T) return;
  const int P = T * k;
  // every lane takes part in each round of the loop (TokenRows asks lanes 0..7),
  // those past the row without loads
  for (int i0 = 0; i0 < n; i0 += 256) {
    const int i = i0 + threadIdx.x;
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0f;
    for (int j0 = 0; j0 < k; j0 += 8) {
      const TokenRows from(row_of_pair, w, w_dt, t * k + j0, k - j0, P);
      using V = RowVec<DT, N>;
      typename V::Raw raw[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) raw[j] = V::request(V::row(rows, row_stride, from.row[j], n), i);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float v[N];
        V::values(raw[j], v);
        const float wt = from.row[j] >= 0 ? from.w[j] : 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = fmaf(wt, v[e], acc[e]);
      }
    }
    if (i < n) RowVec<OT, N>::template store<false>(out + t * out_stride, i, acc);
  }
}

// The gradients of out[t] = sum_j w[t, j] rows[row(t, j)]: grad_rows[row] = w g
// (zeros on rows of no expert), grad_w[t, j] = g[t] . rows[row] (0 without an
// expert), fp32 sums in a fixed order.  One workgroup a token; either may be
// null.  Bound by reading the rows and writing their gradients, which pass the
// caches by: kept, this kernel ends earlier but the next one waits for their lines
// to leave.  8192 tokens of 8 rows of 2048 bf16, four sets of inputs in turn: this
// kernel 111 us, kept 98; the combine that follows 56, kept 79; both calls 168, kept 178.
template <int DT, int OT, int N>
__global__ __launch_bounds__(256) void k_combine_grad(const char* g, int64_t g_stride, const char* rows,
                                                      int64_t row_stride, const void* w, int w_dt,
                                                      const int32_t* row_of_pair, int T, int k, int n, char* grad_rows,
                                                      int64_t grad_stride, void* grad_w) {
  __shared__ float part[4][8];
  const int64_t t = grid_row();
  if (t >= T) return;
  const int P = T * k;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int j0 = 0; j0 < k; j0 += 8) {
    const TokenRows to(row_of_pair, grad_rows != nullptr ? w : nullptr, w_dt, t * k + j0, k - j0, P);
    float dot[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int i = threadIdx.x; i < n; i += 256) {
      using V = RowVec<DT, N>;
      using G = RowVec<OT, N>;
      const typename G::Raw graw = G::request(G::row(g + t * g_stride, 0, 0, n), i);
      typename V::Raw raw[8];
      if (grad_w != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) raw[j] = V::request(V::row(rows, row_stride, to.row[j], n), i);
      }
      float gv[N];
      G::values(graw, gv);
      if (grad_rows != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = to.row[j];
          if (r == ~P) continue;
          float v[N];
#pragma unroll
          for (int e = 0; e < N; ++e) v[e] = r >= 0 ? to.w[j] * gv[e] : 0.0f;
          V::template store<true>(grad_rows + (int64_t)(r < 0 ? ~r : r) * grad_stride, i, v);
        }
      }
      if (grad_w != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (to.row[j] < 0) continue;  // (g may hold infinities: 0 in their place is not the same)
          float v[N];
          V::values(raw[j], v);
#pragma unroll
          for (int e = 0; e < N; ++e) dot[j] = fmaf(gv[e], v[e], dot[j]);
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
    const dim3 grid = row_grid(T), wg(256);
    if (H % N == 0 && ((uintptr_t)rows | (uintptr_t)out | (uint64_t)row_stride) % 16 == 0)
      k_combine_tokens<D, O, N><<<grid, wg, 0, st>>>((const char*)rows, row_stride, w, w_dt, row_of_pair, T, k, H / N,
                                                     (char*)out, os);
    else
      k_combine_tokens<D, O, 1><<<grid, wg, 0, st>>>((const char*)rows, row_stride, w, w_dt, row_of_pair, T, k, H,
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
    const dim3 grid = row_grid(T), wg(256);
    const uint64_t read = grad_w != nullptr ? (uintptr_t)rows | (uint64_t)row_stride : 0;
    if (H % N == 0 && ((uintptr_t)g | (uint64_t)g_stride | read | (uintptr_t)grad_rows) % 16 == 0)
      k_combine_grad<D, O, N><<<grid, wg, 0, st>>>((const char*)g, g_stride, (const char*)rows, row_stride, w, w_dt,
                                                   row_of_pair, T, k, H / N, (char*)grad_rows, rs, grad_w);
    else
      k_combine_grad<D, O, 1><<<grid, wg, 0, st>>>((const char*)g, g_stride, (const char*)rows, row_stride, w, w_dt,
                                                   row_of_pair, T, k, H, (char*)grad_rows, rs, grad_w);
    return hipGetLastError();
  });
}

}  // namespace ftm
