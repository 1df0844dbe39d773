// Rows sorted by expert and back: the learned counterpart of the quadrant partition.  A router gives every
// row (token) top_k expert numbers; gunet_expert_sort orders the n = n_tokens * top_k flat positions by expert
// (stable counting sort), dispatch copies each row once per choice into that order, combine adds a row's
// results back with the router's weights, and the two _grad functions are their transposes.
//
// Everything is a gather or scatter of whole rows: no atomics on results, every float sum in one fixed order
// (choice 0 first, float32, rounded once at the end), so results repeat bit for bit.
#include <algorithm>

#include "common.h"
#include "lowp.h"

namespace gunet {
namespace {

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
// Flat positions per thread and round.  Up to 8192 positions one workgroup ranks all of them in one launch (9.4 us for 8192 of 8 experts; two
// launches over tiles of 2048 take 7.6, but a launch costs the host 3.3); longer lists are cut into tiles of 2048, which more
// workgroups share (65536 of 64 experts: 8.6 us, in tiles of 8192 15.0).
constexpr int kSortAlone = 8, kSortShared = 2;
constexpr int kSortTile = kSortThreads * kSortShared;
constexpr int kSortMaxBlocks = 256;
constexpr int kMaxExperts = GUNET_MAX_EXPERTS;             // one thread per expert in the scans
static_assert(kMaxExperts <= kSortThreads, "one thread per expert");
constexpr int kThreads = 256;

struct SortShape {
  int64_t blocks;   // workgroups
  int64_t chunk;    // flat positions per workgroup
  bool alone;       // one workgroup, one round
};

// At most kSortMaxBlocks workgroups (each reads the counts of all others); longer lists make each of them
// walk several tiles.
SortShape sort_shape(int64_t n) {
  SortShape s;
  s.alone = n <= kSortThreads * kSortAlone;
  if (s.alone) {
    s.chunk = kSortThreads * kSortAlone;
    s.blocks = 1;
    return s;
  }
  const int64_t tiles = ceil_div(n, kSortTile);
  const int64_t tiles_per_block = ceil_div(tiles, kSortMaxBlocks);
  s.chunk = tiles_per_block * kSortTile;
  s.blocks = ceil_div(tiles, tiles_per_block);
  return s;
}

__device__ __forceinline__ int clean_key(int key, int n_experts) { return key >= 0 && key < n_experts ? key : -1; }

// Sum over the lanes below in the workgroup, and the total: one value per thread.
__device__ __forceinline__ int block_exclusive(int v, int* wave_sums, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 63) wave_sums[wave] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    const int s = wave_sums[w];
    before += w < wave ? s : 0;
    all += s;
  }
  *total = all;
  return before + incl - v;
}

// Counts per expert of one workgroup's chunk -> hist[block][expert].
__global__ __launch_bounds__(kSortThreads) void k_expert_count(const int32_t* __restrict__ index, int64_t n, int64_t chunk,
                                                               int n_experts, int32_t* __restrict__ hist) {
  extern __shared__ int lds[];
  for (int e = threadIdx.x; e < n_experts; e += kSortThreads) lds[e] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * chunk, end = begin + chunk < n ? begin + chunk : n;
  for (int64_t i = begin + threadIdx.x; i < end; i += kSortThreads) {
    const int key = clean_key(index[i], n_experts);
    if (key >= 0) atomicAdd(&lds[key], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n_experts; e += kSortThreads) hist[static_cast<int64_t>(blockIdx.x) * n_experts + e] = lds[e];
}

// Ranks and writes one workgroup's chunk.  A wave owns 64 * PER consecutive positions of a tile and ranks them 64 at
// a time: lanes with the same key find each other with one ballot per bit of the key, the lowest of them
// claims the group's places from the wave's own counter of that expert.  Then the counters are summed over the
// waves, offset by what earlier tiles, earlier workgroups and smaller experts hold, and every position has
// its row.  Latency-bound.  ALONE: all positions in one round of one workgroup, hist is not used.
template <int PER, bool ALONE>
__global__ __launch_bounds__(kSortThreads) void k_expert_rank(const int32_t* __restrict__ index, int64_t n, int64_t chunk, int n_experts,
                                                              int key_bits, const int32_t* __restrict__ hist,
                                                              int32_t* __restrict__ offsets, int32_t* __restrict__ order,
                                                              int32_t* __restrict__ slot) {
  extern __shared__ int lds[];
  int* const counts = lds;                               // [kSortWaves][n_experts]
  int* const base = counts + kSortWaves * n_experts;     // [n_experts]: next free row of the expert
  int* const before = base + n_experts;                  // [n_experts]: rows that earlier workgroups hold
  int* const sums = before + n_experts;                  // [kSortWaves]
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t begin = blockIdx.x * chunk, end = begin + chunk < n ? begin + chunk : n;

  for (int e = t; e < n_experts; e += kSortThreads) base[e] = before[e] = 0;
  int total = 0;
  if (!ALONE) {
    __syncthreads();
    // threads of one expert share the workgroups' counts out among them (integer sums: any order)
    int width = 1;
    while (width < n_experts) width <<= 1;
    const int e = t & (width - 1), step = kSortThreads / width;
    if (e < n_experts) {
      int all = 0, mine = 0;
      for (int b = t / width; b < static_cast<int>(gridDim.x); b += step) {
        const int c = hist[static_cast<int64_t>(b) * n_experts + e];
        all += c;
        mine += b < static_cast<int>(blockIdx.x) ? c : 0;
      }
      atomicAdd(&base[e], all);
      atomicAdd(&before[e], mine);
    }
    __syncthreads();
    const int count = t < n_experts ? base[t] : 0;
    const int first = block_exclusive(count, sums, &total);
    if (t < n_experts) {
      base[t] = first + before[t];
      if (blockIdx.x == 0) offsets[t] = first;
    }
    if (blockIdx.x == 0 && t == 0) offsets[n_experts] = total;
  }

  for (int64_t tile = begin; tile < end || (ALONE && tile == begin); tile += kSortThreads * PER) {
    __syncthreads();
    for (int i = t; i < kSortWaves * n_experts; i += kSortThreads) counts[i] = 0;
    __syncthreads();
    int key[PER], rank[PER];
    const int64_t at = tile + wave * (64 * PER) + lane;
#pragma unroll
    for (int s = 0; s < PER; ++s) key[s] = at + 64 * s < end ? clean_key(index[at + 64 * s], n_experts) : -1;
#pragma unroll
    for (int s = 0; s < PER; ++s) {
      rank[s] = 0;
      if (__any(key[s] >= 0)) {
        unsigned long long same = __ballot(key[s] >= 0);
        for (int bit = 0; bit < key_bits; ++bit) {
          const unsigned long long ones = __ballot((key[s] >> bit) & 1);
          same &= (key[s] >> bit) & 1 ? ones : ~ones;
        }
        const int leader = key[s] >= 0 ? __ffsll(same) - 1 : lane;
        int first = 0;
        if (key[s] >= 0 && lane == leader) first = atomicAdd(&counts[wave * n_experts + key[s]], __popcll(same));
        first = __shfl(first, leader);
        rank[s] = first + __popcll(same & ((1ull << lane) - 1));
      }
    }
    __syncthreads();
    int mine = 0;
    if (t < n_experts) {
      for (int w = 0; w < kSortWaves; ++w) {
        const int c = counts[w * n_experts + t];
        counts[w * n_experts + t] = mine;
        mine += c;
      }
    }
    if (ALONE) {
      const int first = block_exclusive(mine, sums, &total);
      if (t < n_experts) {
        base[t] = first;
        offsets[t] = first;
      }
      if (t == 0) offsets[n_experts] = total;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < PER; ++s) {
      const int64_t i = at + 64 * s;
      if (i >= end) continue;
      int row = -1;
      if (key[s] >= 0) {
        row = base[key[s]] + counts[wave * n_experts + key[s]] + rank[s];
        order[row] = static_cast<int32_t>(i);
      }
      slot[i] = row;
    }
    __syncthreads();
    if (t < n_experts) base[t] += mine;
  }
  // rows behind the last expert's
  for (int64_t r = total + begin + t; r < n && r < total + end; r += kSortThreads) order[r] = -1;
}

// What the row kernels are given.  slot[t][j] is the row of token t's choice j; a value outside 0..n-1 is a dropped choice.  A row is worked
// on in pieces of N elements: 16 bytes where every row starts on 16 bytes.  Where they do not, dispatch, which writes top_k rows for one it
// reads, takes pieces of the size that rows do start on (13505 x 3 rows of 333 float16: 9.8 us against 13.8 with unaligned 16-byte ones), and
// combine and dispatch's gradient, which read top_k rows for one they write, unaligned 16-byte ones with a short last one (FULL = false;
// 10.3 us against 20.7 with single elements).  Combine's gradient takes those where rows start on 4 bytes (8000 x 4 rows of 1001 float32
// 65 us against 87 with 4-byte pieces, 30000 x 2 of 33 10.1 against 17.0, 8000 x 4 of 500 bf16 21.1 against 29.5), and single
// elements where they start on 2 (333 float16 19.5 against 23.9).
struct RowArgs {
  int64_t n_tokens, n_rows;
  int32_t top_k, n_experts;
  int32_t width, pieces;    // elements and pieces per row
  int32_t lanes_log2;       // lanes that share a token: 2^lanes_log2 <= 64
  const int32_t* slot;
  const int32_t* offsets;   // only offsets[n_experts] is read: the rows behind it are zeroed
};

__device__ __forceinline__ int64_t kept_row(int32_t s, int64_t n_rows) { return s >= 0 && s < n_rows ? s : -1; }

template <typename T>
constexpr int kVec = 16 / sizeof(T);

template <typename T, int N, bool FULL, bool ONCE = false>
__device__ __forceinline__ Pack<T, N> load_piece(const T* row, int piece, int width) {
  const T* const p = row + static_cast<int64_t>(piece) * N;
  if (FULL) return ONCE ? load_pack_once<T, N>(p) : load_pack<T, N>(p);
  Pack<T, N> v = {};
  if (piece * N + N <= width) {
    __builtin_memcpy(&v, p, sizeof(v));
  } else {
#pragma unroll
    for (int c = 0; c < N - 1; ++c)
      if (piece * N + c < width) v.v[c] = p[c];
  }
  return v;
}
template <typename T, int N, bool FULL>
__device__ __forceinline__ void store_piece(T* row, int piece, int width, const Pack<T, N>& v) {
  T* const p = row + static_cast<int64_t>(piece) * N;
  if (FULL) {
    store_pack<T, N>(p, v);
  } else if (piece * N + N <= width) {
    __builtin_memcpy(p, &v, sizeof(v));
  } else {
#pragma unroll
    for (int c = 0; c < N - 1; ++c)
      if (piece * N + c < width) p[c] = v.v[c];
  }
}

// Zeros into the rows that no choice owns (those behind the last expert's).
template <typename T>
__device__ __forceinline__ void zero_tail(const RowArgs& a, T* rows) {
  int64_t used = a.offsets[a.n_experts];
  used = used < 0 ? 0 : used;
  const int64_t end = a.n_rows * a.width;
  for (int64_t i = used * a.width + static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < end; i += static_cast<int64_t>(gridDim.x) * kThreads)
    rows[i] = from_f32<T>(0.0f);
}

// rows[slot[t][j]] = x[t]: a token's row is read once and written top_k times.  HBM-bound: (n_tokens + n) rows.
template <typename T, int N, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_expert_dispatch(RowArgs a, const T* __restrict__ x, T* __restrict__ rows) {
  constexpr int U = 4;
  const int lanes = 1 << a.lanes_log2;
  const int64_t per_block = kThreads >> a.lanes_log2;
  const int sub = threadIdx.x & (lanes - 1);
  for (int64_t t = blockIdx.x * per_block + (threadIdx.x >> a.lanes_log2); t < a.n_tokens; t += gridDim.x * per_block) {
    const T* const src = x + t * a.width;
    for (int u = sub; u < a.pieces; u += U * lanes) {
      Pack<T, N> v[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (u + i * lanes < a.pieces) v[i] = load_piece<T, N, true, ONCE>(src, u + i * lanes, a.width);
      for (int j = 0; j < a.top_k; ++j) {
        const int64_t r = kept_row(a.slot[t * a.top_k + j], a.n_rows);
        if (r < 0) continue;
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (u + i * lanes < a.pieces) store_piece<T, N, true>(rows + r * a.width, u + i * lanes, a.width, v[i]);
      }
    }
  }
  zero_tail<T>(a, rows);
}

// out[t] = sum_j weights[t][j] rows[slot[t][j]] (WEIGHTED), or the plain sum: combine, and dispatch's gradient.
// Four choices' pieces are fetched together, U of each; the sum is float32, choice 0 first, rounded once.
template <typename T, bool FULL, bool WEIGHTED, int U, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_expert_combine(RowArgs a, const T* __restrict__ rows, const float* __restrict__ weights,
                                                             T* __restrict__ out) {
  constexpr int N = kVec<T>;
  const int lanes = 1 << a.lanes_log2;
  const int64_t per_block = kThreads >> a.lanes_log2;
  const int sub = threadIdx.x & (lanes - 1);
  for (int64_t t = blockIdx.x * per_block + (threadIdx.x >> a.lanes_log2); t < a.n_tokens; t += gridDim.x * per_block) {
    for (int u = sub; u < a.pieces; u += U * lanes) {
      float sum[U][N] = {};
      for (int j0 = 0; j0 < a.top_k; j0 += 4) {
        Pack<T, N> v[4][U];
        float w[4];
        bool kept[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t r = j0 + j < a.top_k ? kept_row(a.slot[t * a.top_k + j0 + j], a.n_rows) : -1;
          kept[j] = r >= 0;
          if (!kept[j]) continue;
          w[j] = WEIGHTED ? weights[t * a.top_k + j0 + j] : 1.0f;
#pragma unroll
          for (int i = 0; i < U; ++i)
            if (u + i * lanes < a.pieces) v[j][i] = load_piece<T, N, FULL, ONCE>(rows + r * a.width, u + i * lanes, a.width);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (kept[j])
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
              for (int c = 0; c < N; ++c)
                sum[i][c] = WEIGHTED ? fmaf(w[j], to_f32(v[j][i].v[c]), sum[i][c]) : sum[i][c] + to_f32(v[j][i].v[c]);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (u + i * lanes >= a.pieces) continue;
        Pack<T, N> o;
#pragma unroll
        for (int c = 0; c < N; ++c) o.v[c] = from_f32<T>(sum[i][c]);
        store_piece<T, N, FULL>(out + t * a.width, u + i * lanes, a.width, o);
      }
    }
  }
}

template <int CTRL>
__device__ __forceinline__ float from_lane(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
// Sum over each aligned group of `lanes` lanes, in all of them: a tree whose first four steps are lane permutations of the vector unit
// (neighbour, pair, mirror of 8, mirror of 16: within the finished smaller groups all lanes are equal).
__device__ __forceinline__ float sum_over_lanes(float v, int lanes) {
  if (lanes > 1) v += from_lane<0xB1>(v);
  if (lanes > 2) v += from_lane<0x4E>(v);
  if (lanes > 4) v += from_lane<0x141>(v);
  if (lanes > 8) v += from_lane<0x140>(v);
  if (lanes > 16) v += __shfl_xor(v, 16);
  if (lanes > 32) v += __shfl_xor(v, 32);
  return v;
}

// Combine's gradient: grad_rows[slot[t][j]] = weights[t][j] grad[t], grad_weights[t][j] = <grad[t], rows[slot[t][j]]>
// (0 where the choice was dropped).  One pass: a token's gradient is read once per four choices, each choice's row read once
// and its gradient written once.  The dot product is a float32 sum per lane, then a fixed tree over the lanes.
template <typename T, int N, bool FULL, int U, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_expert_combine_grad(RowArgs a, const T* __restrict__ grad, const T* __restrict__ rows,
                                                                  const float* __restrict__ weights, T* __restrict__ grad_rows,
                                                                  float* __restrict__ grad_weights) {
  const int lanes = 1 << a.lanes_log2;
  const int64_t per_block = kThreads >> a.lanes_log2;
  const int sub = threadIdx.x & (lanes - 1);
  for (int64_t t = blockIdx.x * per_block + (threadIdx.x >> a.lanes_log2); t < a.n_tokens; t += gridDim.x * per_block) {
    for (int j0 = 0; j0 < a.top_k; j0 += 4) {
      float dot[4] = {}, w[4];
      int64_t r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        r[j] = j0 + j < a.top_k ? kept_row(a.slot[t * a.top_k + j0 + j], a.n_rows) : -1;
        w[j] = r[j] >= 0 ? weights[t * a.top_k + j0 + j] : 0.0f;
      }
      for (int u = sub; u < a.pieces; u += U * lanes) {
        Pack<T, N> g[U], v[4][U];
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (u + i * lanes < a.pieces) g[i] = load_piece<T, N, FULL, ONCE>(grad + t * a.width, u + i * lanes, a.width);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r[j] >= 0)
#pragma unroll
            for (int i = 0; i < U; ++i)
              if (u + i * lanes < a.pieces) v[j][i] = load_piece<T, N, FULL, ONCE>(rows + r[j] * a.width, u + i * lanes, a.width);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (r[j] < 0) continue;
#pragma unroll
          for (int i = 0; i < U; ++i) {
            if (u + i * lanes >= a.pieces) continue;
            Pack<T, N> o;
#pragma unroll
            for (int c = 0; c < N; ++c) {
              dot[j] = fmaf(to_f32(g[i].v[c]), to_f32(v[j][i].v[c]), dot[j]);
              o.v[c] = from_f32<T>(w[j] * to_f32(g[i].v[c]));
            }
            store_piece<T, N, FULL>(grad_rows + r[j] * a.width, u + i * lanes, a.width, o);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        dot[j] = sum_over_lanes(dot[j], lanes);
        if (sub == 0 && j0 + j < a.top_k) grad_weights[t * a.top_k + j0 + j] = r[j] >= 0 ? dot[j] : 0.0f;
      }
    }
  }
  zero_tail<T>(a, grad_rows);
}

int check_shape(const char* fn, int64_t n_tokens, int32_t top_k, int32_t n_experts) {
  GUNET_REQUIRE(n_tokens >= 0 && top_k >= 1 && n_experts >= 1, "%s: n_tokens >= 0, top_k >= 1 and n_experts >= 1 (got %lld, %d, %d)", fn,
                static_cast<long long>(n_tokens), top_k, n_experts);
  GUNET_REQUIRE(n_tokens <= INT32_MAX / top_k, "%s: n_tokens * top_k exceeds int32", fn);
  return GUNET_OK;
}

int check_rows(const char* fn, int32_t dtype, int64_t n_tokens, int32_t top_k, int32_t n_experts, int64_t width) {
  GUNET_TRY(check_shape(fn, n_tokens, top_k, n_experts));
  GUNET_REQUIRE(dtype_valid(dtype), "%s: dtype %d is none of GUNET_DTYPE_*", fn, dtype);
  GUNET_REQUIRE(width >= 0 && width <= (1 << 30), "%s: width %lld (0..2^30)", fn, static_cast<long long>(width));
  return GUNET_OK;
}

bool aligned(std::initializer_list<const void*> ptrs, size_t bytes) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % bytes != 0) return false;
  return true;
}

RowArgs row_args(int64_t n_tokens, int32_t top_k, int32_t n_experts, int64_t width, int per_piece, const int32_t* slot, const int32_t* offsets) {
  RowArgs a = {};
  a.n_tokens = n_tokens;
  a.n_rows = n_tokens * top_k;
  a.top_k = top_k;
  a.n_experts = n_experts;
  a.width = static_cast<int32_t>(width);
  a.pieces = static_cast<int32_t>(ceil_div(width, per_piece));
  a.slot = slot;
  a.offsets = offsets;
  while (a.lanes_log2 < 6 && (1 << a.lanes_log2) < a.pieces) ++a.lanes_log2;
  return a;
}

// One token per group of lanes, up to a million workgroups; beyond that the kernels loop.
unsigned row_grid(const RowArgs& a) {
  return static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(1, ceil_div(a.n_tokens, kThreads >> a.lanes_log2)), int64_t{1} << 20));
}

// Calls f with a tag of the element type and the elements of the largest piece (16, 4 or 2 bytes) that every row starts on.
template <typename F>
int by_type(int32_t dtype, int64_t width, std::initializer_list<const void*> ptrs, F f) {
  const size_t size = dtype_size(dtype);
  const bool full = aligned(ptrs, 16) && width * size % 16 == 0, dwords = aligned(ptrs, 4) && width * size % 4 == 0;
  switch (dtype) {
    case GUNET_DTYPE_F32: return full ? f(TypeTag<float, 4>{}) : f(TypeTag<float, 1>{});
    case GUNET_DTYPE_BF16: return full ? f(TypeTag<__bf16, 8>{}) : dwords ? f(TypeTag<__bf16, 2>{}) : f(TypeTag<__bf16, 1>{});
    default: return full ? f(TypeTag<_Float16, 8>{}) : dwords ? f(TypeTag<_Float16, 2>{}) : f(TypeTag<_Float16, 1>{});
  }
}

// Rows of that many pieces are worked on two pieces a lane at a time: combine of 16384 x 4 rows of 2048 bf16 76 us against 83, of 4096 x 2 rows
// of 1024 4.9 against 5.3 (256 float32, 64 pieces: 66 against 52); combine's gradient from twice as many on: 146 against 153, but
// 12.3 against 9.2 at 128 pieces; with single elements four a lane from 400 on: 8000 x 4 rows of 1001 bf16 37.8 against 54.1, of 501 22.6 against
// 29.8, but 13.0 against 11.0 at 201.
constexpr int kWidePieces = 128;

// Where the rows are more than the L2s hold (8 x 4 MB) everything is read past the caches, which are then left to what is written.  bf16 rows of 1 KB,
// combine / its gradient (us): 8 MB 5.9 / 8.1 against 5.1 / 7.2 through the caches, 32 MB 11.1 / 19.1 against 13.9 / 19.1, 200 MB 51.5 / 88
// against 53.6 / 101, 400 MB 98 / 194 against 107 / 194; 16384 x 4 rows of 4 KB dispatched 54 against 67, combine's gradient 112 against 134.
bool read_once(const RowArgs& a, int32_t dtype) {
  return a.n_rows * a.width * static_cast<int64_t>(dtype_size(dtype)) >= (int64_t{32} << 20);
}

int key_bits_of(int n_experts) {
  int bits = 0;
  while ((1 << bits) < n_experts) ++bits;
  return bits;
}

template <bool WEIGHTED>
int run_combine(const char* fn, const void* rows, int32_t dtype, const float* weights, const int32_t* slot, int64_t n_tokens, int32_t top_k,
                int64_t width, void* out, gunet_stream_t stream) {
  GUNET_TRY(check_rows(fn, dtype, n_tokens, top_k, 1, width));
  if (n_tokens == 0 || width == 0) return GUNET_OK;
  GUNET_REQUIRE(rows && slot && out && (weights || !WEIGHTED), "%s: null pointer", fn);
  GUNET_REQUIRE(aligned({rows, out}, dtype_size(dtype)), "%s: a tensor is not aligned to its type", fn);
  return by_type(dtype, width, {rows, out}, [&](auto tag) {
    using Tag = decltype(tag);
    using T = typename Tag::type;
    constexpr bool kFull = Tag::vec == kVec<T>;
    const RowArgs a = row_args(n_tokens, top_k, 0, width, kVec<T>, slot, nullptr);
    const bool wide = a.pieces >= kWidePieces, once = kFull && read_once(a, dtype);
    auto* const kernel = wide ? (once ? &k_expert_combine<T, kFull, WEIGHTED, 2, kFull> : &k_expert_combine<T, kFull, WEIGHTED, 2, false>)
                              : (once ? &k_expert_combine<T, kFull, WEIGHTED, 1, kFull> : &k_expert_combine<T, kFull, WEIGHTED, 1, false>);
    kernel<<<row_grid(a), kThreads, 0, as_stream(stream)>>>(a, static_cast<const T*>(rows), weights, static_cast<T*>(out));
    GUNET_LAUNCH_CHECK();
    return GUNET_OK;
  });
}

}  // namespace
}  // namespace gunet

using namespace gunet;

extern "C" {

size_t gunet_expert_sort_workspace_bytes(int64_t n_tokens, int32_t top_k, int32_t n_experts) {
  if (check_shape("expert_sort", n_tokens, top_k, n_experts) != GUNET_OK || n_experts > kMaxExperts) return 0;
  const SortShape s = sort_shape(n_tokens * top_k);
  return s.alone ? 0 : static_cast<size_t>(s.blocks) * n_experts * sizeof(int32_t);
}

int gunet_expert_sort(const int32_t* expert_index, int64_t n_tokens, int32_t top_k, int32_t n_experts, int32_t* offsets, int32_t* order,
                      int32_t* slot, void* workspace, size_t workspace_bytes, gunet_stream_t stream) {
  StreamDeviceGuard device_guard(as_stream(stream));
  GUNET_TRY(check_shape("expert_sort", n_tokens, top_k, n_experts));
  if (n_experts > kMaxExperts) {
    set_error("expert_sort: %d experts, at most %d are implemented", n_experts, kMaxExperts);
    return GUNET_ERR_UNSUPPORTED;
  }
  const int64_t n = n_tokens * top_k;
  GUNET_REQUIRE(offsets && (n == 0 || (expert_index && order && slot)), "expert_sort: null pointer");
  const SortShape s = sort_shape(n);
  const size_t need = gunet_expert_sort_workspace_bytes(n_tokens, top_k, n_experts);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    set_error("expert_sort: workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : size_t{0}, need);
    return GUNET_ERR_WORKSPACE;
  }
  GUNET_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 4 == 0, "expert_sort: workspace is not 4-byte aligned");
  int32_t* const hist = static_cast<int32_t*>(workspace);
  const unsigned grid = static_cast<unsigned>(s.blocks);
  if (!s.alone) {
    k_expert_count<<<grid, kSortThreads, n_experts * sizeof(int), as_stream(stream)>>>(expert_index, n, s.chunk, n_experts, hist);
    GUNET_LAUNCH_CHECK();
  }
  const size_t lds = (static_cast<size_t>(kSortWaves + 2) * n_experts + kSortWaves) * sizeof(int);
  auto* const rank = !s.alone         ? &k_expert_rank<kSortShared, false>
                     : n <= kSortTile ? &k_expert_rank<kSortShared, true>      // one token: 3.5 us against 4.0 with eight rounds to skip
                                      : &k_expert_rank<kSortAlone, true>;
  if (lds > (size_t{64} << 10))   // 910 experts and more
    GUNET_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(rank), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
  rank<<<grid, kSortThreads, lds, as_stream(stream)>>>(expert_index, n, s.chunk, n_experts, key_bits_of(n_experts), hist, offsets,
                                                               order, slot);
  GUNET_LAUNCH_CHECK();
  return GUNET_OK;
}

int gunet_expert_dispatch(const void* x, int32_t dtype, const int32_t* offsets, const int32_t* slot, int64_t n_tokens, int32_t top_k,
                          int32_t n_experts, int64_t width, void* rows, gunet_stream_t stream) {
  StreamDeviceGuard device_guard(as_stream(stream));
  GUNET_TRY(check_rows("expert_dispatch", dtype, n_tokens, top_k, n_experts, width));
  if (n_tokens == 0 || width == 0) return GUNET_OK;
  GUNET_REQUIRE(x && offsets && slot && rows, "expert_dispatch: null pointer");
  GUNET_REQUIRE(aligned({x, rows}, dtype_size(dtype)), "expert_dispatch: a tensor is not aligned to its type");
  return by_type(dtype, width, {x, rows}, [&](auto tag) {
    using Tag = decltype(tag);
    using T = typename Tag::type;
    const RowArgs a = row_args(n_tokens, top_k, n_experts, width, Tag::vec, slot, offsets);
    constexpr bool kFull = Tag::vec == kVec<T>;
    auto* const kernel = kFull && read_once(a, dtype) ? &k_expert_dispatch<T, Tag::vec, kFull> : &k_expert_dispatch<T, Tag::vec, false>;
    kernel<<<row_grid(a), kThreads, 0, as_stream(stream)>>>(a, static_cast<const T*>(x), static_cast<T*>(rows));
    GUNET_LAUNCH_CHECK();
    return GUNET_OK;
  });
}

int gunet_expert_dispatch_grad(const void* grad_rows, int32_t dtype, const int32_t* slot, int64_t n_tokens, int32_t top_k, int64_t width,
                               void* grad_x, gunet_stream_t stream) {
  StreamDeviceGuard device_guard(as_stream(stream));
  return run_combine<false>("expert_dispatch_grad", grad_rows, dtype, nullptr, slot, n_tokens, top_k, width, grad_x, stream);
}

int gunet_expert_combine(const void* rows, int32_t dtype, const float* weights, const int32_t* slot, int64_t n_tokens, int32_t top_k,
                         int64_t width, void* out, gunet_stream_t stream) {
  StreamDeviceGuard device_guard(as_stream(stream));
  return run_combine<true>("expert_combine", rows, dtype, weights, slot, n_tokens, top_k, width, out, stream);
}

int gunet_expert_combine_grad(const void* grad_out, const void* rows, int32_t dtype, const float* weights, const int32_t* offsets,
                              const int32_t* slot, int64_t n_tokens, int32_t top_k, int32_t n_experts, int64_t width, void* grad_rows,
                              float* grad_weights, gunet_stream_t stream) {
  StreamDeviceGuard device_guard(as_stream(stream));
  GUNET_TRY(check_rows("expert_combine_grad", dtype, n_tokens, top_k, n_experts, width));
  if (n_tokens == 0) return GUNET_OK;
  GUNET_REQUIRE(weights && offsets && slot && grad_weights && (width == 0 || (grad_out && rows && grad_rows)),
                "expert_combine_grad: null pointer");
  GUNET_REQUIRE(aligned({grad_out, rows, grad_rows}, dtype_size(dtype)), "expert_combine_grad: a tensor is not aligned to its type");
  return by_type(dtype, width, {grad_out, rows, grad_rows}, [&](auto tag) {
    using Tag = decltype(tag);
    using T = typename Tag::type;
    constexpr bool kFull = Tag::vec == kVec<T>, kSingle = sizeof(T) == 2 && Tag::vec == 1, kWhole = kFull || kSingle;
    constexpr int N = kSingle ? 1 : kVec<T>, kWide = kSingle ? 4 : 2;
    const RowArgs a = row_args(n_tokens, top_k, n_experts, width, N, slot, offsets);
    const bool wide = a.pieces >= (kSingle ? 400 : 2 * kWidePieces), once = kFull && read_once(a, dtype);
    auto* const kernel = wide ? (once ? &k_expert_combine_grad<T, N, kWhole, kWide, kFull> : &k_expert_combine_grad<T, N, kWhole, kWide, false>)
                              : (once ? &k_expert_combine_grad<T, N, kWhole, 1, kFull> : &k_expert_combine_grad<T, N, kWhole, 1, false>);
    kernel<<<row_grid(a), kThreads, 0, as_stream(stream)>>>(
        a, static_cast<const T*>(grad_out), static_cast<const T*>(rows), weights, static_cast<T*>(grad_rows), grad_weights);
    GUNET_LAUNCH_CHECK();
    return GUNET_OK;
  });
}

}  // extern "C"
