// Microscaled 4-bit floating point (OCP MXFP4): quantisation, and Dense on 4-bit weights.
//
// A block is 32 consecutive columns of a row.  With amax its largest magnitude the block's scale is
// 2^e, e = floor(log2 amax) - 2 (never below -127), kept as the byte e + 127; an element is x / 2^e rounded to
// nearest even on {0, .5, 1, 1.5, 2, 3, 4, 6} and saturated at 6, kept as a sign bit and the level's number.
// A block with a NaN or an infinity has the scale byte 255, and all of it reads as NaN.
//
// Layout: codes [rows][blocks][16 bytes], the even column in the low four bits; scales [ceil(blocks / 8)][rows][8]:
// the eight scales of one row's 256 columns side by side, so that the fragments of a matrix
// instruction fetch theirs as one dword per lane, contiguous over the rows.
//
// Products run on v_mfma_scale_f32_32x32x64_f8f6f4 with fp4 operands: a lane holds one block (16 bytes) of one row per operand and
// the instruction multiplies by both blocks' scales, so the data goes from memory to the matrix core as
// it lies; sums are float32.
#include <algorithm>

#include "common.h"
#include "lowp.h"

namespace gunet {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 32;                // columns that share a scale
constexpr int kTileBlocks = 8;            // blocks of a K tile: 256 columns, one 8-byte group of scales
constexpr int64_t kMaxK = int64_t{1} << 22;

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

inline int64_t blocks_of(int64_t k) { return ceil_div(k, kBlock); }
inline int64_t code_bytes(int64_t rows, int64_t k) { return rows * blocks_of(k) * 16; }
inline int64_t scale_bytes(int64_t rows, int64_t k) { return ceil_div(blocks_of(k), kTileBlocks) * rows * 8; }

__device__ __forceinline__ float scale_value(uint32_t byte) { return __uint_as_float(byte == 0 ? 0x00400000u : byte << 23); }

// ---- quantisation ------------------------------------------------------------------------------------

struct QuantArgs {
  int64_t rows;           // rows of x per group
  int64_t rows_out;       // rows of codes and scales per group (> rows where rows are sorted by expert)
  int32_t k, blocks;
  int32_t top_k;
  const int32_t* slot;    // [rows][top_k] rows to write, or null: row r goes to row r
};

// Four lanes share a block, eight elements each: the block's amax takes two exchanges inside a group of four lanes, the codes of
// a lane are one dword.  HBM-bound: x is read once, 17/32 byte per element written (per choice, where rows are
// sorted by expert: quantising on the way replaces a dispatch of the unquantised rows).
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void k_mxfp4_quantize(QuantArgs a, const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales) {
  const int64_t parts = static_cast<int64_t>(a.blocks) * 4;    // eight-element pieces per row
  const int64_t group = blockIdx.y;
  x += group * a.rows * a.k;
  codes += group * a.rows_out * a.blocks * 16;
  const int tiles = (a.blocks + kTileBlocks - 1) / kTileBlocks;
  scales += group * tiles * a.rows_out * 8;
  // the four lanes of a block run the same iterations: the step is a multiple of four
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < a.rows * parts; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = i / parts;
    const int part = static_cast<int>(i - row * parts);
    const int block = part >> 2, col = part * 8;
    float v[8];
    const T* src = x + row * a.k + col;
    if (VEC && col + 8 <= a.k) {
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int p = 0; p < 8 / kPer; ++p) {
        const Pack<T, kPer> q = load_pack<T, kPer>(src + p * kPer);
#pragma unroll
        for (int c = 0; c < kPer; ++c) v[p * kPer + c] = to_f32(q.v[c]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = col + c < a.k ? to_f32(src[c]) : 0.0f;
    }
    // magnitudes as integers: NaN sorts above infinity, infinity above every number
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < 8; ++c) top = max(top, __float_as_uint(v[c]) & 0x7FFFFFFFu);
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1)));
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2)));
    const int exponent = static_cast<int>(top >> 23);
    const uint32_t byte = exponent == 255 ? 255u : static_cast<uint32_t>(max(exponent - 2, 0));
    uint32_t word = 0;
    if (exponent != 255) {
      const float s = scale_value(byte);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], s, 0);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], s, 1);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], s, 2);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], s, 3);
    }
    const int copies = a.slot ? a.top_k : 1;
    for (int j = 0; j < copies; ++j) {
      int64_t r = row;
      if (a.slot) {
        r = a.slot[row * a.top_k + j];
        if (r < 0 || r >= a.rows_out) continue;
      }
      reinterpret_cast<uint32_t*>(codes)[r * parts + part] = word;
      uint8_t* const s8 = scales + (static_cast<int64_t>(block / kTileBlocks) * a.rows_out + r) * 8;
      if ((part & 3) == 0) s8[block % kTileBlocks] = static_cast<uint8_t>(byte);
      // the scales behind the last block belong to no column: 0, so that they never read as NaN
      if (part == static_cast<int>(parts) - 1)
        for (int b = block % kTileBlocks + 1; b < kTileBlocks; ++b) s8[b] = 0;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_mxfp4_dequantize(int64_t rows, int32_t k, int32_t blocks, const uint8_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales, T* __restrict__ out) {
  const int64_t parts = static_cast<int64_t>(blocks) * 4;
  const int64_t group = blockIdx.y;
  out += group * rows * k;
  codes += group * rows * blocks * 16;
  scales += group * ((blocks + kTileBlocks - 1) / kTileBlocks) * rows * 8;
  const bool vec = k % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < rows * parts; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = i / parts;
    const int part = static_cast<int>(i - row * parts);
    const int block = part >> 2, col = part * 8;
    const uint32_t word = reinterpret_cast<const uint32_t*>(codes)[i];
    const uint32_t byte = scales[(static_cast<int64_t>(block / kTileBlocks) * rows + row) * 8 + block % kTileBlocks];
    const float s = scale_value(byte);
    const auto v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 0);
    const auto v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 1);
    const auto v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 2);
    const auto v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 3);
    const float nan = __uint_as_float(0x7FC00000u);
    const float v[8] = {v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
    Pack<T, 8> o;
#pragma unroll
    for (int c = 0; c < 8; ++c) o.v[c] = from_f32<T>(byte == 255 ? nan : v[c]);
    T* const dst = out + row * k + col;
    if (vec && col + 8 <= k) {
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int p = 0; p < 8 / kPer; ++p) {
        Pack<T, kPer> q;
#pragma unroll
        for (int c = 0; c < kPer; ++c) q.v[c] = o.v[p * kPer + c];
        store_pack<T, kPer>(dst + p * kPer, q);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (col + c < k) dst[c] = o.v[c];
    }
  }
}

// ---- the product -------------------------------------------------------------------------------------

// out[r][n] = act(sum_k x[r][k] w[g][n][k] + bias[g][n]) for the rows of group g.
struct ProductArgs {
  const uint8_t* x_codes;     // [rows][blocks * 16]
  const uint8_t* x_scales;    // [tiles][rows][8]
  const uint8_t* w_codes;     // [groups][n_out][blocks * 16]
  const uint8_t* w_scales;    // [groups][tiles][n_out][8]
  const float* bias;          // [groups][n_out] or null
  void* out;                  // [rows][n_out]
  const int32_t* offsets;     // [groups + 1] first row of each group, or null: one group of all rows
  int64_t rows;
  int32_t n_out, blocks, tiles, groups;
  int32_t act, out_dtype;
  int64_t row_tiles;          // upper bound, over all groups
  int32_t col_tiles;
};

struct RowTile {
  int group;        // == groups: rows behind the last group, written as zeros
  int64_t row0;
  int rows;
};

// Row tile number `tile` of the groups' rows cut into tiles of at most `size` rows: every wave finds it by itself, 64 groups at a
// time.  Offsets are taken into 0..rows, so no value of theirs leads out of a tensor.
__device__ __forceinline__ bool find_row_tile(const ProductArgs& a, int size, int64_t tile, RowTile* out) {
  if (a.offsets == nullptr) {
    out->group = 0;
    out->row0 = tile * size;
    out->rows = static_cast<int>(a.rows - out->row0 < size ? a.rows - out->row0 : size);
    return out->rows > 0;
  }
  const int lane = threadIdx.x & 63;
  int done = 0;
  for (int first = 0; first <= a.groups; first += 64) {
    const int g = first + lane;
    int begin = 0, end = 0;
    if (g <= a.groups) {
      const int rows = static_cast<int>(a.rows);
      begin = min(max(a.offsets[g], 0), rows);
      end = g < a.groups ? min(max(a.offsets[g + 1], 0), rows) : rows;
    }
    const int tiles = end > begin ? (end - begin + size - 1) / size : 0;
    int upto = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(upto, d);
      if (lane >= d) upto += up;
    }
    const unsigned long long past = __ballot(done + upto > tile);
    if (past) {
      const int l = __ffsll(past) - 1;
      out->group = __builtin_amdgcn_readfirstlane(first + l);
      const int row0 = __shfl(begin, l) + (static_cast<int>(tile) - done - __shfl(upto - tiles, l)) * size;
      out->row0 = __builtin_amdgcn_readfirstlane(row0);
      out->rows = __builtin_amdgcn_readfirstlane(min(size, __shfl(end, l) - row0));
      return true;
    }
    done += __shfl(upto, 63);
  }
  return false;
}

__device__ __forceinline__ void store_out(void* out, int dtype, int64_t at, float v) {
  if (dtype == GUNET_DTYPE_F32)
    static_cast<float*>(out)[at] = v;
  else if (dtype == GUNET_DTYPE_BF16)
    static_cast<__bf16*>(out)[at] = from_f32<__bf16>(v);
  else
    static_cast<_Float16*>(out)[at] = from_f32<_Float16>(v);
}

template <bool ANY_ACT>
__device__ __forceinline__ float finish(float v, float bias, int act) {
  v += bias;
  if (ANY_ACT) return activate_any(v, act);
  return act == GUNET_ACT_RELU ? fmaxf(v, 0.0f) : v;
}

__device__ __forceinline__ v16f mfma_fp4(uint4 a, uint4 b, v16f c, int step, int a_scale, int b_scale) {
  const v8i av = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w), 0, 0, 0, 0};
  const v8i bv = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w), 0, 0, 0, 0};
  switch (step) {   // the byte of the scale dwords is part of the instruction
    case 0: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, 0, a_scale, 0, b_scale);
    case 1: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, 1, a_scale, 1, b_scale);
    case 2: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, 2, a_scale, 2, b_scale);
    default: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, 3, a_scale, 3, b_scale);
  }
}

// The simple form: a wave computes 32 rows x 32 columns straight from memory.  Within a K tile of 8 blocks half-wave h takes
// blocks 4h..4h+3, one per instruction, so its four scales are one dword.
template <bool ANY_ACT>
__global__ __launch_bounds__(kThreads) void k_mxfp4_product(ProductArgs a) {
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int wave = threadIdx.x >> 6;
  RowTile t;
  if (!find_row_tile(a, 32, blockIdx.x / a.col_tiles, &t)) return;
  const int col0 = static_cast<int>(blockIdx.x % a.col_tiles) * 128 + wave * 32;
  if (col0 >= a.n_out) return;
  const int col = col0 + r;
  if (t.group == a.groups) {
    if (col < a.n_out)
      for (int i = h; i < t.rows; i += 2) store_out(a.out, a.out_dtype, (t.row0 + i) * a.n_out + col, 0.0f);
    return;
  }
  const bool row_ok = r < t.rows, col_ok = col < a.n_out;
  const uint4* xc = reinterpret_cast<const uint4*>(a.x_codes) + (t.row0 + r) * a.blocks;
  const uint4* wc = reinterpret_cast<const uint4*>(a.w_codes) + (static_cast<int64_t>(t.group) * a.n_out + col) * a.blocks;
  v16f acc = {};
  for (int kt = 0; kt < a.tiles; ++kt) {
    int xs = 0, ws = 0;
    if (row_ok) xs = reinterpret_cast<const int*>(a.x_scales)[(static_cast<int64_t>(kt) * a.rows + t.row0 + r) * 2 + h];
    if (col_ok) ws = reinterpret_cast<const int*>(a.w_scales)[((static_cast<int64_t>(t.group) * a.tiles + kt) * a.n_out + col) * 2 + h];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int b = kt * kTileBlocks + 4 * h + s;
      uint4 xv = {}, wv = {};
      if (row_ok && b < a.blocks) xv = xc[b];
      if (col_ok && b < a.blocks) wv = wc[b];
      acc = mfma_fp4(xv, wv, acc, s, xs, ws);
    }
  }
  if (!col_ok) return;
  const float bias = a.bias ? a.bias[static_cast<int64_t>(t.group) * a.n_out + col] : 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = (i & 3) + 8 * (i >> 2) + 4 * h;
    if (row < t.rows) store_out(a.out, a.out_dtype, (t.row0 + row) * a.n_out + col, finish<ANY_ACT>(acc[i], bias, a.act));
  }
}

// ---- host side ---------------------------------------------------------------------------------------

int check_matrix(const char* fn, int64_t groups, int64_t rows, int64_t k) {
  GUNET_REQUIRE(groups >= 0 && groups <= 65535, "%s: %lld groups (0..65535)", fn, static_cast<long long>(groups));
  GUNET_REQUIRE(rows >= 0 && rows <= INT32_MAX, "%s: %lld rows", fn, static_cast<long long>(rows));
  GUNET_REQUIRE(k >= 1 && k <= kMaxK, "%s: k = %lld (1..%lld)", fn, static_cast<long long>(k), static_cast<long long>(kMaxK));
  return GUNET_OK;
}

unsigned stride_grid(int64_t items) { return static_cast<unsigned>(std::min<int64_t>(ceil_div(items, kThreads), 1 << 16)); }

// x [groups][rows][k] -> codes, scales of rows_out rows per group (slot: where each row's copies go).
int launch_quantize(const void* x, int32_t dtype, int64_t groups, int64_t rows, int64_t rows_out, int32_t k, int32_t top_k,
                    const int32_t* slot, void* codes, void* scales, hipStream_t stream) {
  QuantArgs a = {};
  a.rows = rows;
  a.rows_out = rows_out;
  a.k = k;
  a.blocks = static_cast<int32_t>(blocks_of(k));
  a.top_k = top_k;
  a.slot = slot;
  const dim3 grid(stride_grid(rows * a.blocks * 4), static_cast<unsigned>(groups));
  const size_t size = dtype_size(dtype);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (k * size) % 16 == 0;
  uint8_t* const c = static_cast<uint8_t*>(codes);
  uint8_t* const s = static_cast<uint8_t*>(scales);
#define GUNET_QUANTIZE(T)                                                                        \
  if (vec)                                                                                       \
    k_mxfp4_quantize<T, true><<<grid, kThreads, 0, stream>>>(a, static_cast<const T*>(x), c, s); \
  else                                                                                           \
    k_mxfp4_quantize<T, false><<<grid, kThreads, 0, stream>>>(a, static_cast<const T*>(x), c, s)
  if (dtype == GUNET_DTYPE_F32) {
    GUNET_QUANTIZE(float);
  } else if (dtype == GUNET_DTYPE_BF16) {
    GUNET_QUANTIZE(__bf16);
  } else {
    GUNET_QUANTIZE(_Float16);
  }
#undef GUNET_QUANTIZE
  GUNET_LAUNCH_CHECK();
  return GUNET_OK;
}

int launch_product(ProductArgs a, hipStream_t stream) {
  constexpr int kRows = 32, kCols = 128;
  a.row_tiles = a.offsets ? std::min<int64_t>(a.rows, a.rows / kRows + a.groups + 1) : ceil_div(a.rows, kRows);
  a.col_tiles = static_cast<int32_t>(ceil_div(a.n_out, kCols));
  GUNET_REQUIRE(a.row_tiles * a.col_tiles <= INT32_MAX, "mxfp4 product: %lld x %d is more than one launch holds",
                static_cast<long long>(a.rows), a.n_out);
  const unsigned grid = static_cast<unsigned>(a.row_tiles * a.col_tiles);
  if (act_tuned(a.act))
    k_mxfp4_product<false><<<grid, kThreads, 0, stream>>>(a);
  else
    k_mxfp4_product<true><<<grid, kThreads, 0, stream>>>(a);
  GUNET_LAUNCH_CHECK();
  return GUNET_OK;
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

// Quantises x into the workspace and multiplies: both entry points.
int run_dense(const char* fn, const void* x, int32_t dtype, int64_t x_rows, int64_t rows, int32_t top_k, const int32_t* slot,
              const int32_t* offsets, int32_t groups, int32_t k, const uint8_t* w_codes, const uint8_t* w_scales, const float* bias,
              int32_t n_out, int32_t activation, void* out, int32_t out_dtype, void* workspace, size_t workspace_bytes,
              hipStream_t stream) {
  GUNET_REQUIRE(dtype_valid(dtype) && dtype_valid(out_dtype), "%s: dtypes %d, %d are not GUNET_DTYPE_*", fn, dtype, out_dtype);
  GUNET_REQUIRE(act_valid(activation), "%s: activation %d", fn, activation);
  GUNET_REQUIRE(n_out >= 1, "%s: n_out = %d", fn, n_out);
  GUNET_TRY(check_matrix(fn, groups, rows, k));
  if (rows == 0) return GUNET_OK;
  GUNET_REQUIRE(x && w_codes && w_scales && out, "%s: null pointer", fn);
  GUNET_REQUIRE(reinterpret_cast<uintptr_t>(w_codes) % 16 == 0 && reinterpret_cast<uintptr_t>(w_scales) % 8 == 0,
                "%s: codes must lie on 16 bytes, scales on 8", fn);
  GUNET_REQUIRE(reinterpret_cast<uintptr_t>(x) % dtype_size(dtype) == 0 && reinterpret_cast<uintptr_t>(out) % dtype_size(out_dtype) == 0,
                "%s: x or out is not aligned to its type", fn);
  const int64_t codes = align256(code_bytes(rows, k)), need = codes + scale_bytes(rows, k);
  if (workspace == nullptr || workspace_bytes < static_cast<size_t>(need)) {
    set_error("%s: workspace of %zu bytes, %lld are needed", fn, workspace ? workspace_bytes : size_t{0}, static_cast<long long>(need));
    return GUNET_ERR_WORKSPACE;
  }
  GUNET_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: workspace is not 16-byte aligned", fn);
  uint8_t* const x_codes = static_cast<uint8_t*>(workspace);
  GUNET_TRY(launch_quantize(x, dtype, 1, x_rows, rows, k, top_k, slot, x_codes, x_codes + codes, stream));
  ProductArgs a = {};
  a.x_codes = x_codes;
  a.x_scales = x_codes + codes;
  a.w_codes = w_codes;
  a.w_scales = w_scales;
  a.bias = bias;
  a.out = out;
  a.offsets = offsets;
  a.rows = rows;
  a.n_out = n_out;
  a.blocks = static_cast<int32_t>(blocks_of(k));
  a.tiles = static_cast<int32_t>(ceil_div(a.blocks, kTileBlocks));
  a.groups = groups;
  a.act = activation;
  a.out_dtype = out_dtype;
  return launch_product(a, stream);
}

}  // namespace
}  // namespace gunet

using namespace gunet;

extern "C" {

size_t gunet_mxfp4_code_bytes(int64_t groups, int64_t rows, int32_t k) {
  if (check_matrix("mxfp4_code_bytes", groups, rows, k) != GUNET_OK) return 0;
  return static_cast<size_t>(groups) * code_bytes(rows, k);
}

size_t gunet_mxfp4_scale_bytes(int64_t groups, int64_t rows, int32_t k) {
  if (check_matrix("mxfp4_scale_bytes", groups, rows, k) != GUNET_OK) return 0;
  return static_cast<size_t>(groups) * scale_bytes(rows, k);
}

int gunet_mxfp4_quantize(const void* x, int32_t dtype, int64_t groups, int64_t rows, int32_t k, uint8_t* codes, uint8_t* scales,
                         gunet_stream_t stream) {
  StreamDeviceGuard device_guard(as_stream(stream));
  GUNET_REQUIRE(dtype_valid(dtype), "mxfp4_quantize: dtype %d is none of GUNET_DTYPE_*", dtype);
  GUNET_TRY(check_matrix("mxfp4_quantize", groups, rows, k));
  if (groups == 0 || rows == 0) return GUNET_OK;
  GUNET_REQUIRE(x && codes && scales, "mxfp4_quantize: null pointer");
  GUNET_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(x) % dtype_size(dtype) == 0,
                "mxfp4_quantize: codes must lie on 16 bytes, scales on 8, x on its type's size");
  return launch_quantize(x, dtype, groups, rows, rows, k, 1, nullptr, codes, scales, as_stream(stream));
}

int gunet_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t groups, int64_t rows, int32_t k, void* out, int32_t dtype,
                           gunet_stream_t stream) {
  StreamDeviceGuard device_guard(as_stream(stream));
  GUNET_REQUIRE(dtype_valid(dtype), "mxfp4_dequantize: dtype %d is none of GUNET_DTYPE_*", dtype);
  GUNET_TRY(check_matrix("mxfp4_dequantize", groups, rows, k));
  if (groups == 0 || rows == 0) return GUNET_OK;
  GUNET_REQUIRE(codes && scales && out, "mxfp4_dequantize: null pointer");
  GUNET_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(out) % dtype_size(dtype) == 0,
                "mxfp4_dequantize: codes must lie on 16 bytes, scales on 8, out on its type's size");
  const int32_t blocks = static_cast<int32_t>(blocks_of(k));
  const dim3 grid(stride_grid(rows * blocks * 4), static_cast<unsigned>(groups));
  hipStream_t s = as_stream(stream);
  if (dtype == GUNET_DTYPE_F32)
    k_mxfp4_dequantize<float><<<grid, kThreads, 0, s>>>(rows, k, blocks, codes, scales, static_cast<float*>(out));
  else if (dtype == GUNET_DTYPE_BF16)
    k_mxfp4_dequantize<__bf16><<<grid, kThreads, 0, s>>>(rows, k, blocks, codes, scales, static_cast<__bf16*>(out));
  else
    k_mxfp4_dequantize<_Float16><<<grid, kThreads, 0, s>>>(rows, k, blocks, codes, scales, static_cast<_Float16*>(out));
  GUNET_LAUNCH_CHECK();
  return GUNET_OK;
}

size_t gunet_mxfp4_dense_workspace_bytes(int64_t rows, int32_t k) {
  if (check_matrix("mxfp4_dense_workspace_bytes", 1, rows, k) != GUNET_OK) return 0;
  return static_cast<size_t>(align256(code_bytes(rows, k)) + scale_bytes(rows, k));
}

int gunet_mxfp4_dense_forward(const void* x, int32_t dtype, int64_t rows, int32_t k, const uint8_t* w_codes, const uint8_t* w_scales,
                              const float* bias, int32_t n_out, int32_t activation, void* out, int32_t out_dtype, void* workspace,
                              size_t workspace_bytes, gunet_stream_t stream) {
  StreamDeviceGuard device_guard(as_stream(stream));
  return run_dense("mxfp4_dense", x, dtype, rows, rows, 1, nullptr, nullptr, 1, k, w_codes, w_scales, bias, n_out, activation, out, out_dtype,
                   workspace, workspace_bytes, as_stream(stream));
}

int gunet_mxfp4_expert_dense_forward(const void* x, int32_t dtype, const int32_t* offsets, const int32_t* slot, int64_t n_tokens, int32_t top_k,
                                     int32_t n_experts, int32_t k, const uint8_t* w_codes, const uint8_t* w_scales, const float* bias,
                                     int32_t n_out, int32_t activation, void* out, int32_t out_dtype, void* workspace,
                                     size_t workspace_bytes, gunet_stream_t stream) {
  StreamDeviceGuard device_guard(as_stream(stream));
  GUNET_REQUIRE(n_tokens >= 0 && top_k >= 1 && n_experts >= 1 && n_tokens <= INT32_MAX / top_k,
                "mxfp4_expert_dense: n_tokens = %lld, top_k = %d, n_experts = %d", static_cast<long long>(n_tokens), top_k, n_experts);
  GUNET_REQUIRE(offsets || n_tokens == 0, "mxfp4_expert_dense: null pointer");
  const int64_t rows = n_tokens * top_k;
  return run_dense("mxfp4_expert_dense", x, dtype, slot ? n_tokens : rows, rows, top_k, slot, offsets, n_experts, k, w_codes, w_scales, bias,
                   n_out, activation, out, out_dtype, workspace, workspace_bytes, as_stream(stream));
}

}  // extern "C"
