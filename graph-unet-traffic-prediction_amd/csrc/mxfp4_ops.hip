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
#include <type_traits>

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

// Eight elements of a row from column `col` on (columns past k read as 0): the lane's share of its block.
template <typename T, bool VEC>
__device__ __forceinline__ Pack<T, 8> load_eight(const T* row, int col, int k) {
  Pack<T, 8> v;
  if (col + 8 <= k) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int p = 0; p < 8; p += kPer) {
      Pack<T, kPer> q;
      if (VEC)
        q = load_pack<T, kPer>(row + col + p);
      else
        __builtin_memcpy(&q, row + col + p, sizeof(q));     // an unaligned load
#pragma unroll
      for (int c = 0; c < kPer; ++c) v.v[p + c] = q.v[c];
    }
  } else {
#pragma unroll
    for (int c = 0; c < 8; ++c) v.v[c] = col + c < k ? row[col + c] : static_cast<T>(0.0f);
  }
  return v;
}

// The value of a neighbour among four lanes: CTRL 0xB1 exchanges lanes 0, 1 and 2, 3, CTRL 0x4E the two pairs.
template <int CTRL>
__device__ __forceinline__ uint32_t of_four(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, true));
}

// Four neighbouring lanes hold a block, eight elements each: returns the lane's eight codes and the block's scale byte.  Two-byte types stay as
// they are, two to a register: the instruction converts them from that (both types exactly, as the float32 form does).
template <typename T>
__device__ __forceinline__ uint32_t quantize_eight(const Pack<T, 8>& v, uint32_t* byte) {
  // magnitudes as integers: NaN sorts above infinity, infinity above every number
  uint32_t top = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int c = 0; c < 8; ++c) top = max(top, __float_as_uint(v.v[c]) & 0x7FFFFFFFu);
  } else {
    typedef uint16_t Two __attribute__((ext_vector_type(2)));
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    Two most = {0, 0};
#pragma unroll
    for (int c = 0; c < 4; ++c) most = __builtin_elementwise_max(most, __builtin_bit_cast(Two, w[c] & 0x7FFF7FFFu));
    top = max(most[0], most[1]);
  }
  top = max(top, of_four<0xB1>(top));
  top = max(top, of_four<0x4E>(top));
  int exponent;      // of the float32 value
  if constexpr (sizeof(T) == 4)
    exponent = static_cast<int>(top >> 23);
  else if constexpr (std::is_same<T, __bf16>::value)
    exponent = static_cast<int>(top >> 7);
  else
    exponent = top >= 0x7C00u ? 255 : static_cast<int>(__float_as_uint(to_f32(__builtin_bit_cast(_Float16, static_cast<uint16_t>(top)))) >> 23);
  *byte = exponent == 255 ? 255u : static_cast<uint32_t>(max(exponent - 2, 0));
  if (exponent == 255) return 0;
  const float s = scale_value(*byte);
  uint32_t word = 0;
  if constexpr (sizeof(T) == 4) {
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v.v[0], v.v[1], s, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v.v[2], v.v[3], s, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v.v[4], v.v[5], s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v.v[6], v.v[7], s, 3);
  } else {
    typedef T Two __attribute__((ext_vector_type(2)));
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3];      // a bit cast of a vector's element itself takes element 0
    const Two a = __builtin_bit_cast(Two, w0), b = __builtin_bit_cast(Two, w1), c = __builtin_bit_cast(Two, w2), d = __builtin_bit_cast(Two, w3);
    if constexpr (std::is_same<T, __bf16>::value) {
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, a, s, 0);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, b, s, 1);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, c, s, 2);
      return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, d, s, 3);
    } else {
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, a, s, 0);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, b, s, 1);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, c, s, 2);
      return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, d, s, 3);
    }
  }
}

// Four lanes share a block: its amax takes two exchanges inside a group of four lanes, the codes of a lane are one dword.  HBM-bound: x
// is read once, 17/32 byte per element written (per choice, where rows are sorted by expert: quantising on the way
// replaces a dispatch of the unquantised rows).  8192 x 8192 bf16 in 31.6 us, 5.4 TB/s (36.8 with its elements widened to float32 first).
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
    const int block = part >> 2;
    uint32_t byte;
    const uint32_t word = quantize_eight(load_eight<T, VEC>(x + row * a.k, part * 8, a.k), &byte);
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

// The inverse: a lane writes 16 bytes, 4 or 8 values of one block (8 float32 values a lane, in two stores whose lanes lie 32 bytes apart, took
// 35 us for 4096 x 8192 where this takes 27.6, 5.5 TB/s), past the caches (quantised and read back 57.6 us against 63).  Rows that do not start on 16 bytes: unaligned stores, 28.5 us at 8191.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_mxfp4_dequantize(int64_t rows, int32_t k, int32_t blocks, const uint8_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales, T* __restrict__ out) {
  constexpr int kPer = 16 / sizeof(T);
  using Word = typename std::conditional<kPer == 8, uint32_t, uint16_t>::type;
  const int64_t parts = static_cast<int64_t>(blocks) * (kBlock / kPer);
  const int64_t group = blockIdx.y;
  out += group * rows * k;
  codes += group * rows * blocks * 16;
  scales += group * ((blocks + kTileBlocks - 1) / kTileBlocks) * rows * 8;
  const bool vec = k % kPer == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < rows * parts; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = i / parts;
    const int part = static_cast<int>(i - row * parts);
    const int block = part / (kBlock / kPer), col = part * kPer;
    const uint32_t word = reinterpret_cast<const Word*>(codes)[i];
    const uint32_t byte = scales[(static_cast<int64_t>(block / kTileBlocks) * rows + row) * 8 + block % kTileBlocks];
    const float s = scale_value(byte), nan = __uint_as_float(0x7FC00000u);
    const auto v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 0);
    const auto v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 1);
    float v[8] = {v0[0], v0[1], v1[0], v1[1]};
    if (kPer == 8) {
      const auto v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 2);
      const auto v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 3);
      v[4] = v2[0], v[5] = v2[1], v[6] = v3[0], v[7] = v3[1];
    }
    Pack<T, kPer> o;
#pragma unroll
    for (int c = 0; c < kPer; ++c) o.v[c] = from_f32<T>(byte == 255 ? nan : v[c]);
    T* const dst = out + row * k + col;
    if (vec) {      // k is a multiple of kPer: all of the piece or none
      if (col < k) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, o), reinterpret_cast<u32x4*>(dst));
    } else if (col + kPer <= k) {
      __builtin_memcpy(dst, &o, sizeof(o));          // an unaligned store
    } else {
#pragma unroll
      for (int c = 0; c < kPer; ++c)
        if (col + c < k) dst[c] = o.v[c];
    }
  }
}

// ---- the product -------------------------------------------------------------------------------------

// out[r][n] = act(sum_k x[r][k] w[g][n][k] + bias[g][n]) for the rows of group g.
struct ProductArgs {
  const void* x;              // for the form that quantises on the way: [rows][k], or with slot [rows / top_k][k]
  const int32_t* slot;        // [rows] or null: row r is a copy of the one whose choice has slot r
  int32_t k, top_k;
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
  int32_t col_tiles;
  int32_t out_wide;           // every row of out starts on 16 bytes
};

struct RowTile {
  int group;        // == groups: rows behind the last group, written as zeros
  int64_t row0;
  int rows;
};

// First and last row of group g (g == groups: the rows behind the last group).  Offsets are taken into 0..rows, so no value of theirs leads
// out of a tensor.
__device__ __forceinline__ void group_rows(const ProductArgs& a, int g, int* begin, int* end) {
  *begin = *end = 0;
  if (g > a.groups) return;
  const int rows = static_cast<int>(a.rows);
  *begin = min(max(a.offsets[g], 0), rows);
  *end = g < a.groups ? min(max(a.offsets[g + 1], 0), rows) : rows;
}

// Row tiles that rows begin .. end - 1 are cut into (unsigned: the sum may pass 2^31).
__device__ __forceinline__ int tiles_of(int begin, int end, int size) {
  return end > begin ? static_cast<int>((static_cast<uint32_t>(end - begin) + size - 1) / static_cast<uint32_t>(size)) : 0;
}

// Number of row tiles of at most `size` rows that the groups' rows are cut into.
__device__ __forceinline__ int count_row_tiles(const ProductArgs& a, int size) {
  if (a.offsets == nullptr) return static_cast<int>((a.rows + size - 1) / size);
  int mine = 0;
  for (int g = threadIdx.x & 63; g <= a.groups; g += 64) {
    int begin, end;
    group_rows(a, g, &begin, &end);
    mine += tiles_of(begin, end, size);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) mine += __shfl_xor(mine, d);
  return __builtin_amdgcn_readfirstlane(mine);
}

// Row tile number `tile`: every wave finds it by itself, 64 groups at a time.
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
    int begin, end;
    group_rows(a, first + lane, &begin, &end);
    const int tiles = tiles_of(begin, end, size);
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

// The row of x that row r is a copy of; there are 16 slots at most.
__device__ __forceinline__ int64_t source_row(const ProductArgs& a, int64_t r) {
  if (a.slot == nullptr) return r;
  int at = 0;
  for (int j = 0; j < static_cast<int>(a.rows); ++j) at = a.slot[j] == r ? j : at;
  return at / a.top_k;
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

// 16 bytes per lane from memory straight into LDS: lane l's land at lds_base + 16 l.  The compiler does not see the load: the caller
// waits for it before a barrier.  What lies out of the buffer's range reads as zeros.
// The compiler does not look into the asm for hazards either: m0 has to be written one wait state before a load to LDS, and scalar registers
// that the vector unit wrote (readfirstlane) five before a load that reads them.
// m0 is a reserved register, so the compiler warns that it keeps nothing in it across the asm: nothing here asks it to.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma_to_lds(u32x4 rsrc, uint32_t lds_base, uint32_t lane_off, uint32_t uniform_off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds_base), "v"(lane_off), "s"(rsrc), "s"(uniform_off)
               : "memory", "m0");
}
#pragma clang diagnostic pop
// Waits until at most N of this wave's loads are on their way and its LDS reads are done, then for the other waves.
template <int N>
__device__ __forceinline__ void wait_and_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
__device__ __forceinline__ u32x4 rsrc_of(const void* p, uint32_t bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  u32x4 r = {static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at))),
             static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32) & 0xFFFF)),
             static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(bytes))), 0x00020000u};
  return r;
}

// LDS by its byte address.  Volatile, so that the compiler keeps the order of what different lanes of a wave write and read (the hardware does) and
// neither merges nor cuts the accesses; through LDS's own address space, since a volatile access through a plain pointer becomes a
// flat one, which waits for the wave's stores to memory as well.
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at) {
  return *(const volatile __attribute__((address_space(3))) V*)(static_cast<uintptr_t>(at));
}
template <typename V>
__device__ __forceinline__ void lds_write(uint32_t at, V v) {
  *(volatile __attribute__((address_space(3))) V*)(static_cast<uintptr_t>(at)) = v;
}

constexpr int kBand = 4;
// Widest rows and most columns of the form by rows (rows_form), which makes one buffer of all the weights.
constexpr int64_t kRowsMaxK = 2048, kRowsMaxColumns = 8192;
// A lane offset past every buffer here, and still a 32-bit one with the K axis added: a tile's 256 rows, all the columns of the form by rows.
constexpr uint32_t kOutOfRange = 0x7FFFFFF0u;
static_assert(256 * (kMaxK / 2) <= kOutOfRange && kRowsMaxColumns * (kRowsMaxK / 2) <= kOutOfRange && kMaxK / 2 <= UINT32_MAX - kOutOfRange, "past every buffer");

// The tiled form: a workgroup of WM x WN waves computes BM rows x BN columns, a wave FM x FN fragments of 32 x 32.  K tiles of 256
// columns (128 bytes a row, and 8 bytes of scales) go through STAGES LDS buffers, filled by direct loads STAGES - 1 tiles ahead of the
// one being multiplied; one barrier per tile.  A row's eight blocks lie in LDS permuted by the row's number (block b at place
// b ^ (row / 2 & 7)), which spreads any 16 neighbouring rows that a fragment load reads one block of over all 64 banks
// (two rows of 128 bytes span them once).  The weights are the instruction's first operand, so that a lane ends up with four
// neighbouring columns of one output row.
template <int WM, int WN, int FM, int FN, int STAGES>
struct TileShape {
  static constexpr int BM = WM * FM * 32, BN = WN * FN * 32, NW = WM * WN;
  static constexpr int SA = (BM + 127) / 128, SB = (BN + 127) / 128;          // scale pieces of 128 rows
  static constexpr int kScales = (BM + BN) * 128, kBuf = kScales + (SA + SB) * 1024;
  // On the way out a wave has its share of one buffer: one or two pieces of 32 rows of 128 bytes at most, and the bias of its columns.
  static constexpr int kOutBytes = kBuf / NW / 16 * 16, kPiece = 32 * 128, kPieces = (kOutBytes - FN * 128) / kPiece >= 2 ? 2 : 1;
  static_assert(kOutBytes >= kPiece + FN * 128, "no room for the way out");
  static constexpr int kLds = STAGES * kBuf, kPerCu = (160 << 10) / kLds;    // workgroups per CU
};

template <int WM, int WN, int FM, int FN, int STAGES, bool ANY_ACT>
__global__ __launch_bounds__(64 * WM * WN, (TileShape<WM, WN, FM, FN, STAGES>::kPerCu * WM * WN / 4)) void k_mxfp4_tile(ProductArgs a) {
  using S = TileShape<WM, WN, FM, FN, STAGES>;
  constexpr int BM = S::BM, BN = S::BN, NW = S::NW, SA = S::SA, SB = S::SB;
  constexpr int CA = BM / 8 / NW, CB = BN / 8 / NW;                          // 8-row pieces per wave
  constexpr int kLoads = CA + CB + 1;                                        // loads per wave and K tile
  constexpr uint32_t kScales = S::kScales, kBuf = S::kBuf;
  static_assert(NW % 2 == 0, "a wave's 8-row pieces must all have the parity of its number");
  static_assert(SA + SB <= NW, "one scale piece per wave");
  static_assert((STAGES - 2) * kLoads < 64, "vmcnt counts to 63");
  static_assert(FN <= 2, "one lane per column of the wave's bias");
  extern __shared__ __attribute__((aligned(128))) char mx_smem[];
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const uint32_t stride = static_cast<uint32_t>(a.blocks) * 16;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)mx_smem));
  const int my_block = (lane & 7) ^ (((wave & 1) << 2) + (lane >> 4));   // place ^ (row / 2 & 7)
  const uint32_t lane_off = static_cast<uint32_t>(wave * 8 + (lane >> 3)) * stride + my_block * 16;
  // the wave's scale piece (waves beyond SA + SB repeat one: every wave has the same number of loads on its way)
  const int piece = wave % (SA + SB);
  const bool x_piece = piece < SA;
  const uint32_t scale_off = static_cast<uint32_t>(x_piece ? piece : piece - SA) * 1024 + lane * 16;
  const int64_t scale_step = (x_piece ? a.rows : static_cast<int64_t>(a.n_out)) * 8;

  // Consecutive workgroups go to different XCDs: each XCD gets a run of tiles, walked in bands of 4 row tiles, so that the tiles in
  // flight on an XCD share their operands in its L2.
  const int64_t row_tiles = count_row_tiles(a, BM), all = row_tiles * a.col_tiles, run = (all + 7) / 8;
  const int64_t tile = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= run || tile >= all) return;
  const int64_t band = tile / (kBand * a.col_tiles), in_band = tile - band * kBand * a.col_tiles;
  const int64_t band_rows = min(static_cast<int64_t>(kBand), row_tiles - band * kBand);
  RowTile t;
  if (!find_row_tile(a, BM, band * kBand + in_band % band_rows, &t)) return;
  const int col0 = static_cast<int>(in_band / band_rows) * BN;
  const int cols = min(BN, a.n_out - col0);
  if (t.group == a.groups) {
    for (int i = threadIdx.x; i < t.rows * BN; i += 64 * NW)
      if (i % BN < cols) store_out(a.out, a.out_dtype, (t.row0 + i / BN) * a.n_out + col0 + i % BN, 0.0f);
    return;
  }
  const int64_t w_row0 = static_cast<int64_t>(t.group) * a.n_out + col0;
  const u32x4 x_rsrc = rsrc_of(a.x_codes + t.row0 * stride, static_cast<uint32_t>(t.rows) * stride);
  const u32x4 w_rsrc = rsrc_of(a.w_codes + w_row0 * stride, static_cast<uint32_t>(cols) * stride);
  const uint8_t* const scales = x_piece ? a.x_scales + t.row0 * 8 : a.w_scales + (static_cast<int64_t>(t.group) * a.tiles * a.n_out + col0) * 8;
  const auto fetch = [&](int kt, int buf) __attribute__((always_inline)) {
    const uint32_t base = lds0 + buf * kBuf + wave * 1024;
    const bool tail = (kt + 1) * kTileBlocks > a.blocks;       // the last tile of a row that ends inside it
    const bool none = tail && kt * kTileBlocks + my_block >= a.blocks;
    const uint32_t step = 8 * NW * stride;
#pragma unroll
    for (int i = 0; i < CA; ++i) dma_to_lds(x_rsrc, base + i * NW * 1024, none ? kOutOfRange : lane_off + i * step, kt * 128);
#pragma unroll
    for (int i = 0; i < CB; ++i) dma_to_lds(w_rsrc, base + BM * 128 + i * NW * 1024, none ? kOutOfRange : lane_off + i * step, kt * 128);
    dma_to_lds(rsrc_of(scales + kt * scale_step, static_cast<uint32_t>(x_piece ? t.rows : cols) * 8), lds0 + buf * kBuf + kScales + piece * 1024,
               scale_off, 0);
  };

  v16f acc[FN][FM];
#pragma unroll
  for (int n = 0; n < FN; ++n)
#pragma unroll
    for (int m = 0; m < FM; ++m) acc[n][m] = v16f{};
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < a.tiles) fetch(s, s);
  int buf = 0;
  for (int kt = 0; kt < a.tiles; ++kt) {
    if (kt + STAGES - 2 < a.tiles)
      wait_and_barrier<(STAGES - 2) * kLoads>();
    else
      wait_and_barrier<0>();
    if (kt + STAGES - 1 < a.tiles) fetch(kt + STAGES - 1, buf == 0 ? STAGES - 1 : buf - 1);
    const char* const base = mx_smem + buf * kBuf;
    int xs[FM], ws[FN];
#pragma unroll
    for (int f = 0; f < FM; ++f) xs[f] = *reinterpret_cast<const int*>(base + kScales + ((wm * FM + f) * 32 + r) * 8 + h * 4);
#pragma unroll
    for (int f = 0; f < FN; ++f) ws[f] = *reinterpret_cast<const int*>(base + kScales + SA * 1024 + ((wn * FN + f) * 32 + r) * 8 + h * 4);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int place = ((4 * h + s) ^ (r >> 1 & 7)) * 16;
      uint4 xf[FM], wf[FN];
#pragma unroll
      for (int f = 0; f < FM; ++f) xf[f] = *reinterpret_cast<const uint4*>(base + ((wm * FM + f) * 32 + r) * 128 + place);
#pragma unroll
      for (int f = 0; f < FN; ++f) wf[f] = *reinterpret_cast<const uint4*>(base + (BM + (wn * FN + f) * 32 + r) * 128 + place);
#pragma unroll
      for (int n = 0; n < FN; ++n)
#pragma unroll
        for (int m = 0; m < FM; ++m) acc[n][m] = mfma_fp4(wf[n], xf[m], acc[n][m], s, ws[n], xs[m]);
    }
    buf = buf == STAGES - 1 ? 0 : buf + 1;
  }
  wait_and_barrier<0>();       // every wave has read its last K tile: LDS is free

  // Lane (r, h) holds row r of a fragment, columns 8 j + 4 h + 0..3 in acc[4 j .. 4 j + 3]: stored from there a wave's 8-byte pieces would
  // touch 32 rows per instruction.  They go through LDS (a region per wave) in pieces of 32 rows x 128 bytes, 16-byte chunks permuted by the
  // row against the banks, and leave 16 bytes a lane as whole lines (8192^3: 0.12 ms less than stores from the fragments), past the caches, which have the operands to hold (16 experts, 268 MB of results: 237 us against 248).
  const uint32_t stage = lds0 + wave * S::kOutBytes, bias_at = stage + S::kPieces * S::kPiece;
  const int wave_col = wn * FN * 32, wave_cols = min(FN * 32, cols - wave_col);
  if (lane < FN * 32) lds_write(bias_at + lane * 4, a.bias && lane < wave_cols ? a.bias[w_row0 + wave_col + lane] : 0.0f);
  const int64_t out0 = (t.row0 + wm * FM * 32) * a.n_out + col0 + wave_col;

  // Fragment row m from column fragment n0 on, in type T: to LDS in 32 rows of kRow bytes, and out through emit(LDS address, kRow, chunk mask)
  const auto piece_out = [&](auto tag, int m, int n0, int which, bool activate, auto emit) __attribute__((always_inline)) {
    using T = typename decltype(tag)::type;
    constexpr int P = sizeof(T) == 4 ? 1 : FN, kRow = P * 32 * sizeof(T), kTurn = kRow / 16 - 1;
    const uint32_t base = stage + which * S::kPiece;
#pragma unroll
    for (int n = 0; n < P; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        typedef T Four __attribute__((ext_vector_type(4)));
        const f32x4n b = lds_read<f32x4n>(bias_at + ((n0 + n) * 32 + 8 * j + 4 * h) * 4);
        Four v;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float sum = acc[n0 + n][m][4 * j + c] + b[c];
          v[c] = from_f32<T>(activate && a.act == GUNET_ACT_RELU ? fmaxf(sum, 0.0f) : sum);
        }
        const int byte = (n * 32 + 8 * j + 4 * h) * sizeof(T);
        lds_write(base + r * kRow + ((byte >> 4 ^ (r * kRow / 128 & kTurn)) << 4) + (byte & 15), v);
      }
    emit(base, kRow, kTurn);
  };
  const auto wide = [&](auto tag) __attribute__((always_inline)) {
    using T = typename decltype(tag)::type;
    constexpr int P = sizeof(T) == 4 ? 1 : FN;
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
      for (int n = 0; n < FN; n += P)
        piece_out(tag, m, n, (m * FN + n) / P % S::kPieces, true, [&](uint32_t base, int row_bytes, int turn) __attribute__((always_inline)) {
          const int lanes = row_bytes / 16, rows = t.rows - (wm * FM + m) * 32;
          const int chunk = lane % lanes, col = n * 32 + chunk * (16 / sizeof(T));
          T* const out = static_cast<T*>(a.out) + out0 + static_cast<int64_t>(m) * 32 * a.n_out + col;
#pragma unroll
          for (int i = 0; i < lanes / 2; ++i) {
            const int row = (i * 64 + lane) / lanes;
            const u32x4 v = lds_read<u32x4>(base + row * row_bytes + ((chunk ^ (row * row_bytes / 128 & turn)) << 4));
            if (row < rows && col < wave_cols) __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(out + static_cast<int64_t>(row) * a.n_out));
          }
        });
  };
  if (!ANY_ACT && a.out_wide) {
    if (a.out_dtype == GUNET_DTYPE_F32)
      wide(TypeTag<float, 4>{});
    else if (a.out_dtype == GUNET_DTYPE_BF16)
      wide(TypeTag<__bf16, 8>{});
    else
      wide(TypeTag<_Float16, 8>{});
  } else {
    // rows that do not start on 16 bytes, and the activations with code of their own: element by element, still along the rows
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
      for (int n = 0; n < FN; ++n)
        piece_out(TypeTag<float, 4>{}, m, n, 0, false, [&](uint32_t base, int row_bytes, int turn) __attribute__((always_inline)) {
          const int rows = min(32, t.rows - (wm * FM + m) * 32);
#pragma nounroll
          for (int i = lane; i < rows * 32; i += 64) {
            const int row = i / 32, col = i % 32;
            const float v = lds_read<float>(base + row * row_bytes + ((col >> 2 ^ (row & turn)) << 4) + (col & 3) * 4);
            const int c = n * 32 + col;
            if (c < wave_cols) store_out(a.out, a.out_dtype, out0 + static_cast<int64_t>(m * 32 + row) * a.n_out + c, finish<ANY_ACT>(v, 0.0f, a.act));
          }
        });
  }
}

typedef float v4f __attribute__((ext_vector_type(4)));
__device__ __forceinline__ v4f mfma16_fp4(u32x4 a, u32x4 b, v4f c, int step, int a_scale, int b_scale) {
  const v8i av = {static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]), static_cast<int>(a[3]), 0, 0, 0, 0};
  const v8i bv = {static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3]), 0, 0, 0, 0};
  switch (step) {
    case 0: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, a_scale, 0, b_scale);
    case 1: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 1, a_scale, 1, b_scale);
    case 2: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 2, a_scale, 2, b_scale);
    default: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 3, a_scale, 3, b_scale);
  }
}

// The form for few rows, where the time is the weights' bytes: a workgroup computes 16 columns for up to 16 * MF rows, its NW waves
// share the K axis out among them in turns of 512 columns (v_mfma_scale_f32_16x16x128: quarter-wave q takes blocks 4 q + s of 16, s = 0..3, its
// scales again one dword), straight from memory to registers with the next turn's loads on their way, and add their parts through LDS in
// wave order.  No barrier inside the K loop.
// XT = void: x comes quantised.  Else x is of that type, and every workgroup quantises its rows (16 at most in all, MF = 1) into LDS while its
// first weights are on their way, which saves the launch (and the time) of doing it before.
template <int MF, int NW, typename XT, bool VEC, bool ANY_ACT>
__global__ __launch_bounds__(64 * NW) void k_mxfp4_skinny(ProductArgs a) {
  constexpr bool kRaw = !std::is_same<XT, void>::value;
  __shared__ __attribute__((aligned(16))) float parts[NW][MF][16][16 + 4];    // [wave][row fragment][row][column]
  extern __shared__ __attribute__((aligned(16))) char raw_smem[];              // kRaw: codes [rows][blocks][16], scales [rows][tiles][8]
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  RowTile t;
  if (!find_row_tile(a, 16 * MF, blockIdx.x / a.col_tiles, &t)) return;
  const int col0 = static_cast<int>(blockIdx.x % a.col_tiles) * 16;
  const int cols = min(16, a.n_out - col0);
  v4f acc[MF];
#pragma unroll
  for (int m = 0; m < MF; ++m) acc[m] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  if (t.group < a.groups) {
    const uint32_t stride = static_cast<uint32_t>(a.blocks) * 16;
    const int64_t w_row0 = static_cast<int64_t>(t.group) * a.n_out + col0;
    const BufferRsrc xr = buffer_of(kRaw ? nullptr : a.x_codes + t.row0 * stride, static_cast<uint32_t>(t.rows) * stride);
    const BufferRsrc wr = buffer_of(a.w_codes + w_row0 * stride, static_cast<uint32_t>(cols) * stride);
    const uint8_t* const xs_base = kRaw ? nullptr : a.x_scales + t.row0 * 8;
    const uint8_t* const ws_base = a.w_scales + (static_cast<int64_t>(t.group) * a.tiles * a.n_out + col0) * 8;
    char* const raw_scales = raw_smem + (kRaw ? t.rows * static_cast<int>(stride) : 0);
    const int turns = (a.blocks + 15) / 16;
    struct Turn {
      u32x4 w[4], x[MF][4];
      int ws, xs[MF];
    };
    // 256 columns per group of scales: quarter-waves 0, 1 read the turn's first group, 2, 3 its second, which a short row may not have
    const auto fetch = [&](int turn, Turn& f) __attribute__((always_inline)) {
      const int64_t kt = 2 * turn + (q >> 1);
      const bool have = kt < a.tiles;
      f.ws = have && r < cols ? *reinterpret_cast<const int*>(ws_base + (kt * a.n_out + r) * 8 + (q & 1) * 4) : 0;
      if constexpr (!kRaw) {
#pragma unroll
        for (int m = 0; m < MF; ++m)
          f.xs[m] = have && m * 16 + r < t.rows ? *reinterpret_cast<const int*>(xs_base + (kt * a.rows + m * 16 + r) * 8 + (q & 1) * 4) : 0;
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int block = turn * 16 + 4 * q + s;
        f.w[s] = __builtin_amdgcn_raw_buffer_load_b128(wr, block < a.blocks ? r * stride + block * 16 : kOutOfRange, 0, 0);
        if constexpr (!kRaw) {
#pragma unroll
          for (int m = 0; m < MF; ++m)
            f.x[m][s] = __builtin_amdgcn_raw_buffer_load_b128(xr, block < a.blocks ? (m * 16 + r) * stride + block * 16 : kOutOfRange, 0, 0);
        }
      }
    };
    const auto multiply = [&](int turn, Turn& f) __attribute__((always_inline)) {
      if constexpr (kRaw) {     // lanes of rows that are not there repeat the last one: their results are not stored
        const int row = min(r, t.rows - 1), kt = 2 * turn + (q >> 1);
        f.xs[0] = kt < a.tiles ? *reinterpret_cast<const int*>(raw_scales + (row * a.tiles + kt) * 8 + (q & 1) * 4) : 0;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int block = turn * 16 + 4 * q + s;
          f.x[0][s] = block < a.blocks ? *reinterpret_cast<const u32x4*>(raw_smem + row * stride + block * 16) : u32x4{0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int m = 0; m < MF; ++m) acc[m] = mfma16_fp4(f.w[s], f.x[m][s], acc[m], s, f.ws, f.xs[m]);
    };
    Turn even, odd;
    int turn = wave;
    if (turn < turns) fetch(turn, even);
    if constexpr (kRaw) {
      const int row_parts = a.blocks * 4;
      for (int i = threadIdx.x; i < t.rows * row_parts; i += 64 * NW) {
        const int row = i / row_parts, part = i - row * row_parts, block = part >> 2;
        uint32_t byte;
        const uint32_t word = quantize_eight(load_eight<XT, VEC>(static_cast<const XT*>(a.x) + source_row(a, t.row0 + row) * a.k, part * 8, a.k), &byte);
        *reinterpret_cast<uint32_t*>(raw_smem + row * stride + part * 4) = word;
        char* const s8 = raw_scales + row * a.tiles * 8;
        if ((part & 3) == 0) s8[block] = static_cast<char>(byte);
        if (part == row_parts - 1)
          for (int b = block + 1; b < a.tiles * kTileBlocks; ++b) s8[b] = 0;
      }
      __syncthreads();
    }
    while (turn < turns) {
      if (turn + NW < turns) fetch(turn + NW, odd);
      multiply(turn, even);
      turn += NW;
      if (turn >= turns) break;
      if (turn + NW < turns) fetch(turn + NW, even);
      multiply(turn, odd);
      turn += NW;
    }
  }
  // lane (r, q) holds row r of the fragment, columns 4 q .. 4 q + 3
#pragma unroll
  for (int m = 0; m < MF; ++m) *reinterpret_cast<v4f*>(&parts[wave][m][r][4 * q]) = acc[m];
  __syncthreads();
  for (int i = threadIdx.x; i < MF * 256; i += 64 * NW) {
    const int m = i >> 8, row = (i >> 4) & 15, col = i & 15;
    if (m * 16 + row >= t.rows || col >= cols) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += parts[w][m][row][col];
    if (t.group < a.groups) {
      const float b = a.bias ? a.bias[static_cast<int64_t>(t.group) * a.n_out + col0 + col] : 0.0f;
      v = finish<ANY_ACT>(v, b, a.act);
    }
    store_out(a.out, a.out_dtype, (t.row0 + m * 16 + row) * a.n_out + col0 + col, v);
  }
}

// The form for small weights and any number of rows of one group: a workgroup quantises its 16 * MF rows of x into LDS and computes all their
// columns (or every gridDim.y-th share of them), so x is read once and never written in 4 bits, and one launch does it all.  A wave takes 16
// columns at a time over the whole K axis (v_mfma_scale_f32_16x16x128, as above), their weights from the L2s straight to registers, a turn
// ahead.  Rows lie in LDS an odd number of 16 bytes apart, so that the 16 rows a fragment reads one block of lie on all 64 banks.
constexpr int kRowsWaves = 8;
template <int MF, typename XT, bool VEC, bool ANY_ACT>
__global__ __launch_bounds__(64 * kRowsWaves) void k_mxfp4_rows(ProductArgs a) {
  constexpr int NW = kRowsWaves;
  extern __shared__ __attribute__((aligned(16))) char rows_smem[];      // codes [rows][pitch], scales [rows][tiles][8]
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (16 * MF);
  const int rows = static_cast<int>(min(static_cast<int64_t>(16 * MF), a.rows - row0));
  const uint32_t stride = static_cast<uint32_t>(a.blocks) * 16, pitch = (a.blocks | 1) * 16;
  char* const lds_scales = rows_smem + 16 * MF * pitch;
  const int scale_pitch = a.tiles * 8;
  const int turns = (a.blocks + 15) / 16, sets = (a.n_out + 15) / 16, step = NW * gridDim.y;
  struct Turn {
    u32x4 w[4];
    int ws;
  };
  const BufferRsrc wr = buffer_of(a.w_codes, static_cast<uint32_t>(a.n_out) * stride);
  const auto fetch = [&](int set, int turn, Turn& f) __attribute__((always_inline)) {
    const int kt = 2 * turn + (q >> 1), col = set * 16 + r;
    f.ws = kt < a.tiles && col < a.n_out ? *reinterpret_cast<const int*>(a.w_scales + (static_cast<int64_t>(kt) * a.n_out + col) * 8 + (q & 1) * 4) : 0;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int block = turn * 16 + 4 * q + s;
      f.w[s] = __builtin_amdgcn_raw_buffer_load_b128(wr, block < a.blocks ? col * stride + block * 16 : kOutOfRange, 0, 0);
    }
  };
  Turn even, odd;
  int set = static_cast<int>(blockIdx.y) * NW + wave;
  if (set < sets) fetch(set, 0, even);
  const int row_parts = a.blocks * 4;
  for (int i = threadIdx.x; i < rows * row_parts; i += 64 * NW) {
    const int row = i / row_parts, part = i - row * row_parts, block = part >> 2;
    uint32_t byte;
    const uint32_t word = quantize_eight(load_eight<XT, VEC>(static_cast<const XT*>(a.x) + (row0 + row) * a.k, part * 8, a.k), &byte);
    *reinterpret_cast<uint32_t*>(rows_smem + row * pitch + part * 4) = word;
    char* const s8 = lds_scales + row * scale_pitch;
    if ((part & 3) == 0) s8[block] = static_cast<char>(byte);
    if (part == row_parts - 1)
      for (int b = block + 1; b < scale_pitch; ++b) s8[b] = 0;
  }
  __syncthreads();
  v4f acc[MF];
#pragma unroll
  for (int m = 0; m < MF; ++m) acc[m] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const auto multiply = [&](int turn, Turn& f) __attribute__((always_inline)) {
    const int kt = 2 * turn + (q >> 1);
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      const int row = min(m * 16 + r, rows - 1);        // lanes of rows that are not there repeat the last one: their results are not stored
      const int xs = kt < a.tiles ? *reinterpret_cast<const int*>(lds_scales + row * scale_pitch + kt * 8 + (q & 1) * 4) : 0;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int block = turn * 16 + 4 * q + s;
        const u32x4 x = block < a.blocks ? *reinterpret_cast<const u32x4*>(rows_smem + row * pitch + block * 16) : u32x4{0, 0, 0, 0};
        acc[m] = mfma16_fp4(f.w[s], x, acc[m], s, f.ws, xs);
      }
    }
  };
  // lane (r, q) holds row r of a fragment, columns 4 q .. 4 q + 3
  const auto columns_out = [&](int at) __attribute__((always_inline)) {
    const int col = at * 16 + 4 * q;
    float b[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) b[c] = a.bias && col + c < a.n_out ? a.bias[col + c] : 0.0f;
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      if (m * 16 + r < rows && col < a.n_out) {
        const int64_t out = (row0 + m * 16 + r) * a.n_out + col;
        float v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = finish<ANY_ACT>(acc[m][c], b[c], a.act);
        const auto four = [&](auto* p) __attribute__((always_inline)) {
          using T = typename std::remove_pointer<decltype(p)>::type;
          Pack<T, 4> o;
#pragma unroll
          for (int c = 0; c < 4; ++c) o.v[c] = from_f32<T>(v[c]);
          store_pack<T, 4>(p + out, o);
        };
        if (!a.out_wide) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (col + c < a.n_out) store_out(a.out, a.out_dtype, out + c, v[c]);
        } else if (a.out_dtype == GUNET_DTYPE_F32) {
          four(static_cast<float*>(a.out));
        } else if (a.out_dtype == GUNET_DTYPE_BF16) {
          four(static_cast<__bf16*>(a.out));
        } else {
          four(static_cast<_Float16*>(a.out));
        }
      }
      acc[m] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
  };
  int turn = 0;
  const auto advance = [&](Turn& now, Turn& next) __attribute__((always_inline)) {
    const int at = set, turn_now = turn;
    if (++turn == turns) {
      turn = 0;
      set += step;
    }
    if (set < sets) fetch(set, turn, next);
    multiply(turn_now, now);
    if (turn == 0) columns_out(at);
  };
  while (set < sets) {
    advance(even, odd);
    if (set >= sets) break;
    advance(odd, even);
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

constexpr int64_t kCus = 256;     // compute units

// The forms of the product: quantising x inside (kRaw*, by the number of waves), by rows (kRows*, by the rows of a workgroup), 16 columns a workgroup
// (kSkinny*: rows, waves), tiles.
enum Form { kRaw4, kRaw8, kRaw16, kRows16, kRows32, kSkinny16x2, kSkinny16x4, kSkinny32x4, kSkinny32x8, kTile32x128, kTile64x128, kTile64x64, kTile128x128, kTile256x256 };
struct FormShape {
  const char* name;
  int rows, cols, waves;    // what a workgroup computes (kRows*: its 16 * kRowsWaves columns, at most), and its waves
};
constexpr FormShape kForms[] = {{"raw 4 waves", 16, 16, 4}, {"raw 8 waves", 16, 16, 8}, {"raw 16 waves", 16, 16, 16},
                                {"rows 16", 16, 16 * kRowsWaves, kRowsWaves}, {"rows 32", 32, 16 * kRowsWaves, kRowsWaves},
                                {"skinny 16 rows 2 waves", 16, 16, 2}, {"skinny 16 rows 4 waves", 16, 16, 4}, {"skinny 32 rows 4 waves", 32, 16, 4},
                                {"skinny 32 rows 8 waves", 32, 16, 8}, {"tile 32 x 128", 32, 128, 4}, {"tile 64 x 128", 64, 128, 4},
                                {"tile 64 x 64", 64, 64, 4}, {"tile 128 x 128", 128, 128, 8}, {"tile 256 x 256", 256, 256, 8}};
static_assert(sizeof(kForms) / sizeof(*kForms) == kTile256x256 + 1, "a shape for each form");

// What the choice of a form goes by.
struct ProductSize {
  int64_t rows, k, n_out;
  int64_t groups;           // experts, or 0: one matrix for all rows
};

// Workgroups of a form.  Experts: at most so many row tiles, whichever way the rows fall; what is not needed ends at once.
int64_t form_grid(Form form, const ProductSize& p) {
  const FormShape& f = kForms[form];
  const int64_t row_tiles = p.groups ? std::min<int64_t>(p.rows, p.rows / f.rows + p.groups + 1) : ceil_div(p.rows, f.rows);
  const int64_t all = row_tiles * ceil_div(p.n_out, f.cols);
  return form >= kTile32x128 ? ceil_div(all, 8) * 8 : all;      // tiles: a run for each XCD
}
// Whether one launch holds them: it has less than 2^32 threads (by rows they are fewer, rows_form).
bool form_fits(Form form, const ProductSize& p) { return form_grid(form, p) * kForms[form].waves * 64 <= UINT32_MAX; }

template <Form FORM, int WM, int WN, int FM, int FN, int STAGES>
int launch_tile(ProductArgs a, int64_t grid, hipStream_t stream) {
  using S = TileShape<WM, WN, FM, FN, STAGES>;
  static_assert(kForms[FORM].rows == S::BM && kForms[FORM].cols == S::BN && kForms[FORM].waves == S::NW, "the form's shape is the kernel's");
  a.col_tiles = static_cast<int32_t>(ceil_div(a.n_out, S::BN));
  auto* const kernel = act_tuned(a.act) ? &k_mxfp4_tile<WM, WN, FM, FN, STAGES, false> : &k_mxfp4_tile<WM, WN, FM, FN, STAGES, true>;
  if (S::kLds > (64 << 10))
    GUNET_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds));
  kernel<<<static_cast<unsigned>(grid), 64 * S::NW, S::kLds, stream>>>(a);
  GUNET_LAUNCH_CHECK();
  return GUNET_OK;
}

template <Form FORM, int MF, int NW, typename XT = void, bool VEC = false>
int launch_skinny(ProductArgs a, int64_t grid, hipStream_t stream, size_t lds = 0) {
  static_assert(kForms[FORM].rows == 16 * MF && kForms[FORM].cols == 16 && kForms[FORM].waves == NW, "the form's shape is the kernel's");
  a.col_tiles = static_cast<int32_t>(ceil_div(a.n_out, 16));
  auto* const kernel = act_tuned(a.act) ? &k_mxfp4_skinny<MF, NW, XT, VEC, false> : &k_mxfp4_skinny<MF, NW, XT, VEC, true>;
  kernel<<<static_cast<unsigned>(grid), 64 * NW, lds, stream>>>(a);
  GUNET_LAUNCH_CHECK();
  return GUNET_OK;
}

// Whether the product quantises x on its way.  Every workgroup does all of it (of its expert's rows), so it pays for little x only; it saves a launch,
// of which the host makes one in 3.5 us.  Whole bf16 call, one launch against two, in a captured graph (us): 1 x 4096 x 4096 4.8 / 6.6,
// 2 x 8192 x 8192 13.0 / 13.7, 4 x 4096 x 4096 5.7 / 7.1, 16 x 1024 x 8192 5.9 / 6.5, 16 x 1024 x 1024 3.9 / 5.0; 1 token x 2 of 8 experts 2048 -> 4096
// 4.3 / 7.1, 4 x 4 of 32 1024 -> 2048 8.2 / 8.5; called one by one 7.7 / 11.9, experts 8.7 / 12.0.  At twice as much x
// 4 x 8192 x 4096 8.8 / 9.0, 16 x 2048 x 8192 8.9 / 7.5; 4 x 4 of 16 experts 2048 -> 4096 15.9 / 14.8.
constexpr int64_t kRawElements = 16384;
bool raw_form(int64_t rows, int64_t k) { return rows <= 16 && rows * k <= kRawElements; }

// Whether one group's product runs by rows in one launch.  Against a launch that quantises and one that multiplies (bf16, captured, us): 24 x 128 x 128
// 3.1 / 5.0, 300 x 512 x 512 4.3 / 6.2, 1000 x 256 x 1024 4.7 / 5.9, 3410 x 128 x 128 3.5 / 5.9, 3410 x 256 x 256 4.6 / 6.0, 13505 x 256 x 256 8.4 / 9.2,
// 24000 x 512 x 128 11.8 / 13.8, 96493 x 64 x 64 13.5 / 15.2, 96493 x 512 x 64 31.5 / 37.4; called one by one about 9 / 11.7.  Beyond, where
// every 16 or 32 rows read all weights anew and rows are written in pieces of 16 columns: 3410 x 256 x 1024 8.6 / 7.2, 8000 x 512 x 512 11.4 / 10.4,
// 13505 x 256 x 512 13.2 / 10.3, 48332 x 512 x 192 27.1 / 25.2, 96493 x 128 x 128 20.0 / 18.7, 300 x 2048 x 256 9.2 / 7.1.
bool rows_form(int64_t rows, int64_t k, int64_t n_out) {
  const bool k_fits = k <= 1024 || (k <= kRowsMaxK && rows >= 1024);
  if (rows > 1 << 26) return false;       // one launch holds 2^32 threads
  if (n_out <= 64) return k_fits;
  if (n_out <= 128) return k_fits && rows <= (k <= 1024 ? 32768 : 16384);
  if (n_out <= 256) return k <= 1024 && rows * n_out <= 3500000;
  return n_out <= kRowsMaxColumns && k <= 1024 && rows * n_out <= (k <= 512 ? 512000000 : 170000000) / std::max<int64_t>(k, 128);
}

// 16 rows a workgroup and each wave 16 columns, while that makes few workgroups (or the columns are few and the quantisation is most of it); else 32, and
// the columns shared out over what fills the chip twice.
Form choose_rows(const ProductSize& p) {
  const bool small = ceil_div(p.rows, 16) * ceil_div(p.n_out, 16 * kRowsWaves) <= kCus * 3 / 2 || (p.n_out <= 64 && p.k >= 256 && p.k <= 1024);
  return small ? kRows16 : kRows32;
}
template <typename XT, bool VEC>
int launch_rows(ProductArgs a, Form form, hipStream_t stream) {
  a.out_wide = reinterpret_cast<uintptr_t>(a.out) % (4 * dtype_size(a.out_dtype)) == 0 && a.n_out % 4 == 0;
  const bool small = form == kRows16;
  const int64_t shares = ceil_div(a.n_out, 16 * kRowsWaves), tiles = ceil_div(a.rows, small ? 16 : 32);
  const int64_t split = small ? shares : std::max<int64_t>(1, std::min(shares, 2 * kCus / tiles));
  const size_t lds = static_cast<size_t>(small ? 16 : 32) * ((a.blocks | 1) * 16 + a.tiles * 8);
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(split));
  const bool any = !act_tuned(a.act);
  auto* const kernel = small ? (any ? &k_mxfp4_rows<1, XT, VEC, true> : &k_mxfp4_rows<1, XT, VEC, false>)
                             : (any ? &k_mxfp4_rows<2, XT, VEC, true> : &k_mxfp4_rows<2, XT, VEC, false>);
  kernel<<<grid, 64 * kRowsWaves, lds, stream>>>(a);
  GUNET_LAUNCH_CHECK();
  return GUNET_OK;
}

// One group: sixteen waves quantise faster than eight, where they are a CU's only ones: 4 x 4096 x 1024 4.4 us against 4.8, 1 x 8192 x 1024 5.2 against
// 5.5, 1 x 4096 x 4096 4.8 both; with two workgroups to a CU 1 x 8192 x 8192 12.8 against 11.9, 16 x 1024 x 8192 7.0 against 5.9.  (Four waves: 4 x 4096 x 1024 6.0.)
// Experts, of which most have a row or two here: four waves, 1 token x 4 of 32 experts 2048 -> 4096 6.6 us against 8.3 with eight, and eight where
// few workgroups have long rows, 1 x 2 of 8 4096 -> 4096 6.4 against 7.3; in two launches 9.1 and 8.5.
Form choose_raw(const ProductSize& p) {
  const int64_t col_tiles = ceil_div(p.n_out, 16);
  if (p.groups) return p.k > 2048 && std::min<int64_t>(p.rows, p.groups + 1) * col_tiles <= 2 * kCus ? kRaw8 : kRaw4;
  return p.rows * p.k > 4096 && col_tiles <= kCus ? kRaw16 : kRaw8;
}
template <typename XT, bool VEC>
int launch_raw(const ProductArgs& a, Form form, int64_t grid, hipStream_t stream) {
  const size_t lds = static_cast<size_t>(a.rows) * (a.blocks * 16 + a.tiles * 8);
  if (form == kRaw4) return launch_skinny<kRaw4, 1, 4, XT, VEC>(a, grid, stream, lds);
  if (form == kRaw8) return launch_skinny<kRaw8, 1, 8, XT, VEC>(a, grid, stream, lds);
  return launch_skinny<kRaw16, 1, 16, XT, VEC>(a, grid, stream, lds);
}
// The forms that take x as it is.
template <typename XT>
int launch_unquantised(const ProductArgs& a, Form form, int64_t grid, hipStream_t stream) {
  const bool vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.k * sizeof(XT) % 16 == 0;
  if (form <= kRaw16) return vec ? launch_raw<XT, true>(a, form, grid, stream) : launch_raw<XT, false>(a, form, grid, stream);
  return vec ? launch_rows<XT, true>(a, form, stream) : launch_rows<XT, false>(a, form, stream);
}

// Which form.  Rows per group decide how many rows a tile can fill, the number of tiles whether they fill the chip (256 CUs).
// Measured, product alone (us):
//   rows x k x n         16 columns a workgroup   64 x 64   128 x 128   256 x 256
//   1 x 4096 x 4096              3.4                7.6       12.4        26.4
//   32 x 4096 x 4096             5.7                7.7       13.0        26.7
//   64 x 4096 x 4096             8.6                7.8       13.3        26.6
//   256 x 4096 x 4096           26.5                8.9       14.3        27.6
//   2048 x 8192 x 1024                             18.8       25.1        48.6
//   4096 x 4096 x 4096                             79.8       48.5        37.7
//   8192 x 8192 x 8192                              540        326         258
// with the quantisation:                  64 x 64   64 x 128   128 x 128   256 x 256
//   512 x 4096 x 4096                       14.8       17.1        18.6        32.0
//   1024 x 4096 x 4096                      24.7       19.1        21.4        34.3
//   2048 x 4096 x 4096                      43.9       37.0        29.8        36.6
//   13505 x 256 x 256 float32               11.8       10.4        10.7        14.1
//   48332 x 256 x 256 float32                          24.4        24.6        25.9
//   96493 x 128 x 128 float32               28.8       24.4        24.4        29.7
//   16384 x 2048 x 1024                                49.8        44.3        42.0
//   16384 x 2048 x 1152                                53.2        50.1        55.7
//   8192 x 8192 x 2176                                  143         136         148
// and experts with their quantisation, by average rows per expert:
//                           16 columns   32 x 128   64 x 128   64 x 64   128 x 128   256 x 256
//   32 of 2048 -> 4096:  1        20.1       22.5       20.7      20.4        29.3        41.7
//                        4        35.4       34.9       39.7      39.7        39.1        48.5
//                        8        41.8       36.4       40.8      40.7        41.1        49.2
//                       16        56.4       40.0       43.5      45.1        43.0        51.0
//                       32        87.3       43.8       44.5      47.5        47.5        52.9
//                       64         147       57.5       47.6      58.1        53.9        57.9
//                      128         269       88.6       65.4      86.4        62.7        68.2
//                      256                    157        107       152         101        91.7
//   64 of 1024 -> 1024:  3        13.6       12.5       12.7
//                       16                   16.1       14.0      14.6        14.7
//                       48                   19.8       15.8                  19.8
//    8 of 4096 -> 2048, too few tiles of 128 columns to fill the chip:
//                        4        12.9       13.6       17.5
//                       32                   14.2       18.0      14.0        19.4
// Two and three rows each, where 32 x 128 begins, 16 columns / 32 x 128: 32 of 2048 -> 4096 27.0 / 29.3 and 29.8 / 30.3, 64 of 1024 -> 4096 32.4 / 28.0 and
// 35.0 / 32.2, 64 of 1024 -> 1024 11.6 / 10.7 and 12.2 / 11.0, 128 of 512 -> 2048 28.0 / 20.9 and 29.7 / 21.5, 128 of 2048 -> 1408 36.1 / 32.8 and 38.8 / 33.7.
// A CU takes in about 50 bytes a ns whatever the form, so a product of few tiles gains by smaller ones as long as each has a CU of its
// own: 32 rows x 16 columns, eight waves sharing K, against 64 x 64, whole call (us): 64 x 8192 x 1024 11.6 / 16.9, 128 x 8192 x 1024 12.2 / 17.3,
// 256 x 2048 x 512 6.8 / 8.1, 512 x 8192 x 256 16.2 / 19.9; and where there are two to a CU 128 x 8192 x 2048 20.0 / 16.8.
Form choose_quantised(const ProductSize& p) {
  const bool experts = p.groups > 0;
  const int64_t per_group = experts ? ceil_div(p.rows, p.groups) : p.rows;
  const auto tiles = [&](int64_t m, int64_t n) { return (experts ? p.rows / m + p.groups / 2 : ceil_div(p.rows, m)) * ceil_div(p.n_out, n); };
  const int64_t expert_tiles = p.groups * ceil_div(p.n_out, 128);      // if each expert's rows fit one row tile
  if (expert_tiles >= kCus && per_group >= 2 && per_group <= 96) {
    // experts have uneven numbers of rows, so 32 rows hold most of them up to an average of 12 only; where there are many tiles to hide in, of 24
    return per_group < 12 || (per_group <= 24 && expert_tiles >= 4 * kCus) ? kTile32x128 : kTile64x128;
  }
  if (per_group <= (experts ? 6 : 16)) {
    // two waves a workgroup stream as well as four once there are four workgroups per CU, and leave more of them side by side: 35.5 us
    // against 41.6 for 32 experts of 4 rows each
    return std::min<int64_t>(p.rows, p.rows / 16 + std::max<int64_t>(1, p.groups)) * ceil_div(p.n_out, 16) >= 1024 ? kSkinny16x2 : kSkinny16x4;
  }
  if ((ceil_div(p.rows, 32) + p.groups) * ceil_div(p.n_out, 16) <= kCus) return kSkinny32x8;
  if (!experts && p.rows <= 32) return kSkinny32x4;
  // 256 x 256 tiles go over the chip in rounds of 256 and take 1.6 times as long as 128 x 128 ones, which go in rounds of 512
  const int64_t t256 = tiles(256, 256), t128 = tiles(128, 128), t64 = tiles(64, 128);
  if (per_group >= 256 && t256 >= kCus && 8 * ceil_div(t256, kCus) <= 5 * ceil_div(t128, 2 * kCus)) return kTile256x256;
  if (p.n_out > 64 && t64 > kCus && t64 <= 3 * kCus) return kTile64x128;     // three of them to a CU: one round
  if ((experts || p.rows >= 96) && t128 >= kCus) return kTile128x128;
  return kTile64x64;
}

Form choose_form(const ProductSize& p) {
  if (raw_form(p.rows, p.k)) return choose_raw(p);
  return p.groups == 0 && rows_form(p.rows, p.k, p.n_out) ? choose_rows(p) : choose_quantised(p);
}

int launch_quantised(ProductArgs a, Form form, int64_t grid, hipStream_t stream) {
  a.out_wide = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.n_out * dtype_size(a.out_dtype) % 16 == 0;
  switch (form) {
    case kSkinny16x2: return launch_skinny<kSkinny16x2, 1, 2>(a, grid, stream);
    case kSkinny16x4: return launch_skinny<kSkinny16x4, 1, 4>(a, grid, stream);
    case kSkinny32x4: return launch_skinny<kSkinny32x4, 2, 4>(a, grid, stream);
    case kSkinny32x8: return launch_skinny<kSkinny32x8, 2, 8>(a, grid, stream);
    case kTile32x128: return launch_tile<kTile32x128, 1, 4, 1, 1, 3>(a, grid, stream);
    case kTile64x128: return launch_tile<kTile64x128, 2, 2, 1, 2, 2>(a, grid, stream);
    case kTile64x64: return launch_tile<kTile64x64, 2, 2, 1, 1, 4>(a, grid, stream);
    case kTile128x128: return launch_tile<kTile128x128, 2, 4, 2, 1, 2>(a, grid, stream);
    default: return launch_tile<kTile256x256, 2, 4, 4, 2, 2>(a, grid, stream);
  }
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
  ProductArgs a = {};
  a.x = x;
  a.slot = slot;
  a.k = k;
  a.top_k = top_k;
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
  const ProductSize size = {rows, k, n_out, offsets ? groups : 0};
  const Form form = choose_form(size);
  GUNET_REQUIRE(form_fits(form, size), "%s: %lld rows x %d columns are more than one launch holds", fn, static_cast<long long>(rows), n_out);
  const int64_t grid = form_grid(form, size);
  const int64_t codes = align256(code_bytes(rows, k)), need = form <= kRaw16 && offsets == nullptr ? 0 : codes + scale_bytes(rows, k);
  if (need > 0 && (workspace == nullptr || workspace_bytes < static_cast<size_t>(need))) {
    set_error("%s: workspace of %zu bytes, %lld are needed", fn, workspace ? workspace_bytes : size_t{0}, static_cast<long long>(need));
    return GUNET_ERR_WORKSPACE;
  }
  GUNET_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: workspace is not 16-byte aligned", fn);
  if (form <= kRows32) {
    if (dtype == GUNET_DTYPE_F32) return launch_unquantised<float>(a, form, grid, stream);
    if (dtype == GUNET_DTYPE_BF16) return launch_unquantised<__bf16>(a, form, grid, stream);
    return launch_unquantised<_Float16>(a, form, grid, stream);
  }
  uint8_t* const x_codes = static_cast<uint8_t*>(workspace);
  GUNET_TRY(launch_quantize(x, dtype, 1, x_rows, rows, k, top_k, slot, x_codes, x_codes + codes, stream));
  a.x_codes = x_codes;
  a.x_scales = x_codes + codes;
  return launch_quantised(a, form, grid, stream);
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
  const dim3 grid(stride_grid(rows * blocks * (dtype == GUNET_DTYPE_F32 ? 8 : 4)), static_cast<unsigned>(groups));
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
  if (check_matrix("mxfp4_dense_workspace_bytes", 1, rows, k) != GUNET_OK || raw_form(rows, k)) return 0;
  return static_cast<size_t>(align256(code_bytes(rows, k)) + scale_bytes(rows, k));
}

size_t gunet_mxfp4_expert_dense_workspace_bytes(int64_t rows, int32_t k) {
  if (check_matrix("mxfp4_expert_dense_workspace_bytes", 1, rows, k) != GUNET_OK) return 0;
  return static_cast<size_t>(align256(code_bytes(rows, k)) + scale_bytes(rows, k));
}

const char* gunet_mxfp4_form(int64_t rows, int32_t k, int32_t n_out, int32_t n_experts) {
  if (check_matrix("mxfp4_form", n_experts, rows, k) != GUNET_OK || rows == 0 || n_out < 1) return "";
  const ProductSize size = {rows, k, n_out, n_experts};
  const Form form = choose_form(size);
  return form_fits(form, size) ? kForms[form].name : "";
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
