// seqcommon.h -- what the sequence operators over packs share: element types, vector loads, the
// 32x32 matrix-core tiles and the pack arrays.
//
// Pack arrays of one boundary mask (kl_pack_layout): ids[i] = the pack of row i (-1 before the first
// pack), starts[p] = the first row of pack p, and starts[p] = num_rows for every p past the last pack
// up to starts[num_rows]: rows [starts[p], starts[p+1]) are pack p, also where p does not exist (none).
#pragma once

#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace kl {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// the vectors of one element type: V8 is a matrix-core operand fragment, V4 four neighbours
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  typedef f32x4 V4;
  typedef f32x8 V8;
};
template <>
struct Vec<f16_t> {
  typedef f16x4 V4;
  typedef f16x8 V8;
};
template <>
struct Vec<bf16_t> {
  typedef bf16x4 V4;
  typedef bf16x8 V8;
};
template <typename T>
using V4 = typename Vec<T>::V4;
template <typename T>
using V8 = typename Vec<T>::V8;

// acc (32 x 32) += A (32 x 16) * B (16 x 32).  Lane l holds A[l % 32][8 * (l / 32) + e] and
// B[8 * (l / 32) + e][l % 32], e = 0..7, and of acc the column l % 32 at the rows
// 8 * (r / 4) + 4 * (l / 32) + r % 4, r = 0..15.  The sum over the 16 inner indices does not depend
// on their order, so any permutation of them is right where A and B use the same one.
// float has no 16-deep product: eight 2-deep ones, step e taking the inner indices e and 8 + e.
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 acc) {
#pragma unroll
  for (int e = 0; e < 8; e++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
  return acc;
}

// the row of accumulator register r in lane half h, and the inner index that a fragment made of the
// eight accumulator registers 8 * s .. 8 * s + 7 holds at element e: the same permutation
__device__ __forceinline__ constexpr int acc_row(int r, int h) { return 8 * (r / 4) + 4 * h + r % 4; }

// An accumulator half (registers 8 * s .. 8 * s + 7) as an operand: rows 16 * s .. 16 * s + 15 of acc
// become the 16 inner indices, in the order of acc_row, with no exchange between lanes.
template <typename T>
__device__ __forceinline__ V8<T> acc_frag(const f32x16 &acc, int s) {
  f32x8 v;
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = acc[8 * s + e];
  return __builtin_convertvector(v, V8<T>);
}

// A tile of rows of DP elements in LDS, laid out so that both ways of reading it spread over the 64 banks.  A
// row fragment reads one 16-byte piece of 32 rows (16 rows at a time: 16 different places of the 256 bytes), a
// column fragment of a 16-bit type four neighbouring pieces of four rows (again 16 places): piece p of row r lies
// at place p ^ swizzle(r).  float: rows are a piece longer than DP; its column fragments read 32 neighbouring
// words of two rows, two places in conflict at most, and its products are too slow for that to matter.
template <typename T, int DP>
struct Tile {
  static constexpr int E = 16 / (int)sizeof(T);  // elements per piece
  static constexpr int LD = sizeof(T) == 4 ? DP + E : DP;
  __device__ static __forceinline__ int swizzle(int r) {
    if constexpr (sizeof(T) == 4) return 0;
    if constexpr (DP == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
    if constexpr (DP == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    return (r >> 2) & 3;
  }
  // the place of piece p of row r
  __device__ static __forceinline__ int piece(int r, int p) { return r * LD + (p ^ swizzle(r)) * E; }
  __device__ static __forceinline__ int at(int r, int c) { return piece(r, c / E) + c % E; }

  // Row fragment: element e = tile[row][col + e].
  __device__ static __forceinline__ V8<T> row_frag(const T *tile, int row, int col) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 a = *reinterpret_cast<const f32x4 *>(tile + piece(row, col / 4));
      const f32x4 b = *reinterpret_cast<const f32x4 *>(tile + piece(row, col / 4 + 1));
      return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    } else {
      return *reinterpret_cast<const V8<T> *>(tile + piece(row, col / 8));
    }
  }

  // Column fragment: element e = tile[row0 + acc_row(e, h)][col0 + l % 32], the A operand of the transposed
  // tile whose inner indices are in the order of acc_frag.  16-bit types: the transposed LDS read gives lane
  // i of 16 the column i of a 4 x 16 block whose rows four lanes each address, which is just the run of four
  // rows that acc_row holds together.
  __device__ static __forceinline__ V8<T> col_frag(T *tile, int row0, int col0) {
    const int l = threadIdx.x & 63, h = l >> 5;
    if constexpr (sizeof(T) == 4) {
      f32x8 v;
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = tile[at(row0 + acc_row(e, h), col0 + (l & 31))];
      return v;
    } else {
      const int i = l & 15, r = row0 + 4 * h + i / 4, c = col0 + (l & 16) + (i & 3) * 4;
      typedef __attribute__((address_space(3))) i16x4 lds4;
      union {
        i16x4 u[2];
        V8<T> v;
      } x;
      x.u[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(tile + at(r, c)));
      x.u[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(tile + at(r + 8, c)));
      return x.v;
    }
  }
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

// sum and maximum over the two halves that hold a column: lanes l and l ^ 32
__device__ __forceinline__ float half_sum(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}
__device__ __forceinline__ float half_max(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}

// Strided heads: element (row, head, i) of a (rows, heads, dim) tensor lies at row * row_stride +
// head * head_stride + i.
struct Heads {
  int64_t row, head;
};
// (rows, heads, dim) whose rows of a head all start at multiples of 16 bytes
inline bool whole_pieces(const void *p, int64_t rows, int64_t heads, Heads st, size_t esize) {
  return rows == 0 || heads == 0 ||
         ((uintptr_t)p % 16 == 0 && (rows == 1 || st.row * esize % 16 == 0) && (heads == 1 || st.head * esize % 16 == 0));
}

// any element of a 16-byte piece that is an infinity or a NaN
template <typename T>
__device__ __forceinline__ bool piece_bad(u32x4 w) {
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      bad |= (w[i] & 0x7f800000u) == 0x7f800000u;
    } else {
      constexpr uint32_t m = std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;
      bad |= (w[i] & m) == m;
      bad |= (w[i] & (m << 16)) == (m << 16);
    }
  }
  return bad != 0;
}

// What is the same in every lane, as such: loops and addresses made of it stay in scalar registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// f(T()) for the element type of a tensor
template <typename F>
inline int with_type(kl_dtype dtype, const char *func, F f) {
  switch (dtype) {
    case KL_F32: return f(float());
    case KL_F16: return f(f16_t());
    case KL_BF16: return f(bf16_t());
    default: set_error(std::string(func) + ": expected a Half, BFloat16 or Float tensor"); return KL_E_INVALID;
  }
}

}  // namespace kl
