// What the history model's kernels (learning.hip) share: the element types and the
// matrix-instruction operands ("quads").
//
// Operand convention of the 16x16 matrix instructions here: lane l holds index
// l % 16 of the operand's outer dimension and 4 consecutive entries of the
// contracted one from 4 * (l / 16): a quad.  The accumulator of lane l is column
// l % 16, rows 4 * (l / 16) + 0..3, which is a quad of its transpose, so the result
// of one product is an operand of the next without leaving its registers.  bf16
// joins two quads (32 contracted entries, the order inside the sum being free)
// into one 16x16x32 instruction; fp32 issues a 16x16x4 instruction per entry.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tmpc {

typedef __bf16 bf16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 16 bytes of a row, as global memory and LDS move them
template <typename E>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int PIECE = 4;  // elements of 16 bytes
  typedef f32x4 quad;
  typedef f32x4 piece;
  typedef float piece_u __attribute__((ext_vector_type(4), aligned(4)));  // at any element
};
template <>
struct Elem<bf16> {
  static constexpr int PIECE = 8;
  typedef bf16x4 quad;
  typedef bf16x8 piece;
  typedef __bf16 piece_u __attribute__((ext_vector_type(8), aligned(2)));
};
template <typename E>
using quad_t = typename Elem<E>::quad;
template <typename E>
using piece_t = typename Elem<E>::piece;

// elements c .. c + PIECE - 1 of a row of `width` elements, zeros past its end;
// `live` false: zeros without a read
template <typename E>
__device__ inline piece_t<E> load_piece(const E* row, int c, int width, bool live) {
  constexpr int P = Elem<E>::PIECE;
  piece_t<E> r;
  if (live && c + P <= width) {
    r = *reinterpret_cast<const typename Elem<E>::piece_u*>(row + c);
  } else {
#pragma unroll
    for (int e = 0; e < P; ++e) r[e] = (live && c + e < width) ? row[c + e] : E(0.0f);
  }
  return r;
}
template <typename E>
__device__ inline void store_piece(E* row, int c, int width, piece_t<E> v) {
  constexpr int P = Elem<E>::PIECE;
  if (c + P <= width) {
    *reinterpret_cast<typename Elem<E>::piece_u*>(row + c) = v;
  } else {
#pragma unroll
    for (int e = 0; e < P; ++e)
      if (c + e < width) row[c + e] = v[e];
  }
}
// 4 elements from column c on, the accumulator's shape
__device__ inline void store_quad(float* row, int c, int width, f32x4 v) {
  typedef float q_u __attribute__((ext_vector_type(4), aligned(4)));
  if (c + 4 <= width) {
    *reinterpret_cast<q_u*>(row + c) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < width) row[c + e] = v[e];
  }
}
__device__ inline bf16x4 to_bf16(f32x4 v) {
  bf16x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = (bf16)v[e];
  return r;
}
__device__ inline void store_quad(bf16* row, int c, int width, f32x4 v) {
  typedef __bf16 q_u __attribute__((ext_vector_type(4), aligned(2)));
  const bf16x4 b = to_bf16(v);
  if (c + 4 <= width) {
    *reinterpret_cast<q_u*>(row + c) = b;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < width) row[c + e] = b[e];
  }
}
__device__ inline f32x4 load_quad_f32(const float* row, int c, int width) {
  typedef float q_u __attribute__((ext_vector_type(4), aligned(4)));
  if (c + 4 <= width) return *reinterpret_cast<const q_u*>(row + c);
  f32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = c + e < width ? row[c + e] : 0.0f;
  return r;
}
// fp32 accumulator -> operand quad (rounds to nearest for bf16)
template <typename E>
__device__ inline quad_t<E> to_quad(f32x4 v);
template <>
__device__ inline f32x4 to_quad<float>(f32x4 v) {
  return v;
}
template <>
__device__ inline bf16x4 to_quad<bf16>(f32x4 v) {
  return to_bf16(v);
}
__device__ inline f32x4 to_f32(f32x4 v) { return v; }
__device__ inline f32x4 to_f32(bf16x4 v) {
  f32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = (float)v[e];
  return r;
}

// quad (row0 + l % 16, col0 + 4 (l / 16) ..) of a row-major LDS tile of pitch ld
template <typename E>
__device__ inline quad_t<E> lds_quad(const E* tile, int ld, int row0, int col0, int lane) {
  return *reinterpret_cast<const quad_t<E>*>(tile + (row0 + (lane & 15)) * ld + col0 + 4 * (lane >> 4));
}
// quad of the transpose: outer index col0 + l % 16, contracted rows row0 + 4 (l / 16) ..
__device__ inline f32x4 lds_quad_t(const float* tile, int ld, int row0, int col0, int lane) {
  const float* p = tile + (row0 + 4 * (lane >> 4)) * ld + col0 + (lane & 15);
  f32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = p[e * ld];
  return r;
}
// the LDS transpose read: of 16 lanes, lane 4 r + c gives the address of row r,
// columns 4 c .. 4 c + 3, and lane i receives column i of the 4 rows
__device__ inline bf16x4 lds_quad_t(const bf16* tile, int ld, int row0, int col0, int lane) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const bf16* p = tile + (row0 + 4 * (lane >> 4) + ((lane & 15) >> 2)) * ld + col0 + 4 * (lane & 3);
  return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}

// acc += A B over 32 contracted entries (two quads of each operand)
__device__ inline f32x4 mma2(bf16x4 a0, bf16x4 a1, bf16x4 b0, bf16x4 b1, f32x4 acc) {
  const bf16x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
  const bf16x8 b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
}
__device__ inline f32x4 mma2(f32x4 a0, f32x4 a1, f32x4 b0, f32x4 b1, f32x4 acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a0[e], b0[e], acc, 0, 0, 0);
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a1[e], b1[e], acc, 0, 0, 0);
  return acc;
}

}  // namespace tmpc
