// Host helpers of the history model's C entry points.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/tmpc.h"
#include "learn_common.hpp"

namespace tmpc {

constexpr int kCUs = 256;

inline size_t align_up(size_t n) { return (n + 255) & ~size_t(255); }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline int launch_status() { return hipGetLastError() == hipSuccess ? TMPC_OK : TMPC_ELAUNCH; }

// Dynamic LDS above the 64 KiB default needs an explicit opt-in per kernel.
template <typename K>
void lds_optin(K kernel, size_t bytes) {
  if (bytes > 65536)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)bytes);
}

// The norms' rows
constexpr int kMaxWidth = 8192;

// f(threads per row, pieces per thread) of the smallest form that holds `width`
template <typename E, typename F>
void with_row(int width, F f) {
  const int pieces = (width + Elem<E>::PIECE - 1) / Elem<E>::PIECE;
  using std::integral_constant;
  if (pieces <= 16) f(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (pieces <= 64) f(integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (pieces <= 128) f(integral_constant<int, 64>(), integral_constant<int, 2>());
  else if (pieces <= 256) f(integral_constant<int, 256>(), integral_constant<int, 1>());
  else if (pieces <= 512) f(integral_constant<int, 256>(), integral_constant<int, 2>());
  else if (pieces <= 1024) f(integral_constant<int, 256>(), integral_constant<int, 4>());
  else f(integral_constant<int, 256>(), integral_constant<int, 8>());
}
// rows that a block of 256 threads has at a time
inline int64_t rows_per_block(int width, int elem_bytes) {
  const int pieces = (width * elem_bytes + 15) / 16;
  return pieces <= 16 ? 16 : pieces <= 128 ? 4 : 1;
}
inline bool norm_shape_ok(int64_t rows, int width) { return rows >= 0 && width >= 1 && width <= kMaxWidth; }

}  // namespace tmpc
