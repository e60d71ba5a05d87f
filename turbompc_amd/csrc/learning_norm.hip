// C ABI of the layer norm and of dropout (include/tmpc.h): argument checks, workspace, launches.
#include <algorithm>
#include <cmath>

#include "layer_norm.hpp"
#include "learn_host.hpp"

namespace tmpc {
namespace {

constexpr int64_t kMaxDropRows = (int64_t(1) << 31) - 1;  // the counter's row word, signed in the indexes
constexpr int kMaxDropWidth = 1 << 24;

// p in 0 .. 1 so that something is kept; p 0: no key is read
bool drop_ok(double p, const int64_t* key) { return p >= 0.0 && nearbyint(p * 65536) < 65536 && (p == 0.0 || key); }
DropKey drop_key(double p, const int64_t* key, uint32_t call) {
  const uint32_t least = (uint32_t)nearbyint(p * 65536);
  return {p > 0.0 ? key : nullptr, call, least, 65536.0f / (float)(65536 - least)};
}

template <typename E>
int dropout_impl(hipStream_t st, int64_t rows, int32_t width, const void* x, int64_t ldx, double p, const int64_t* key,
                 uint32_t call, void* y) {
  if (rows < 0 || rows > kMaxDropRows || width < 1 || width > kMaxDropWidth) return TMPC_EBADSHAPE;
  if (rows == 0) return TMPC_OK;
  if (!x || !y || !key || ldx < 0 || !drop_ok(p, key)) return TMPC_EBADARG;
  const uint32_t pieces = (uint32_t)ceil_div(width, Elem<E>::PIECE);
  DropKey d = drop_key(p, key, call);
  d.key = key;
  const int64_t most = (int64_t(1) << 31) / pieces;  // rows of a launch, whose pieces have 32-bit indexes
  for (int64_t r0 = 0; r0 < rows; r0 += most) {
    const uint32_t n = (uint32_t)(std::min(most, rows - r0) * pieces);
    hipLaunchKernelGGL((dropout_kernel<E>), dim3((unsigned)std::min<int64_t>(ceil_div(n, 256), 1 << 20)), dim3(256), 0, st,
                       n, width, pieces, (uint32_t)r0, (const E*)x, ldx, d, (E*)y);
  }
  return launch_status();
}

// Blocks of the backward pass, whose rows meet in the blocks' partial sums (206848 x 512, bf16, reading s: 237
// to 267 us with 512, 197 with 1024, 209 with 2048, the sums' kernel 4, 5 and 10 us beside them).
constexpr int kNormBlocks = 1024;
int64_t backward_blocks(int64_t rows, int width, int elem_bytes) {
  return std::min<int64_t>(ceil_div(rows, rows_per_block(width, elem_bytes)), kNormBlocks);
}

bool args_ok(const tmpc_layer_norm* a) {
  return a && norm_shape_ok(a->rows, a->width) && (a->p == 0.0 || a->rows <= kMaxDropRows);
}

template <typename E>
int forward_impl(hipStream_t st, const tmpc_layer_norm* a, void* y, void* s, float* stats) {
  if (!args_ok(a)) return TMPC_EBADSHAPE;
  if (a->rows == 0) return TMPC_OK;
  if (!a->x || !a->weight || !y || !s || !(a->eps >= 0.0) || a->ldx < 0 || a->ldr < 0 || !drop_ok(a->p, a->key))
    return TMPC_EBADARG;
  const LayerNormArgs<E> k{a->rows, a->width, (const E*)a->x, (const E*)a->residual, (const E*)a->weight,
                           (const E*)a->bias, a->ldx, a->ldr, (float)a->eps, drop_key(a->p, a->key, a->call), (E*)y,
                           (E*)s, stats};
  with_row<E>(a->width, [&](auto tpr, auto np) {
    const int64_t blocks = ceil_div(a->rows, 256 / tpr());
    hipLaunchKernelGGL((layer_norm_forward_kernel<E, tpr(), np()>), dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)),
                       dim3(256), 0, st, k);
  });
  return launch_status();
}

template <typename E>
int backward_impl(hipStream_t st, const tmpc_layer_norm* a, const void* dy, int64_t lddy, const void* ds, int64_t ldds,
                  const void* s, int64_t lds, const float* stats, void* dx, void* dr, void* dw, void* db, void* ws,
                  size_t wsb) {
  if (!args_ok(a)) return TMPC_EBADSHAPE;
  if (!dw || (a->rows > 0 && (!dy || (!s && !a->x) || !a->weight || !stats || !dx)) || lddy < 0 || ldds < 0 ||
      lds < 0 || a->ldx < 0 || a->ldr < 0 ||
      !drop_ok(a->p, a->key))
    return TMPC_EBADARG;
  const int64_t blocks = backward_blocks(a->rows, a->width, sizeof(E));
  const size_t need = (size_t)blocks * 2 * a->width * sizeof(float);
  if (wsb < need) return TMPC_EWORKSPACE;
  if (need > 0 && !ws) return TMPC_EBADARG;
  float* part = (float*)ws;
  if (a->rows > 0) {
    const LayerNormBwdArgs<E> k{a->rows, a->width, (const E*)dy, (const E*)ds, (const E*)s, (const E*)a->weight, lddy,
                                ldds, lds, (const E*)a->x, (const E*)a->residual, a->ldx, a->ldr, stats,
                                drop_key(a->p, a->key, a->call), (E*)dx, (E*)dr, part};
    with_row<E>(a->width, [&](auto tpr, auto np) {
      hipLaunchKernelGGL((layer_norm_backward_kernel<E, tpr(), np()>), dim3((unsigned)blocks), dim3(256), 0, st, k);
    });
  }
  hipLaunchKernelGGL((layer_norm_dweight_kernel<E>), dim3((unsigned)ceil_div(2 * a->width, 16)), dim3(256), 0, st, part,
                     (int)blocks, a->width, (E*)dw, (E*)db);
  return launch_status();
}

}  // namespace
}  // namespace tmpc

using namespace tmpc;

extern "C" {

size_t tmpc_layer_norm_backward_workspace_bytes(int elem_bytes, int64_t rows, int32_t width) {
  if (!norm_shape_ok(rows, width) || (elem_bytes != 2 && elem_bytes != 4)) return 0;
  return align_up((size_t)backward_blocks(rows, width, elem_bytes) * 2 * width * sizeof(float));
}

#define TMPC_LEARNING_NORM(SFX, E)                                                                                     \
  int tmpc_dropout_##SFX(hipStream_t s, int64_t rows, int32_t width, const void* x, int64_t ldx, double p,             \
                         const int64_t* key, uint32_t call, void* y) {                                                 \
    return dropout_impl<E>(s, rows, width, x, ldx, p, key, call, y);                                                   \
  }                                                                                                                    \
  int tmpc_layer_norm_forward_##SFX(hipStream_t s, const tmpc_layer_norm* a, void* y, void* sum, float* stats) {       \
    return forward_impl<E>(s, a, y, sum, stats);                                                                       \
  }                                                                                                                    \
  int tmpc_layer_norm_backward_##SFX(hipStream_t s, const tmpc_layer_norm* a, const void* dy, int64_t lddy,            \
                                     const void* ds, int64_t ldds, const void* sum, int64_t lds, const float* stats,   \
                                     void* dx, void* dresidual, void* dweight, void* dbias, void* ws, size_t wsb) {    \
    return backward_impl<E>(s, a, dy, lddy, ds, ldds, sum, lds, stats, dx, dresidual, dweight, dbias, ws, wsb);        \
  }
TMPC_LEARNING_NORM(f32, float)
TMPC_LEARNING_NORM(bf16, bf16)

}  // extern "C"
