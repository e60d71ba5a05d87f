// Root-mean-square norm with the residual's addition, forward and backward:
//   s = x + r,  y = s rstd w,  rstd = (mean s^2 + eps)^-1/2;
//   dx = dr = ds + rstd (a - s rstd^2 mean(a s)) with a = dy w,  dw = sum_rows dy s rstd.
// The backward pass reads s as the forward call returned it, in bf16 rounded once: dw is 2.3e-3 off
// where 1.5e-3 is one rounding (dx 1.7e-3); x and r read again instead are a fifth pass to its four.
// Bound by memory: each row is read once and kept in registers between the sum of
// its squares and the write.  206848 rows of 512, bf16: forward 141 us (6.0 TB/s), backward
// 165 us and 21 us for the weight's partial sums (5.2 TB/s over both directions).
#pragma once
#include "learn_common.hpp"

namespace tmpc {

template <typename E>
struct RmsArgs {
  int64_t rows;
  int width;
  const E *x, *r, *w;  // r NULL: no residual
  int64_t ldx, ldr;
  float eps;
  E *y, *s;     // s NULL: not wanted
  float* rstd;  // NULL: not wanted
};

template <typename E>
struct RmsBwdArgs {
  int64_t rows;
  int width;
  const E *dy, *ds, *s, *w;  // ds NULL: zero
  int64_t lddy, ldds, lds_;  // row pitches of dy, ds, s
  const float* rstd;
  E* dx;
  float* part;  // (gridDim.x, width) partial sums of dw
};

// Sum over the TPR threads of a row (TPR a power of two up to 64: within a wave;
// else across the block's waves through LDS).
template <int TPR>
__device__ inline float row_sum(float v, float* red) {
  constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int d = W / 2; d; d >>= 1) v += __shfl_xor(v, d, 64);
  if constexpr (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // the previous row's values have been read
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += red[i];
  }
  return v;
}

// NP pieces of 16 bytes a thread, TPR threads a row, 256 / TPR rows a block.
template <typename E, int TPR, int NP>
__global__ __launch_bounds__(256) void rms_forward_kernel(RmsArgs<E> a) {
  constexpr int P = Elem<E>::PIECE, RPB = 256 / TPR;
  __shared__ float red[4];
  const int lane = threadIdx.x % TPR;
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows; row0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = row0 + threadIdx.x / TPR;
    const bool live = row < a.rows;
    float v[NP][P], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (i * TPR + lane) * P;
      const piece_t<E> px = load_piece(a.x + row * a.ldx, c, a.width, live);
#pragma unroll
      for (int e = 0; e < P; ++e) v[i][e] = (float)px[e];
      if (a.r) {
        const piece_t<E> pr = load_piece(a.r + row * a.ldr, c, a.width, live);
#pragma unroll
        for (int e = 0; e < P; ++e) v[i][e] += (float)pr[e];
      }
#pragma unroll
      for (int e = 0; e < P; ++e) ss += v[i][e] * v[i][e];
    }
    ss = row_sum<TPR>(ss, red);
    const float rstd = 1.0f / sqrtf(ss / (float)a.width + a.eps);
    if (!live) continue;
    if (a.rstd && lane == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (i * TPR + lane) * P;
      if (c >= a.width) continue;
      const piece_t<E> pw = load_piece(a.w, c, a.width, true);
      piece_t<E> py, ps;
#pragma unroll
      for (int e = 0; e < P; ++e) py[e] = (E)(v[i][e] * rstd * (float)pw[e]), ps[e] = (E)v[i][e];
      store_piece(a.y + row * a.width, c, a.width, py);
      if (a.s) store_piece(a.s + row * a.width, c, a.width, ps);
    }
  }
}

template <typename E, int TPR, int NP>
__global__ __launch_bounds__(256) void rms_backward_kernel(RmsBwdArgs<E> a) {
  constexpr int P = Elem<E>::PIECE, RPB = 256 / TPR;
  __shared__ float red[4];
  __shared__ float dws[RPB > 1 ? RPB * TPR * NP * P : 1];
  const int lane = threadIdx.x % TPR;
  float w[NP][P], dw[NP][P];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const piece_t<E> pw = load_piece(a.w, (i * TPR + lane) * P, a.width, true);
#pragma unroll
    for (int e = 0; e < P; ++e) w[i][e] = (float)pw[e], dw[i][e] = 0.0f;
  }
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows; row0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = row0 + threadIdx.x / TPR;
    const bool live = row < a.rows;
    const float rstd = live ? a.rstd[row] : 0.0f;
    float s[NP][P], g[NP][P], as = 0.0f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (i * TPR + lane) * P;
      const piece_t<E> ps = load_piece(a.s + row * a.lds_, c, a.width, live);
      const piece_t<E> pg = load_piece(a.dy + row * a.lddy, c, a.width, live);
#pragma unroll
      for (int e = 0; e < P; ++e) {
        s[i][e] = (float)ps[e] * rstd, g[i][e] = (float)pg[e];
        dw[i][e] += g[i][e] * s[i][e];
        g[i][e] *= w[i][e];
        as += g[i][e] * s[i][e];
      }
    }
    as = row_sum<TPR>(as, red) / (float)a.width;
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (i * TPR + lane) * P;
      if (c >= a.width) continue;
      piece_t<E> pd, px;
      if (a.ds) pd = load_piece(a.ds + row * a.ldds, c, a.width, true);
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float d = rstd * (g[i][e] - s[i][e] * as);
        px[e] = (E)(a.ds ? d + (float)pd[e] : d);
      }
      store_piece(a.dx + row * a.width, c, a.width, px);
    }
  }
  // the block's rows meet in a fixed order
  if constexpr (RPB > 1) {
    const int r = threadIdx.x / TPR;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int e = 0; e < P; ++e) dws[r * TPR * NP * P + (i * TPR + lane) * P + e] = dw[i][e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.width; c += 256) {
      float t = 0.0f;
      for (int k = 0; k < RPB; ++k) t += dws[k * TPR * NP * P + c];
      a.part[(int64_t)blockIdx.x * a.width + c] = t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const int c = (i * TPR + lane) * P + e;
        if (c < a.width) a.part[(int64_t)blockIdx.x * a.width + c] = dw[i][e];
      }
  }
}

// dw[c] = sum over the blocks' partial sums, in order: 16 columns a block, the
// blocks' sums over 16 threads of each column.
template <typename E>
__global__ __launch_bounds__(256) void rms_dweight_kernel(const float* __restrict__ part, int nblocks, int width,
                                                          E* __restrict__ dw) {
  __shared__ float t[16][17];
  const int c = blockIdx.x * 16 + threadIdx.x % 16, k = threadIdx.x / 16;
  float v = 0.0f;
  if (c < width)
    for (int b = k; b < nblocks; b += 16) v += part[(int64_t)b * width + c];
  t[k][threadIdx.x % 16] = v;
  __syncthreads();
  if (k == 0 && c < width) {
    float s = 0.0f;
    for (int i = 0; i < 16; ++i) s += t[i][threadIdx.x];
    dw[c] = (E)s;
  }
}

}  // namespace tmpc
