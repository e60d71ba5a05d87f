// Layer norm with the residual's addition, of x as it is or with elements dropped:
//   s = m x + r,  h = (s - mean s) rstd,  y = h w + b,  rstd = (mean (s - mean s)^2 + eps)^-1/2;
//   dr = ds + rstd (a - mean a - h mean(a h)) with a = dy w,  dx = m dr,
//   dw = sum_rows dy h,  db = sum_rows dy
// (m: dropout.hpp, made again in the backward pass).  A row stays in registers from its one
// read to its write, so the mean is subtracted before the squares are summed: no
// cancellation, whatever the mean.  The backward pass reads s as the forward call returned
// it, or, where that was rounded (bf16), x and r again: s rounded made dw 2.4e-3 off, for narrow rows 3e-3,
// where a rounding is 1.7e-3.  Bound by memory, both passes: 206848 x 512, bf16, with
// dropout: 157 to 172 us (4.9 to 5.4 TB/s over four tensor passes), the gradients 237 us (5.4 TB/s over
// six; 197 with s rounded) and 5 us for the weights' sums; 20705 x 1001, fp32: 57 to 63 us.
#pragma once
#include "dropout.hpp"
#include "rms_norm.hpp"

namespace tmpc {

template <typename E>
struct LayerNormArgs {
  int64_t rows;
  int width;
  const E *x, *r, *w, *b;  // r, b NULL: zero
  int64_t ldx, ldr;
  float eps;
  DropKey drop;
  E *y, *s;
  float* stats;  // (rows, 2): mean, rstd; NULL: not wanted
};

template <typename E>
struct LayerNormBwdArgs {
  int64_t rows;
  int width;
  const E *dy, *ds, *s, *w;  // ds NULL: zero; s NULL: x and r are read
  int64_t lddy, ldds, lds_;
  const E *x, *r;  // r NULL: zero
  int64_t ldx, ldr;
  const float* stats;
  DropKey drop;
  E *dx, *dr;   // dr NULL: not wanted
  float* part;  // (gridDim.x, 2, width) partial sums of dw and db
};

// NP pieces of 16 bytes a thread, TPR threads a row, 256 / TPR rows a block.
template <typename E, int TPR, int NP>
__global__ __launch_bounds__(256) void layer_norm_forward_kernel(LayerNormArgs<E> a) {
  constexpr int P = Elem<E>::PIECE, RPB = 256 / TPR;
  __shared__ float red[4];
  const int lane = threadIdx.x % TPR;
  const Philox rng(a.drop);
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows; row0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = row0 + threadIdx.x / TPR;
    const bool live = row < a.rows;
    float v[NP][P], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (i * TPR + lane) * P;
      const piece_t<E> px = load_piece(a.x + row * a.ldx, c, a.width, live);
#pragma unroll
      for (int e = 0; e < P; ++e) v[i][e] = (float)px[e];
      if (a.drop.key) drop_piece(drop_mask<P>(rng, a.drop, (uint32_t)row, c), a.drop, v[i]);
      if (a.r) {
        const piece_t<E> pr = load_piece(a.r + row * a.ldr, c, a.width, live);
#pragma unroll
        for (int e = 0; e < P; ++e) v[i][e] += (float)pr[e];
      }
#pragma unroll
      for (int e = 0; e < P; ++e) sum += v[i][e];
    }
    const float mean = row_sum<TPR>(sum, red) / (float)a.width;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float d = (i * TPR + lane) * P + e < a.width ? v[i][e] - mean : 0.0f;
        ss += d * d;
      }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(ss, red) / (float)a.width + a.eps);
    if (!live) continue;
    if (a.stats && lane == 0) a.stats[2 * row] = mean, a.stats[2 * row + 1] = rstd;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (i * TPR + lane) * P;
      if (c >= a.width) continue;
      const piece_t<E> pw = load_piece(a.w, c, a.width, true);
      piece_t<E> pb, py, ps;
      if (a.b) pb = load_piece(a.b, c, a.width, true);
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float h = (v[i][e] - mean) * rstd;
        py[e] = (E)(a.b ? h * (float)pw[e] + (float)pb[e] : h * (float)pw[e]), ps[e] = (E)v[i][e];
      }
      store_piece(a.y + row * a.width, c, a.width, py);
      store_piece(a.s + row * a.width, c, a.width, ps);
    }
  }
}

template <typename E, int TPR, int NP>
__global__ __launch_bounds__(256) void layer_norm_backward_kernel(LayerNormBwdArgs<E> a) {
  constexpr int P = Elem<E>::PIECE, RPB = 256 / TPR, ROW = TPR * NP * P;
  __shared__ float red[4];
  __shared__ float sums[RPB > 1 ? RPB * ROW : 1];
  const int lane = threadIdx.x % TPR;
  const Philox rng(a.drop);
  float w[NP][P], dw[NP][P], db[NP][P];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const piece_t<E> pw = load_piece(a.w, (i * TPR + lane) * P, a.width, true);
#pragma unroll
    for (int e = 0; e < P; ++e) w[i][e] = (float)pw[e], dw[i][e] = db[i][e] = 0.0f;
  }
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows; row0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = row0 + threadIdx.x / TPR;
    const bool live = row < a.rows;
    const float mean = live ? a.stats[2 * row] : 0.0f, rstd = live ? a.stats[2 * row + 1] : 0.0f;
    float h[NP][P], g[NP][P], sa = 0.0f, sah = 0.0f;
    uint32_t kept[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (i * TPR + lane) * P;
      const piece_t<E> ps = a.s ? load_piece(a.s + row * a.lds_, c, a.width, live) : load_piece(a.x + row * a.ldx, c, a.width, live);
      const piece_t<E> pg = load_piece(a.dy + row * a.lddy, c, a.width, live);
      float s[P];
#pragma unroll
      for (int e = 0; e < P; ++e) s[e] = (float)ps[e];
      if (a.drop.key) kept[i] = drop_mask<P>(rng, a.drop, (uint32_t)row, c);
      if (!a.s) {
        if (a.drop.key) drop_piece(kept[i], a.drop, s);
        if (a.r) {
          const piece_t<E> pr = load_piece(a.r + row * a.ldr, c, a.width, live);
#pragma unroll
          for (int e = 0; e < P; ++e) s[e] += (float)pr[e];
        }
      }
#pragma unroll
      for (int e = 0; e < P; ++e) {
        h[i][e] = (s[e] - mean) * rstd, g[i][e] = (float)pg[e];  // g is zero past the row's end
        dw[i][e] += g[i][e] * h[i][e], db[i][e] += g[i][e];
        g[i][e] *= w[i][e];
        sa += g[i][e], sah += g[i][e] * h[i][e];
      }
    }
    sa = row_sum<TPR>(sa, red) / (float)a.width;
    sah = row_sum<TPR>(sah, red) / (float)a.width;
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (i * TPR + lane) * P;
      if (c >= a.width) continue;
      piece_t<E> pd, px;
      if (a.ds) pd = load_piece(a.ds + row * a.ldds, c, a.width, true);
      float d[P];
#pragma unroll
      for (int e = 0; e < P; ++e) {
        d[e] = rstd * (g[i][e] - sa - h[i][e] * sah);
        if (a.ds) d[e] += (float)pd[e];
        px[e] = (E)d[e];
      }
      if (a.dr) store_piece(a.dr + row * a.width, c, a.width, px);
      if (a.drop.key) {
        drop_piece(kept[i], a.drop, d);
#pragma unroll
        for (int e = 0; e < P; ++e) px[e] = (E)d[e];
      }
      store_piece(a.dx + row * a.width, c, a.width, px);
    }
  }
  // the block's rows meet in a fixed order
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.width;
  if constexpr (RPB > 1) {
    const int r = threadIdx.x / TPR;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k) __syncthreads();
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int e = 0; e < P; ++e) sums[r * ROW + (i * TPR + lane) * P + e] = k ? db[i][e] : dw[i][e];
      __syncthreads();
      for (int c = threadIdx.x; c < a.width; c += 256) {
        float t = 0.0f;
        for (int j = 0; j < RPB; ++j) t += sums[j * ROW + c];
        part[k * a.width + c] = t;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const int c = (i * TPR + lane) * P + e;
        if (c < a.width) part[c] = dw[i][e], part[a.width + c] = db[i][e];
      }
  }
}

// dw and db: the sums over the blocks' partial sums, in order; 16 columns of the 2 width a block,
// 16 threads a column.  db NULL: not wanted.
template <typename E>
__global__ __launch_bounds__(256) void layer_norm_dweight_kernel(const float* __restrict__ part, int nblocks, int width,
                                                                 E* __restrict__ dw, E* __restrict__ db) {
  __shared__ float t[16][17];
  const int c = blockIdx.x * 16 + threadIdx.x % 16, k = threadIdx.x / 16;
  float v = 0.0f;
  if (c < 2 * width) {
    int b = k;
    for (; b + 7 * 16 < nblocks; b += 8 * 16) {  // eight reads on their way at a time
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = part[(int64_t)(b + i * 16) * 2 * width + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) v += x[i];
    }
    for (; b < nblocks; b += 16) v += part[(int64_t)b * 2 * width + c];
  }
  t[k][threadIdx.x % 16] = v;
  __syncthreads();
  if (k == 0 && c < 2 * width) {
    float s = 0.0f;
    for (int i = 0; i < 16; ++i) s += t[i][threadIdx.x];
    if (c < width) dw[c] = (E)s;
    else if (db) db[c - width] = (E)s;
  }
}

}  // namespace tmpc
