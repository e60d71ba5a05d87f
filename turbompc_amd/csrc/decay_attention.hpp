// Linear attention with a decay for each head.  Problem b, head h, g = log_decay[h]:
//   S_t = e^g S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t        (S fp32, DK x DV).
//
// Chunked form.  Over C steps from the state S_in,
//   O = (Q K^T o Gamma) V + diag(e^{g (i+1)}) Q S_in,  Gamma_ij = e^{g (i-j)} for i >= j, else 0
//   S_out = e^{g L} S_in + K^T diag(e^{g (L-1-j)}) V,  L the chunk's live steps;
// every exponent's factor of g is >= 0, so a strong decay underflows to zero and
// nothing overflows.
//
// Backward.  With D_t = dL/dS_t = e^g D_{t+1} + scale q_t^T do_t,
//   dq_t = scale do_t S_t^T,  dk_t = v_t D_t^T,  dv_t = k_t D_t :
// dq is the same recurrence with (q, k, v) := (do, v, k) from the transposed state;
// dk and dv are the recurrence run backwards in time with (v, do, q) and (k, q, do).
// Backwards the carried matrix is X = e^g D (what the next earlier step starts
// from), which begins as the final state's gradient and ends as the initial
// state's; its powers are i for the rows and L - j in the update.
#pragma once
#include "learn_common.hpp"

namespace tmpc {

// One recurrence: a (query-like), b (key-like), c (value-like).
template <typename E>
struct AttnArgs {
  int B, T, H;
  int da, dc;                // widths of a and b, and of c and the output
  int ga, gb, gc;            // heads that share one of a's (b's, c's) heads
  const E *a, *b, *c;
  int64_t as[3], bs[3], cs[3];  // strides of problem, step, head
  const float* log_decay;    // (H)
  const int32_t* lengths;    // (B) or NULL
  float ss, si, su;          // factors of the scores, of the carried state's part and of the update
  int rev;                   // 1: from the last live step to the first
  const float* s_in;         // (B, H, da, dc), or (B, H, dc, da) with s_in_t; NULL: zero
  int s_in_t;
  float* s_out;              // (B, H, da, dc) or NULL
  void* o;                   // (B, T, H, dc): E, or fp32 with o_f32
  int o_f32;
  int segs, seg_len;         // the steps in segs runs of seg_len (a multiple of the chunk)
  float* seg_state;          // segs > 1: (B, H, segs, da, dc): each run's own sum, then its start
};

// live steps of problem b
template <typename E>
__device__ inline int attn_length(const AttnArgs<E>& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
}

template <typename E>
struct AttnTile {
  static constexpr int C = sizeof(E) == 2 ? 64 : 32;  // steps of a chunk
  static constexpr int PAD = 16 / sizeof(E);          // of an LDS row: its quads spread over the banks
};

__device__ inline float decay_pow(float g, int n) { return n == 0 ? 1.0f : __expf(g * (float)n); }

// A workgroup carries one (problem, head) through its chunks.  Wave w owns NV
// 16-column tiles of the values: S and O need no exchange between waves, only the
// chunk's scores do (LDS).  S stays in registers, in the accumulator's layout, which
// is the operand layout of the product with Q.
template <typename E, int DA, int DC>
struct AttnShape {
  static constexpr int W = DC / 16 < 4 ? DC / 16 : 4;  // waves
  static constexpr int NV = DC / 16 / W;               // value tiles of a wave
  static constexpr int THREADS = 64 * W;
  static constexpr int C = AttnTile<E>::C;
  static constexpr int LDA = DA + AttnTile<E>::PAD, LDC = DC + AttnTile<E>::PAD, LDP = C + AttnTile<E>::PAD;
  static constexpr size_t LDS_STATE = sizeof(E) * (size_t)(C * LDA + C * LDC);
  static constexpr size_t LDS = LDS_STATE + sizeof(E) * (size_t)(C * LDA + C * LDP);
};

// A chunk's rows of one operand on their way from memory through registers to LDS: the
// next chunk's are in flight while this one's are multiplied.  A thread moves N pieces
// of one column, RS rows apart.
template <typename E, int C, int D, int THREADS>
struct AttnRows {
  static constexpr int P = Elem<E>::PIECE, W = D / P, RS = THREADS / W, N = C / RS, LD = D + AttnTile<E>::PAD;
  static_assert(THREADS % W == 0 && C % RS == 0, "whole rows a pass");
  piece_t<E> r[N];
  const E* at;      // this thread's first piece of the next chunk
  int64_t step;     // elements between steps
  int row, c;

  __device__ void init(const E* base, int64_t stride, int t0, int tid) {
    row = tid / W, c = (tid - row * W) * P, step = stride;
    at = base + (t0 + row) * stride + c;
  }
  // the next chunk's rows, n of them live
  __device__ void load(int n, int width) {
    if (n >= C && width == D) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = *reinterpret_cast<const typename Elem<E>::piece_u*>(at + i * RS * step);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = load_piece(at + i * RS * step - c, c, width, row + i * RS < n);
    }
    at += C * step;
  }
  __device__ void store(E* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<piece_t<E>*>(tile + (row + i * RS) * LD + c) = r[i];
  }
};

__device__ inline float uniform(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}

// Powers of a head's decay that every whole chunk needs, of exponents >= 0 alone:
// lag 16 d + lo - 4 hi - r of a score as tile[d] * near[r] (d >= 1; near has 16 more and tile
// 16 fewer), diag[r] on the diagonal tile (0 above it), row i = 16 it + lo of the
// carried state's part as tile[it] * rowf, step j = 16 jt + 4 hi + r of the update as
// tile[CT - 1 - jt] * tail[r].
template <int CT>
struct AttnPowers {
  float tile[CT], near[4], diag[4], rowf, tail[4], chunk;
  __device__ void init(float g, int rev, float ss, float si, float su, int lo, int hi) {
#pragma unroll
    for (int d = 0; d < CT; ++d) tile[d] = uniform(decay_pow(g, 16 * d));
    chunk = uniform(decay_pow(g, 16 * CT));
    rowf = si * decay_pow(g, lo + 1 - rev);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int lag = lo - 4 * hi - r;
      near[r] = ss * decay_pow(g, 16 + lag);
      diag[r] = lag >= 0 ? ss * decay_pow(g, max(lag, 0)) : 0.0f;
      tail[r] = su * decay_pow(g, 15 - 4 * hi - r + rev);
    }
  }
};

// FULL: outputs and the carried state; else the run's own sum alone, into seg_state.
template <typename E, int DA, int DC, bool FULL>
__global__ __launch_bounds__((AttnShape<E, DA, DC>::THREADS), 2) void attn_chunk_kernel(AttnArgs<E> p) {
  using S = AttnShape<E, DA, DC>;
  constexpr int C = S::C, W = S::W, NV = S::NV, LDA = S::LDA, LDC = S::LDC, LDP = S::LDP;
  constexpr int CT = C / 16, KA = DA / 16;
  extern __shared__ __align__(16) char smem[];
  E* tb = reinterpret_cast<E*>(smem);
  E* tc = tb + C * LDA;
  E* ta = tc + C * LDC;
  E* tp = ta + C * LDA;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4;
  const int bh = blockIdx.x / p.segs, seg = blockIdx.x - bh * p.segs;
  const int b = bh / p.H, h = bh - b * p.H;
  const float g = p.log_decay[h];
  const int L = attn_length(p, b);
  const int64_t first = p.rev ? L - 1 : 0, dir = p.rev ? -1 : 1;
  const E* pa = p.a + b * p.as[0] + (h / p.ga) * p.as[2] + first * p.as[1];
  const E* pb = p.b + b * p.bs[0] + (h / p.gb) * p.bs[2] + first * p.bs[1];
  const E* pc = p.c + b * p.cs[0] + (h / p.gc) * p.cs[2] + first * p.cs[1];
  const int64_t orow = (int64_t)p.H * p.dc;
  const int64_t obase = ((int64_t)b * p.T * p.H + h) * p.dc;
  const int col0 = wave * NV * 16;
  const int begin = seg * p.seg_len, end = min(L, begin + p.seg_len);
  const int64_t sbase = (int64_t)bh * p.da * p.dc;
  float* seg_state = p.segs > 1 ? p.seg_state + (int64_t)blockIdx.x * p.da * p.dc : nullptr;

  // S[m][n]: rows 16 m + 4 hi + r, column col0 + 16 n + lo
  f32x4 s[KA][NV];
#pragma unroll
  for (int m = 0; m < KA; ++m)
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * m + 4 * hi + r, col = col0 + 16 * n + lo;
        float v = 0.0f;
        if (FULL && row < p.da && col < p.dc) {
          if (seg_state)
            v = seg_state[(int64_t)row * p.dc + col];
          else if (p.s_in)
            v = p.s_in_t ? p.s_in[sbase + (int64_t)col * p.da + row] : p.s_in[sbase + (int64_t)row * p.dc + col];
        }
        s[m][n][r] = v;
      }

  AttnPowers<CT> pw;
  pw.init(g, p.rev, p.ss, p.si, p.su, lo, hi);
  AttnRows<E, C, DA, S::THREADS> ra, rb;
  AttnRows<E, C, DC, S::THREADS> rc;
  rb.init(pb, dir * p.bs[1], begin, tid);
  rc.init(pc, dir * p.cs[1], begin, tid);
  if constexpr (FULL) ra.init(pa, dir * p.as[1], begin, tid);
  auto fetch = [&](int n) {
    rb.load(n, p.da);
    rc.load(n, p.dc);
    if constexpr (FULL) ra.load(n, p.da);
  };
  if (begin < end) fetch(end - begin);
  int64_t orow0 = obase + (first + dir * (begin + lo)) * orow;  // the output row of tile 0
  for (int t0 = begin; t0 < end; t0 += C) {
    const int n = min(C, end - t0);  // live steps
    rb.store(tb);
    rc.store(tc);
    if constexpr (FULL) ra.store(ta);
    __syncthreads();
    if (t0 + C < end) fetch(end - t0 - C);

    if constexpr (FULL) {
    // scores: tile (it, jt <= it) as its transpose, so that a lane holds 4 consecutive j of
    // one i; rounded to E for the product with V (the output is E as well)
    for (int q = wave; q < CT * (CT + 1) / 2; q += W) {
      int it = 0, jt = q;
      while (jt > it) jt -= ++it;
      float far = pw.tile[0];  // e^{16 g (it - jt - 1)}
#pragma unroll
      for (int d = 1; d < CT - 1; ++d) far = it - jt - 1 == d ? pw.tile[d] : far;
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KA; k += 2)
        acc = mma2(lds_quad(tb, LDA, 16 * jt, 16 * k, lane), lds_quad(tb, LDA, 16 * jt, 16 * k + 16, lane),
                   lds_quad(ta, LDA, 16 * it, 16 * k, lane), lds_quad(ta, LDA, 16 * it, 16 * k + 16, lane), acc);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = it == jt ? acc[r] * pw.diag[r] : acc[r] * (far * pw.near[r]);
      *reinterpret_cast<quad_t<E>*>(tp + (16 * it + lo) * LDP + 16 * jt + 4 * hi) = to_quad<E>(acc);
    }
    __syncthreads();
    }

    // the wave's values, contracted over the steps
    quad_t<E> v[CT][NV];
#pragma unroll
    for (int j = 0; j < CT; ++j)
#pragma unroll
      for (int x = 0; x < NV; ++x) v[j][x] = lds_quad_t(tc, LDC, 16 * j, col0 + 16 * x, lane);

    // O^T tiles: columns i, rows the values
    if constexpr (FULL) {
#pragma unroll
    for (int it = 0; it < CT; ++it) {
      const int i = 16 * it + lo;
      f32x4 acc[NV];
#pragma unroll
      for (int x = 0; x < NV; ++x) acc[x] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KA; k += 2) {
        const quad_t<E> a0 = lds_quad(ta, LDA, 16 * it, 16 * k, lane);
        const quad_t<E> a1 = lds_quad(ta, LDA, 16 * it, 16 * k + 16, lane);
#pragma unroll
        for (int x = 0; x < NV; ++x)  // the state rounds to E as this product's operand only
          acc[x] = mma2(to_quad<E>(s[k][x]), to_quad<E>(s[k + 1][x]), a0, a1, acc[x]);
      }
      const float f = pw.rowf * pw.tile[it];
#pragma unroll
      for (int x = 0; x < NV; ++x) acc[x] *= f;
#pragma unroll
      for (int j = 0; j < CT; j += 2)
        if (j <= it) {  // the odd tile past the diagonal was not written: zero
          const quad_t<E> p0 = lds_quad(tp, LDP, 16 * it, 16 * j, lane);
          const quad_t<E> p1 = j + 1 <= it ? lds_quad(tp, LDP, 16 * it, 16 * j + 16, lane) : to_quad<E>(f32x4{0, 0, 0, 0});
#pragma unroll
          for (int x = 0; x < NV; ++x) acc[x] = mma2(v[j][x], v[j + 1][x], p0, p1, acc[x]);
        }
      if (i < n) {
        const int64_t row = orow0 + dir * 16 * it * orow;
#pragma unroll
        for (int x = 0; x < NV; ++x) {
          const int c = col0 + 16 * x + 4 * hi;
          if (p.o_f32)
            store_quad(reinterpret_cast<float*>(p.o) + row, c, p.dc, acc[x]);
          else
            store_quad(reinterpret_cast<E*>(p.o) + row, c, p.dc, acc[x]);
        }
      }
    }
    }

    // S update.  The decayed values are not exact in bf16: they enter as a sum of three bf16
    // terms (24 bits), for the state is an fp32 result
    const bool whole = n == C;
    const float fl = whole ? pw.chunk : decay_pow(g, n);
#pragma unroll
    for (int m = 0; m < KA; ++m)
#pragma unroll
      for (int x = 0; x < NV; ++x) s[m][x] *= fl;
#pragma unroll
    for (int j = 0; j < CT; j += 2) {
      f32x4 d0, d1;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (whole) {
          d0[r] = pw.tile[CT - 1 - j] * pw.tail[r], d1[r] = pw.tile[CT - 2 - j] * pw.tail[r];
          continue;
        }
        const int j0 = 16 * j + 4 * hi + r;
        d0[r] = p.su * decay_pow(g, max(n - 1 - j0, 0) + p.rev);
        d1[r] = p.su * decay_pow(g, max(n - 17 - j0, 0) + p.rev);
      }
      constexpr int TERMS = sizeof(E) == 2 ? 3 : 1;
      quad_t<E> w0[TERMS][NV], w1[TERMS][NV];
#pragma unroll
      for (int x = 0; x < NV; ++x) {
        f32x4 r0 = to_f32(v[j][x]) * d0, r1 = to_f32(v[j + 1][x]) * d1;
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
          w0[t][x] = to_quad<E>(r0), w1[t][x] = to_quad<E>(r1);
          r0 -= to_f32(w0[t][x]), r1 -= to_f32(w1[t][x]);
        }
      }
#pragma unroll
      for (int m = 0; m < KA; ++m) {
        const quad_t<E> b0 = lds_quad_t(tb, LDA, 16 * j, 16 * m, lane);
        const quad_t<E> b1 = lds_quad_t(tb, LDA, 16 * j + 16, 16 * m, lane);
#pragma unroll
        for (int x = 0; x < NV; ++x)
#pragma unroll
          for (int t = 0; t < TERMS; ++t) s[m][x] = mma2(b0, b1, w0[t][x], w1[t][x], s[m][x]);
      }
    }
    orow0 += dir * C * orow;
    __syncthreads();  // the tiles are free
  }

  if constexpr (FULL) {
    // this run's steps past the end
    const int64_t z0 = max(L, begin), z1 = min(p.T, begin + p.seg_len);
    for (int64_t e = z0 * p.dc + tid; e < z1 * p.dc; e += S::THREADS) {
      const int64_t t = e / p.dc, c = e - t * p.dc;
      if (p.o_f32)
        reinterpret_cast<float*>(p.o)[obase + t * orow + c] = 0.0f;
      else
        reinterpret_cast<E*>(p.o)[obase + t * orow + c] = E(0.0f);
    }
  }
  // the run that holds the last live step has the final state
  float* out = FULL ? (p.s_out && seg == (L > 0 ? (L - 1) / p.seg_len : 0) ? p.s_out + sbase : nullptr) : seg_state;
  if (out) {
#pragma unroll
    for (int m = 0; m < KA; ++m)
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * m + 4 * hi + r, col = col0 + 16 * n + lo;
          if (row < p.da && col < p.dc) out[(int64_t)row * p.dc + col] = s[m][n][r];
        }
  }
}

// Between the passes of a split history: each run's own sum becomes the state it starts
// from.  A thread an element of the state; the loads of eight runs are in flight.
template <typename E>
__global__ __launch_bounds__(256) void attn_scan_kernel(AttnArgs<E> p) {
  const int n = p.da * p.dc, per = (n + 255) / 256;
  const int bh = blockIdx.x / per, e = (blockIdx.x - bh * per) * 256 + threadIdx.x;
  if (e >= n) return;
  const int b = bh / p.H, h = bh - b * p.H;
  const float g = p.log_decay[h];
  const int L = attn_length(p, b);
  float v = 0.0f;
  if (p.s_in) {
    const int row = e / p.dc, col = e - row * p.dc;
    v = p.s_in[(int64_t)bh * n + (p.s_in_t ? col * p.da + row : e)];
  }
  float* x = p.seg_state + (int64_t)bh * p.segs * n + e;
  constexpr int AHEAD = 8;
  for (int i0 = 0; i0 < p.segs; i0 += AHEAD) {
    float u[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) u[i] = i0 + i < p.segs ? x[(int64_t)(i0 + i) * n] : 0.0f;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int seg = i0 + i;
      if (seg < p.segs) {
        x[(int64_t)seg * n] = v;
        const int len = min(max(L - seg * p.seg_len, 0), p.seg_len);
        v = v * decay_pow(g, len) + u[i];
      }
    }
  }
}

// Sums the shared heads' gradients: (tokens, Hk, G, d) fp32 -> (tokens, Hk, d), in order.
template <typename E>
__global__ __launch_bounds__(256) void attn_head_sum_kernel(const float* __restrict__ in, int64_t n, int G, int d,
                                                            E* __restrict__ out) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    const int64_t row = e / d;
    const float* src = in + row * G * d + (e - row * d);
    float v = 0.0f;
    for (int i = 0; i < G; ++i) v += src[(int64_t)i * d];
    out[e] = (E)v;
  }
}

// One step: S := e^g S + k^T v, o = scale q S in place, a (problem, head) a workgroup.
// Bound by the state's read and write.  Thread (row group, 4 columns): the rows of S
// are walked RG at a time, o is summed over the row groups in LDS.
template <typename E>
struct AttnStepArgs {
  int B, H, G, dk, dv;
  const E *q, *k, *v;
  int64_t qs[2], ks[2], vs[2];  // strides of problem, head
  const float* log_decay;
  const uint8_t* active;  // (B) or NULL
  float scale;
  float* state;  // (B, H, dk, dv)
  E* o;          // (B, H, dv)
};

template <typename E>
__global__ __launch_bounds__(256) void attn_step_kernel(AttnStepArgs<E> p) {
  __shared__ float sq[128], sk[128], sv[128], so[256 * 4];
  const int tid = threadIdx.x;
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / p.H), h = (int)(bh - (int64_t)b * p.H), hk = h / p.G;
  E* o = p.o + bh * p.dv;
  if (p.active && !p.active[b]) {
    for (int c = tid; c < p.dv; c += 256) o[c] = E(0.0f);
    return;
  }
  if (tid < p.dk) {
    sq[tid] = (float)p.q[b * p.qs[0] + h * p.qs[1] + tid] * p.scale;
    sk[tid] = (float)p.k[b * p.ks[0] + hk * p.ks[1] + tid];
  }
  if (tid < p.dv) sv[tid] = (float)p.v[b * p.vs[0] + hk * p.vs[1] + tid];
  const float gamma = __expf(p.log_decay[h]);
  __syncthreads();
  float* S = p.state + bh * p.dk * p.dv;
  const int nc = (p.dv + 3) / 4;        // 4-column groups
  const int rg = 256 / nc;              // rows walked at a time (>= 8)
  const int c = (tid % nc) * 4, r0 = tid / nc;
  f32x4 acc = {0, 0, 0, 0};
  if (r0 < rg)
    for (int r = r0; r < p.dk; r += rg) {
      f32x4 x = load_quad_f32(S + (int64_t)r * p.dv, c, p.dv);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = x[e] * gamma + sk[r] * (c + e < p.dv ? sv[c + e] : 0.0f);
        acc[e] += sq[r] * x[e];
      }
      store_quad(S + (int64_t)r * p.dv, c, p.dv, x);
    }
  *reinterpret_cast<f32x4*>(so + tid * 4) = acc;
  __syncthreads();
  if (tid < p.dv) {
    float t = 0.0f;
    for (int r = 0; r < rg; ++r) t += so[(r * nc + tid / 4) * 4 + (tid & 3)];
    o[tid] = (E)t;
  }
}

}  // namespace tmpc
