// Gated delta rule.  Problem b, head h, a_t = exp(g_t) (S fp32, dk x dv):
//   e_t = v_t - a_t k_t S_{t-1},  u_t = beta_t e_t,  S_t = a_t S_{t-1} + k_t^T u_t,  o_t = scale q_t S_t.
//
// Blocks of 16 steps, G_i the sum of g up to step i of the block, Gamma_ij = exp(G_i - G_j) for
// j <= i, else 0.  With A_ij = Gamma_ij (k_i . k_j) beta_j for j < i, the block's steps are
//   E = (I + A)^-1 (V - diag(exp G) K S),  U = diag(beta) E,
//   O = scale (diag(exp G) Q S + (Q K^T o Gamma) U),  S := exp(G_15) S + K^T diag(exp(G_15 - G)) U.
// The inverse is formed by substitution, row by row: its entries stay as small as the recurrence's
// products of (I - beta k^T k), where a product of powers of A would cancel large terms for keys
// that repeat themselves.  Sums of g are held in 64 bits, so that their differences are exact to 32
// also behind a decay of zero (g = -inf, taken as -1e5, whose exponential is zero).
//
// A block is as long as a matrix instruction's tile, so that the chain from state to state stays in a
// wave's registers: S is the operand of K S, whose result is the operand of the product with the
// inverse, whose result is the operand of the state's update.  A wave owns 16 columns of the values and
// walks its head's blocks without meeting the other waves; what depends on the block alone (the
// inverse, Q K^T o Gamma, the powers) is made once a chunk of several blocks, a wave a block, in LDS.
//
// Backward.  With R_t = dL/dS_t from later steps, D_t = R_t + scale q_t^T do_t:
//   du_t = k_t D_t,  y_t = dv_t = beta_t du_t,  R_{t-1} = a_t (D_t - k_t^T y_t),  dbeta_t = du_t . e_t,
//   dq_t = scale do_t S_t^T,  dk_t = u_t D_t^T - a_t y_t S_{t-1}^T,  dg_t = <R_{t-1}, S_{t-1}>.
#pragma once
#include "decay_attention.hpp"

namespace tmpc {

constexpr float kNoDecay = -1e5f;  // a log decay below it is a decay of zero

template <typename E>
struct DeltaArgs {
  int B, T, H, dk, dv;
  int gq, gk, gv;  // heads that share one of q's (k's, v's) heads
  const E *q, *k, *v, *beta;
  const float* g;
  int64_t qs[3], ks[3], vs[3], bs[3], gs[3];  // strides of problem, step, head
  const int32_t* lengths;                     // (B) or NULL
  float scale;
  const float* s_in;  // (B, H, dk, dv) or NULL
  float* s_out;       // (B, H, dk, dv) or NULL
  E* o;               // (B, T, H, dv)
};

template <typename E, int DK, int DV>
struct DeltaShape {
  static constexpr int W = DV / 16, THREADS = 64 * W;  // a wave 16 value columns
  static constexpr int C = AttnTile<E>::C, SUB = C / 16, PAD = AttnTile<E>::PAD;
  static constexpr int LDK = DK + PAD, LDV = DV + PAD;
  static constexpr int LDT = 20;  // pitch of a 16 x 16 fp32 tile: its quads spread over the banks
  static constexpr int LDP = sizeof(E) == 2 ? 24 : 20;
  // floats: the chunk's gates, powers and inverses
  static constexpr int GATES = 4 * C + 4, INV = SUB * 16 * LDT;
};

__device__ inline f32x4 lds_f4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }

// acc += A B over 16 contracted entries in fp32 (a quad of each operand)
__device__ inline f32x4 mma16(f32x4 a, f32x4 b, f32x4 acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], acc, 0, 0, 0);
  return acc;
}

// What a block's products are made of, per chunk in LDS.
struct DeltaGates {
  float *g, *beta;      // the chunk's, zeros past its last live step
  float *from, *to;     // exp(G_i) and exp(G_15 - G_i) of each block
  float* total;         // exp(G_15)
  float* inv;           // tiles of the inverses, pitch LDT
};
template <typename S>
__device__ inline DeltaGates delta_gates(float* base) {
  DeltaGates d;
  d.g = base, d.beta = base + S::C, d.from = base + 2 * S::C, d.to = base + 3 * S::C, d.total = base + 4 * S::C;
  d.inv = base + S::GATES;
  return d;
}

// The chunk's gates on their way from memory to LDS: a thread a step.
template <typename E, int C>
struct DeltaGateRows {
  const float* g;
  const E* beta;
  int64_t gs, bs;
  float vg, vb;
  __device__ void load(int t0, int n, int tid) {
    vg = vb = 0.0f;
    if (tid < n && tid < C) {
      vg = g[(t0 + tid) * gs];
      vb = (float)beta[(t0 + tid) * bs];
    }
  }
  __device__ void store(const DeltaGates& d, int tid) const {
    if (tid < C) d.g[tid] = vg < kNoDecay ? kNoDecay : vg, d.beta[tid] = vb;
  }
};

// Block `sub` of a chunk, by one wave: the powers, and G_i - G_j of a lane's i = lo and j = 4 hi + r.
template <typename S>
__device__ inline f32x4 delta_powers(const DeltaGates& d, int sub, int lane) {
  const int lo = lane & 15, hi = lane >> 4;
  double sum = 0.0, mine = 0.0, at[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    const f32x4 g = lds_f4(d.g + 16 * sub + j);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      sum += (double)g[r];
      if (j + r == lo) mine = sum;
      if (j == 4 * hi) at[r] = sum;
    }
  }
  if (hi == 0) d.from[16 * sub + lo] = __expf((float)mine), d.to[16 * sub + lo] = __expf((float)(sum - mine));
  if (lane == 0) d.total[sub] = __expf((float)sum);
  f32x4 lag;
#pragma unroll
  for (int r = 0; r < 4; ++r) lag[r] = (float)(mine - at[r]);
  return lag;
}

// (I + A)^-1 of a block from A's rows: lane lo has A[lo][4 hi + r] in `a`, zeros from the diagonal on.
// The rows of the inverse (or, with TRANSPOSED, its columns) go to the block's tile.
template <typename S, bool TRANSPOSED>
__device__ inline void delta_inverse(const DeltaGates& d, int sub, f32x4 a, int lane) {
  const int lo = lane & 15, hi = lane >> 4;
  float* tile = d.inv + sub * 16 * S::LDT;
  *reinterpret_cast<f32x4*>(tile + lo * S::LDT + 4 * hi) = a;
  __builtin_amdgcn_wave_barrier();
  float t[16];  // column lo of the inverse
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float v = i == lo ? 1.0f : 0.0f;
#pragma unroll
    for (int j = 0; j < i; j += 4) {
      const f32x4 row = lds_f4(tile + i * S::LDT + j);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (j + r < i) v = fmaf(-row[r], t[j + r], v);
    }
    t[i] = v;
  }
  __builtin_amdgcn_wave_barrier();
  if constexpr (TRANSPOSED) {
    if (hi == 0)
#pragma unroll
      for (int j = 0; j < 16; j += 4)
        *reinterpret_cast<f32x4*>(tile + lo * S::LDT + j) = f32x4{t[j], t[j + 1], t[j + 2], t[j + 3]};
  } else {
    if (hi == 0)
#pragma unroll
      for (int j = 0; j < 16; ++j) tile[j * S::LDT + lo] = t[j];
  }
}

// x (fp32) as an operand of products whose other operand is exact in E: three bf16 terms (24
// bits), or itself.
template <typename E>
struct Terms {
  static constexpr int N = sizeof(E) == 2 ? 3 : 1;
  quad_t<E> t[N];
  __device__ Terms(f32x4 x) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      t[i] = to_quad<E>(x);
      if (i + 1 < N) x -= to_f32(t[i]);
    }
  }
};
// acc += A x over 16 contracted entries, x by its terms
__device__ inline f32x4 mma_terms(bf16x4 a, const Terms<bf16>& x, f32x4 acc) {
  const bf16x4 zero = to_bf16(f32x4{0, 0, 0, 0});
  acc = mma2(a, a, x.t[0], x.t[1], acc);
  return mma2(a, zero, x.t[2], zero, acc);
}
__device__ inline f32x4 mma_terms(f32x4 a, const Terms<float>& x, f32x4 acc) { return mma16(a, x.t[0], acc); }

// K s (rows i of the block at k: 16 x dk, the wave's 16 columns) exact to fp32, and with OT > 0
// (Q s)^T by s's first OT terms.
template <typename E, int KA, int OT>
__device__ inline f32x4 delta_state_products(const E* k, const E* q, int ld, int row0, const f32x4 (&s)[KA][1], f32x4& qs,
                                             int lane) {
  f32x4 x[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
  for (int m = 0; m < KA; m += 2) {
    const quad_t<E> k0 = lds_quad(k, ld, row0, 16 * m, lane), k1 = lds_quad(k, ld, row0, 16 * m + 16, lane);
    quad_t<E> q0, q1;
    if constexpr (OT > 0) q0 = lds_quad(q, ld, row0, 16 * m, lane), q1 = lds_quad(q, ld, row0, 16 * m + 16, lane);
    const Terms<E> a(s[m][0]), b(s[m + 1][0]);
#pragma unroll
    for (int t = 0; t < Terms<E>::N; ++t) {
      x[t & 1] = mma2(k0, k1, a.t[t], b.t[t], x[t & 1]);
      if (t < OT) qs = mma2(a.t[t], b.t[t], q0, q1, qs);
    }
  }
  return x[0] + x[1];
}

// A wave's columns of a history whose state is not finite in the end, by the definition, a step at
// a time: in a block such a step meets the earlier ones with factors of zero, which makes those NaN.
template <typename E, int KA>
__device__ __attribute__((always_inline)) inline void delta_by_step(const DeltaArgs<E>& p, int bh, int tid) {
  const int lo = tid & 15, hi = (tid & 63) >> 4, col0 = (tid >> 6) * 16, c = col0 + lo;
  const int b = bh / p.H, h = bh - b * p.H;
  const int L = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const E* pq = p.q + b * p.qs[0] + (h / p.gq) * p.qs[2];
  const E* pk = p.k + b * p.ks[0] + (h / p.gk) * p.ks[2];
  const E* pv = p.v + b * p.vs[0] + (h / p.gv) * p.vs[2];
  const E* pb = p.beta + b * p.bs[0] + h * p.bs[2];
  const float* pg = p.g + b * p.gs[0] + h * p.gs[2];
  const int64_t size = (int64_t)p.dk * p.dv;
  f32x4 s[KA][1];
  load_state(s, p.s_in ? p.s_in + bh * size : nullptr, false, p.dk, p.dv, col0, lo, hi);
  for (int t = 0; t < L; ++t) {
    const E *qt = pq + t * p.qs[1], *kt = pk + t * p.ks[1];
    const float a = __expf(pg[t * p.gs[1]]), beta = (float)pb[t * p.bs[1]];
    float ks = 0.0f, qs = 0.0f;
#pragma unroll
    for (int m = 0; m < KA; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * m + 4 * hi + r;
        s[m][0][r] *= a;
        if (row < p.dk) ks += (float)kt[row] * s[m][0][r];
      }
    ks += __shfl_xor(ks, 16, 64), ks += __shfl_xor(ks, 32, 64);
    const float u = c < p.dv ? beta * ((float)pv[t * p.vs[1] + c] - ks) : 0.0f;
#pragma unroll
    for (int m = 0; m < KA; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * m + 4 * hi + r;
        if (row < p.dk) s[m][0][r] += (float)kt[row] * u, qs += (float)qt[row] * s[m][0][r];
      }
    qs += __shfl_xor(qs, 16, 64), qs += __shfl_xor(qs, 32, 64);
    if (hi == 0 && c < p.dv) p.o[(((int64_t)b * p.T + t) * p.H + h) * p.dv + c] = (E)(p.scale * qs);
  }
  if (p.s_out) store_state(s, p.s_out + bh * size, p.dk, p.dv, col0, lo, hi);
}

template <typename E, int DK, int DV>
constexpr size_t delta_forward_lds() {
  using S = DeltaShape<E, DK, DV>;
  return sizeof(float) * (S::GATES + S::INV) + sizeof(E) * (2 * S::C * S::LDK + S::C * S::LDV + S::SUB * 16 * S::LDP);
}

// A workgroup a (problem, head).
template <typename E, int DK, int DV, bool VEC>
__global__ __launch_bounds__((DeltaShape<E, DK, DV>::THREADS)) void delta_forward_kernel(DeltaArgs<E> p) {
  using S = DeltaShape<E, DK, DV>;
  constexpr int C = S::C, SUB = S::SUB, KA = DK / 16, LDK = S::LDK, LDV = S::LDV, LDT = S::LDT, LDP = S::LDP;
  extern __shared__ __align__(16) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4, col0 = wave * 16;
  const int bh = blockIdx.x, b = bh / p.H, h = bh - b * p.H;
  const int L = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const DeltaGates d = delta_gates<S>(reinterpret_cast<float*>(smem));
  E* tk = reinterpret_cast<E*>(d.inv + S::INV);
  E* tq = tk + C * LDK;
  E* tv = tq + C * LDK;
  E* tp = tv + C * LDV;  // the blocks' scores, pitch LDP

  AttnRows<E, C, DK, S::THREADS, VEC> rk, rq;
  AttnRows<E, C, DV, S::THREADS, VEC> rv;
  rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], 0, p.dk, tid);
  rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], 0, p.dk, tid);
  rv.init(p.v + b * p.vs[0] + (h / p.gv) * p.vs[2], p.vs[1], 0, p.dv, tid);
  DeltaGateRows<E, C> rg{p.g + b * p.gs[0] + h * p.gs[2], p.beta + b * p.bs[0] + h * p.bs[2], p.gs[1], p.bs[1]};
  auto fetch = [&](int t0) {
    rk.load(L - t0, p.dk), rq.load(L - t0, p.dk), rv.load(L - t0, p.dv), rg.load(t0, L - t0, tid);
  };
  if (L > 0) fetch(0);
  const int64_t size = (int64_t)p.dk * p.dv;
  f32x4 s[KA][1];
  load_state(s, p.s_in ? p.s_in + bh * size : nullptr, false, p.dk, p.dv, col0, lo, hi);
  const int64_t orow = (int64_t)p.H * p.dv, obase = ((int64_t)b * p.T * p.H + h) * p.dv;
  const int oc = col0 + 4 * hi;

  for (int t0 = 0; t0 < L; t0 += C) {
    const int n = min(C, L - t0);
    rk.store(tk), rq.store(tq), rv.store(tv), rg.store(d, tid);
    __syncthreads();
    if (t0 + C < L) fetch(t0 + C);
    for (int sub = wave; 16 * sub < n; sub += S::W) {
      const f32x4 lag = delta_powers<S>(d, sub, lane);
      f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
      for (int m = 0; m < KA; m += 2) {
        const quad_t<E> k0 = lds_quad(tk, LDK, 16 * sub, 16 * m, lane), k1 = lds_quad(tk, LDK, 16 * sub, 16 * m + 16, lane);
        kk = mma2(k0, k1, k0, k1, kk);
        qk = mma2(k0, k1, lds_quad(tq, LDK, 16 * sub, 16 * m, lane), lds_quad(tq, LDK, 16 * sub, 16 * m + 16, lane), qk);
      }
      const f32x4 beta = lds_f4(d.beta + 16 * sub + 4 * hi);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 4 * hi + r;
        kk[r] = j < lo ? kk[r] * __expf(lag[r]) * beta[r] : 0.0f;
        qk[r] = j <= lo ? p.scale * (qk[r] * __expf(lag[r])) : 0.0f;
      }
      *reinterpret_cast<quad_t<E>*>(tp + (16 * sub + lo) * LDP + 4 * hi) = to_quad<E>(qk);
      delta_inverse<S, false>(d, sub, kk, lane);
    }
    __syncthreads();
    for (int sub = 0; 16 * sub < n; ++sub) {
      f32x4 o = {0, 0, 0, 0};
      const f32x4 ks = delta_state_products<E, KA, 1>(tk, tq, LDK, 16 * sub, s, o, lane);
      const f32x4 v = to_f32(lds_quad_t(tv, LDV, 16 * sub, col0, lane));
      const f32x4 x = v - lds_f4(d.from + 16 * sub + 4 * hi) * ks;
      const f32x4 u = lds_f4(d.beta + 16 * sub + 4 * hi) * mma16(lds_f4(d.inv + (16 * sub + lo) * LDT + 4 * hi), x, f32x4{0, 0, 0, 0});
      o *= p.scale * d.from[16 * sub + lo];
      const quad_t<E> pq = *reinterpret_cast<const quad_t<E>*>(tp + (16 * sub + lo) * LDP + 4 * hi);
      if constexpr (sizeof(E) == 2) {
        const bf16x4 uh = to_bf16(u);
        o = mma2(uh, to_bf16(u - to_f32(uh)), pq, pq, o);
      } else {
        o = mma16(u, pq, o);
      }
      const int t = t0 + 16 * sub + lo;
      if (t < L) {
        E* row = p.o + obase + t * orow;
        if (VEC) {
          if (oc < p.dv) *reinterpret_cast<quad_t<E>*>(row + oc) = to_quad<E>(o);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (oc + e < p.dv) row[oc + e] = (E)o[e];
        }
      }
      const Terms<E> w(lds_f4(d.to + 16 * sub + 4 * hi) * u);
      const float total = d.total[sub];
#pragma unroll
      for (int m = 0; m < KA; ++m) s[m][0] = mma_terms(lds_quad_t(tk, LDK, 16 * sub, 16 * m, lane), w, s[m][0] * total);
    }
    __syncthreads();
  }
  zero_rows(p.o, false, sizeof(E), obase, orow, p.dv, L, p.T, tid, S::THREADS);
  // An infinite or NaN value leaves the state so, to the end.
  f32x4 zero = {0, 0, 0, 0};
#pragma unroll
  for (int m = 0; m < KA; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) zero[r] = fmaf(s[m][0][r], 0.0f, zero[r]);
  if (L > 0 && __ballot(!(zero[0] + zero[1] + zero[2] + zero[3] == 0.0f))) {
    __threadfence_block();  // rows written above are written again
    delta_by_step<E, KA>(p, bh, tid);
  } else if (p.s_out) {
    store_state(s, p.s_out + bh * size, p.dk, p.dv, col0, lo, hi);
  }
}

// ---- backward ----
// Three kernels.  The first walks forwards in time as the forward pass does and leaves e_t, the state
// at each chunk's start and do_t . o_t.  The second walks backwards with the state's gradient,
// which gives y = dv and dbeta, and leaves the gradient at each chunk's end: over a block,
//   dU = (I + A')^-T (scale (Q K^T o Gamma)^T dO + diag(exp(G_15 - G)) K R),  A'_ij = beta_i Gamma_ij (k_i . k_j),
//   R := exp(G_15) R + (diag(exp G) scale Q)^T dO - (diag(exp G) K)^T Y,  Y = diag(beta) dU.
// With the state and its gradient known at its ends every chunk then gives its dq and dk by itself:
//   dq_i = scale exp(G_i) do_i S^T + sum_{j <= i} M_ij k_j,  M_ij = scale Gamma_ij (do_i . u_j),
//   dk_j = exp(G_end - G_j) u_j R^T - exp(G_j) y_j S^T + sum_{i >= j} M_ij q_i
//          - sum_{i > j} N_ij k_i - sum_{l < j} N_jl k_l,  N_ij = Gamma_ij (y_i . u_j).
// log_decay's gradient is dg_t = <R_{t-1}, S_{t-1}>; what makes it change from step to step is
// dg_t = dg_{t+1} + do_t . o_t - dv_t . v_t, so it is that sum from the end of each stretch of 256
// steps, where both matrices are at hand in fp32, and o enters it unrounded.  (No values that are not
// finite are looked for here: they may spoil the gradients of their whole history and head.)
template <typename E>
struct DeltaBwdArgs {
  DeltaArgs<E> f;
  const E* d_o;
  int64_t dos[3];
  const float* d_out;  // (B, H, dk, dv) or NULL
  int chunks, segs;    // of T
  E *e;                // (B H, chunks C, DV)
  E *s, *r;            // (B H, chunks, DV, DK): the states at the chunks' starts, their gradients at the ends
  float *w, *z;        // (B H, chunks C): do . o, y . v
  float* s_seg;        // (B H, segs, the wave's registers): the states at the stretches' ends
  float* dot;          // (B H, segs): <R, S> there
  E* y;                // as e, or dv's output (B, T, H, dv)
  int64_t ys[2];       // its strides of (b h) and step, from b and h where it is the output
  int y_width;
  float* y_part;       // (B, T, H, dv) or NULL
  E* dbeta;            // (B, T, H)
  float* dg;           // (B, T, H)
  float* d_in;         // (B, H, dk, dv) or NULL
  void *dq, *dk;       // (B, T, H, dk) of E, or fp32 parts
  int q_part, k_part;
};
constexpr int kDeltaSeg = 256;  // steps

// sum over the 16 lanes of a row
__device__ inline float row16_sum(float v) {
#define TMPC_ROR(n) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + n, 0xf, 0xf, false))
  v += TMPC_ROR(8);
  v += TMPC_ROR(4);
  v += TMPC_ROR(2);
  v += TMPC_ROR(1);
#undef TMPC_ROR
  return v;
}

// The wave's 16 columns of a state, rounded, as rows of a (DV, DK) matrix.
template <typename E, int DK, int KA>
__device__ inline void store_columns(E* dst, const f32x4 (&s)[KA][1], int col0, int lo, int hi) {
#pragma unroll
  for (int m = 0; m < KA; ++m)
    *reinterpret_cast<quad_t<E>*>(dst + (col0 + lo) * DK + 16 * m + 4 * hi) = to_quad<E>(s[m][0]);
}

// Rows of a tile in LDS to memory: `n` of them, row t at dst + t pitch.
template <typename R, typename E>
__device__ inline void copy_out(const R& map, const E* tile, E* dst, int64_t pitch, int n, int width) {
  constexpr int P = Elem<E>::PIECE;
  if (map.row >= R::RS) return;
#pragma unroll
  for (int i = 0; i < R::N; ++i) {
    const int row = map.row + i * R::RS;
    if (row < n && map.c < width)
      store_piece(dst + row * pitch, map.c, width, *reinterpret_cast<const piece_t<E>*>(tile + row * R::LD + map.c));
  }
  (void)P;
}

template <typename E, int DK, int DV>
constexpr size_t delta_states_lds() {
  using S = DeltaShape<E, DK, DV>;
  return sizeof(float) * (S::GATES + 2 * S::INV + S::W * S::C) + sizeof(E) * (2 * S::C * S::LDK + 2 * S::C * S::LDV);
}

template <typename E, int DK, int DV, bool VEC>
__global__ __launch_bounds__((DeltaShape<E, DK, DV>::THREADS)) void delta_states_kernel(DeltaBwdArgs<E> a) {
  using S = DeltaShape<E, DK, DV>;
  constexpr int C = S::C, KA = DK / 16, LDK = S::LDK, LDV = S::LDV, LDT = S::LDT, SEG = kDeltaSeg / C;
  extern __shared__ __align__(16) char smem[];
  const DeltaArgs<E>& p = a.f;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4, col0 = wave * 16;
  const int bh = blockIdx.x, b = bh / p.H, h = bh - b * p.H;
  const int L = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const DeltaGates d = delta_gates<S>(reinterpret_cast<float*>(smem));
  float* tp = d.inv + S::INV;  // the blocks' scores
  float* sums = tp + S::INV;   // (waves, steps)
  E* tk = reinterpret_cast<E*>(sums + S::W * C);
  E* tq = tk + C * LDK;
  E* tv = tq + C * LDK;
  E* tdo = tv + C * LDV;

  AttnRows<E, C, DK, S::THREADS, VEC> rk, rq;
  AttnRows<E, C, DV, S::THREADS, VEC> rv, rdo;
  rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], 0, p.dk, tid);
  rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], 0, p.dk, tid);
  rv.init(p.v + b * p.vs[0] + (h / p.gv) * p.vs[2], p.vs[1], 0, p.dv, tid);
  rdo.init(a.d_o + b * a.dos[0] + h * a.dos[2], a.dos[1], 0, p.dv, tid);
  DeltaGateRows<E, C> rg{p.g + b * p.gs[0] + h * p.gs[2], p.beta + b * p.bs[0] + h * p.bs[2], p.gs[1], p.bs[1]};
  auto fetch = [&](int t0) {
    rk.load(L - t0, p.dk), rq.load(L - t0, p.dk), rv.load(L - t0, p.dv), rdo.load(L - t0, p.dv), rg.load(t0, L - t0, tid);
  };
  if (L > 0) fetch(0);
  f32x4 s[KA][1];
  load_state(s, p.s_in ? p.s_in + bh * ((int64_t)p.dk * p.dv) : nullptr, false, p.dk, p.dv, col0, lo, hi);

  for (int t0 = 0; t0 < L; t0 += C) {
    const int n = min(C, L - t0), chunk = t0 / C;
    rk.store(tk), rq.store(tq), rv.store(tv), rdo.store(tdo), rg.store(d, tid);
    store_columns<E, DK>(a.s + ((int64_t)bh * a.chunks + chunk) * DK * DV, s, col0, lo, hi);
    __syncthreads();
    if (t0 + C < L) fetch(t0 + C);
    for (int sub = wave; 16 * sub < n; sub += S::W) {
      const f32x4 lag = delta_powers<S>(d, sub, lane);
      f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
      for (int m = 0; m < KA; m += 2) {
        const quad_t<E> k0 = lds_quad(tk, LDK, 16 * sub, 16 * m, lane), k1 = lds_quad(tk, LDK, 16 * sub, 16 * m + 16, lane);
        kk = mma2(k0, k1, k0, k1, kk);
        qk = mma2(k0, k1, lds_quad(tq, LDK, 16 * sub, 16 * m, lane), lds_quad(tq, LDK, 16 * sub, 16 * m + 16, lane), qk);
      }
      const f32x4 beta = lds_f4(d.beta + 16 * sub + 4 * hi);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 4 * hi + r;
        kk[r] = j < lo ? kk[r] * __expf(lag[r]) * beta[r] : 0.0f;
        qk[r] = j <= lo ? p.scale * (qk[r] * __expf(lag[r])) : 0.0f;
      }
      *reinterpret_cast<f32x4*>(tp + (16 * sub + lo) * LDT + 4 * hi) = qk;
      delta_inverse<S, false>(d, sub, kk, lane);
    }
    __syncthreads();
    for (int sub = 0; 16 * sub < n; ++sub) {
      f32x4 o = {0, 0, 0, 0};
      const f32x4 ks = delta_state_products<E, KA, Terms<E>::N>(tk, tq, LDK, 16 * sub, s, o, lane);
      const f32x4 v = to_f32(lds_quad_t(tv, LDV, 16 * sub, col0, lane));
      const f32x4 x = v - lds_f4(d.from + 16 * sub + 4 * hi) * ks;
      const f32x4 e = mma16(lds_f4(d.inv + (16 * sub + lo) * LDT + 4 * hi), x, f32x4{0, 0, 0, 0});
      const f32x4 u = lds_f4(d.beta + 16 * sub + 4 * hi) * e;
      // these columns of V are this wave's alone and have been read
#pragma unroll
      for (int r = 0; r < 4; ++r) tv[(16 * sub + 4 * hi + r) * LDV + col0 + lo] = (E)e[r];
      o *= p.scale * d.from[16 * sub + lo];
      o = mma16(u, lds_f4(tp + (16 * sub + lo) * LDT + 4 * hi), o);
      o *= to_f32(lds_quad(tdo, LDV, 16 * sub, col0, lane));
      float w = o[0] + o[1] + o[2] + o[3];
      w += __shfl_xor(w, 16, 64), w += __shfl_xor(w, 32, 64);
      if (hi == 0) sums[wave * C + 16 * sub + lo] = w;
      const Terms<E> du(lds_f4(d.to + 16 * sub + 4 * hi) * u);
      const float total = d.total[sub];
#pragma unroll
      for (int m = 0; m < KA; ++m) s[m][0] = mma_terms(lds_quad_t(tk, LDK, 16 * sub, 16 * m, lane), du, s[m][0] * total);
    }
    if ((chunk + 1) % SEG == 0 || t0 + C >= L) {
      f32x4* dst = reinterpret_cast<f32x4*>(a.s_seg + ((int64_t)bh * a.segs + chunk / SEG) * DK * DV) + wave * KA * 64 + lane;
#pragma unroll
      for (int m = 0; m < KA; ++m) dst[m * 64] = s[m][0];
    }
    __syncthreads();
    copy_out(rv, tv, a.e + ((int64_t)bh * a.chunks + chunk) * C * DV, DV, n, DV);
    if (tid < n) {
      float w = 0.0f;
#pragma unroll
      for (int i = 0; i < S::W; ++i) w += sums[i * C + tid];
      a.w[(int64_t)bh * a.chunks * C + t0 + tid] = w;
    }
  }
}

template <typename E, int DK, int DV>
constexpr size_t delta_reverse_lds() {
  using S = DeltaShape<E, DK, DV>;
  return sizeof(float) * (S::GATES + 2 * S::INV + 2 * S::W * S::C + 8) + sizeof(E) * (2 * S::C * S::LDK + 3 * S::C * S::LDV);
}

template <typename E, int DK, int DV, bool VEC>
__global__ __launch_bounds__((DeltaShape<E, DK, DV>::THREADS)) void delta_reverse_kernel(DeltaBwdArgs<E> a) {
  using S = DeltaShape<E, DK, DV>;
  constexpr int C = S::C, KA = DK / 16, LDK = S::LDK, LDV = S::LDV, LDT = S::LDT, SEG = kDeltaSeg / C;
  extern __shared__ __align__(16) char smem[];
  const DeltaArgs<E>& p = a.f;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4, col0 = wave * 16;
  const int bh = blockIdx.x, b = bh / p.H, h = bh - b * p.H;
  const int L = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const DeltaGates d = delta_gates<S>(reinterpret_cast<float*>(smem));
  float* tp = d.inv + S::INV;         // the blocks' scores, transposed
  float* sum_beta = tp + S::INV;      // (waves, steps)
  float* sum_z = sum_beta + S::W * C;
  float* sum_dot = sum_z + S::W * C;  // (waves)
  E* tk = reinterpret_cast<E*>(sum_dot + 8);
  E* tq = tk + C * LDK;
  E* tv = tq + C * LDK;
  E* tdo = tv + C * LDV;
  E* te = tdo + C * LDV;

  AttnRows<E, C, DK, S::THREADS, VEC> rk, rq;
  AttnRows<E, C, DV, S::THREADS, VEC> rv, rdo;
  AttnRows<E, C, DV, S::THREADS, true> re;
  rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], 0, p.dk, tid);
  rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], 0, p.dk, tid);
  rv.init(p.v + b * p.vs[0] + (h / p.gv) * p.vs[2], p.vs[1], 0, p.dv, tid);
  rdo.init(a.d_o + b * a.dos[0] + h * a.dos[2], a.dos[1], 0, p.dv, tid);
  re.init(a.e + (int64_t)bh * a.chunks * C * DV, DV, 0, DV, tid);
  const E *bk = rk.base, *bq = rq.base, *bv = rv.base, *bdo = rdo.base, *be = re.base;
  DeltaGateRows<E, C> rg{p.g + b * p.gs[0] + h * p.gs[2], p.beta + b * p.bs[0] + h * p.bs[2], p.gs[1], p.bs[1]};
  auto fetch = [&](int t0) {
    rk.base = bk + t0 * p.ks[1], rq.base = bq + t0 * p.qs[1], rv.base = bv + t0 * p.vs[1];
    rdo.base = bdo + t0 * a.dos[1], re.base = be + (int64_t)t0 * DV;
    rk.load(L - t0, p.dk), rq.load(L - t0, p.dk), rv.load(L - t0, p.dv), rdo.load(L - t0, p.dv), re.load(L - t0, DV);
    rg.load(t0, L - t0, tid);
  };
  const int last = L > 0 ? (L - 1) / C : -1;
  if (last >= 0) fetch(last * C);
  const int64_t size = (int64_t)p.dk * p.dv;
  f32x4 s[KA][1];
  load_state(s, a.d_out ? a.d_out + bh * size : nullptr, false, p.dk, p.dv, col0, lo, hi);
  E* yrow = a.y + (a.y_part ? bh * a.ys[0] : b * a.ys[0] + (int64_t)h * p.dv);

  for (int chunk = last; chunk >= 0; --chunk) {
    const int t0 = chunk * C, n = min(C, L - t0);
    rk.store(tk), rq.store(tq), rv.store(tv), rdo.store(tdo), re.store(te), rg.store(d, tid);
    store_columns<E, DK>(a.r + ((int64_t)bh * a.chunks + chunk) * DK * DV, s, col0, lo, hi);
    const bool seg_end = (chunk + 1) % SEG == 0 || chunk == last;
    if (seg_end) {
      const f32x4* src = reinterpret_cast<const f32x4*>(a.s_seg + ((int64_t)bh * a.segs + chunk / SEG) * DK * DV) + wave * KA * 64 + lane;
      float dot = 0.0f;
#pragma unroll
      for (int m = 0; m < KA; ++m) {
        const f32x4 x = src[m * 64];
#pragma unroll
        for (int r = 0; r < 4; ++r) dot += x[r] * s[m][0][r];
      }
#pragma unroll
      for (int i = 32; i; i >>= 1) dot += __shfl_xor(dot, i, 64);
      if (lane == 0) sum_dot[wave] = dot;
    }
    __syncthreads();
    if (seg_end && tid == 0) {
      float dot = 0.0f;
      for (int i = 0; i < S::W; ++i) dot += sum_dot[i];
      a.dot[(int64_t)bh * a.segs + chunk / SEG] = dot;
    }
    if (chunk > 0) fetch(t0 - C);
    for (int sub = wave; 16 * sub < n; sub += S::W) {
      const f32x4 lag = delta_powers<S>(d, sub, lane);
      f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
      for (int m = 0; m < KA; m += 2) {
        const quad_t<E> k0 = lds_quad(tk, LDK, 16 * sub, 16 * m, lane), k1 = lds_quad(tk, LDK, 16 * sub, 16 * m + 16, lane);
        kk = mma2(k0, k1, k0, k1, kk);
        qk = mma2(lds_quad(tq, LDK, 16 * sub, 16 * m, lane), lds_quad(tq, LDK, 16 * sub, 16 * m + 16, lane), k0, k1, qk);
      }
      const float beta = d.beta[16 * sub + lo];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int x = 4 * hi + r;
        kk[r] = x < lo ? kk[r] * __expf(lag[r]) * beta : 0.0f;
        qk[r] = x >= lo ? p.scale * (qk[r] * __expf(-lag[r])) : 0.0f;  // row lo is the key's
      }
      *reinterpret_cast<f32x4*>(tp + (16 * sub + lo) * LDT + 4 * hi) = qk;
      delta_inverse<S, true>(d, sub, kk, lane);
    }
    __syncthreads();
    for (int sub = (n - 1) / 16; sub >= 0; --sub) {
      f32x4 none;
      const f32x4 from = lds_f4(d.from + 16 * sub + 4 * hi);
      const f32x4 g = to_f32(lds_quad_t(tdo, LDV, 16 * sub, col0, lane));
      f32x4 x = lds_f4(d.to + 16 * sub + 4 * hi) * delta_state_products<E, KA, 0>(tk, tq, LDK, 16 * sub, s, none, lane);
      x = mma16(lds_f4(tp + (16 * sub + lo) * LDT + 4 * hi), g, x);
      const f32x4 du = mma16(lds_f4(d.inv + (16 * sub + lo) * LDT + 4 * hi), x, f32x4{0, 0, 0, 0});
      const f32x4 y = lds_f4(d.beta + 16 * sub + 4 * hi) * du;
      const f32x4 pe = du * to_f32(lds_quad_t(te, LDV, 16 * sub, col0, lane));
      const f32x4 pv = y * to_f32(lds_quad_t(tv, LDV, 16 * sub, col0, lane));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 16 * sub + 4 * hi + r;
        const float sb = row16_sum(pe[r]), sz = row16_sum(pv[r]);
        if (lo == 0) sum_beta[wave * C + t] = sb, sum_z[wave * C + t] = sz;
        tdo[t * LDV + col0 + lo] = (E)y[r];  // these columns of dO are this wave's alone and have been read
        if (a.y_part && t < n && col0 + lo < p.dv)
          a.y_part[(((int64_t)b * p.T + t0 + t) * p.H + h) * p.dv + col0 + lo] = y[r];
      }
      const Terms<E> wq(p.scale * from * g), wk(-(from * y));
      const float total = d.total[sub];
#pragma unroll
      for (int m = 0; m < KA; ++m) {
        const quad_t<E> qt = lds_quad_t(tq, LDK, 16 * sub, 16 * m, lane), kt = lds_quad_t(tk, LDK, 16 * sub, 16 * m, lane);
        s[m][0] *= total;
        if constexpr (sizeof(E) == 2) {
#pragma unroll
          for (int t = 0; t < 3; ++t) s[m][0] = mma2(qt, kt, wq.t[t], wk.t[t], s[m][0]);
        } else {
          s[m][0] = mma16(kt, wk.t[0], mma16(qt, wq.t[0], s[m][0]));
        }
      }
    }
    __syncthreads();
    copy_out(rdo, tdo, yrow + t0 * a.ys[1], a.ys[1], n, a.y_width);
    if (tid < n) {
      float sb = 0.0f, sz = 0.0f;
#pragma unroll
      for (int i = 0; i < S::W; ++i) sb += sum_beta[i * C + tid], sz += sum_z[i * C + tid];
      a.dbeta[((int64_t)b * p.T + t0 + tid) * p.H + h] = (E)sb;
      a.z[(int64_t)bh * a.chunks * C + t0 + tid] = sz;
    }
  }
  if (a.d_in) store_state(s, a.d_in + bh * size, p.dk, p.dv, col0, lo, hi);
  for (int t = L + tid; t < p.T; t += S::THREADS) a.dbeta[((int64_t)b * p.T + t) * p.H + h] = E(0.0f);
  const int64_t orow = (int64_t)p.H * p.dv, obase = ((int64_t)b * p.T * p.H + h) * p.dv;
  if (a.y_part) zero_rows(a.y_part, true, 4, obase, orow, p.dv, L, p.T, tid, S::THREADS);
  else zero_rows(a.y, false, sizeof(E), obase, orow, p.dv, L, p.T, tid, S::THREADS);
}

// log_decay's gradient: a wave a stretch, four steps a lane; in 64 bits, for the terms are.
template <typename E>
__global__ __launch_bounds__(64) void delta_dgate_kernel(DeltaBwdArgs<E> a, int rows) {
  const DeltaArgs<E>& p = a.f;
  const int seg = blockIdx.x % a.segs, bh = blockIdx.x / a.segs, b = bh / p.H, h = bh - b * p.H, lane = threadIdx.x;
  const int L = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const int t0 = seg * kDeltaSeg + lane * 4;
  const int64_t at = (int64_t)bh * rows + t0;
  double x[4], sum = 0.0;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    if (t0 + i < L) sum += (double)a.w[at + i] - (double)a.z[at + i];
    x[i] = sum;
  }
  double after = sum;  // this lane's and the later ones' terms
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    const double v = __shfl_down(after, i, 64);
    if (lane + i < 64) after += v;
  }
  after -= sum;
  if (seg * kDeltaSeg < L) after += (double)a.dot[(int64_t)bh * a.segs + seg];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + i;
    if (t >= p.T) break;
    float v = 0.0f;
    if (t < L && !(p.g[b * p.gs[0] + t * p.gs[1] + h * p.gs[2]] < kNoDecay)) v = (float)(after + x[i]);
    a.dg[((int64_t)b * p.T + t) * p.H + h] = v;
  }
}

template <typename E, int DK, int DV>
constexpr size_t delta_dqk_lds() {
  using S = DeltaShape<E, DK, DV>;
  return 8 * S::C + 4 * 3 * S::C + sizeof(E) * (2 * S::C * S::LDK + 3 * S::C * S::LDV + DV * S::LDK);
}

// dq and dk of a chunk: a wave 16 rows (and with fp32 chunks of 32 steps half of the columns).
template <typename E, int DK, int DV, bool VEC>
__global__ __launch_bounds__(256) void delta_dqk_kernel(DeltaBwdArgs<E> a) {
  using S = DeltaShape<E, DK, DV>;
  constexpr int C = S::C, CT = C / 16, WC = 4 / CT, KT = DK / 16 / WC, VA = DV / 16, LDK = S::LDK, LDV = S::LDV;
  extern __shared__ __align__(16) char smem[];
  const DeltaArgs<E>& p = a.f;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4;
  const int chunk = blockIdx.x % a.chunks, bh = blockIdx.x / a.chunks, b = bh / p.H, h = bh - b * p.H;
  const int L = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const int t0 = chunk * C, n = min(C, L - t0);
  const int64_t orow = (int64_t)p.H * p.dk, obase = ((int64_t)b * p.T * p.H + h) * p.dk;
  const int64_t z0 = max(L, t0), z1 = min(p.T, t0 + C);
  zero_rows(a.dq, a.q_part, sizeof(E), obase, orow, p.dk, z0, z1, tid, 256);
  zero_rows(a.dk, a.k_part, sizeof(E), obase, orow, p.dk, z0, z1, tid, 256);
  if (n <= 0) return;
  double* G = reinterpret_cast<double*>(smem);
  float* beta = reinterpret_cast<float*>(G + C);
  float* from = beta + C;
  float* to = from + C;
  E* tk = reinterpret_cast<E*>(to + C);
  E* tq = tk + C * LDK;
  E* tu = tq + C * LDK;
  E* tdo = tu + C * LDV;
  E* ty = tdo + C * LDV;
  E* ts = ty + C * LDV;  // a state or its gradient, (DV, DK)

  AttnRows<E, C, DK, 256, VEC> rk, rq;
  AttnRows<E, C, DV, 256, VEC> rdo;
  AttnRows<E, C, DV, 256, true> re;
  AttnRows<E, C, DV, 256, false> ry;
  rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], t0, p.dk, tid);
  rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], t0, p.dk, tid);
  rdo.init(a.d_o + b * a.dos[0] + h * a.dos[2], a.dos[1], t0, p.dv, tid);
  re.init(a.e + (int64_t)bh * a.chunks * C * DV, DV, t0, DV, tid);
  const E* y = a.y + (a.y_part ? bh * a.ys[0] : b * a.ys[0] + (int64_t)h * p.dv);
  rk.load(n, p.dk), rq.load(n, p.dk), rdo.load(n, p.dv), re.load(n, DV);
  AttnRows<E, C, DV, 256, true> ryv;
  const bool yv = a.y_part || (VEC && p.dv % Elem<E>::PIECE == 0);
  if (yv) ryv.init(y, a.ys[1], t0, a.y_width, tid), ryv.load(n, a.y_width);
  else ry.init(y, a.ys[1], t0, a.y_width, tid), ry.load(n, a.y_width);
  // rows of the state: DV of DK elements, whole pieces
  constexpr int P = Elem<E>::PIECE, SP = (DV * DK / P + 255) / 256;
  piece_t<E> sp[SP];
  const E* src = a.s + ((int64_t)bh * a.chunks + chunk) * DK * DV;
  auto state_load = [&](const E* from_) {
#pragma unroll
    for (int i = 0; i < SP; ++i)
      if ((i * 256 + tid) * P < DV * DK) sp[i] = *reinterpret_cast<const piece_t<E>*>(from_ + (i * 256 + tid) * P);
  };
  auto state_store = [&]() {
#pragma unroll
    for (int i = 0; i < SP; ++i) {
      const int e = (i * 256 + tid) * P;
      if (e < DV * DK) *reinterpret_cast<piece_t<E>*>(ts + e / DK * LDK + e % DK) = sp[i];
    }
  };
  state_load(src);
  if (wave == 0) {
    const bool live = lane < n;
    float g = live ? p.g[b * p.gs[0] + (t0 + lane) * p.gs[1] + h * p.gs[2]] : 0.0f;
    g = g < kNoDecay ? kNoDecay : g;
    double sum = (double)g;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
      const double v = __shfl_up(sum, i, 64);
      if (lane >= i) sum += v;
    }
    const double end = __shfl(sum, 63, 64);
    if (lane < C) {
      G[lane] = sum, from[lane] = __expf((float)sum), to[lane] = __expf((float)(end - sum));
      beta[lane] = live ? (float)p.beta[b * p.bs[0] + (t0 + lane) * p.bs[1] + h * p.bs[2]] : 0.0f;
    }
  }
  rk.store(tk), rq.store(tq), rdo.store(tdo);
  if (yv) ryv.store(ty);
  else ry.store(ty);
  state_store();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < re.N; ++i) {
    const float f = re.row < re.RS ? beta[re.row + i * re.RS] : 0.0f;
#pragma unroll
    for (int e = 0; e < P; ++e) re.r[i][e] = (E)((float)re.r[i][e] * f);
  }
  re.store(tu);
  state_load(a.r + ((int64_t)bh * a.chunks + chunk) * DK * DV);
  __syncthreads();

  const int it = wave / WC, kt0 = (wave % WC) * KT, row = 16 * it + lo;
  const double mine = G[row];
  // the scores as operands: outer index this wave's rows, contracted the chunk's steps
  quad_t<E> m[CT], mt[CT], nn[CT];
#pragma unroll
  for (int jt = 0; jt < CT; ++jt) {
    f32x4 s1 = {0, 0, 0, 0}, s2 = {0, 0, 0, 0}, s3 = {0, 0, 0, 0}, s4 = {0, 0, 0, 0};
    const bool below = jt <= it, above = jt >= it;
#pragma unroll
    for (int v = 0; v < VA; v += 2) {
      auto two = [&](const E* x, int r0, quad_t<E>& x0, quad_t<E>& x1) {
        x0 = lds_quad(x, LDV, r0, 16 * v, lane), x1 = lds_quad(x, LDV, r0, 16 * v + 16, lane);
      };
      quad_t<E> x0, x1, y0, y1;
      if (below) {
        two(tu, 16 * jt, x0, x1);
        two(tdo, 16 * it, y0, y1), s1 = mma2(x0, x1, y0, y1, s1);
        two(ty, 16 * it, y0, y1), s2 = mma2(x0, x1, y0, y1, s2);
      }
      if (above) {
        two(tu, 16 * it, x0, x1);
        two(tdo, 16 * jt, y0, y1), s3 = mma2(y0, y1, x0, x1, s3);
        two(ty, 16 * jt, y0, y1), s4 = mma2(y0, y1, x0, x1, s4);
      }
    }
    f32x4 nsum;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = 16 * jt + 4 * hi + r;
      const float lag = (float)(mine - G[j]);
      const float back = __expf(lag), ahead = __expf(-lag);
      s1[r] = below && j <= row ? p.scale * back * s1[r] : 0.0f;
      s3[r] = above && j >= row ? p.scale * ahead * s3[r] : 0.0f;
      nsum[r] = j < row ? -back * s2[r] : j > row ? -ahead * s4[r] : 0.0f;
    }
    m[jt] = to_quad<E>(s1), mt[jt] = to_quad<E>(s3), nn[jt] = to_quad<E>(nsum);
  }
  f32x4 aq[KT], ak[KT];
  const float ff = from[row], ft = to[row];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    aq[kt] = ak[kt] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < VA; v += 2) {
      const quad_t<E> s0 = lds_quad_t(ts, LDK, 16 * v, 16 * (kt0 + kt), lane);
      const quad_t<E> s1 = lds_quad_t(ts, LDK, 16 * v + 16, 16 * (kt0 + kt), lane);
      aq[kt] = mma2(s0, s1, lds_quad(tdo, LDV, 16 * it, 16 * v, lane), lds_quad(tdo, LDV, 16 * it, 16 * v + 16, lane), aq[kt]);
      ak[kt] = mma2(s0, s1, lds_quad(ty, LDV, 16 * it, 16 * v, lane), lds_quad(ty, LDV, 16 * it, 16 * v + 16, lane), ak[kt]);
    }
    aq[kt] *= p.scale * ff, ak[kt] *= -ff;
  }
  __syncthreads();
  state_store();
  __syncthreads();
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    f32x4 r = {0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < VA; v += 2)
      r = mma2(lds_quad_t(ts, LDK, 16 * v, 16 * (kt0 + kt), lane), lds_quad_t(ts, LDK, 16 * v + 16, 16 * (kt0 + kt), lane),
               lds_quad(tu, LDV, 16 * it, 16 * v, lane), lds_quad(tu, LDV, 16 * it, 16 * v + 16, lane), r);
    ak[kt] += ft * r;
#pragma unroll
    for (int j = 0; j < CT; j += 2) {
      const quad_t<E> k0 = lds_quad_t(tk, LDK, 16 * j, 16 * (kt0 + kt), lane), k1 = lds_quad_t(tk, LDK, 16 * j + 16, 16 * (kt0 + kt), lane);
      const quad_t<E> q0 = lds_quad_t(tq, LDK, 16 * j, 16 * (kt0 + kt), lane), q1 = lds_quad_t(tq, LDK, 16 * j + 16, 16 * (kt0 + kt), lane);
      aq[kt] = mma2(k0, k1, m[j], m[j + 1], aq[kt]);
      ak[kt] = mma2(k0, k1, nn[j], nn[j + 1], ak[kt]);
      ak[kt] = mma2(q0, q1, mt[j], mt[j + 1], ak[kt]);
    }
    if (row < n) {
      const int64_t at = obase + (t0 + row) * orow;
      const int c = 16 * (kt0 + kt) + 4 * hi;
      if (a.q_part) store_quad((float*)a.dq + at, c, p.dk, aq[kt]);
      else store_quad((E*)a.dq + at, c, p.dk, aq[kt]);
      if (a.k_part) store_quad((float*)a.dk + at, c, p.dk, ak[kt]);
      else store_quad((E*)a.dk + at, c, p.dk, ak[kt]);
    }
  }
}

// One step, S := a S + k^T u, u = beta (v - a k S), o = scale q S, in place: a (problem, head) a workgroup, thread
// (row group, 4 columns) with NR rows of S in registers between its one read and its write;
// k S and q S are summed over the row groups in LDS together, o = scale (a q S + (q . k) u).
// Bound by the state's read and write.
template <typename E>
struct DeltaStepArgs {
  int B, H, gq, gk, gv, dk, dv;
  const E *q, *k, *v, *beta;
  const float* g;
  int64_t qs[2], ks[2], vs[2], bs[2], gs[2];  // strides of problem, head
  const uint8_t* active;                      // (B) or NULL
  float scale;
  float* state;  // (B, H, dk, dv)
  E* o;          // (B, H, dv)
};

template <typename E, int NR>
__global__ __launch_bounds__(256) void delta_step_kernel(DeltaStepArgs<E> p) {
  __shared__ float sq[128], sk[128], sdot[4];
  __shared__ f32x4 sks[256], sqs[256];
  const int tid = threadIdx.x, bh = blockIdx.x, b = bh / p.H, h = bh - b * p.H;
  E* o = p.o + (int64_t)bh * p.dv;
  if (p.active && !p.active[b]) {
    for (int c = tid; c < p.dv; c += 256) o[c] = E(0.0f);
    return;
  }
  const int nc = (p.dv + 3) / 4, rg = 256 / nc;  // 4-column groups, rows walked at a time
  const int c = (tid % nc) * 4, r0 = tid / nc;
  float* S = p.state + (int64_t)bh * p.dk * p.dv;
  f32x4 s[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = r0 + i * rg;
    s[i] = r0 < rg && r < p.dk ? load_quad_f32(S + (int64_t)r * p.dv, c, p.dv) : f32x4{0, 0, 0, 0};
  }
  float dot = 0.0f;
  if (tid < p.dk) {
    const float q = (float)p.q[b * p.qs[0] + (h / p.gq) * p.qs[1] + tid], k = (float)p.k[b * p.ks[0] + (h / p.gk) * p.ks[1] + tid];
    sq[tid] = q, sk[tid] = k, dot = q * k;
  }
#pragma unroll
  for (int w = 32; w; w >>= 1) dot += __shfl_xor(dot, w, 64);
  if ((tid & 63) == 0) sdot[tid >> 6] = dot;
  const float a = __expf(p.g[b * p.gs[0] + h * p.gs[1]]), beta = (float)p.beta[b * p.bs[0] + h * p.bs[1]];
  const E* pv = p.v + b * p.vs[0] + (h / p.gv) * p.vs[1];
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = c + e < p.dv ? (float)pv[c + e] : 0.0f;
  __syncthreads();
  f32x4 ks = {0, 0, 0, 0}, qs = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = r0 + i * rg;
    if (r0 < rg && r < p.dk) {
      s[i] *= a;
      ks += sk[r] * s[i], qs += sq[r] * s[i];
    }
  }
  sks[tid] = ks, sqs[tid] = qs;
  __syncthreads();
  if (r0 >= rg) return;
  ks = f32x4{0, 0, 0, 0};
  for (int r = 0; r < rg; ++r) ks += sks[r * nc + c / 4];
  const f32x4 u = beta * (v - ks);
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = r0 + i * rg;
    if (r < p.dk) store_quad(S + (int64_t)r * p.dv, c, p.dv, s[i] + sk[r] * u);
  }
  if (r0 == 0) {
    qs = f32x4{0, 0, 0, 0};
    for (int r = 0; r < rg; ++r) qs += sqs[r * nc + c / 4];
    store_quad(o, c, p.dv, p.scale * (qs + (sdot[0] + sdot[1]) * u));
  }
}

}  // namespace tmpc
