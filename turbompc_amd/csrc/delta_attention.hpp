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

// Block `sub` of a chunk, by one wave: the powers, and the ratio Gamma_ij of a lane's i = lo and
// j = 4 hi + r as exponents' differences (a double each, rounded once).
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
  f32x4 ratio;
#pragma unroll
  for (int r = 0; r < 4; ++r) ratio[r] = __expf((float)(mine - at[r]));
  return ratio;
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
      const f32x4 ratio = delta_powers<S>(d, sub, lane);
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
        kk[r] = j < lo ? kk[r] * ratio[r] * beta[r] : 0.0f;
        qk[r] = j <= lo ? p.scale * (qk[r] * ratio[r]) : 0.0f;
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
