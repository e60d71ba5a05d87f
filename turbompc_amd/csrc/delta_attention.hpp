// Gated delta rule.  Problem b, head h, a_t = exp(g_t) (S fp32, dk x dv):
//   e_t = v_t - a_t k_t S_{t-1},  u_t = beta_t e_t,  S_t = a_t S_{t-1} + k_t^T u_t,  o_t = scale q_t S_t.
//
// Blocks of 16 NB steps, G_i the sum of g up to step i of the block, Gamma_ij = exp(G_i - G_j) for
// j <= i, else 0.  With A_ij = Gamma_ij (k_i . k_j) beta_j for j < i, the block's steps are
//   E = (I + A)^-1 (V - diag(exp G) K S),  U = diag(beta) E,
//   O = scale (diag(exp G) Q S + (Q K^T o Gamma) U),  S := exp(G_end) S + K^T diag(exp(G_end - G)) U.
// The inverses of the 16 x 16 tiles on the diagonal are formed by substitution, row by row: their
// entries stay as small as the recurrence's products of (I - beta k^T k), where a product of powers of A
// would cancel large terms for keys that repeat themselves.  Sums of g are held in 64 bits, so that
// their differences are exact to 32 also behind a decay of zero (g = -inf, taken as -1e5, whose
// exponential is zero).
//
// Blocks are short, so that the chain from state to state stays in a wave's registers: S is the
// operand of K S, whose result is the operand of the product with the inverse, whose result is the operand
// of the state's update.  A wave owns 16 columns of the values and walks its head's blocks without
// meeting the other waves; what depends on the block alone (the inverse, Q K^T o Gamma, the powers) is
// made once a chunk of several blocks, the waves sharing it out, in LDS.  In bf16 the state, an fp32
// result, enters products as three bf16 terms (24 bits); a block has two tiles there, so that they are
// formed half as often.
//
// Backward.  With R_t = dL/dS_t from later steps, D_t = R_t + scale q_t^T do_t:
//   du_t = k_t D_t,  y_t = dv_t = beta_t du_t,  R_{t-1} = a_t (D_t - k_t^T y_t),  dbeta_t = du_t . e_t,
//   dq_t = scale do_t S_t^T,  dk_t = u_t D_t^T - a_t y_t S_{t-1}^T,  dg_t = <R_{t-1}, S_{t-1}>.
#pragma once
#include <type_traits>

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
  int vec;            // rows of whole pieces at 4-byte addresses, all operands'
  const float* s_in;  // (B, H, dk, dv) or NULL
  float* s_out;       // (B, H, dk, dv) or NULL
  E* o;               // (B, T, H, dv)
  int segs, seg_len;  // the steps in segs runs of seg_len (a multiple of kDeltaSeg)
  float* seg_state;   // segs > 1: (B H, segs, DK, DV): each run's own sum, then the state it starts from
  float* seg_map;     // segs > 1: (B H, segs, DK, DK): what a run does to the state it starts from
};
constexpr int kDeltaSeg = 256;  // steps

template <typename E>
__device__ inline int delta_length(const DeltaArgs<E>& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
}

template <typename E, int DK, int DV>
struct DeltaShape {
  static constexpr int W = DV / 16, THREADS = 64 * W;  // a wave 16 value columns
  static constexpr int C = AttnTile<E>::C, PAD = AttnTile<E>::PAD;
  static constexpr int NB = sizeof(E) == 2 ? 2 : 1, BS = 16 * NB, NBLK = C / BS, TRI = NB * (NB + 1) / 2;
  static constexpr int LDK = DK + PAD, LDV = DV + PAD;
  static constexpr int LDT = 20, TILE = 16 * LDT;  // a 16 x 16 fp32 tile, its quads spread over the banks
  static constexpr int LDP = sizeof(E) == 2 ? 24 : 20, TILE_P = 16 * LDP;  // one of E
  static constexpr int GATES = 2 * C + 3 * C + 4;  // floats
  static constexpr int INV = NBLK * TRI * TILE, SCORES = NBLK * TRI * TILE_P;
  // waves of a SIMD that the registers hold
  static constexpr int WAVES_FORWARD = DK <= 64 ? (W == 8 ? 4 : 3) : 2, WAVES_BACKWARD = DK <= 64 ? 3 : 2;
};
// tile (i, j <= i) of a block
constexpr int tri(int i, int j) { return i * (i + 1) / 2 + j; }

__device__ inline f32x4 lds_f4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }

// acc += A B over 16 contracted entries in fp32 (a quad of each operand)
__device__ inline f32x4 mma16(f32x4 a, f32x4 b, f32x4 acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], acc, 0, 0, 0);
  return acc;
}

// The same value, which the compiler takes for another: what is computed from it is computed where it is
// used, and not before the loop around, to be kept in (or spilled from) registers through all of it.
__device__ inline int here(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// A chunk's gates in LDS: the sums of g from each block's start, beta (zeros past the last live
// step), exp(G), exp(G_end - G), exp(G_end).
struct DeltaGates {
  double* G;
  float *beta, *from, *to, *total;
};
template <typename S>
__device__ inline DeltaGates delta_gates(char* base) {
  DeltaGates d;
  d.G = reinterpret_cast<double*>(base), d.beta = reinterpret_cast<float*>(d.G + S::C);
  d.from = d.beta + S::C, d.to = d.from + S::C, d.total = d.to + S::C;
  return d;
}

template <int CTRL>
__device__ inline double dpp_f64(double v) {  // zero where there is no such lane
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t l = __builtin_amdgcn_update_dpp(0, (uint32_t)u, CTRL, 0xf, 0xf, true);
  const uint32_t h = __builtin_amdgcn_update_dpp(0, (uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)h << 32 | l);
}
__device__ inline double lane_f64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t l = __builtin_amdgcn_readlane((uint32_t)u, lane), h = __builtin_amdgcn_readlane((uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)h << 32 | l);
}

// The chunk's gates on their way from memory to LDS: the first wave's lanes a step each.
template <typename E, typename S>
struct DeltaGateRows {
  const float* g;
  const E* beta;
  int64_t gs, bs;
  float vg, vb;
  __device__ void load(int t0, int n, int tid) {
    vg = vb = 0.0f;
    if (tid < n && tid < S::C) vg = g[(t0 + tid) * gs], vb = (float)beta[(t0 + tid) * bs];
  }
  __device__ void store(const DeltaGates& d, int tid) const {
    if (tid >= 64) return;
    double x = vg < kNoDecay ? kNoDecay : vg;
    x += dpp_f64<0x111>(x);  // within 16 lanes
    x += dpp_f64<0x112>(x);
    x += dpp_f64<0x114>(x);
    x += dpp_f64<0x118>(x);
    double end;
    const double e0 = lane_f64(x, 15), e1 = lane_f64(x, 31), e2 = lane_f64(x, 47), e3 = lane_f64(x, 63);
    if constexpr (S::NB == 2) {
      if (tid & 16) x += tid & 32 ? e2 : e0;
      end = tid & 32 ? e2 + e3 : e0 + e1;
    } else {
      end = tid & 32 ? (tid & 16 ? e3 : e2) : (tid & 16 ? e1 : e0);
    }
    if (tid < S::C) {
      d.G[tid] = x, d.beta[tid] = vb, d.from[tid] = __expf((float)x), d.to[tid] = __expf((float)(end - x));
      if (tid % S::BS == 0) d.total[tid / S::BS] = __expf((float)end);
    }
  }
};

// G_i - G_j for a lane's i = i0 + lo and j = j0 + 4 hi + r
__device__ inline f32x4 delta_lag(const DeltaGates& d, int i0, int j0, int lane) {
  const double mine = d.G[i0 + (lane & 15)];
  const double* at = d.G + j0 + 4 * (lane >> 4);
  f32x4 lag;
#pragma unroll
  for (int r = 0; r < 4; ++r) lag[r] = (float)(mine - at[r]);
  return lag;
}

// (X Y^T)^T of 16 rows of each: lane lo has row y0 + lo of Y, and of X rows x0 + 4 hi + r
template <typename E, int D>
__device__ inline f32x4 row_products(const E* x, int x0, const E* y, int y0, int ld, int lane) {
  f32x4 t = {0, 0, 0, 0};
#pragma unroll
  for (int m = 0; m < D; m += 32)
    t = mma2(lds_quad(x, ld, x0, m, lane), lds_quad(x, ld, x0, m + 16, lane), lds_quad(y, ld, y0, m, lane),
             lds_quad(y, ld, y0, m + 16, lane), t);
  return t;
}

// f(0) ... f(N - 1) with constants
template <int N, typename F, int I = 0>
__device__ inline void steps(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    steps<N, F, I + 1>(f);
  }
}
// lane I's of each 16
template <int I>
__device__ inline float row_lane(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x150 + I, 0xf, 0xf, true));
}

// The inverse of I + A for block `blk` of a chunk, by one wave, into its tiles at `inv`.  A_ij has
// beta_j, or with REVERSE beta_i, and the inverse's transpose is left.
template <typename E, typename S, int DK, bool REVERSE>
__device__ inline void delta_inverse(const DeltaGates& d, float* inv, const E* tk, int blk, int lane) {
  constexpr int NB = S::NB, LDT = S::LDT;
  const int lo = lane & 15, hi = lane >> 4, r0 = blk * S::BS;
  float* tiles = inv + blk * S::TRI * S::TILE;
  auto a_tile = [&](int i, int j) {
    f32x4 a = row_products<E, DK>(tk, r0 + 16 * j, tk, r0 + 16 * i, S::LDK, lane);
    const f32x4 lag = delta_lag(d, r0 + 16 * i, r0 + 16 * j, lane);
    const float bi = d.beta[r0 + 16 * i + lo];
    const f32x4 bj = lds_f4(d.beta + r0 + 16 * j + 4 * hi);
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] = i > j || 4 * hi + r < lo ? a[r] * __expf(lag[r]) * (REVERSE ? bi : bj[r]) : 0.0f;
    return a;
  };
  auto rows = [&](int k) { return reinterpret_cast<f32x4*>(tiles + k * S::TILE + lo * LDT + 4 * hi); };
  auto columns = [&](int k) { return lds_quad_t(tiles + k * S::TILE, LDT, 0, 0, lane); };
  f32x4 a10, a[NB][4], t[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) *rows(tri(i, i)) = a_tile(i, i);
  if constexpr (NB == 2) a10 = a_tile(1, 0);
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < NB; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) a[i][j] = lds_f4(tiles + tri(i, i) * S::TILE + lo * LDT + 4 * j);  // row lo
#pragma unroll
    for (int r = 0; r < 4; ++r) t[i][r] = 4 * hi + r == lo ? 1.0f : 0.0f;
  }
  // row lo of the inverse, columns 4 hi + r: takes off A[lo][j] times row j, which is final by then
  steps<15>([&](auto j) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) t[i][r] = fmaf(-a[i][j() / 4][j() % 4], row_lane<j()>(t[i][r]), t[i][r]);
  });
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < NB; ++i) *rows(tri(i, i)) = t[i];
  f32x4 corner;
  if constexpr (NB == 2) {  // the corner: -T11 A10 T00
    __builtin_amdgcn_wave_barrier();
    const f32x4 zero = {0, 0, 0, 0}, y = mma16(a10, columns(tri(0, 0)), zero);
    corner = REVERSE ? -mma16(t[1], y, zero) : -mma16(y, t[1], zero);
    *rows(tri(1, 0)) = corner;
  }
  if constexpr (REVERSE) {
    __builtin_amdgcn_wave_barrier();
    f32x4 c[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) c[i] = columns(tri(i, i));
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < NB; ++i) *rows(tri(i, i)) = c[i];
  }
}

// A chunk's rows of one operand on their way from memory through registers to LDS, as AttnRows moves
// them; whether they are whole pieces at 4-byte addresses is asked at run time (a variant of every kernel for
// it would double what there is to compile).
template <typename E, int C, int D, int THREADS>
struct DeltaRows {
  static constexpr int P = Elem<E>::PIECE, W = D / P, RS = THREADS / W < C ? THREADS / W : C, N = C / RS;
  static constexpr int LD = D + AttnTile<E>::PAD;
  static_assert(THREADS % W == 0 && C % RS == 0, "whole rows a pass");
  piece_t<E> r[N];
  const E* base;  // step 0
  int64_t step;   // elements between steps
  int width, row, c;
  bool vec;

  __device__ void init(const E* b, int64_t stride, int d, bool whole, int tid) {
    row = tid / W, c = (tid - row * W) * P, step = stride, base = b, width = d, vec = whole;
  }
  // rows t0 ..., n of them live (zeros behind them)
  __device__ void load(int t0, int n) {
    const __amdgpu_buffer_rsrc_t rs = buffer_at(base + t0 * step);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int t = row + i * RS;
      const unsigned at = t < n && c < width && row < RS ? (unsigned)((t * step + c) * (int64_t)sizeof(E)) : kNowhere;
      if (vec) {
        r[i] = __builtin_bit_cast(piece_t<E>, __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0));
      } else {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const unsigned ae = c + e < width && at != kNowhere ? at + e * (unsigned)sizeof(E) : kNowhere;
          if constexpr (sizeof(E) == 4)
            r[i][e] = __builtin_bit_cast(float, (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rs, ae, 0, 0));
          else
            r[i][e] = __builtin_bit_cast(bf16, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rs, ae, 0, 0));
        }
      }
    }
  }
  __device__ void store(E* tile) const {
    if (RS * W < THREADS && row >= RS) return;
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<piece_t<E>*>(tile + (row + i * RS) * LD + c) = r[i];
  }
};

// x (fp32) as an operand of products whose other operand is exact in E: itself, or three bf16 terms, the
// upper 8 bits of what is left each time (24 bits together; cut off, not rounded: the terms' sum is
// exact all the same, and a pair of them is one byte permutation).
template <typename E>
struct Terms;
template <>
struct Terms<float> {
  static constexpr int N = 1;
  f32x4 t[1];
  __device__ Terms() {}
  __device__ Terms(f32x4 x) : t{x} {}
};
template <>
struct Terms<bf16> {
  static constexpr int N = 3;
  bf16x4 t[3];
  __device__ Terms() {}
  __device__ Terms(f32x4 x) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const u4 b = __builtin_bit_cast(u4, x);
      const u32x2 p = {__builtin_amdgcn_perm(b[1], b[0], 0x07060302u), __builtin_amdgcn_perm(b[3], b[2], 0x07060302u)};
      t[i] = __builtin_bit_cast(bf16x4, p);
      if (i < 2) x -= __builtin_bit_cast(f32x4, b & 0xffff0000u);
    }
  }
};

// acc += sum over NB tiles of A_i x_i, 16 contracted entries each, x by its terms
template <int NB>
__device__ inline f32x4 mma_terms(const bf16x4 (&a)[NB], const Terms<bf16> (&x)[NB], f32x4 acc) {
  static_assert(NB == 2, "pairs");
#pragma unroll
  for (int t = 0; t < 3; ++t) acc = mma2(a[0], a[1], x[0].t[t], x[1].t[t], acc);
  return acc;
}
template <int NB>
__device__ inline f32x4 mma_terms(const f32x4 (&a)[NB], const Terms<float> (&x)[NB], f32x4 acc) {
#pragma unroll
  for (int i = 0; i < NB; ++i) acc = mma16(a[i], x[i].t[0], acc);
  return acc;
}

// For the block's tiles i: K_i s (16 rows, the wave's 16 columns) exact to fp32, and with OT > 0
// (Q_i s)^T by s's first OT terms.
template <typename E, typename S, int KA, int OT>
__device__ inline void delta_state_products(const E* k, const E* q, int row0, const f32x4 (&s)[KA][1], f32x4 (&ks)[S::NB],
                                            f32x4 (&qs)[S::NB], int lane) {
#pragma unroll
  for (int i = 0; i < S::NB; ++i) ks[i] = qs[i] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int m = 0; m < KA; m += 2) {
    const Terms<E> a(s[m][0]), b(s[m + 1][0]);
#pragma unroll
    for (int i = 0; i < S::NB; ++i) {
      const int r0 = row0 + 16 * i;
      const quad_t<E> k0 = lds_quad(k, S::LDK, r0, 16 * m, lane), k1 = lds_quad(k, S::LDK, r0, 16 * m + 16, lane);
#pragma unroll
      for (int t = 0; t < Terms<E>::N; ++t) ks[i] = mma2(k0, k1, a.t[t], b.t[t], ks[i]);
      if constexpr (OT > 0) {
        const quad_t<E> q0 = lds_quad(q, S::LDK, r0, 16 * m, lane), q1 = lds_quad(q, S::LDK, r0, 16 * m + 16, lane);
#pragma unroll
        for (int t = 0; t < OT; ++t) qs[i] = mma2(a.t[t], b.t[t], q0, q1, qs[i]);
      }
    }
  }
}

// e = (I + A)^-1 x over the block's tiles, from the inverse's tiles or with REVERSE its transpose's
template <typename S, bool REVERSE>
__device__ inline void delta_solve(const float* tiles, const f32x4 (&x)[S::NB], f32x4 (&e)[S::NB], int lane) {
  const float* at = tiles + (lane & 15) * S::LDT + 4 * (lane >> 4);
#pragma unroll
  for (int i = 0; i < S::NB; ++i) {
    e[i] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < S::NB; ++j)
      if (REVERSE ? j >= i : j <= i) e[i] = mma16(lds_f4(at + (REVERSE ? tri(j, i) : tri(i, j)) * S::TILE), x[j], e[i]);
  }
}

// A wave's columns of a history whose state is not finite in the end, by the definition, a step at
// a time: in a block such a step meets the earlier ones with factors of zero, which makes those NaN.
template <typename E, int KA, int DV>
__device__ __attribute__((always_inline)) inline void delta_by_step(const DeltaArgs<E>& p, int block, int tid) {
  const int lo = tid & 15, hi = (tid & 63) >> 4, col0 = (tid >> 6) * 16, c = col0 + lo;
  const int bh = block / p.segs, seg = block - bh * p.segs, b = bh / p.H, h = bh - b * p.H;
  const int L = delta_length(p, b);
  const E* pq = p.q + b * p.qs[0] + (h / p.gq) * p.qs[2];
  const E* pk = p.k + b * p.ks[0] + (h / p.gk) * p.ks[2];
  const E* pv = p.v + b * p.vs[0] + (h / p.gv) * p.vs[2];
  const E* pb = p.beta + b * p.bs[0] + h * p.bs[2];
  const float* pg = p.g + b * p.gs[0] + h * p.gs[2];
  const int64_t size = (int64_t)p.dk * p.dv;
  f32x4 s[KA][1];
  if (p.segs > 1) load_state(s, p.seg_state + block * (int64_t)(KA * 16 * DV), false, KA * 16, DV, col0, lo, hi);
  else load_state(s, p.s_in ? p.s_in + bh * size : nullptr, false, p.dk, p.dv, col0, lo, hi);
  for (int t = seg * p.seg_len; t < min(L, (seg + 1) * p.seg_len); ++t) {
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
  if (p.s_out && seg == (L - 1) / p.seg_len) store_state(s, p.s_out + bh * size, p.dk, p.dv, col0, lo, hi);
}

template <typename E, int DK, int DV>
constexpr size_t delta_forward_lds() {
  using S = DeltaShape<E, DK, DV>;
  return sizeof(float) * (S::GATES + S::INV) + sizeof(E) * (S::SCORES + 2 * S::C * S::LDK + S::C * S::LDV);
}

// A workgroup a run of a (problem, head).
template <typename E, int DK, int DV>
__global__ __launch_bounds__((DeltaShape<E, DK, DV>::THREADS), (DeltaShape<E, DK, DV>::WAVES_FORWARD)) void delta_forward_kernel(
    DeltaArgs<E> p) {
  using S = DeltaShape<E, DK, DV>;
  constexpr int C = S::C, NB = S::NB, KA = DK / 16, LDK = S::LDK, LDV = S::LDV, LDP = S::LDP;
  extern __shared__ __align__(16) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4, col0 = wave * 16;
  const int bh = blockIdx.x / p.segs, seg = blockIdx.x - bh * p.segs, b = bh / p.H, h = bh - b * p.H;
  const int begin = seg * p.seg_len, L = min(delta_length(p, b), begin + p.seg_len);  // the run's end
  const DeltaGates d = delta_gates<S>(smem);
  float* inv = reinterpret_cast<float*>(smem) + S::GATES;
  E* tp = reinterpret_cast<E*>(inv + S::INV);  // the blocks' scores
  E* tk = tp + S::SCORES;
  E* tq = tk + C * LDK;
  E* tv = tq + C * LDK;

  DeltaRows<E, C, DK, S::THREADS> rk, rq;
  DeltaRows<E, C, DV, S::THREADS> rv;
  rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], p.dk, p.vec, tid);
  rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], p.dk, p.vec, tid);
  rv.init(p.v + b * p.vs[0] + (h / p.gv) * p.vs[2], p.vs[1], p.dv, p.vec, tid);
  DeltaGateRows<E, S> rg{p.g + b * p.gs[0] + h * p.gs[2], p.beta + b * p.bs[0] + h * p.bs[2], p.gs[1], p.bs[1]};
  auto fetch = [&](int t0) {
    rk.load(t0, L - t0), rq.load(t0, L - t0), rv.load(t0, L - t0), rg.load(t0, L - t0, tid);
  };
  if (begin < L) fetch(begin);
  f32x4 s[KA][1];
  if (p.segs > 1) load_state(s, p.seg_state + blockIdx.x * (int64_t)(DK * DV), false, DK, DV, col0, lo, hi);
  else load_state(s, p.s_in ? p.s_in + bh * ((int64_t)p.dk * p.dv) : nullptr, false, p.dk, p.dv, col0, lo, hi);
  const int64_t orow = (int64_t)p.H * p.dv, obase = ((int64_t)b * p.T * p.H + h) * p.dv;
  const int oc = col0 + 4 * hi;
  const unsigned ooff = oc < p.dv ? (unsigned)((lo * orow + oc) * sizeof(E)) : kNowhere;
  const unsigned otile = (unsigned)(16 * orow * sizeof(E));

  for (int t0 = begin; t0 < L; t0 += C) {
    const int n = min(C, L - t0);
    rk.store(tk), rq.store(tq), rv.store(tv), rg.store(d, tid);
    __syncthreads();
    for (int task = wave; task < 2 * S::NBLK; task += S::W) {
      const int blk = task % S::NBLK, r0 = blk * S::BS, lane = here(tid & 63), lo = lane & 15, hi = lane >> 4;
      if (r0 >= n) continue;
      if (task < S::NBLK) {
        delta_inverse<E, S, DK, false>(d, inv, tk, blk, lane);
        continue;
      }
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j <= i; ++j) {
          f32x4 x = row_products<E, DK>(tk, r0 + 16 * j, tq, r0 + 16 * i, LDK, lane);
          const f32x4 lag = delta_lag(d, r0 + 16 * i, r0 + 16 * j, lane);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = i > j || 4 * hi + r <= lo ? p.scale * (x[r] * __expf(lag[r])) : 0.0f;
          *reinterpret_cast<quad_t<E>*>(tp + (blk * S::TRI + tri(i, j)) * S::TILE_P + lo * LDP + 4 * hi) = to_quad<E>(x);
        }
    }
    __syncthreads();
    if (t0 + C < L) fetch(t0 + C);
    const __amdgpu_buffer_rsrc_t rs = buffer_at(p.o + obase + t0 * orow);
#pragma unroll 1
    for (int blk = 0; blk * S::BS < n; ++blk) {
      const int r0 = blk * S::BS, lane = here(tid & 63), lo = lane & 15, hi = lane >> 4, col0 = here(wave) * 16;
      f32x4 o[NB], x[NB], u[NB];
      delta_state_products<E, S, KA, Terms<E>::N == 3 ? 2 : 1>(tk, tq, r0, s, x, o, lane);
#pragma unroll
      for (int i = 0; i < NB; ++i)
        x[i] = to_f32(lds_quad_t(tv, LDV, r0 + 16 * i, col0, lane)) - lds_f4(d.from + r0 + 16 * i + 4 * hi) * x[i];
      delta_solve<S, false>(inv + blk * S::TRI * S::TILE, x, u, lane);
      Terms<E> w[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        u[i] *= lds_f4(d.beta + r0 + 16 * i + 4 * hi);
        w[i] = Terms<E>(lds_f4(d.to + r0 + 16 * i + 4 * hi) * u[i]);
      }
      const float total = d.total[blk];
#pragma unroll
      for (int m = 0; m < KA; ++m) {
        quad_t<E> kt[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) kt[i] = lds_quad_t(tk, LDK, r0 + 16 * i, 16 * m, lane);
        s[m][0] = mma_terms(kt, w, s[m][0] * total);
      }
      // outputs, bf16: the scores are rounded, the state and u enter by two terms (16 bits)
      Terms<E> ut[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) ut[i] = Terms<E>(u[i]);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        o[i] *= p.scale * d.from[r0 + 16 * i + lo];
        const E* pt = tp + (blk * S::TRI + tri(i, 0)) * S::TILE_P + lo * LDP + 4 * hi;
#pragma unroll
        for (int j = 0; j <= i; ++j) {
          const quad_t<E> pq = *reinterpret_cast<const quad_t<E>*>(pt + j * S::TILE_P);
          if constexpr (sizeof(E) == 2) o[i] = mma2(ut[j].t[0], ut[j].t[1], pq, pq, o[i]);
          else o[i] = mma16(u[j], pq, o[i]);
        }
        const unsigned at = r0 + 16 * i + lo < n && ooff != kNowhere ? ooff + (blk * NB + i) * otile : kNowhere;
        if (p.vec) {
          if constexpr (sizeof(E) == 4) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o[i]), rs, at, 0, 0);
          else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, to_bf16(o[i])), rs, at, 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned ae = oc + e < p.dv && at != kNowhere ? at + e * (unsigned)sizeof(E) : kNowhere;
            const float f = o[i][e];
            if constexpr (sizeof(E) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, f), rs, ae, 0, 0);
            else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (bf16)f), rs, ae, 0, 0);
          }
        }
      }
    }
    __syncthreads();
  }
  // What follows makes its indexes and reads its arguments again: they would be kept through every chunk.
  auto* args = __builtin_amdgcn_kernarg_segment_ptr();
  int etid = tid, block = blockIdx.x;
  asm volatile("" : "+v"(etid), "+s"(args), "+s"(block));
  const DeltaArgs<E>& a = *(const DeltaArgs<E>*)args;
  const int ebh = block / a.segs, eseg = block - ebh * a.segs, eb = ebh / a.H, eL = delta_length(a, eb);
  const int ebegin = eseg * a.seg_len;
  zero_rows(a.o, false, sizeof(E), ((int64_t)eb * a.T * a.H + (ebh - eb * a.H)) * a.dv, (int64_t)a.H * a.dv, a.dv, max(eL, ebegin),
            min((int64_t)a.T, (int64_t)ebegin + a.seg_len), etid, S::THREADS);
  // An infinite or NaN value leaves the state so, to the end.
  f32x4 zero = {0, 0, 0, 0};
#pragma unroll
  for (int m = 0; m < KA; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) zero[r] = fmaf(s[m][0][r], 0.0f, zero[r]);
  if (ebegin < eL && __ballot(!(zero[0] + zero[1] + zero[2] + zero[3] == 0.0f))) {
    __threadfence_block();  // rows written above are written again
    delta_by_step<E, KA, DV>(a, block, etid);
  } else if (a.s_out && eseg == (eL > 0 ? (eL - 1) / a.seg_len : 0)) {  // the run that holds the last live step
    store_state(s, a.s_out + ebh * ((int64_t)a.dk * a.dv), a.dk, a.dv, (etid >> 6) * 16, etid & 15, (etid & 63) >> 4);
  }
}

// A long history of few heads does not fill the chip: it is cut into runs.  A run is a linear map of the
// state it starts from, S -> M S + N: a first pass makes each run's M (its columns start from the unit
// matrix, with values of zero) and N (from zero), a scan carries the states through, and the outputs
// start from those.  A wave 16 columns of [N | M].
template <typename E, int DK>
constexpr size_t delta_run_lds() {
  using S = DeltaShape<E, DK, 64>;
  return sizeof(float) * (S::GATES + S::INV) + sizeof(E) * (S::C * S::LDK + S::C * S::LDV);
}
template <typename E, int DK>
__global__ __launch_bounds__(256, DK <= 64 ? 3 : 2) void delta_run_kernel(DeltaArgs<E> p, int DV) {
  using S = DeltaShape<E, DK, 64>;
  constexpr int C = S::C, NB = S::NB, KA = DK / 16, LDK = S::LDK, LDV = S::LDV;
  extern __shared__ __align__(16) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4;
  const int bh = blockIdx.x / p.segs, seg = blockIdx.x - bh * p.segs, b = bh / p.H, h = bh - b * p.H;
  const int begin = seg * p.seg_len, L = min(delta_length(p, b), begin + p.seg_len);
  const int tile = blockIdx.y * 4 + wave, unit = tile * 16 - DV;  // the first of its columns of the unit matrix
  const DeltaGates d = delta_gates<S>(smem);
  float* inv = reinterpret_cast<float*>(smem) + S::GATES;
  E* tk = reinterpret_cast<E*>(inv + S::INV);
  E* tv = tk + C * LDK;
  DeltaRows<E, C, DK, 256> rk;
  DeltaRows<E, C, 64, 256> rv;
  const int c0 = blockIdx.y * 64;
  rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], p.dk, p.vec, tid);
  rv.init(p.v + b * p.vs[0] + (h / p.gv) * p.vs[2] + min(c0, p.dv), p.vs[1], min(max(p.dv - c0, 0), 64), p.vec, tid);
  DeltaGateRows<E, S> rg{p.g + b * p.gs[0] + h * p.gs[2], p.beta + b * p.bs[0] + h * p.bs[2], p.gs[1], p.bs[1]};
  auto fetch = [&](int t0) { rk.load(t0, L - t0), rv.load(t0, L - t0), rg.load(t0, L - t0, tid); };
  if (begin < L) fetch(begin);
  f32x4 s[KA][1];
#pragma unroll
  for (int m = 0; m < KA; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) s[m][0][r] = 16 * m + 4 * hi + r == unit + lo ? 1.0f : 0.0f;
  for (int t0 = begin; t0 < L; t0 += C) {
    const int n = min(C, L - t0);
    rk.store(tk), rv.store(tv), rg.store(d, tid);
    __syncthreads();
    if (wave < S::NBLK && wave * S::BS < n) delta_inverse<E, S, DK, false>(d, inv, tk, wave, here(lane));
    __syncthreads();
    if (t0 + C < L) fetch(t0 + C);
#pragma unroll 1
    for (int blk = 0; blk * S::BS < n; ++blk) {
      const int r0 = blk * S::BS, lane = here(tid & 63), hi = lane >> 4, col0 = here(wave) * 16;
      f32x4 none[NB], x[NB], u[NB];
      delta_state_products<E, S, KA, 0>(tk, tk, r0, s, x, none, lane);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const f32x4 v = to_f32(lds_quad_t(tv, LDV, r0 + 16 * i, col0, lane));  // zeros for the unit matrix' columns
        x[i] = v - lds_f4(d.from + r0 + 16 * i + 4 * hi) * x[i];
      }
      delta_solve<S, false>(inv + blk * S::TRI * S::TILE, x, u, lane);
      Terms<E> w[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i)
        w[i] = Terms<E>(lds_f4(d.to + r0 + 16 * i + 4 * hi) * (lds_f4(d.beta + r0 + 16 * i + 4 * hi) * u[i]));
      const float total = d.total[blk];
#pragma unroll
      for (int m = 0; m < KA; ++m) {
        quad_t<E> kt[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) kt[i] = lds_quad_t(tk, LDK, r0 + 16 * i, 16 * m, lane);
        s[m][0] = mma_terms(kt, w, s[m][0] * total);
      }
    }
    __syncthreads();
  }
  if (unit >= 0) {
    if (unit < DK) store_state(s, p.seg_map + blockIdx.x * (int64_t)(DK * DK), DK, DK, unit, lo, hi);
  } else {
    store_state(s, p.seg_state + blockIdx.x * (int64_t)(DK * DV), DK, DV, tile * 16, lo, hi);
  }
}

// The same backwards in time: what a run adds to the gradient of the state that it starts from.
template <typename E, int DK>
constexpr size_t delta_reverse_run_lds() {
  using S = DeltaShape<E, DK, 64>;
  return sizeof(float) * (S::GATES + S::INV) + sizeof(E) * (Terms<E>::N * S::SCORES + 2 * S::C * S::LDK + S::C * S::LDV);
}

// Between the passes: each run's sum becomes the state it starts from (REVERSE: the state's gradient
// that it ends with, through the maps' transposes), for 16 columns a workgroup; its waves share the rows out.
template <int DK, bool REVERSE>
__global__ __launch_bounds__(256) void delta_scan_kernel(const float* map, float* state, int segs, int DV, const float* start,
                                                         int dk, int dv) {
  constexpr int KA = DK / 16, MT = (KA + 3) / 4, LD = DK + 4;
  __shared__ __align__(16) float ts[2][16 * LD];  // (column, row)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4;
  const int tiles = DV / 16, bh = blockIdx.x / tiles, col = (blockIdx.x - bh * tiles) * 16 + lo;
  map += (int64_t)bh * segs * DK * DK, state += (int64_t)bh * segs * DK * DV;
  const int first = REVERSE ? segs - 1 : 0, dir = REVERSE ? -1 : 1;
  f32x4 a[MT][KA], n[MT], s[MT];
  auto load = [&](int seg) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = wave + 4 * i;
      if (m >= KA) continue;
#pragma unroll
      for (int k = 0; k < KA; ++k) {
        const float* x = map + (int64_t)seg * DK * DK;
        if constexpr (REVERSE) {
#pragma unroll
          for (int r = 0; r < 4; ++r) a[i][k][r] = x[(16 * k + 4 * hi + r) * DK + 16 * m + lo];
        } else {
          a[i][k] = *reinterpret_cast<const f32x4*>(x + (16 * m + lo) * DK + 16 * k + 4 * hi);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) n[i][r] = state[(int64_t)seg * DK * DV + (16 * m + 4 * hi + r) * DV + col];
    }
  };
  load(first);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * (wave + 4 * i) + 4 * hi + r;
      s[i][r] = start && row < dk && col < dv ? start[((int64_t)bh * dk + row) * dv + col] : 0.0f;
    }
  for (int j = 0; j < segs; ++j) {
    const int seg = first + dir * j;
    float* t = ts[j & 1];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = wave + 4 * i;
      if (m < KA) *reinterpret_cast<f32x4*>(t + lo * LD + 16 * m + 4 * hi) = s[i];
    }
    __syncthreads();
    f32x4 all[KA];
#pragma unroll
    for (int k = 0; k < KA; ++k) all[k] = lds_f4(t + lo * LD + 16 * k + 4 * hi);
    f32x4 next[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = wave + 4 * i;
      if (m >= KA) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) state[(int64_t)seg * DK * DV + (16 * m + 4 * hi + r) * DV + col] = s[i][r];
      next[i] = n[i];
#pragma unroll
      for (int k = 0; k < KA; ++k) next[i] = mma16(a[i][k], all[k], next[i]);
    }
    if (j + 1 < segs) load(seg + dir);
#pragma unroll
    for (int i = 0; i < MT; ++i) s[i] = next[i];
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
  float* r_seg;        // f.segs > 1: as f.seg_state, of the state's gradient at the runs' ends
  void *dq, *dk;       // (B, T, H, dk) of E, or fp32 parts
  int q_part, k_part;
};
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

template <typename E, int DK, int DV>
__global__ __launch_bounds__((DeltaShape<E, DK, DV>::THREADS), (DeltaShape<E, DK, DV>::WAVES_BACKWARD)) void delta_states_kernel(
    DeltaBwdArgs<E> a) {
  using S = DeltaShape<E, DK, DV>;
  constexpr int C = S::C, NB = S::NB, KA = DK / 16, LDK = S::LDK, LDV = S::LDV, LDT = S::LDT, SEG = kDeltaSeg / C;
  extern __shared__ __align__(16) char smem[];
  const DeltaArgs<E>& p = a.f;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4, col0 = wave * 16;
  const int bh = blockIdx.x / p.segs, seg = blockIdx.x - bh * p.segs, b = bh / p.H, h = bh - b * p.H;
  const int begin = seg * p.seg_len, L = min(delta_length(p, b), begin + p.seg_len);  // the run's end
  const DeltaGates d = delta_gates<S>(smem);
  float* inv = reinterpret_cast<float*>(smem) + S::GATES;
  float* tp = inv + S::INV;   // the blocks' scores
  float* sums = tp + S::INV;  // (waves, steps)
  E* tk = reinterpret_cast<E*>(sums + S::W * C);
  E* tq = tk + C * LDK;
  E* tv = tq + C * LDK;
  E* tdo = tv + C * LDV;

  DeltaRows<E, C, DK, S::THREADS> rk, rq;
  DeltaRows<E, C, DV, S::THREADS> rv, rdo;
  rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], p.dk, p.vec, tid);
  rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], p.dk, p.vec, tid);
  rv.init(p.v + b * p.vs[0] + (h / p.gv) * p.vs[2], p.vs[1], p.dv, p.vec, tid);
  rdo.init(a.d_o + b * a.dos[0] + h * a.dos[2], a.dos[1], p.dv, p.vec, tid);
  DeltaGateRows<E, S> rg{p.g + b * p.gs[0] + h * p.gs[2], p.beta + b * p.bs[0] + h * p.bs[2], p.gs[1], p.bs[1]};
  auto fetch = [&](int t0) {
    rk.load(t0, L - t0), rq.load(t0, L - t0), rv.load(t0, L - t0), rdo.load(t0, L - t0), rg.load(t0, L - t0, tid);
  };
  if (begin < L) fetch(begin);
  f32x4 s[KA][1];
  if (p.segs > 1) load_state(s, p.seg_state + blockIdx.x * (int64_t)(DK * DV), false, DK, DV, col0, lo, hi);
  else load_state(s, p.s_in ? p.s_in + bh * ((int64_t)p.dk * p.dv) : nullptr, false, p.dk, p.dv, col0, lo, hi);

  for (int t0 = begin; t0 < L; t0 += C) {
    const int n = min(C, L - t0), chunk = t0 / C;
    rk.store(tk), rq.store(tq), rv.store(tv), rdo.store(tdo), rg.store(d, tid);
    store_columns<E, DK>(a.s + ((int64_t)bh * a.chunks + chunk) * DK * DV, s, col0, lo, hi);
    __syncthreads();
    for (int task = wave; task < 2 * S::NBLK; task += S::W) {
      const int blk = task % S::NBLK, r0 = blk * S::BS, lane = here(tid & 63), lo = lane & 15, hi = lane >> 4;
      if (r0 >= n) continue;
      if (task < S::NBLK) {
        delta_inverse<E, S, DK, false>(d, inv, tk, blk, lane);
        continue;
      }
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j <= i; ++j) {
          f32x4 x = row_products<E, DK>(tk, r0 + 16 * j, tq, r0 + 16 * i, LDK, lane);
          const f32x4 lag = delta_lag(d, r0 + 16 * i, r0 + 16 * j, lane);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = i > j || 4 * hi + r <= lo ? p.scale * (x[r] * __expf(lag[r])) : 0.0f;
          *reinterpret_cast<f32x4*>(tp + (blk * S::TRI + tri(i, j)) * S::TILE + lo * LDT + 4 * hi) = x;
        }
    }
    __syncthreads();
    if (t0 + C < L) fetch(t0 + C);
#pragma unroll 1
    for (int blk = 0; blk * S::BS < n; ++blk) {
      const int r0 = blk * S::BS, lane = here(tid & 63), lo = lane & 15, hi = lane >> 4, col0 = here(wave) * 16;
      f32x4 o[NB], x[NB], u[NB];
      delta_state_products<E, S, KA, Terms<E>::N>(tk, tq, r0, s, x, o, lane);
#pragma unroll
      for (int i = 0; i < NB; ++i)
        x[i] = to_f32(lds_quad_t(tv, LDV, r0 + 16 * i, col0, lane)) - lds_f4(d.from + r0 + 16 * i + 4 * hi) * x[i];
      delta_solve<S, false>(inv + blk * S::TRI * S::TILE, x, u, lane);
      Terms<E> w[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        // these columns of V are this wave's alone and have been read: e takes their place
#pragma unroll
        for (int r = 0; r < 4; ++r) tv[(r0 + 16 * i + 4 * hi + r) * LDV + col0 + lo] = (E)u[i][r];
        u[i] *= lds_f4(d.beta + r0 + 16 * i + 4 * hi);
        w[i] = Terms<E>(lds_f4(d.to + r0 + 16 * i + 4 * hi) * u[i]);
      }
      const float total = d.total[blk];
#pragma unroll
      for (int m = 0; m < KA; ++m) {
        quad_t<E> kt[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) kt[i] = lds_quad_t(tk, LDK, r0 + 16 * i, 16 * m, lane);
        s[m][0] = mma_terms(kt, w, s[m][0] * total);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        o[i] *= p.scale * d.from[r0 + 16 * i + lo];
#pragma unroll
        for (int j = 0; j <= i; ++j)
          o[i] = mma16(u[j], lds_f4(tp + (blk * S::TRI + tri(i, j)) * S::TILE + lo * LDT + 4 * hi), o[i]);
        o[i] *= to_f32(lds_quad(tdo, LDV, r0 + 16 * i, col0, lane));
        float w1 = o[i][0] + o[i][1] + o[i][2] + o[i][3];
        w1 += __shfl_xor(w1, 16, 64), w1 += __shfl_xor(w1, 32, 64);
        if (hi == 0) sums[wave * C + r0 + 16 * i + lo] = w1;
      }
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

// The inverses' transposes and the scores, transposed and by their terms, of a chunk's blocks.
template <typename E, typename S, int DK>
__device__ inline void delta_reverse_setup(const DeltaGates& d, float* inv, E* tp, const E* tk, const E* tq, int n, float scale,
                                           int wave, int tid) {
  for (int task = wave; task < 2 * S::NBLK; task += S::W) {
    const int blk = task % S::NBLK, r0 = blk * S::BS, lane = here(tid & 63), lo = lane & 15, hi = lane >> 4;
    if (r0 >= n) continue;
    if (task < S::NBLK) {
      delta_inverse<E, S, DK, true>(d, inv, tk, blk, lane);
      continue;
    }
#pragma unroll
    for (int i = 0; i < S::NB; ++i)
#pragma unroll
      for (int j = 0; j <= i; ++j) {  // lane lo has the key's row
        f32x4 x = row_products<E, DK>(tq, r0 + 16 * i, tk, r0 + 16 * j, S::LDK, lane);
        const f32x4 lag = delta_lag(d, r0 + 16 * j, r0 + 16 * i, lane);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = i > j || 4 * hi + r >= lo ? scale * (x[r] * __expf(-lag[r])) : 0.0f;
        const Terms<E> terms(x);
#pragma unroll
        for (int t = 0; t < Terms<E>::N; ++t)
          *reinterpret_cast<quad_t<E>*>(tp + ((blk * S::TRI + tri(i, j)) * Terms<E>::N + t) * S::TILE_P + lo * S::LDP + 4 * hi) = terms.t[t];
      }
  }
}

// dU of a block, and dO's columns as operands
template <typename E, typename S, int KA>
__device__ inline void delta_reverse_solve(const DeltaGates& d, const float* inv, const E* tp, const E* tk, const E* tdo, int blk,
                                           const f32x4 (&s)[KA][1], quad_t<E> (&g)[S::NB], f32x4 (&du)[S::NB], int col0, int lane) {
  constexpr int NB = S::NB, TERMS = Terms<E>::N;
  const int r0 = blk * S::BS, lo = lane & 15, hi = lane >> 4;
  f32x4 x[NB], none[NB];
  delta_state_products<E, S, KA, 0>(tk, tk, r0, s, x, none, lane);
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    g[i] = lds_quad_t(tdo, S::LDV, r0 + 16 * i, col0, lane);
    x[i] *= lds_f4(d.to + r0 + 16 * i + 4 * hi);
  }
  const E* pt = tp + blk * S::TRI * TERMS * S::TILE_P + lo * S::LDP + 4 * hi;
  auto score = [&](int i, int j, int t) { return *reinterpret_cast<const quad_t<E>*>(pt + (tri(i, j) * TERMS + t) * S::TILE_P); };
  if constexpr (NB == 2) {
    const quad_t<E> zero = to_quad<E>(f32x4{0, 0, 0, 0});
#pragma unroll
    for (int t = 0; t < 3; ++t) x[0] = mma2(score(0, 0, t), score(1, 0, t), g[0], g[1], x[0]);
    x[1] = mma2(score(1, 1, 0), score(1, 1, 1), g[1], g[1], x[1]);
    x[1] = mma2(score(1, 1, 2), zero, g[1], zero, x[1]);
  } else {
    x[0] = mma16(score(0, 0, 0), g[0], x[0]);
  }
  delta_solve<S, true>(inv + blk * S::TRI * S::TILE, x, du, lane);
}

// R := exp(G_end) R + (diag(exp G) scale Q)^T dO - (diag(exp G) K)^T Y
template <typename E, typename S, int KA>
__device__ inline void delta_reverse_update(const DeltaGates& d, const E* tk, const E* tq, int blk, float scale,
                                            const quad_t<E> (&g)[S::NB], const f32x4 (&du)[S::NB], f32x4 (&s)[KA][1], int lane) {
  constexpr int NB = S::NB;
  const int r0 = blk * S::BS, hi = lane >> 4;
  Terms<E> wq[NB], wk[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const f32x4 from = lds_f4(d.from + r0 + 16 * i + 4 * hi);
    wq[i] = Terms<E>(scale * from * to_f32(g[i]));
    wk[i] = Terms<E>(-(from * (lds_f4(d.beta + r0 + 16 * i + 4 * hi) * du[i])));
  }
  const float total = d.total[blk];
#pragma unroll
  for (int m = 0; m < KA; ++m) {
    quad_t<E> qt[NB], kt[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      qt[i] = lds_quad_t(tq, S::LDK, r0 + 16 * i, 16 * m, lane);
      kt[i] = lds_quad_t(tk, S::LDK, r0 + 16 * i, 16 * m, lane);
    }
    s[m][0] = mma_terms(kt, wk, mma_terms(qt, wq, s[m][0] * total));
  }
}

template <typename E, int DK, int DV>
constexpr size_t delta_reverse_lds() {
  using S = DeltaShape<E, DK, DV>;
  return sizeof(float) * (S::GATES + S::INV + 2 * S::W * S::C + 8) +
         sizeof(E) * (Terms<E>::N * S::SCORES + 2 * S::C * S::LDK + 3 * S::C * S::LDV);
}

template <typename E, int DK, int DV>
__global__ __launch_bounds__((DeltaShape<E, DK, DV>::THREADS), (DeltaShape<E, DK, DV>::WAVES_BACKWARD)) void delta_reverse_kernel(
    DeltaBwdArgs<E> a) {
  using S = DeltaShape<E, DK, DV>;
  constexpr int C = S::C, NB = S::NB, KA = DK / 16, LDK = S::LDK, LDV = S::LDV, LDP = S::LDP, SEG = kDeltaSeg / C;
  constexpr int TERMS = Terms<E>::N;
  extern __shared__ __align__(16) char smem[];
  const DeltaArgs<E>& p = a.f;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4, col0 = wave * 16;
  const int bh = blockIdx.x / p.segs, seg = blockIdx.x - bh * p.segs, b = bh / p.H, h = bh - b * p.H;
  const int begin = seg * p.seg_len, L = min(delta_length(p, b), begin + p.seg_len);  // the run's end
  const DeltaGates d = delta_gates<S>(smem);
  float* inv = reinterpret_cast<float*>(smem) + S::GATES;
  float* sum_beta = inv + S::INV;     // (waves, steps)
  float* sum_z = sum_beta + S::W * C;
  float* sum_dot = sum_z + S::W * C;  // (waves)
  E* tp = reinterpret_cast<E*>(sum_dot + 8);  // the blocks' scores, transposed, by their terms
  E* tk = tp + TERMS * S::SCORES;
  E* tq = tk + C * LDK;
  E* tv = tq + C * LDK;
  E* tdo = tv + C * LDV;
  E* te = tdo + C * LDV;

  DeltaRows<E, C, DK, S::THREADS> rk, rq;
  DeltaRows<E, C, DV, S::THREADS> rv, rdo;
  DeltaRows<E, C, DV, S::THREADS> re;
  rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], p.dk, p.vec, tid);
  rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], p.dk, p.vec, tid);
  rv.init(p.v + b * p.vs[0] + (h / p.gv) * p.vs[2], p.vs[1], p.dv, p.vec, tid);
  rdo.init(a.d_o + b * a.dos[0] + h * a.dos[2], a.dos[1], p.dv, p.vec, tid);
  re.init(a.e + (int64_t)bh * a.chunks * C * DV, DV, DV, true, tid);
  DeltaGateRows<E, S> rg{p.g + b * p.gs[0] + h * p.gs[2], p.beta + b * p.bs[0] + h * p.bs[2], p.gs[1], p.bs[1]};
  auto fetch = [&](int t0) {
    rk.load(t0, L - t0), rq.load(t0, L - t0), rv.load(t0, L - t0), rdo.load(t0, L - t0), re.load(t0, L - t0);
    rg.load(t0, L - t0, tid);
  };
  const int last = begin < L ? (L - 1) / C : -1;
  if (last >= 0) fetch(last * C);
  const int64_t size = (int64_t)p.dk * p.dv;
  f32x4 s[KA][1];
  if (p.segs > 1) load_state(s, a.r_seg + blockIdx.x * (int64_t)(DK * DV), false, DK, DV, col0, lo, hi);
  else load_state(s, a.d_out ? a.d_out + bh * size : nullptr, false, p.dk, p.dv, col0, lo, hi);
  E* yrow = a.y + (a.y_part ? bh * a.ys[0] : b * a.ys[0] + (int64_t)h * p.dv);

  for (int chunk = last; chunk * C >= begin; --chunk) {
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
    delta_reverse_setup<E, S, DK>(d, inv, tp, tk, tq, n, p.scale, wave, tid);
    __syncthreads();
    if (t0 > begin) fetch(t0 - C);
#pragma unroll 1
    for (int blk = (n - 1) / S::BS; blk >= 0; --blk) {
      const int r0 = blk * S::BS, lane = here(tid & 63), lo = lane & 15, hi = lane >> 4, col0 = here(wave) * 16;
      f32x4 du[NB];
      quad_t<E> g[NB];
      delta_reverse_solve<E, S, KA>(d, inv, tp, tk, tdo, blk, s, g, du, col0, lane);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const f32x4 y = lds_f4(d.beta + r0 + 16 * i + 4 * hi) * du[i];
        const f32x4 pe = du[i] * to_f32(lds_quad_t(te, LDV, r0 + 16 * i, col0, lane));
        const f32x4 pv = y * to_f32(lds_quad_t(tv, LDV, r0 + 16 * i, col0, lane));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = r0 + 16 * i + 4 * hi + r;
          const float sb = row16_sum(pe[r]), sz = row16_sum(pv[r]);
          if (lo == 0) sum_beta[wave * C + t] = sb, sum_z[wave * C + t] = sz;
          tdo[t * LDV + col0 + lo] = (E)y[r];  // these columns of dO are this wave's alone and have been read
          if (a.y_part && t < n && col0 + lo < p.dv)
            a.y_part[(((int64_t)b * p.T + t0 + t) * p.H + h) * p.dv + col0 + lo] = y[r];
        }
      }
      delta_reverse_update<E, S, KA>(d, tk, tq, blk, p.scale, g, du, s, lane);
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
  if (a.d_in && seg == 0) store_state(s, a.d_in + bh * size, p.dk, p.dv, col0, lo, hi);
  const int z0 = max(delta_length(p, b), begin), z1 = (int)min((int64_t)p.T, (int64_t)begin + p.seg_len);
  for (int t = z0 + tid; t < z1; t += S::THREADS) a.dbeta[((int64_t)b * p.T + t) * p.H + h] = E(0.0f);
  const int64_t orow = (int64_t)p.H * p.dv, obase = ((int64_t)b * p.T * p.H + h) * p.dv;
  if (a.y_part) zero_rows(a.y_part, true, 4, obase, orow, p.dv, z0, z1, tid, S::THREADS);
  else zero_rows(a.y, false, sizeof(E), obase, orow, p.dv, z0, z1, tid, S::THREADS);
}

template <typename E, int DK>
__global__ __launch_bounds__(256, DK <= 64 ? 3 : 2) void delta_reverse_run_kernel(DeltaBwdArgs<E> a, int DV) {
  using S = DeltaShape<E, DK, 64>;
  constexpr int C = S::C, NB = S::NB, KA = DK / 16, LDK = S::LDK, LDV = S::LDV, TERMS = Terms<E>::N;
  extern __shared__ __align__(16) char smem[];
  const DeltaArgs<E>& p = a.f;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int bh = blockIdx.x / p.segs, seg = blockIdx.x - bh * p.segs, b = bh / p.H, h = bh - b * p.H;
  const int begin = seg * p.seg_len, L = min(delta_length(p, b), begin + p.seg_len);
  const DeltaGates d = delta_gates<S>(smem);
  float* inv = reinterpret_cast<float*>(smem) + S::GATES;
  E* tp = reinterpret_cast<E*>(inv + S::INV);
  E* tk = tp + TERMS * S::SCORES;
  E* tq = tk + C * LDK;
  E* tdo = tq + C * LDK;
  DeltaRows<E, C, DK, 256> rk, rq;
  DeltaRows<E, C, 64, 256> rdo;
  const int c0 = blockIdx.y * 64;
  rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], p.dk, p.vec, tid);
  rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], p.dk, p.vec, tid);
  rdo.init(a.d_o + b * a.dos[0] + h * a.dos[2] + min(c0, p.dv), a.dos[1], min(max(p.dv - c0, 0), 64), p.vec, tid);
  DeltaGateRows<E, S> rg{p.g + b * p.gs[0] + h * p.gs[2], p.beta + b * p.bs[0] + h * p.bs[2], p.gs[1], p.bs[1]};
  auto fetch = [&](int t0) { rk.load(t0, L - t0), rq.load(t0, L - t0), rdo.load(t0, L - t0), rg.load(t0, L - t0, tid); };
  const int last = begin < L ? (L - 1) / C : -1;
  if (last >= 0) fetch(last * C);
  f32x4 s[KA][1];
#pragma unroll
  for (int m = 0; m < KA; ++m) s[m][0] = f32x4{0, 0, 0, 0};
  for (int chunk = last; chunk * C >= begin; --chunk) {
    const int t0 = chunk * C, n = min(C, L - t0);
    rk.store(tk), rq.store(tq), rdo.store(tdo), rg.store(d, tid);
    __syncthreads();
    delta_reverse_setup<E, S, DK>(d, inv, tp, tk, tq, n, p.scale, wave, tid);
    __syncthreads();
    if (t0 > begin) fetch(t0 - C);
#pragma unroll 1
    for (int blk = (n - 1) / S::BS; blk >= 0; --blk) {
      f32x4 du[NB];
      quad_t<E> g[NB];
      const int lane = here(tid & 63), col0 = here(wave) * 16;
      delta_reverse_solve<E, S, KA>(d, inv, tp, tk, tdo, blk, s, g, du, col0, lane);
      delta_reverse_update<E, S, KA>(d, tk, tq, blk, p.scale, g, du, s, lane);
    }
    __syncthreads();
  }
  const int col0 = c0 + wave * 16;
  if (col0 < DV) store_state(s, a.r_seg + blockIdx.x * (int64_t)(DK * DV), DK, DV, col0, tid & 15, (tid & 63) >> 4);
}

// log_decay's gradient: a wave a stretch, four steps a lane; in 64 bits, for the terms are.
template <typename E>
__global__ __launch_bounds__(64) void delta_dgate_kernel(DeltaBwdArgs<E> a, int rows) {
  const DeltaArgs<E>& p = a.f;
  const int seg = blockIdx.x % a.segs, bh = blockIdx.x / a.segs, b = bh / p.H, h = bh - b * p.H, lane = threadIdx.x;
  const int L = delta_length(p, b);
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
template <typename E, int DK, int DV>
__global__ __launch_bounds__(256) void delta_dqk_kernel(DeltaBwdArgs<E> a) {
  using S = DeltaShape<E, DK, DV>;
  constexpr int C = S::C, CT = C / 16, WC = 4 / CT, KT = DK / 16 / WC, VA = DV / 16, LDK = S::LDK, LDV = S::LDV;
  extern __shared__ __align__(16) char smem[];
  const DeltaArgs<E>& p = a.f;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4;
  const int chunk = blockIdx.x % a.chunks, bh = blockIdx.x / a.chunks, b = bh / p.H, h = bh - b * p.H;
  const int L = delta_length(p, b);
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

  DeltaRows<E, C, DK, 256> rk, rq;
  DeltaRows<E, C, DV, 256> rdo, re, ry;
  rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], p.dk, p.vec, tid);
  rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], p.dk, p.vec, tid);
  rdo.init(a.d_o + b * a.dos[0] + h * a.dos[2], a.dos[1], p.dv, p.vec, tid);
  re.init(a.e + (int64_t)bh * a.chunks * C * DV, DV, DV, true, tid);
  ry.init(a.y + (a.y_part ? bh * a.ys[0] : b * a.ys[0] + (int64_t)h * p.dv), a.ys[1], a.y_width, a.y_part || p.vec, tid);
  rk.load(t0, n), rq.load(t0, n), rdo.load(t0, n), re.load(t0, n), ry.load(t0, n);
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
  ry.store(ty);
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
