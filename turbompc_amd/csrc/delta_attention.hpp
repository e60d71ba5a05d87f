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
// of the state's update.  A wave owns 16 columns of the values and walks its head's blocks.  The chain
// leaves each SIMD waiting, so it has nothing else to do: further waves, the helpers, bring the next
// block's rows to LDS and make what depends on its blocks alone (the inverses, Q K^T o Gamma, the
// powers) while the walkers work on this one.  In bf16 the state, an fp32
// result, enters products as three bf16 terms (24 bits); a block has two tiles there, so that they are
// formed half as often.
//
// What bounds it: a walker's vector instructions and the latency of its chain (4000 to 4900 cycles a block of
// 32 steps with two workgroups on a CU, the vector units busy for 70% of them), not memory.  Forward, 64
// problems of 1024 steps, 8 heads of 64 / 64, bf16, whose bytes take 58 us at a copy's rate: with blocks of 16
// steps 214 us, of 32 145 us, their inverses by whole rows 137 us, with helpers 104 to 126 us.  The helpers cost where workgroups are
// many and short (2048 ragged histories of 101, 4 heads of 64 / 128: 297 us without them, 304 to 333 with; 1024 of
// 51 in fp32, 4 heads of 33 / 57: 84 and 101), and a second form of every kernel was not worth that.
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
// Steps of a stretch: a state kept in fp32 each (1/4 of the bytes of the bf16 states at every 64 steps), and at
// most so many terms of the gates' gradients summed up from one exact value.  Runs are whole stretches.
constexpr int kDeltaSeg = 256;

template <typename E>
__device__ inline int delta_length(const DeltaArgs<E>& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
}

template <typename E, int DK, int DV>
struct DeltaShape {
  static constexpr int W = DV / 16, HELPERS = 3;  // walkers, a wave 16 value columns, and helpers
  static constexpr int WALKERS = 64 * W, THREADS = 64 * (W + HELPERS);
  static constexpr int PAD = AttnTile<E>::PAD;
  static constexpr int NB = sizeof(E) == 2 ? 2 : 1, C = 16 * NB, TRI = NB * (NB + 1) / 2;  // a block's tiles and steps
  static constexpr int LDK = DK + PAD, LDV = DV + PAD;
  static constexpr int LDT = 20, TILE = 16 * LDT;  // a 16 x 16 fp32 tile, its quads spread over the banks
  static constexpr int LDP = 20, TILE_P = 16 * LDP;  // one of E
  // of a buffer, of which there are two: floats of the gates and the inverses; elements of E of the scores
  static constexpr int GATES = 6 * C + 4, INV = TRI * TILE, SCORES = TRI * TILE_P;
  // registers for two workgroups of seven waves on a CU, or one of eleven; five-wave ones are short of nothing
  static constexpr int WAVES_PER_SIMD = W == 2 ? 2 : 3;
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

// A block's gates in LDS: the sums of g from its start (as two floats), beta (zeros past the
// last live step), exp(G), exp(G_end - G), exp(G_end).
struct DeltaGates {
  float2* G;
  float *beta, *from, *to, *total;
};
template <typename S>
__device__ inline DeltaGates delta_gates(float* base) {
  DeltaGates d;
  d.G = reinterpret_cast<float2*>(base), d.beta = base + 2 * S::C;
  d.from = d.beta + S::C, d.to = d.from + S::C, d.total = d.to + S::C;
  return d;
}

// Every wave of the workgroup, each from its own place in the code: the walkers and the helpers meet here.
__device__ inline void meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// A launch's threads stay within 32 bits: many workgroups lie in rows of kFlatGrid.
constexpr int64_t kFlatGrid = 1 << 22;
__device__ inline int64_t flat_block() { return blockIdx.y * kFlatGrid + blockIdx.x; }

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

// A block's gates on their way from memory to LDS, a lane a step: by the first helper, which makes the
// inverses too.  The second and third move the rows, and the second makes the scores.
template <typename E, typename S>
struct DeltaGateRows {
  const float* g;
  const E* beta;
  int64_t gs, bs;
  float vg, vb;
  // from here on g and beta are the lane's own, and move from block to block
  __device__ void start(int64_t t, bool back) {
    g += t * gs, beta += t * bs;
    gs *= back ? -S::C : S::C, bs *= back ? -S::C : S::C;
  }
  __device__ void load(int n, int lane) {  // the next block's, n of its steps live
    vg = vb = 0.0f;
    if (lane < n && lane < S::C) vg = *g, vb = (float)*beta;
    g += gs, beta += bs;
  }
  // the sums and the powers, in registers
  float2 sum;
  float from, to, total, vb_scanned;
  __device__ void scan(int lane) {
    double x = vg < kNoDecay ? kNoDecay : vg;
    x += dpp_f64<0x111>(x);  // within 16 lanes
    x += dpp_f64<0x112>(x);
    x += dpp_f64<0x114>(x);
    x += dpp_f64<0x118>(x);
    double end = lane_f64(x, 15);
    if constexpr (S::NB == 2) {
      const double second = lane_f64(x, 31);
      if (lane >= 16) x += end;
      end += second;
    }
    const float top = (float)x;
    sum = make_float2(top, (float)(x - top)), vb_scanned = vb;
    from = __expf((float)x), to = __expf((float)(end - x)), total = __expf((float)end);
  }
  __device__ void store(const DeltaGates& d, int lane) const {
    if (lane < S::C) d.G[lane] = sum, d.beta[lane] = vb_scanned, d.from[lane] = from, d.to[lane] = to;
    if (lane == 0) *d.total = total;
  }
};

// Gamma_ij for a lane's i = i0 + lo and j = j0 + 4 hi + r, or with SWAP the other way round
template <bool SWAP>
__device__ inline f32x4 delta_ratio(const DeltaGates& d, int i0, int j0, int lane) {
  const float2 mine = d.G[i0 + (lane & 15)];
  const f32x4* at = reinterpret_cast<const f32x4*>(d.G + j0 + 4 * (lane >> 4));
  const f32x4 a = at[0], b = at[1];
  const f32x4 top = {a[0], a[2], b[0], b[2]}, rest = {a[1], a[3], b[1], b[3]};
  f32x4 ratio;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float lag = (mine.x - top[r]) + (mine.y - rest[r]);
    ratio[r] = __expf(SWAP ? -lag : lag);
  }
  return ratio;
}

// f(0) ... f(N - 1) with constants
template <int N, typename F, int I = 0>
__device__ inline void steps(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    steps<N, F, I + 1>(f);
  }
}
// x += a times x of lane I of each 16, y += b times y's.  (The wait is that of a lane permutation behind a
// vector write of its operand; a value that one of these writes is read eight of them later.)
template <int I>
__device__ inline void subtract_row(f32x4& x, float a, f32x4& y, float b) {
#define TMPC_ROW(v, f) "v_fmac_f32_dpp " v ", " v ", " f " row_newbcast:%10 row_mask:0xf bank_mask:0xf\n\t"
  float x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3], y0 = y[0], y1 = y[1], y2 = y[2], y3 = y[3];
  asm("s_nop 1\n\t" TMPC_ROW("%0", "%8") TMPC_ROW("%1", "%8") TMPC_ROW("%2", "%8") TMPC_ROW("%3", "%8") TMPC_ROW("%4", "%9")
          TMPC_ROW("%5", "%9") TMPC_ROW("%6", "%9") TMPC_ROW("%7", "%9")
      : "+v"(x0), "+v"(x1), "+v"(x2), "+v"(x3), "+v"(y0), "+v"(y1), "+v"(y2), "+v"(y3)
      : "v"(a), "v"(b), "n"(I));
#undef TMPC_ROW
  x = f32x4{x0, x1, x2, x3}, y = f32x4{y0, y1, y2, y3};
}

// (X Y^T)^T of 16 rows of each, from their quads: a lane has Y's row lo, and of X rows 4 hi + r
template <typename E, int KA>
__device__ inline f32x4 row_products(const quad_t<E> (&x)[KA], const quad_t<E> (&y)[KA]) {
  f32x4 t = {0, 0, 0, 0};
#pragma unroll
  for (int m = 0; m < KA; m += 2) t = mma2(x[m], x[m + 1], y[m], y[m + 1], t);
  return t;
}

// Which of a block's scores are made: none, those of j <= i, or those of j < i and apart from them each step's own.
enum DeltaScores { NO_SCORES, ALL_SCORES, EARLIER_SCORES };
struct DeltaNone {
  template <typename... A>
  __device__ void operator()(A...) const {}
};

// What the walkers need of a block, by one wave.  INVERSE: the tiles on the diagonal of (I + A)^-1 - I, or with
// REVERSE of (I + A')^-T - I, and the other tile of -A, or of -A'^T; each has beta of the column.  SCORES: put(tile
// (i, j), values) with scale (q_i . k_j) Gamma_ij, a lane having i = lo and j = 4 hi + r, or with REVERSE j = lo and
// i = 4 hi + r; own(i, scale (q_i . k_i)).
template <typename E, typename S, int DK, bool REVERSE, bool INVERSE, DeltaScores SCORES, typename Put, typename Own>
__device__ inline void delta_setup(const DeltaGates& d, float* inv, const E* tk, const E* tq, float scale, int lane, Put put, Own own) {
  constexpr int NB = S::NB, LDT = S::LDT, KA = DK / 16;
  const int lo = lane & 15, hi = lane >> 4;
  quad_t<E> k[NB][KA];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int m = 0; m < KA; ++m) k[i][m] = lds_quad(tk, S::LDK, 16 * i, 16 * m, lane);
  if constexpr (SCORES != NO_SCORES) {
    constexpr int AFTER = SCORES == EARLIER_SCORES ? 1 : 0;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      quad_t<E> q[KA];
#pragma unroll
      for (int m = 0; m < KA; ++m) q[m] = lds_quad(tq, S::LDK, 16 * i, 16 * m, lane);
#pragma unroll
      for (int j = 0; j <= i; ++j) {
        f32x4 x = REVERSE ? row_products<E, KA>(q, k[j]) : row_products<E, KA>(k[j], q);
        const f32x4 ratio = delta_ratio<REVERSE>(d, REVERSE ? 16 * j : 16 * i, REVERSE ? 16 * i : 16 * j, lane);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = 4 * hi + r;
          if (AFTER && i == j && at == lo) own(16 * i + lo, scale * x[r]);
          x[r] = i > j || (REVERSE ? at >= lo + AFTER : at + AFTER <= lo) ? scale * (x[r] * ratio[r]) : 0.0f;
        }
        put(tri(i, j), x);
      }
    }
  }
  if constexpr (INVERSE) {
    auto rows = [&](int k) { return reinterpret_cast<f32x4*>(inv + k * S::TILE + lo * LDT + 4 * hi); };
    auto a_tile = [&](int i, int j) {  // lane: row 16 i + lo, columns 16 j + 4 hi + r
      f32x4 a = row_products<E, KA>(k[j], k[i]);
      const f32x4 ratio = delta_ratio<REVERSE>(d, 16 * i, 16 * j, lane), beta = lds_f4(d.beta + 16 * j + 4 * hi);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        a[r] = i != j || (REVERSE ? 4 * hi + r > lo : 4 * hi + r < lo) ? -(a[r] * ratio[r] * beta[r]) : 0.0f;
      return a;
    };
#pragma unroll
    for (int i = 0; i < NB; ++i) *rows(tri(i, i)) = a_tile(i, i);
    if constexpr (NB == 2) *rows(tri(1, 0)) = REVERSE ? a_tile(0, 1) : a_tile(1, 0);
    f32x4 a[NB][4], t[2];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i < NB)
#pragma unroll
        for (int j = 0; j < 4; ++j) a[i][j] = lds_f4(inv + tri(i, i) * S::TILE + lo * LDT + 4 * j);  // -A's row lo
#pragma unroll
      for (int r = 0; r < 4; ++r) t[i][r] = 4 * hi + r == lo ? 1.0f : 0.0f;
    }
    // row lo of the inverse, columns 4 hi + r: takes off A[lo][j] times row j, which is final by then
    steps<15>([&](auto n) {
      constexpr int j = REVERSE ? 15 - n() : n();
      subtract_row<j>(t[0], a[0][j / 4][j % 4], t[1], a[NB - 1][j / 4][j % 4]);
    });
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < NB; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) t[i][r] = 4 * hi + r == lo ? 0.0f : t[i][r];
      *rows(tri(i, i)) = t[i];
    }
  }
}

// A block's rows of one operand on their way from memory through registers to LDS, by two helpers; whether
// they are whole pieces at 4-byte addresses is asked at run time (a variant of every kernel for
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
  unsigned off;   // bytes of the thread's first piece
  bool vec;

  __device__ void init(const E* b, int64_t stride, int d, bool whole, int tid) {
    row = tid / W, c = (tid - row * W) * P, step = stride, base = b, width = d, vec = whole;
    off = c < width && row < RS ? (unsigned)(row * (int)step + c) * (unsigned)sizeof(E) : kNowhere;
  }
  // rows t0 ..., n of them live (zeros behind them)
  __device__ void load(int64_t t0, int n) {
    const __amdgpu_buffer_rsrc_t rs = buffer_at(base + t0 * step);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned at = row + i * RS < n ? off : kNowhere, past = (unsigned)(i * RS * (int)step) * (unsigned)sizeof(E);
      if (vec) {
        r[i] = __builtin_bit_cast(piece_t<E>, __builtin_amdgcn_raw_buffer_load_b128(rs, at, past, 0));
      } else {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const unsigned ae = c + e < width && at != kNowhere ? at + e * (unsigned)sizeof(E) : kNowhere;
          if constexpr (sizeof(E) == 4)
            r[i][e] = __builtin_bit_cast(float, (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rs, ae, past, 0));
          else
            r[i][e] = __builtin_bit_cast(bf16, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rs, ae, past, 0));
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

// An fp32 value where elements of E are kept: itself, or its bits as two halves.
template <typename E>
__device__ inline E upper(float v) {
  if constexpr (sizeof(E) == 4) return v;
  else return __builtin_bit_cast(bf16, (uint16_t)(__builtin_bit_cast(uint32_t, v) >> 16));
}
__device__ inline bf16 lower(float v) { return __builtin_bit_cast(bf16, (uint16_t)__builtin_bit_cast(uint32_t, v)); }
__device__ inline float joined(bf16 high, bf16 low) {
  return __builtin_bit_cast(float, (uint32_t)__builtin_bit_cast(uint16_t, high) << 16 | __builtin_bit_cast(uint16_t, low));
}

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
__device__ inline void delta_state_products(const E* k, const E* q, const f32x4 (&s)[KA][1], f32x4 (&ks)[S::NB],
                                            f32x4 (&qs)[S::NB], int lane) {
#pragma unroll
  for (int i = 0; i < S::NB; ++i) ks[i] = qs[i] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int m = 0; m < KA; m += 2) {
    const Terms<E> a(s[m][0]), b(s[m + 1][0]);
#pragma unroll
    for (int i = 0; i < S::NB; ++i) {
      const int r0 = 16 * i;
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

// e = (I + A)^-1 (w + c), or with REVERSE by (I + A')^-T, over the block's tiles, from what delta_setup left.  With PARTS
// c := e - w, summed up by itself (where w is far larger, c would be lost in it); without, w is not used.  (PARTS
// everywhere: 315 in place of 304 us for the outputs of 2048 ragged histories of 101, 4 heads of 64 / 128.)
template <typename S, bool REVERSE, bool PARTS>
__device__ inline void delta_solve(const float* inv, const f32x4 (&w)[S::NB], f32x4 (&c)[S::NB], f32x4 (&e)[S::NB], int lane) {
  const float* at = inv + (lane & 15) * S::LDT + 4 * (lane >> 4);
  auto tile = [&](int i, f32x4 t) {
    if constexpr (PARTS) {
      c[i] = mma16(t, c[i] + w[i], c[i]), e[i] = c[i] + w[i];
    } else {
      e[i] = mma16(t, c[i], c[i]);
    }
  };
  if constexpr (S::NB == 2) {
    constexpr int first = REVERSE ? 1 : 0, second = 1 - first;
    const f32x4 t0 = lds_f4(at + tri(first, first) * S::TILE), corner = lds_f4(at + tri(1, 0) * S::TILE);
    const f32x4 t1 = lds_f4(at + tri(second, second) * S::TILE);
    tile(first, t0);
    c[second] = mma16(corner, e[first], c[second]);
    tile(second, t1);
  } else {
    tile(0, lds_f4(at));
  }
}

// K^T as operands, and s := total s + K^T w
template <typename E, typename S, int KA>
__device__ inline void transposed_rows(const E* k, quad_t<E> (&kt)[KA][S::NB], int lane) {
#pragma unroll
  for (int m = 0; m < KA; ++m)
#pragma unroll
    for (int i = 0; i < S::NB; ++i) kt[m][i] = lds_quad_t(k, S::LDK, 16 * i, 16 * m, lane);
}
template <typename E, int KA, int NB>
__device__ inline void delta_state_update(const quad_t<E> (&kt)[KA][NB], const Terms<E> (&w)[NB], float total, f32x4 (&s)[KA][1]) {
#pragma unroll
  for (int m = 0; m < KA; ++m) s[m][0] = mma_terms(kt[m], w, s[m][0] * total);
}

// Zero rows [z0, z1) of an output, four columns a thread.
template <typename T>
__device__ inline void zero_quads(T* base, int64_t pitch, int d, int64_t z0, int64_t z1, int tid, int threads) {
  const int q = (d + 3) / 4, per = threads / q, r = tid / q, c = (tid - r * q) * 4;
  if (r >= per) return;
  for (int64_t t = z0 + r; t < z1; t += per) store_quad(base + t * pitch, c, d, f32x4{0, 0, 0, 0});
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

// ---- backward ----
// Four kernels (and the sums over heads that share one of q's, k's or v's).  The first walks forwards in
// time as the forward pass does and leaves x_t = a_t k_t S_{t-1} (so e_t = v_t - x_t), the state at each chunk's start
// and the first of dg's terms below.  The second walks backwards with the state's gradient,
// which gives y = dv and dbeta, and leaves the gradient at each chunk's end and dg's other terms: over a block,
//   dU = (I + A')^-T (scale (Q K^T o Gamma)^T dO + diag(exp(G_end - G)) K R),  A'_ij = beta_i Gamma_ij (k_i . k_j),
//   R := exp(G_end) R + (diag(exp G) scale Q)^T dO - (diag(exp G) K)^T Y,  Y = diag(beta) dU.
// With the state and its gradient known at its ends every chunk then gives its dq and dk by itself:
//   dq_i = scale exp(G_i) do_i S^T + sum_{j <= i} M_ij k_j,  M_ij = scale Gamma_ij (do_i . u_j),
//   dk_j = exp(G_end - G_j) u_j R^T - exp(G_j) y_j S^T + sum_{i >= j} M_ij q_i
//          - sum_{i > j} N_ij k_i - sum_{l < j} N_jl k_l,  N_ij = Gamma_ij (y_i . u_j).
// The last: log_decay's gradient is dg_t = <R_{t-1}, S_{t-1}>, known from fp32 matrices at the ends of each stretch of
// 256 steps, and from step to step dg_t - dg_{t+1} = do_t . o_t - y_t . v_t.  Taken so, what a step has in o_t
// from itself and in v_t from itself cancels, and where decays are strong that is nearly all: at
// log_decay -8 dg was 1e-4 off, at -20 it was lost.  With both parts left out
//   dg_t = dg_{t+1} + w_t - z_t,  w_t = scale a_t do_t . (q_t S_{t-1}),  z_t = y_t . x_t + u_t . (k_t R_t),
// whose terms have the decays of the gradients that they lead to or from.  They come by themselves from the
// block's sums: w_t with the scores of j < t, and with T = (I + A)^-1, c = diag(exp G) K S and what the tiles before
// add to it, x = c - (T - I) (V - c), so that e = V - x; k_t R_t = du_t - scale (q_t . k_t) do_t likewise.
// (No values that are not finite are looked for here: they may spoil the gradients of their whole history and head.)
template <typename E>
struct DeltaBwdArgs {
  DeltaArgs<E> f;
  const E* d_o;
  int64_t dos[3];
  const float* d_out;  // (B, H, dk, dv) or NULL
  int chunks, stretches;  // of T
  E *x, *x_low;        // (B H, chunks C, DV): x_t, fp32 (in bf16 its upper and its lower halves)
  E *s, *r;            // (B H, chunks, DV, DK): the states at the chunks' starts, their gradients at the ends; in
  uint8_t *s_low, *r_low;  // bf16 the upper halves of fp32, and the next 8 bits here
  float *w, *z;        // (B H, chunks C): the parts of dg_t - dg_{t+1}
  float* s_seg;        // (B H, stretches, the walkers' registers): the states at their ends
  float* dot;          // (B H, stretches): <R, S> there
  float* dot0;         // (B H, 8): at the history's start, the walkers' parts
  E* y;                // as e, or dv's output (B, T, H, dv)
  int64_t ys[2];       // its strides of (b h) and step, from b and h where it is the output
  int y_width;
  E* y_low;            // in bf16 what y's rounding leaves, laid out as x
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

// The wave's 16 columns of a state as rows of a (DV, DK) matrix; in bf16 rounded to 24 bits, which are two terms.
template <typename E, int DK, int KA>
__device__ inline void store_columns(E* dst, uint8_t* low, const f32x4 (&s)[KA][1], int col0, int lo, int hi) {
#pragma unroll
  for (int m = 0; m < KA; ++m) {
    const int at = (col0 + lo) * DK + 16 * m + 4 * hi;
    if constexpr (sizeof(E) == 4) {
      *reinterpret_cast<f32x4*>(dst + at) = s[m][0];
    } else {
      const u32x4 b = __builtin_bit_cast(u32x4, s[m][0]) + 0x80u;
      *reinterpret_cast<u32x2*>(dst + at) = u32x2{__builtin_amdgcn_perm(b[1], b[0], 0x07060302u), __builtin_amdgcn_perm(b[3], b[2], 0x07060302u)};
      const uint32_t b01 = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0501u), b23 = __builtin_amdgcn_perm(b[3], b[2], 0x05010c0cu);
      *reinterpret_cast<uint32_t*>(low + at) = b01 | b23;
    }
  }
}
// The second terms of 8 elements kept so: exact in bf16.
__device__ inline bf16x8 second_terms(bf16x8 upper, u32x2 low) {
  const u32x4 u = __builtin_bit_cast(u32x4, upper);
  u32x4 r;
  steps<4>([&](auto n) {
    constexpr int i = n();
    const uint32_t b = low[i / 2];
    const uint32_t x0 = __builtin_amdgcn_perm(u[i], b, 0x0504000cu | (2 * i % 4) << 8), x1 = __builtin_amdgcn_perm(u[i], b, 0x0706000cu | (2 * i % 4 + 1) << 8);
    const float t0 = __builtin_bit_cast(float, x0) - __builtin_bit_cast(float, u[i] << 16);
    const float t1 = __builtin_bit_cast(float, x1) - __builtin_bit_cast(float, u[i] & 0xffff0000u);
    r[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, t1), __builtin_bit_cast(uint32_t, t0), 0x07060302u);
  });
  return __builtin_bit_cast(bf16x8, r);
}

// Rows of a tile in LDS to memory: `n` of them, row t at dst + t pitch.
template <typename R, typename E>
__device__ inline void copy_out(const R& map, const E* tile, E* dst, int64_t pitch, int n, int width) {
  if (map.row >= R::RS) return;
#pragma unroll
  for (int i = 0; i < R::N; ++i) {
    const int row = map.row + i * R::RS;
    if (row < n && map.c < width)
      store_piece(dst + row * pitch, map.c, width, *reinterpret_cast<const piece_t<E>*>(tile + row * R::LD + map.c));
  }
}

// A long history of few heads does not fill the chip: it is cut into runs.  A run is a linear map of the
// state it starts from, S -> M S + N: a first pass (WALK_RUN) makes each run's M (its columns start from the
// unit matrix, with values of zero) and N (from zero), a scan carries the states through, and the
// outputs start from those.  There a wave has 16 columns of [N | M].
enum DeltaWalk { WALK_OUT, WALK_STATES, WALK_RUN };

template <typename E, int DK, int DV, int MODE>
struct DeltaWalkLds {
  using S = DeltaShape<E, DK, DV>;
  static constexpr bool SCORES = MODE != WALK_RUN, DO = MODE == WALK_STATES;
  static constexpr int TERMS = (Terms<E>::N + 1) / 2;  // of the outputs' scores: in bf16 two
  // a buffer's bytes: gates, inverses, scores (of E, or for the states fp32), sums, rows of K, V, Q, dO
  static constexpr size_t inv = sizeof(float) * S::GATES, scores = inv + sizeof(float) * S::INV;
  static constexpr size_t sums = scores + (MODE == WALK_OUT ? sizeof(E) * TERMS * S::SCORES : DO ? sizeof(float) * S::INV : 0);
  static constexpr size_t k = sums + (DO ? sizeof(float) * S::W * S::C : 0), v = k + sizeof(E) * S::C * S::LDK;
  static constexpr size_t q = v + sizeof(E) * S::C * S::LDV, d_o = q + (SCORES ? sizeof(E) * S::C * S::LDK : 0);
  static constexpr size_t bytes = d_o + (DO ? sizeof(E) * S::C * S::LDV : 0), all = 2 * bytes;
};

// A workgroup a run of a (problem, head).
template <typename E, int DK, int DV, int MODE>
__global__ __launch_bounds__((DeltaShape<E, DK, DV>::THREADS), (DeltaShape<E, DK, DV>::WAVES_PER_SIMD)) void delta_walk_kernel(
    DeltaBwdArgs<E> a, int run_width) {
  using S = DeltaShape<E, DK, DV>;
  using M = DeltaWalkLds<E, DK, DV, MODE>;
  constexpr int C = S::C, NB = S::NB, KA = DK / 16, LDV = S::LDV, LDT = S::LDT, LDP = S::LDP, CK = AttnTile<E>::C;
  extern __shared__ __align__(16) char smem[];
  const DeltaArgs<E>& p = a.f;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bh = blockIdx.x / p.segs, seg = blockIdx.x - bh * p.segs, b = bh / p.H, h = bh - b * p.H;
  const int begin = seg * p.seg_len, L = min(delta_length(p, b), begin + p.seg_len);  // the run's end
  const int blocks = begin < L ? (L - begin + C - 1) / C : 0;
  if (MODE == WALK_RUN && seg == p.segs - 1 && !a.r_seg) return;  // no run starts from it, nor has its gradient at its end
  struct Buffer {
    DeltaGates d;
    float *inv, *sums;
    char* scores;
    E *k, *v, *q, *d_o;
  };
  auto buffer = [&](int i) {
    char* x = smem + (i & 1) * M::bytes;
    return Buffer{delta_gates<S>((float*)x), (float*)(x + M::inv), (float*)(x + M::sums), x + M::scores, (E*)(x + M::k),
                  (E*)(x + M::v), (E*)(x + M::q), (E*)(x + M::d_o)};
  };

  if (wave >= S::W) {  // ---- a helper
    constexpr int THREADS = 128;
    const int helper = wave - S::W, htid = tid - S::WALKERS - 64;
    if (helper == 0) {
      __builtin_amdgcn_s_setprio(3);  // the longest way from meeting to meeting
      DeltaGateRows<E, S> rg{p.g + b * p.gs[0] + h * p.gs[2], p.beta + b * p.bs[0] + h * p.bs[2], p.gs[1], p.bs[1]};
      rg.start(begin + lane, false);
      auto fetch = [&](int c) { rg.load(L - begin - c * C, lane); };
      auto setup = [&](int c) {
        const Buffer x = buffer(c);
        delta_setup<E, S, DK, false, true, NO_SCORES>(x.d, x.inv, x.k, x.q, p.scale, here(lane), DeltaNone(), DeltaNone());
      };
      if (blocks > 0) fetch(0), rg.scan(lane), rg.store(buffer(0).d, lane);
      meet();
      if (blocks > 1) fetch(1);
      if (blocks > 0) setup(0);
      if (blocks > 1) rg.scan(lane);
      meet();
      for (int c = 0; c < blocks; ++c) {
        if (c + 1 < blocks) rg.store(buffer(c + 1).d, lane);
        meet();
        if (c + 2 < blocks) fetch(c + 2);
        if (c + 1 < blocks) setup(c + 1);
        if (c + 2 < blocks) rg.scan(lane);
        meet();
      }
      return;
    }
    DeltaRows<E, C, DK, THREADS> rk, rq;
    DeltaRows<E, C, DV, THREADS> rv, rdo;
    const int c0 = MODE == WALK_RUN ? blockIdx.y * DV : 0;  // the first of the workgroup's columns
    rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], p.dk, p.vec, htid);
    rv.init(p.v + b * p.vs[0] + (h / p.gv) * p.vs[2] + min(c0, p.dv), p.vs[1], min(max(p.dv - c0, 0), DV), p.vec, htid);
    if constexpr (M::SCORES) rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], p.dk, p.vec, htid);
    if constexpr (M::DO) rdo.init(a.d_o + b * a.dos[0] + h * a.dos[2], a.dos[1], p.dv, p.vec, htid);
    auto fetch = [&](int c) {
      const int t0 = begin + c * C;
      rk.load(t0, L - t0), rv.load(t0, L - t0);
      if constexpr (M::SCORES) rq.load(t0, L - t0);
      if constexpr (M::DO) rdo.load(t0, L - t0);
    };
    auto stage = [&](int c) {
      const Buffer x = buffer(c);
      rk.store(x.k), rv.store(x.v);
      if constexpr (M::SCORES) rq.store(x.q);
      if constexpr (M::DO) rdo.store(x.d_o);
    };
    auto setup = [&](int c) {
      const Buffer x = buffer(c);
      [[maybe_unused]] const int lane = here(tid & 63), lo = lane & 15, hi = lane >> 4;
      auto put = [&](int tile, f32x4 s) {
        if constexpr (M::DO) {
          *reinterpret_cast<f32x4*>((float*)x.scores + tile * S::TILE + lo * LDT + 4 * hi) = s;
        } else {
          const Terms<E> terms(s);
#pragma unroll
          for (int t = 0; t < M::TERMS; ++t)
            *reinterpret_cast<quad_t<E>*>((E*)x.scores + (tile * M::TERMS + t) * S::TILE_P + lo * LDP + 4 * hi) = terms.t[t];
        }
      };
      if constexpr (M::SCORES)
        if (helper == 1)
          delta_setup<E, S, DK, false, false, M::DO ? EARLIER_SCORES : ALL_SCORES>(x.d, x.inv, x.k, x.q, p.scale, lane, put, DeltaNone());
    };
    auto results = [&](int c) {  // of a block that the walkers have left
      if constexpr (M::DO) {
        const Buffer x = buffer(c);
        const int t0 = begin + c * C, n = min(C, L - t0);
        const int64_t at = ((int64_t)bh * a.chunks * CK + t0) * DV;
        copy_out(rv, x.v, a.x + at, DV, n, DV);
        if constexpr (sizeof(E) == 2) copy_out(rdo, x.d_o, a.x_low + at, DV, n, DV);
        if (htid < n) {
          float w = 0.0f;
#pragma unroll
          for (int i = 0; i < S::W; ++i) w += x.sums[i * C + htid];
          a.w[(int64_t)bh * a.chunks * CK + t0 + htid] = w;
        }
      }
    };
    if (blocks > 0) fetch(0), stage(0);
    meet();
    if (blocks > 1) fetch(1);
    if (blocks > 0) setup(0);
    meet();
    for (int c = 0; c < blocks; ++c) {
      if (c > 0) results(c - 1);
      if (c + 1 < blocks) stage(c + 1);
      meet();
      if (c + 2 < blocks) fetch(c + 2);
      if (c + 1 < blocks) setup(c + 1);
      meet();
    }
    if (blocks > 0) results(blocks - 1);
    return;
  }

  // ---- a walker
  f32x4 s[KA][1];
  const int unit = MODE == WALK_RUN ? (blockIdx.y * S::W + wave) * 16 - run_width : 0;  // its first column of the unit matrix
  {
    const int lo = lane & 15, hi = lane >> 4;
    if constexpr (MODE == WALK_RUN) {
#pragma unroll
      for (int m = 0; m < KA; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[m][0][r] = 16 * m + 4 * hi + r == unit + lo ? 1.0f : 0.0f;
    } else if (p.segs > 1) {
      load_state(s, p.seg_state + blockIdx.x * (int64_t)(DK * DV), false, DK, DV, wave * 16, lo, hi);
    } else {
      load_state(s, p.s_in ? p.s_in + bh * ((int64_t)p.dk * p.dv) : nullptr, false, p.dk, p.dv, wave * 16, lo, hi);
    }
  }
  const int64_t orow = (int64_t)p.H * p.dv, obase = ((int64_t)b * p.T * p.H + h) * p.dv;
  const int oc = wave * 16 + 4 * (lane >> 4);
  const unsigned ooff = oc < p.dv ? (unsigned)(((lane & 15) * (int)orow + oc) * (int)sizeof(E)) : kNowhere;
  const unsigned otile = (unsigned)(16 * (int)orow * (int)sizeof(E));
  meet();
  meet();
  for (int c = 0; c < blocks; ++c) {
    const int t0 = begin + c * C, n = min(C, L - t0);
    const Buffer x = buffer(c);
    if (M::DO && t0 % CK == 0) {
      const int64_t at = ((int64_t)bh * a.chunks + t0 / CK) * DK * DV;
      store_columns<E, DK>(a.s + at, a.s_low + at, s, wave * 16, lane & 15, lane >> 4);
    }
    const __amdgpu_buffer_rsrc_t rs = buffer_at(MODE == WALK_OUT ? p.o + obase + t0 * orow : nullptr);
    const int lane = here(tid & 63), lo = lane & 15, hi = lane >> 4, col0 = wave * 16;
    f32x4 o[NB], v[NB], held[NB], u[NB];  // held: - a_t k_t S_{t-1}, where the outputs alone are made v_t less that
    // the state, u and the scores enter outputs of bf16 by two terms (16 bits: the scores by one made outputs of
    // heads of 16, or of short histories, 2.5e-3 off where a rounding is 1.66e-3)
    constexpr int OT = MODE == WALK_RUN ? 0 : M::DO ? Terms<E>::N : (Terms<E>::N + 1) / 2;
    meet();
    delta_state_products<E, S, KA, OT>(x.k, x.q, s, held, o, lane);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      v[i] = to_f32(lds_quad_t(x.v, LDV, 16 * i, col0, lane));
      held[i] *= -lds_f4(x.d.from + 16 * i + 4 * hi);
      if constexpr (!M::DO) held[i] += v[i];
    }
    quad_t<E> kt[KA][NB];  // read ahead of their use
    transposed_rows<E, S, KA>(x.k, kt, lane);
    f32x4 beta[NB], to[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) beta[i] = lds_f4(x.d.beta + 16 * i + 4 * hi), to[i] = lds_f4(x.d.to + 16 * i + 4 * hi);
    const float total = *x.d.total;
    delta_solve<S, false, M::DO>(x.inv, v, held, u, lane);
    Terms<E> w[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      // these columns of V are this wave's alone and have been read: x takes their place
      if constexpr (M::DO)
#pragma unroll
        for (int r = 0; r < 4; ++r) x.v[(16 * i + 4 * hi + r) * LDV + col0 + lo] = upper<E>(-held[i][r]);
      u[i] *= beta[i];
      w[i] = Terms<E>(to[i] * u[i]);
    }
    delta_state_update<E, KA, NB>(kt, w, total, s);
    if constexpr (MODE == WALK_OUT) {
      Terms<E> ut[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) ut[i] = Terms<E>(u[i]);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        o[i] *= p.scale * x.d.from[16 * i + lo];
        const E* pt = (const E*)x.scores + lo * LDP + 4 * hi;
        auto score = [&](int j, int t) { return *reinterpret_cast<const quad_t<E>*>(pt + (tri(i, j) * M::TERMS + t) * S::TILE_P); };
        if constexpr (sizeof(E) == 2) {
#pragma unroll
          for (int j = 0; j <= i; ++j) o[i] = mma2(ut[j].t[0], ut[j].t[1], score(j, 0), score(j, 0), o[i]);
          const quad_t<E> zero = to_quad<E>(f32x4{0, 0, 0, 0});
          if (i == 0) o[i] = mma2(ut[0].t[0], zero, score(0, 1), zero, o[i]);
          else o[i] = mma2(ut[0].t[0], ut[1].t[0], score(0, 1), score(1, 1), o[i]);
        } else {
#pragma unroll
          for (int j = 0; j <= i; ++j) o[i] = mma16(u[j], score(j, 0), o[i]);
        }
        const unsigned at = 16 * i + lo < n ? ooff : kNowhere, past = i * otile;
        if (p.vec) {
          if constexpr (sizeof(E) == 4) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o[i]), rs, at, past, 0);
          else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, to_bf16(o[i])), rs, at, past, 0);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const unsigned ae = oc + r < p.dv && at != kNowhere ? at + r * (unsigned)sizeof(E) : kNowhere;
            const float f = o[i][r];
            if constexpr (sizeof(E) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, f), rs, ae, past, 0);
            else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (bf16)f), rs, ae, past, 0);
          }
        }
      }
    }
    if constexpr (M::DO) {  // a_t do_t . (scale q_t S_{t-1}), unrounded
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        o[i] *= p.scale * x.d.from[16 * i + lo];
#pragma unroll
        for (int j = 0; j <= i; ++j)
          o[i] = mma16(u[j], lds_f4((const float*)x.scores + (tri(i, j)) * S::TILE + lo * LDT + 4 * hi), o[i]);
        o[i] *= to_f32(lds_quad(x.d_o, LDV, 16 * i, col0, lane));
        float w1 = o[i][0] + o[i][1] + o[i][2] + o[i][3];
        w1 += __shfl_xor(w1, 16, 64), w1 += __shfl_xor(w1, 32, 64);
        if (hi == 0) x.sums[wave * C + 16 * i + lo] = w1;
        if constexpr (sizeof(E) == 2)  // and so for dO
#pragma unroll
          for (int r = 0; r < 4; ++r) x.d_o[(16 * i + 4 * hi + r) * LDV + col0 + lo] = lower(-held[i][r]);
      }
    }
    if (M::DO && ((t0 + C) % kDeltaSeg == 0 || t0 + C >= L)) {
      f32x4* dst = reinterpret_cast<f32x4*>(a.s_seg + ((int64_t)bh * a.stretches + t0 / kDeltaSeg) * DK * DV) + wave * KA * 64 + lane;
#pragma unroll
      for (int m = 0; m < KA; ++m) dst[m * 64] = s[m][0];
    }
    meet();
  }
  if constexpr (MODE == WALK_RUN) {
    const int lo = lane & 15, hi = lane >> 4;
    if (unit >= 0) {
      if (unit < DK) store_state(s, p.seg_map + blockIdx.x * (int64_t)(DK * DK), DK, DK, unit, lo, hi);
    } else {
      store_state(s, p.seg_state + blockIdx.x * (int64_t)(DK * run_width), DK, run_width, unit + run_width, lo, hi);
    }
  }
  if constexpr (MODE == WALK_OUT) {
    // What follows makes its indexes and reads its arguments again: they would be kept through every chunk.
    auto* args = __builtin_amdgcn_kernarg_segment_ptr();
    int etid = tid, block = blockIdx.x;
    asm volatile("" : "+v"(etid), "+s"(args), "+s"(block));
    const DeltaArgs<E>& f = ((const DeltaBwdArgs<E>*)args)->f;
    const int ebh = block / f.segs, eseg = block - ebh * f.segs, eb = ebh / f.H, eL = delta_length(f, eb);
    const int ebegin = eseg * f.seg_len;
    zero_quads(f.o + ((int64_t)eb * f.T * f.H + (ebh - eb * f.H)) * f.dv, (int64_t)f.H * f.dv, f.dv, max(eL, ebegin),
               min((int64_t)f.T, (int64_t)ebegin + f.seg_len), etid, S::WALKERS);
    // An infinite or NaN value leaves the state so, to the end.
    f32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int m = 0; m < KA; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) zero[r] = fmaf(s[m][0][r], 0.0f, zero[r]);
    if (ebegin < eL && __ballot(!(zero[0] + zero[1] + zero[2] + zero[3] == 0.0f))) {
      __threadfence_block();  // rows written above are written again
      delta_by_step<E, KA, DV>(f, block, etid);
    } else if (f.s_out && eseg == (eL > 0 ? (eL - 1) / f.seg_len : 0)) {  // the run that holds the last live step
      store_state(s, f.s_out + ebh * ((int64_t)f.dk * f.dv), f.dk, f.dv, (etid >> 6) * 16, etid & 15, (etid & 63) >> 4);
    }
  }
}

// Between the passes: each run's sum becomes the state it starts from (REVERSE: the state's gradient
// that it ends with, through the maps' transposes), for 16 columns a workgroup; its waves share the rows out.
// Bound by the chain: 2.9 us a run of 128 x 128 (64 dependent matrix instructions, a meeting, the states'
// stores), with the next run's map and sum on their way meanwhile.  16 heads, 16 runs: 46 us.
template <int DK, bool REVERSE>
__global__ __launch_bounds__(256, 1) void delta_scan_kernel(const float* map, float* state, int segs, int DV, const float* start,
                                                         int dk, int dv) {
  constexpr int KA = DK / 16, MT = (KA + 3) / 4, LD = DK + 4;
  __shared__ __align__(16) float ts[2][16 * LD];  // (column, row)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4;
  const int tiles = DV / 16, bh = blockIdx.x / tiles, col = (blockIdx.x - bh * tiles) * 16 + lo;
  map += (int64_t)bh * segs * DK * DK, state += (int64_t)bh * segs * DK * DV;
  const int first = REVERSE ? segs - 1 : 0, dir = REVERSE ? -1 : 1;
  struct Run {
    f32x4 map[MT][KA], sum[MT];
  } even, odd;  // a run's and, on its way meanwhile, the next one's
  f32x4 s[MT];
  auto load = [&](int seg, Run& run) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = wave + 4 * i;
      if (KA % 4 != 0 && m >= KA) continue;
#pragma unroll
      for (int k = 0; k < KA; ++k) {
        const float* x = map + (int64_t)seg * DK * DK;
        if constexpr (REVERSE) {
#pragma unroll
          for (int r = 0; r < 4; ++r) run.map[i][k][r] = x[(16 * k + 4 * hi + r) * DK + 16 * m + lo];
        } else {
          run.map[i][k] = *reinterpret_cast<const f32x4*>(x + (16 * m + lo) * DK + 16 * k + 4 * hi);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) run.sum[i][r] = state[(int64_t)seg * DK * DV + (16 * m + 4 * hi + r) * DV + col];
    }
  };
  load(first, even);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * (wave + 4 * i) + 4 * hi + r;
      s[i][r] = start && row < dk && col < dv ? start[((int64_t)bh * dk + row) * dv + col] : 0.0f;
    }
  auto step = [&](int j, const Run& run, Run& ahead) {
    const int seg = first + dir * j;
    float* t = ts[j & 1];
    // the last run's own are nobody's start; a branch in place of the min would wait for all at its end
    load(first + dir * min(j + 1, segs - 2), ahead);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = wave + 4 * i;
      if (KA % 4 == 0 || m < KA) *reinterpret_cast<f32x4*>(t + lo * LD + 16 * m + 4 * hi) = s[i];
    }
    __syncthreads();
    f32x4 all[KA];
#pragma unroll
    for (int k = 0; k < KA; ++k) all[k] = lds_f4(t + lo * LD + 16 * k + 4 * hi);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = wave + 4 * i;
      if (KA % 4 != 0 && m >= KA) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) state[(int64_t)seg * DK * DV + (16 * m + 4 * hi + r) * DV + col] = s[i][r];
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KA; ++k) acc = mma16(run.map[i][k], all[k], acc);
      s[i] = acc + run.sum[i];
    }
  };
  for (int j = 0; j < segs; j += 2) {
    step(j, even, odd);
    if (j + 1 < segs) step(j + 1, odd, even);
  }
}

// dU of a block, dO's columns as operands, and with PARTS x_t = k_t R_t
template <typename E, typename S, int KA, bool PARTS>
__device__ inline void delta_reverse_solve(const DeltaGates& d, const float* inv, const float* own, const E* tp, const E* tk,
                                           const E* tdo, const f32x4 (&s)[KA][1], quad_t<E> (&g)[S::NB], f32x4 (&du)[S::NB],
                                           f32x4 (&x)[S::NB], int col0, int lane) {
  constexpr int NB = S::NB, TERMS = Terms<E>::N;
  const int lo = lane & 15, hi = lane >> 4;
  f32x4 w[NB], none[NB];
  delta_state_products<E, S, KA, 0>(tk, tk, s, x, none, lane);
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    g[i] = lds_quad_t(tdo, S::LDV, 16 * i, col0, lane);
    x[i] *= lds_f4(d.to + 16 * i + 4 * hi), w[i] = lds_f4(own + 16 * i + 4 * hi) * to_f32(g[i]);
  }
  const E* pt = tp + lo * S::LDP + 4 * hi;
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
  if constexpr (!PARTS)
#pragma unroll
    for (int i = 0; i < NB; ++i) x[i] += w[i];
  delta_solve<S, true, PARTS>(inv, w, x, du, lane);
}

// R := exp(G_end) R + (diag(exp G) scale Q)^T dO - (diag(exp G) K)^T Y
template <typename E, typename S, int KA>
__device__ inline void delta_reverse_update(const DeltaGates& d, const E* tk, const E* tq, float scale,
                                            const quad_t<E> (&g)[S::NB], const f32x4 (&du)[S::NB], f32x4 (&s)[KA][1], int lane) {
  constexpr int NB = S::NB;
  const int hi = lane >> 4;
  Terms<E> wq[NB], wk[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const f32x4 from = lds_f4(d.from + 16 * i + 4 * hi);
    wq[i] = Terms<E>(scale * from * to_f32(g[i]));
    wk[i] = Terms<E>(-(from * (lds_f4(d.beta + 16 * i + 4 * hi) * du[i])));
  }
  const float total = *d.total;
#pragma unroll
  for (int m = 0; m < KA; ++m) {
    quad_t<E> qt[NB], kt[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      qt[i] = lds_quad_t(tq, S::LDK, 16 * i, 16 * m, lane);
      kt[i] = lds_quad_t(tk, S::LDK, 16 * i, 16 * m, lane);
    }
    s[m][0] = mma_terms(kt, wk, mma_terms(qt, wq, s[m][0] * total));
  }
}

template <typename E, int DK, int DV, bool RUN>
struct DeltaReverseLds {
  using S = DeltaShape<E, DK, DV>;
  static constexpr int TERMS = sizeof(E) == 2 ? 2 : 1;  // elements of E that hold an x
  // a buffer's bytes: gates, inverses, scores by their terms, the steps' own and sums, rows of K, Q, dO, V, x
  static constexpr size_t inv = sizeof(float) * S::GATES, scores = inv + sizeof(float) * S::INV;
  static constexpr size_t sums = scores + sizeof(E) * Terms<E>::N * S::SCORES;
  static constexpr size_t k = sums + sizeof(float) * (S::C + (RUN ? 0 : 2 * S::W * S::C + 16)), q = k + sizeof(E) * S::C * S::LDK;
  static constexpr size_t d_o = q + sizeof(E) * S::C * S::LDK, v = d_o + sizeof(E) * S::C * S::LDV;
  static constexpr size_t x = v + (RUN ? 0 : sizeof(E) * S::C * S::LDV);
  static constexpr size_t bytes = x + (RUN ? 0 : sizeof(E) * TERMS * S::C * S::LDV), all = 2 * bytes;
};

// The walk backwards (64 problems of 1024 steps, 8 heads of 64 / 64, bf16: 189 to 224 us, where the walk for
// the states takes 151 to 176; both are bound as the forward walk); RUN: what a run adds to the gradient of the
// state that it starts from, alone.
template <typename E, int DK, int DV, bool RUN>
__global__ __launch_bounds__((DeltaShape<E, DK, DV>::THREADS), (DeltaShape<E, DK, DV>::WAVES_PER_SIMD)) void delta_reverse_kernel(
    DeltaBwdArgs<E> a, int run_width) {
  using S = DeltaShape<E, DK, DV>;
  using M = DeltaReverseLds<E, DK, DV, RUN>;
  constexpr int C = S::C, NB = S::NB, KA = DK / 16, LDV = S::LDV, LDP = S::LDP, TERMS = Terms<E>::N, CK = AttnTile<E>::C;
  extern __shared__ __align__(16) char smem[];
  const DeltaArgs<E>& p = a.f;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bh = blockIdx.x / p.segs, seg = blockIdx.x - bh * p.segs, b = bh / p.H, h = bh - b * p.H;
  const int begin = seg * p.seg_len, L = min(delta_length(p, b), begin + p.seg_len);  // the run's end
  const int blocks = begin < L ? (L - begin + C - 1) / C : 0, last = begin / C + blocks - 1;  // block `last` comes first
  if (RUN && seg == 0) return;  // no run ends where it starts
  const int c0 = RUN ? blockIdx.y * DV : 0;  // the first of the workgroup's columns
  struct Buffer {
    DeltaGates d;
    float *inv, *own, *beta, *z, *dot;
    E *scores, *k, *q, *d_o, *v, *x;
  };
  auto buffer = [&](int i) {
    char* x = smem + (i & 1) * M::bytes;
    float *own = (float*)(x + M::sums), *sums = own + C;
    return Buffer{delta_gates<S>((float*)x), (float*)(x + M::inv), own, sums, sums + S::W * C, sums + 2 * S::W * C, (E*)(x + M::scores),
                  (E*)(x + M::k), (E*)(x + M::q), (E*)(x + M::d_o), (E*)(x + M::v), (E*)(x + M::x)};
  };
  auto ends = [&](int t0, int of) { return (t0 + C) % of == 0 || t0 + C >= L; };

  if (wave >= S::W) {  // ---- a helper
    constexpr int THREADS = 128;
    const int helper = wave - S::W, htid = tid - S::WALKERS - 64;
    if (helper == 0) {
      __builtin_amdgcn_s_setprio(3);  // the longest way from meeting to meeting
      DeltaGateRows<E, S> rg{p.g + b * p.gs[0] + h * p.gs[2], p.beta + b * p.bs[0] + h * p.bs[2], p.gs[1], p.bs[1]};
      rg.start((int64_t)last * C + lane, true);
      auto fetch = [&](int c) { rg.load(L - (last - c) * C, lane); };
      auto setup = [&](int c) {
        const Buffer x = buffer(c);
        delta_setup<E, S, DK, true, true, NO_SCORES>(x.d, x.inv, x.k, x.q, p.scale, here(lane), DeltaNone(), DeltaNone());
      };
      if (blocks > 0) fetch(0), rg.scan(lane), rg.store(buffer(0).d, lane);
      meet();
      if (blocks > 1) fetch(1);
      if (blocks > 0) setup(0);
      if (blocks > 1) rg.scan(lane);
      meet();
      for (int c = 0; c < blocks; ++c) {
        if (c + 1 < blocks) rg.store(buffer(c + 1).d, lane);
        meet();
        if (c + 2 < blocks) fetch(c + 2);
        if (c + 1 < blocks) setup(c + 1);
        if (c + 2 < blocks) rg.scan(lane);
        meet();
      }
      return;
    }
    DeltaRows<E, C, DK, THREADS> rk, rq;
    DeltaRows<E, C, DV, THREADS> rdo, rv, rx[M::TERMS];
    rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], p.dk, p.vec, htid);
    rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], p.dk, p.vec, htid);
    rdo.init(a.d_o + b * a.dos[0] + h * a.dos[2] + min(c0, p.dv), a.dos[1], min(max(p.dv - c0, 0), DV), p.vec, htid);
    if constexpr (!RUN) {
      rv.init(p.v + b * p.vs[0] + (h / p.gv) * p.vs[2], p.vs[1], p.dv, p.vec, htid);
#pragma unroll
      for (int t = 0; t < M::TERMS; ++t) rx[t].init((t ? a.x_low : a.x) + (int64_t)bh * a.chunks * CK * DV, DV, DV, true, htid);
    }
    auto fetch = [&](int c) {
      const int t0 = (last - c) * C;
      rk.load(t0, L - t0), rq.load(t0, L - t0), rdo.load(t0, L - t0);
      if constexpr (!RUN) {
        rv.load(t0, L - t0);
#pragma unroll
        for (int t = 0; t < M::TERMS; ++t) rx[t].load(t0, L - t0);
      }
    };
    auto stage = [&](int c) {
      const Buffer x = buffer(c);
      rk.store(x.k), rq.store(x.q), rdo.store(x.d_o);
      if constexpr (!RUN) {
        rv.store(x.v);
#pragma unroll
        for (int t = 0; t < M::TERMS; ++t) rx[t].store(x.x + t * C * LDV);
      }
    };
    auto setup = [&](int c) {
      const Buffer x = buffer(c);
      [[maybe_unused]] const int lane = here(tid & 63), lo = lane & 15, hi = lane >> 4;
      auto put = [&](int tile, f32x4 s) {
        const Terms<E> terms(s);
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
          *reinterpret_cast<quad_t<E>*>(x.scores + (tile * TERMS + t) * S::TILE_P + lo * LDP + 4 * hi) = terms.t[t];
      };
      auto own = [&](int i, float v) { x.own[i] = v; };
      if (helper == 1) delta_setup<E, S, DK, true, false, EARLIER_SCORES>(x.d, x.inv, x.k, x.q, p.scale, lane, put, own);
    };
    E* yrow = a.y + (a.y_part ? bh * a.ys[0] : b * a.ys[0] + (int64_t)h * p.dv);
    auto results = [&](int c) {  // of a block that the walkers have left
      if constexpr (!RUN) {
        const Buffer x = buffer(c);
        const int t0 = (last - c) * C, n = min(C, L - t0);
        copy_out(rdo, x.d_o, yrow + t0 * a.ys[1], a.ys[1], n, a.y_width);
        if constexpr (sizeof(E) == 2) copy_out(rv, x.v, a.y_low + ((int64_t)bh * a.chunks * CK + t0) * DV, DV, n, DV);
        if (htid < n) {
          float sb = 0.0f, sz = 0.0f;
#pragma unroll
          for (int i = 0; i < S::W; ++i) sb += x.beta[i * C + htid], sz += x.z[i * C + htid];
          a.dbeta[((int64_t)b * p.T + t0 + htid) * p.H + h] = (E)sb;
          a.z[(int64_t)bh * a.chunks * CK + t0 + htid] = sz;
        }
        if (htid == 0 && ends(t0, kDeltaSeg)) {
          float dot = 0.0f;
          for (int i = 0; i < S::W; ++i) dot += x.dot[i];
          a.dot[(int64_t)bh * a.stretches + t0 / kDeltaSeg] = dot;
        }
      }
    };
    if (blocks > 0) fetch(0), stage(0);
    meet();
    if (blocks > 1) fetch(1);
    if (blocks > 0) setup(0);
    meet();
    for (int c = 0; c < blocks; ++c) {
      if (c > 0) results(c - 1);
      if (c + 1 < blocks) stage(c + 1);
      meet();
      if (c + 2 < blocks) fetch(c + 2);
      if (c + 1 < blocks) setup(c + 1);
      meet();
    }
    if (blocks > 0) results(blocks - 1);
    return;
  }

  // ---- a walker
  const int64_t size = (int64_t)p.dk * p.dv;
  f32x4 s[KA][1];
  if constexpr (RUN) {
#pragma unroll
    for (int m = 0; m < KA; ++m) s[m][0] = f32x4{0, 0, 0, 0};
  } else if (p.segs > 1) {
    load_state(s, a.r_seg + blockIdx.x * (int64_t)(DK * DV), false, DK, DV, wave * 16, lane & 15, lane >> 4);
  } else {
    load_state(s, a.d_out ? a.d_out + bh * size : nullptr, false, p.dk, p.dv, wave * 16, lane & 15, lane >> 4);
  }
  meet();
  meet();
  for (int c = 0; c < blocks; ++c) {
    const int t0 = (last - c) * C, n = min(C, L - t0);
    const Buffer x = buffer(c);
    if constexpr (!RUN) {
      if (ends(t0, CK)) {
        const int64_t at = ((int64_t)bh * a.chunks + t0 / CK) * DK * DV;
        store_columns<E, DK>(a.r + at, a.r_low + at, s, wave * 16, lane & 15, lane >> 4);
      }
      if (ends(t0, kDeltaSeg)) {
        const f32x4* src = reinterpret_cast<const f32x4*>(a.s_seg + ((int64_t)bh * a.stretches + t0 / kDeltaSeg) * DK * DV) + wave * KA * 64 + lane;
        float dot = 0.0f;
#pragma unroll
        for (int m = 0; m < KA; ++m) {
          const f32x4 y = src[m * 64];
#pragma unroll
          for (int r = 0; r < 4; ++r) dot += y[r] * s[m][0][r];
        }
#pragma unroll
        for (int i = 32; i; i >>= 1) dot += __shfl_xor(dot, i, 64);
        if (lane == 0) x.dot[wave] = dot;
      }
    }
    const int lane = here(tid & 63), lo = lane & 15, hi = lane >> 4, col0 = wave * 16;
    f32x4 du[NB], kr[NB];
    quad_t<E> g[NB];
    meet();
    delta_reverse_solve<E, S, KA, !RUN>(x.d, x.inv, x.own, x.scores, x.k, x.d_o, s, g, du, kr, col0, lane);
    if constexpr (!RUN) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const f32x4 beta = lds_f4(x.d.beta + 16 * i + 4 * hi), y = beta * du[i];
        const quad_t<E> high = lds_quad_t(x.x, LDV, 16 * i, col0, lane);
        f32x4 held = to_f32(high);
        if constexpr (M::TERMS == 2) {
          const quad_t<E> low = lds_quad_t(x.x + C * LDV, LDV, 16 * i, col0, lane);
#pragma unroll
          for (int r = 0; r < 4; ++r) held[r] = joined(high[r], low[r]);
        }
        const f32x4 e = to_f32(lds_quad_t(x.v, LDV, 16 * i, col0, lane)) - held;
        const f32x4 pe = du[i] * e, pz = y * held + beta * e * kr[i];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = 16 * i + 4 * hi + r;
          const float sb = row16_sum(pe[r]), sz = row16_sum(pz[r]);
          if (lo == 0) x.beta[wave * C + t] = sb, x.z[wave * C + t] = sz;
          // these columns of dO and V are this wave's alone and have been read
          const E top = (E)y[r];
          x.d_o[t * LDV + col0 + lo] = top;
          if constexpr (sizeof(E) == 2) x.v[t * LDV + col0 + lo] = (E)(y[r] - (float)top);
          if (a.y_part && t < n && col0 + lo < p.dv)
            a.y_part[(((int64_t)b * p.T + t0 + t) * p.H + h) * p.dv + col0 + lo] = y[r];
        }
      }
    }
    delta_reverse_update<E, S, KA>(x.d, x.k, x.q, p.scale, g, du, s, lane);
    meet();
  }
  if constexpr (RUN) {
    const int col0 = c0 + wave * 16;
    if (col0 < run_width) store_state(s, a.r_seg + blockIdx.x * (int64_t)(DK * run_width), DK, run_width, col0, lane & 15, lane >> 4);
  } else {
    if (a.d_in && seg == 0) store_state(s, a.d_in + bh * size, p.dk, p.dv, wave * 16, lane & 15, lane >> 4);
    if (seg == 0 && L > 0) {
      float dot = 0.0f;
      if (p.s_in) {
        f32x4 y[KA][1];
        load_state(y, p.s_in + bh * size, false, p.dk, p.dv, wave * 16, lane & 15, lane >> 4);
#pragma unroll
        for (int m = 0; m < KA; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) dot += y[m][0][r] * s[m][0][r];
#pragma unroll
        for (int i = 32; i; i >>= 1) dot += __shfl_xor(dot, i, 64);
      }
      if (lane == 0) a.dot0[bh * (int64_t)8 + wave] = dot;
    }
    const int z0 = max(delta_length(p, b), begin), z1 = (int)min((int64_t)p.T, (int64_t)begin + p.seg_len);
    for (int t = z0 + tid; t < z1; t += S::WALKERS) a.dbeta[((int64_t)b * p.T + t) * p.H + h] = E(0.0f);
    const int64_t orow = (int64_t)p.H * p.dv, obase = ((int64_t)b * p.T * p.H + h) * p.dv;
    if (a.y_part) zero_quads(a.y_part + obase, orow, p.dv, z0, z1, tid, S::WALKERS);
    else zero_quads(a.y + obase, orow, p.dv, z0, z1, tid, S::WALKERS);
  }
}

// sum over the lanes behind this one, or before it
template <bool BEHIND>
__device__ inline double other_lanes(double v, int lane) {
  double sum = v;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    const double u = BEHIND ? __shfl_down(sum, i, 64) : __shfl_up(sum, i, 64);
    if (BEHIND ? lane + i < 64 : lane >= i) sum += u;
  }
  const double u = BEHIND ? __shfl_down(sum, 1, 64) : __shfl_up(sum, 1, 64);
  return (BEHIND ? lane < 63 : lane > 0) ? u : 0.0;
}

// log_decay's gradient: a wave a stretch, four steps a lane; in 64 bits, for the terms are.  It is known at both
// ends of a stretch from the states there, and the terms w - z lead from step to step; each of these numbers is
// off by some of its own last bits.  So the two sums, from either end, are weighted by the squares of what
// has gone into the other one: a large end (a final state's gradient behind decays that leave nothing of it)
// spoils nothing beyond its own step.
template <typename E>
__global__ __launch_bounds__(64) void delta_dgate_kernel(DeltaBwdArgs<E> a, int rows, int walkers) {
  const DeltaArgs<E>& p = a.f;
  const int block = (int)flat_block(), bh = block / a.stretches, seg = block - bh * a.stretches;
  if (bh >= p.B * p.H) return;
  const int b = bh / p.H, h = bh - b * p.H, lane = threadIdx.x;
  const int L = delta_length(p, b);
  const int t0 = seg * kDeltaSeg + lane * 4;
  const int64_t at = (int64_t)bh * rows + t0;
  double term[4], square[4], sum = 0.0, squares = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double w = t0 + i < L ? a.w[at + i] : 0.0, z = t0 + i < L ? a.z[at + i] : 0.0;
    term[i] = w - z, square[i] = w * w + z * z;
    sum += term[i], squares += square[i];
  }
  double start = 0.0, end = 0.0;
  if (seg * kDeltaSeg < L) {
    const float* dot = a.dot + (int64_t)bh * a.stretches + seg;
    end = dot[0];
    if (seg > 0) start = dot[-1];
    else for (int i = 0; i < walkers; ++i) start += (double)a.dot0[bh * (int64_t)8 + i];
  }
  // from the start to before this lane's steps, and from the end to behind them
  double from_start = start - other_lanes<false>(sum, lane), weight_end = start * start + other_lanes<false>(squares, lane);
  double from_end[4], weight_start[4], later = end + other_lanes<true>(sum, lane);
  double more = end * end + other_lanes<true>(squares, lane);
#pragma unroll
  for (int i = 3; i >= 0; --i) from_end[i] = later += term[i], weight_start[i] = more += square[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + i;
    if (t >= p.T) break;
    const double all = weight_start[i] + weight_end;
    const double dg = all > 0.0 ? (from_start * weight_start[i] + from_end[i] * weight_end) / all : from_end[i];
    // it has a_t as a factor: zero where that is below the least normal number
    const bool decays = t < L && !(__expf(p.g[b * p.gs[0] + t * p.gs[1] + h * p.gs[2]]) < 0x1p-126f);
    a.dg[((int64_t)b * p.T + t) * p.H + h] = decays ? (float)dg : 0.0f;
    from_start -= term[i], weight_end += square[i];
  }
}

template <typename E, int DK, int DV>
struct DeltaDqkShape {
  static constexpr int C = AttnTile<E>::C, CT = C / 16, PAD = AttnTile<E>::PAD, TERMS = sizeof(E) == 2 ? 2 : 1;
  static constexpr int WC = sizeof(E) == 2 || DK == 32 ? 2 : 4, KT = DK / 16 / WC;  // waves that share 16 rows' columns, tiles of each
  static constexpr int WAVES = CT * WC, THREADS = 64 * WAVES;
  static constexpr int HV = DV < 64 ? DV : 64;                                // values in LDS at a time
  static constexpr int SV = sizeof(E) == 2 && DK == 128 && HV == 64 ? 32 : HV;  // of these, of a state
  static constexpr int LDK = DK + PAD, LDV = HV + PAD, LDC = C + PAD;
  // tiles of the scores on and below the diagonal, and those right of it that a pair of tiles begins with
  static constexpr int LOWER = CT * (CT + 1) / 2, TILES = LOWER + CT / 2, MINE = (TILES + WAVES - 1) / WAVES;
  // rows of dO, y and e (these by their terms) and a state's part; then the scores by theirs, K and Q in their place
  static constexpr size_t FIRST = sizeof(E) * ((1 + 2 * TERMS) * C * LDV + TERMS * SV * LDK);
  static constexpr size_t SECOND = sizeof(E) * (2 * TERMS * C * LDC + 2 * C * LDK);
  static constexpr size_t LDS = 8 * C + 4 * 3 * C + (FIRST > SECOND ? FIRST : SECOND);
  static constexpr int FIT = 160 * 1024 / LDS * THREADS / 256, WAVES_PER_SIMD = FIT > 4 ? 4 : FIT;  // by LDS and registers
};

// dq and dk of a chunk.  beta_j stays out of the operands (u_j = beta_j e_j).  In bf16 the states, y, e and the scores M
// and N enter by two terms, so that dq and dk are off by their own rounding (1.66e-3; with y and the states by one
// term 2.1e-3 and 2.3e-3).  The waves share the scores out and exchange them in LDS, half of the values' columns at a
// time where they are 128: every wave for itself needed more registers than there are.  Bound by memory
// where heads are 64 wide: 64 problems of 1024 steps, 8 heads of 64 / 64, 190 to 215 us for 0.87 GB, of which the second
// terms are 0.13 (the states' as whole bf16 0.20 GB and 198 to 220); 2048 ragged histories of 101, 4 heads of 64 / 128,
// 504 to 518 us; 256 of 41, 4 of 32 / 49, fp32, 31 us.
template <typename E, int DK, int DV>
__global__ __launch_bounds__((DeltaDqkShape<E, DK, DV>::THREADS), (DeltaDqkShape<E, DK, DV>::WAVES_PER_SIMD)) void delta_dqk_kernel(DeltaBwdArgs<E> a) {
  using S = DeltaDqkShape<E, DK, DV>;
  constexpr int C = S::C, CT = S::CT, WC = S::WC, KT = S::KT, THREADS = S::THREADS, HV = S::HV, SV = S::SV;
  constexpr int LDK = S::LDK, LDV = S::LDV, LDC = S::LDC, P = Elem<E>::PIECE, TERMS = S::TERMS;
  extern __shared__ __align__(16) char smem[];
  const DeltaArgs<E>& p = a.f;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lo = lane & 15, hi = lane >> 4;
  const int block = (int)flat_block(), bh = block / a.chunks, chunk = block - bh * a.chunks, b = bh / p.H, h = bh - b * p.H;
  if (b >= p.B) return;
  const int L = delta_length(p, b);
  const int t0 = chunk * C, n = min(C, L - t0);
  const int64_t orow = (int64_t)p.H * p.dk, obase = ((int64_t)b * p.T * p.H + h) * p.dk;
  const int64_t z0 = max(L, t0), z1 = min(p.T, t0 + C);
  auto zero = [&](void* out, bool part) {
    if (part) zero_quads((float*)out + obase, orow, p.dk, z0, z1, tid, THREADS);
    else zero_quads((E*)out + obase, orow, p.dk, z0, z1, tid, THREADS);
  };
  if (z0 < z1) zero(a.dq, a.q_part), zero(a.dk, a.k_part);
  if (n <= 0) return;
  double* G = reinterpret_cast<double*>(smem);
  float* beta = reinterpret_cast<float*>(G + C);
  float* from = beta + C;
  float* to = from + C;
  E* tdo = reinterpret_cast<E*>(to + C);
  E* ty = tdo + C * LDV;              // TERMS of them
  E* te = ty + TERMS * C * LDV;       // and of these
  E* ts = te + TERMS * C * LDV;       // a state's or its gradient's, (SV, DK) each
  E* tm = reinterpret_cast<E*>(to + C);  // M by its terms, -N by its terms
  E* tk = tm + 2 * TERMS * C * LDC;
  E* tq = tk + C * LDK;

  DeltaRows<E, C, HV, THREADS> rdo, rv, ry[TERMS], rx[TERMS];
  const int64_t rows = ((int64_t)bh * a.chunks * C + t0) * DV;
  auto rows_load = [&](int v0) {  // columns v0 ... of the values
    const int left = min(max(p.dv - v0, 0), HV), from0 = min(v0, p.dv);
    rdo.init(a.d_o + b * a.dos[0] + h * a.dos[2] + from0, a.dos[1], left, p.vec, tid);
    rv.init(p.v + b * p.vs[0] + (h / p.gv) * p.vs[2] + from0, p.vs[1], left, p.vec, tid);
    if (a.y_part) ry[0].init(a.y + bh * a.ys[0] + v0, a.ys[1], HV, true, tid);
    else ry[0].init(a.y + b * a.ys[0] + (int64_t)h * p.dv + from0, a.ys[1], left, p.vec, tid);
    rdo.load(t0, n), rv.load(t0, n), ry[0].load(t0, n);
#pragma unroll
    for (int t = 0; t < TERMS; ++t) rx[t].init((t ? a.x_low : a.x) + rows + v0, DV, HV, true, tid), rx[t].load(0, n);
    if constexpr (TERMS == 2) ry[1].init(a.y_low + rows + v0, DV, HV, true, tid), ry[1].load(0, n);
  };
  auto rows_store = [&]() {
    rdo.store(tdo);
#pragma unroll
    for (int i = 0; i < rv.N; ++i)
#pragma unroll
      for (int c = 0; c < P; ++c) {  // e = v - x
        if constexpr (TERMS == 2) {
          const float e = (float)rv.r[i][c] - joined(rx[0].r[i][c], rx[1].r[i][c]);
          rx[0].r[i][c] = (bf16)e, rx[1].r[i][c] = (bf16)(e - (float)rx[0].r[i][c]);
        } else {
          rx[0].r[i][c] = rv.r[i][c] - rx[0].r[i][c];
        }
      }
#pragma unroll
    for (int t = 0; t < TERMS; ++t) rx[t].store(te + t * C * LDV), ry[t].store(ty + t * C * LDV);
  };
  // SV rows of a state (by its terms) on their way to LDS: S's, then R's, then the next ones
  constexpr int SP = (SV * DK / P + THREADS - 1) / THREADS, PARTS = 2 * DV / SV;
  piece_t<E> sp[SP];
  [[maybe_unused]] u32x2 sp_low[SP];
  const int64_t state = ((int64_t)bh * a.chunks + chunk) * DK * DV;
  auto state_load = [&](int part) {
    const int64_t at = state + part / 2 * SV * DK;
#pragma unroll
    for (int i = 0; i < SP; ++i) {
      const int e = (i * THREADS + tid) * P;
      if (e >= SV * DK) continue;
      sp[i] = *reinterpret_cast<const piece_t<E>*>((part & 1 ? a.r : a.s) + at + e);
      if constexpr (TERMS == 2) sp_low[i] = *reinterpret_cast<const u32x2*>((part & 1 ? a.r_low : a.s_low) + at + e);
    }
  };
  auto state_store = [&]() {
#pragma unroll
    for (int i = 0; i < SP; ++i) {
      const int e = (i * THREADS + tid) * P;
      if (e >= SV * DK) continue;
      E* dst = ts + e / DK * LDK + e % DK;
      *reinterpret_cast<piece_t<E>*>(dst) = sp[i];
      if constexpr (TERMS == 2) *reinterpret_cast<piece_t<E>*>(dst + SV * LDK) = second_terms(sp[i], sp_low[i]);
    }
  };
  rows_load(0);
  state_load(0);
  if (wave == 0) {
    const bool live = lane < n;
    float g = live ? p.g[b * p.gs[0] + (t0 + lane) * p.gs[1] + h * p.gs[2]] : 0.0f;
    const float bt = live ? (float)p.beta[b * p.bs[0] + (t0 + lane) * p.bs[1] + h * p.bs[2]] : 0.0f;
    g = g < kNoDecay ? kNoDecay : g;
    double sum = (double)g;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
      const double v = __shfl_up(sum, i, 64);
      if (lane >= i) sum += v;
    }
    const double end = __shfl(sum, 63, 64);
    if (lane < C) G[lane] = sum, from[lane] = __expf((float)sum), to[lane] = __expf((float)(end - sum)), beta[lane] = bt;
  }

  const int it = wave / WC, kt0 = (wave % WC) * KT, row = 16 * it + lo;
  // R's part is scaled by exp(G_end - G_j) beta_j, S's by -exp(G_j): kept apart until the sums are whole
  f32x4 aq[KT], as[KT], ar[KT], s1[S::MINE], s2[S::MINE];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) aq[kt] = as[kt] = ar[kt] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < S::MINE; ++k) s1[k] = s2[k] = f32x4{0, 0, 0, 0};
  // this wave's tiles of the scores: rows 16 ti, columns 16 tj; not live: all zeros
  int ti[S::MINE], tj[S::MINE];
  bool live[S::MINE];
#pragma unroll
  for (int k = 0; k < S::MINE; ++k) {
    const int t = wave + k * S::WAVES;
    ti[k] = t >= S::LOWER ? 2 * (t - S::LOWER) : t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0;
    tj[k] = t >= S::LOWER ? ti[k] + 1 : t - tri(ti[k], 0);
    live[k] = t < S::LOWER && 16 * ti[k] < n;
  }
  DeltaRows<E, C, DK, THREADS> rk, rq;
  // two quads of each of an operand's terms
  auto two = [&](const E* z, int ld, int r0, int c0, int lane, quad_t<E> (&x)[2]) {
    x[0] = lds_quad(z, ld, r0, c0, lane), x[1] = lds_quad(z, ld, r0, c0 + 16, lane);
  };
#pragma unroll 1
  for (int part = 0; part < PARTS; part += 2 * HV / SV) {  // HV values
    if (part > 0) rows_load(part / 2 * SV);  // (not ahead of their use: held in registers they cost 566 us for 512)
    __syncthreads();
    rows_store();
#pragma unroll
    for (int sub = 0; sub < 2 * HV / SV; ++sub) {
      if (sub > 0) __syncthreads();
      state_store();
      __syncthreads();
      if (part + sub + 1 < PARTS) state_load(part + sub + 1);
      if (16 * it >= n) continue;
      const int lane = here(tid & 63);
#pragma unroll
      for (int v = 0; v < SV; v += 32) {
        const int col = sub / 2 * SV + v;
        quad_t<E> x[3][2];  // this wave's rows of dO and y (by its terms), or of e's terms
        if (sub & 1) {
#pragma unroll
          for (int t = 0; t < TERMS; ++t) two(te + t * C * LDV, LDV, 16 * it, col, lane, x[t]);
        } else {
          two(tdo, LDV, 16 * it, col, lane, x[0]);
#pragma unroll
          for (int t = 0; t < TERMS; ++t) two(ty + t * C * LDV, LDV, 16 * it, col, lane, x[1 + t]);
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int t = 0; t < TERMS; ++t) {  // the state's first term with all of theirs, the second with their first
            const quad_t<E> s0 = lds_quad_t(ts + t * SV * LDK, LDK, v, 16 * (kt0 + kt), lane);
            const quad_t<E> s1 = lds_quad_t(ts + t * SV * LDK, LDK, v + 16, 16 * (kt0 + kt), lane);
            if (sub & 1) {
#pragma unroll
              for (int u = 0; u < (t ? 1 : TERMS); ++u) ar[kt] = mma2(s0, s1, x[u][0], x[u][1], ar[kt]);
            } else {
              aq[kt] = mma2(s0, s1, x[0][0], x[0][1], aq[kt]);
#pragma unroll
              for (int u = 0; u < (t ? 1 : TERMS); ++u) as[kt] = mma2(s0, s1, x[1 + u][0], x[1 + u][1], as[kt]);
            }
          }
      }
    }
#pragma unroll
    for (int k = 0; k < S::MINE; ++k) {
      if (!live[k]) continue;
      const int lane = here(tid & 63);
#pragma unroll
      for (int v = 0; v < HV; v += 32) {
        quad_t<E> g[2], y[TERMS][2], e[TERMS][2];
        two(tdo, LDV, 16 * ti[k], v, lane, g);
#pragma unroll
        for (int t = 0; t < TERMS; ++t) two(ty + t * C * LDV, LDV, 16 * ti[k], v, lane, y[t]), two(te + t * C * LDV, LDV, 16 * tj[k], v, lane, e[t]);
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
          s1[k] = mma2(e[t][0], e[t][1], g[0], g[1], s1[k]);
#pragma unroll
          for (int u = 0; u < (t ? 1 : TERMS); ++u) s2[k] = mma2(e[t][0], e[t][1], y[u][0], y[u][1], s2[k]);
        }
      }
    }
  }
  rk.init(p.k + b * p.ks[0] + (h / p.gk) * p.ks[2], p.ks[1], p.dk, p.vec, tid);
  rq.init(p.q + b * p.qs[0] + (h / p.gq) * p.qs[2], p.qs[1], p.dk, p.vec, tid);
  rk.load(t0, n), rq.load(t0, n);
  const float ff = from[row], ft = to[row], bt = beta[row];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) aq[kt] *= p.scale * ff, ar[kt] = ft * bt * ar[kt] - ff * as[kt];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < S::MINE; ++k) {
    if (wave + k * S::WAVES >= S::TILES) continue;
    const int i = 16 * ti[k] + lo, j0 = 16 * tj[k] + 4 * hi;
    f32x4 m = {0, 0, 0, 0}, nn = {0, 0, 0, 0};
    if (live[k]) {
      const f32x4 bj = lds_f4(beta + j0);
      const double mine = G[i];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = j0 + r;
        const float ratio = __expf((float)(mine - G[j])) * bj[r];
        m[r] = j <= i ? p.scale * ratio * s1[k][r] : 0.0f;
        nn[r] = j < i ? -ratio * s2[k][r] : 0.0f;
      }
    }
    const Terms<E> m_terms(m), n_terms(nn);
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
      *reinterpret_cast<quad_t<E>*>(tm + t * C * LDC + i * LDC + j0) = m_terms.t[t];
      *reinterpret_cast<quad_t<E>*>(tm + (TERMS + t) * C * LDC + i * LDC + j0) = n_terms.t[t];
    }
  }
  rk.store(tk), rq.store(tq);
  __syncthreads();
  if (16 * it >= n) return;
#pragma unroll
  for (int jt = 0; jt < CT; jt += 2) {
    if (16 * jt >= n) continue;
    const bool below = jt <= it, above = jt + 1 >= it;  // tiles left of the diagonal, or below it and read across
    const int lane = here(tid & 63);
    quad_t<E> m[TERMS][2], mt[TERMS][2], nl[TERMS][2], nt[TERMS][2];
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
      const E *zm = tm + t * C * LDC, *zn = tm + (TERMS + t) * C * LDC;
      if (below) two(zm, LDC, 16 * it, 16 * jt, lane, m[t]), two(zn, LDC, 16 * it, 16 * jt, lane, nl[t]);
      if (above) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          mt[t][u] = lds_quad_t(zm, LDC, 16 * (jt + u), 16 * it, lane), nt[t][u] = lds_quad_t(zn, LDC, 16 * (jt + u), 16 * it, lane);
      }
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int col = 16 * (kt0 + kt);
      const quad_t<E> k0 = lds_quad_t(tk, LDK, 16 * jt, col, lane), k1 = lds_quad_t(tk, LDK, 16 * jt + 16, col, lane);
      if (below) {
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
          aq[kt] = mma2(k0, k1, m[t][0], m[t][1], aq[kt]);
          ar[kt] = mma2(k0, k1, nl[t][0], nl[t][1], ar[kt]);
        }
      }
      if (above) {
        const quad_t<E> q0 = lds_quad_t(tq, LDK, 16 * jt, col, lane), q1 = lds_quad_t(tq, LDK, 16 * jt + 16, col, lane);
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
          ar[kt] = mma2(k0, k1, nt[t][0], nt[t][1], ar[kt]);
          ar[kt] = mma2(q0, q1, mt[t][0], mt[t][1], ar[kt]);
        }
      }
    }
  }
  if (row >= n) return;
  const int64_t at = obase + (t0 + row) * orow;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    const int c = 16 * (kt0 + kt) + 4 * hi;
    if (a.q_part) store_quad((float*)a.dq + at, c, p.dk, aq[kt]);
    else store_quad((E*)a.dq + at, c, p.dk, aq[kt]);
    if (a.k_part) store_quad((float*)a.dk + at, c, p.dk, ar[kt]);
    else store_quad((E*)a.dk + at, c, p.dk, ar[kt]);
  }
}

// One step, S := a S + k^T u, u = beta (v - a k S), o = scale q S, in place: a (problem, head) a workgroup, thread
// (row group, 4 columns) with NR rows of S in registers between its one read and its write;
// k S and q S are summed over the row groups in LDS together, o = scale (a q S + (q . k) u).
// Bound by the state's read and write: 4096 problems, a quarter of them idle, 8 heads of 64 x 64: 148 to 153
// us, 5.2 TB/s.
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
