// Gated feed-forward block  y = (act(x Wg^T) o (x Wu^T)) Wd^T  and its backward pass:
//   dh = dy Wd;  dG = dh o U o act'(G);  dU = dh o act(G);
//   dx = dG Wg + dU Wu;  dWg = dG^T x;  dWu = dU^T x;  dWd = dy^T h.
// Both projections, the activation and the product are one kernel: a column tile of
// the product holds 16 columns of the gate next to the same 16 of the other
// projection, so a lane has both values of a feature.  The product dy Wd ends in the
// derivatives, so dh is never written; h is formed again there from the saved G, U.
// Every matrix here is multiplied in the layout it is stored in: an operand whose
// contracted index is its row (W in dx, every operand of the weight gradients) is
// staged as it lies and read from LDS transposed.
// Bound by the matrix units where the widths are large (gemm_wide.hpp), by the (M, F)
// arrays of the backward pass at 20705 x 512 x 1408 (545 us a training step, 1.0 GB of them
// among it), and by latency on small shapes: 64 rows of 256 x 683 5.0 and 6.3 us for the two kernels.
#pragma once
#include "learn_common.hpp"

namespace tmpc {

enum { ACT_SILU = 0, ACT_GELU = 1 };

// act(g) and its derivative
template <int ACT>
__device__ inline void act_both(float g, float& a, float& d) {
  if constexpr (ACT == ACT_SILU) {
    const float sg = 1.0f / (1.0f + __expf(-g));
    a = g * sg;
    d = sg * (1.0f + g * (1.0f - sg));
  } else {
    const float phi = 0.5f * erfcf(-0.70710678118654752f * g);
    a = g * phi;
    d = phi + g * (0.39894228040143268f * __expf(-0.5f * g * g));
  }
}
template <int ACT>
__device__ inline float act_only(float g) {
  if constexpr (ACT == ACT_SILU) return g / (1.0f + __expf(-g));
  return g * (0.5f * erfcf(-0.70710678118654752f * g));
}

// out (M, N) = sum over segments s of A_s B_s, K contracted entries each.
//   A_s (M, K) of pitch lda, or (K, M) with AT; B_s (N, K) of pitch ldb, or (K, N) with BT.
// DUAL: B_0, B_1 are the two projections (no segments).
template <typename E>
struct GemmArgs {
  int64_t M;
  int N, nseg;
  int pair;          // 1: two products A_0^T B_0 -> o0 and A_1^T B_0 -> o1, the grid's x twice as long
  int64_t K;
  const E *A[2], *B[2];
  int64_t lda, ldb;
  // outputs; pitches in elements
  E *o0, *o1, *o2;
  float *g, *u;      // the saved projections: fp32, for rounding them would double the gradients' error
  int64_t ldo, ldg;  // pitches of o* and of g, u
  float* part;       // split over K: (splits, 1 + pair, M, N) partial sums
  int64_t k_split;   // contracted entries of a split (a multiple of the K tile)
};

enum GemmEpi {
  EPI_STORE = 0,     // o0 = acc
  EPI_GATE = 1,      // DUAL: o0 = act(G) o U
  EPI_GATE_SAVE = 2, // and g = G, u = U
  EPI_DGATE = 3,     // acc = dh: o0 = dG, o1 = dU, o2 = h from the saved g, u
  EPI_PART = 4       // part[split] = acc
};

template <typename E>
constexpr int kGemmBK = 128 / sizeof(E);  // contracted entries of a step

// The operand tile of one K step: global memory -> registers -> LDS.
template <typename E, int BR, int BK, int THREADS, bool TR, bool DUAL>
struct Stage {
  static constexpr int P = Elem<E>::PIECE, PAD = 16 / sizeof(E);
  static constexpr int LD = TR ? BR + PAD : BK + PAD;
  static constexpr int ELEMS = TR ? BK * LD : BR * LD;
  static constexpr int NP = BR * BK / P / THREADS;
  static_assert(NP * THREADS * P == BR * BK, "a whole number of pieces a thread");
  piece_t<E> r[NP];

  // Rows r0 .. of an operand with `rows` rows (outer index) and K contracted entries, zeros
  // past K.  Which of the three ways is the same for the whole tile, and none branches
  // between its loads, so that all of them are in flight together.
  __device__ void load(const E* const* src, int seg, int64_t ld, int64_t r0, int64_t rows, int64_t k0, int64_t K, int tid) {
    const int rl = (int)(rows - r0 < BR ? rows - r0 : BR), kl = (int)(K - k0 < BK ? K - k0 : BK);  // live ones, >= 1
    const int width = TR ? rl : kl, deep = TR ? kl : rl;  // of a stored row; stored rows
    // piece i's place in the tile, and its row of the operand (past the edge: the last one)
    auto piece = [&](int i, int& row, int& c) -> const E* {
      const int e = tid + i * THREADS, w = (TR ? BR : BK) / P;
      row = e / w, c = (e - row * w) * P;
      if constexpr (DUAL) {  // 16 rows of the one, 16 of the other
        const int f = (row >> 5) * 16 + (row & 15);
        return src[(row >> 4) & 1] + (r0 + min(f, deep - 1)) * ld + k0;
      } else {
        const int64_t f = min(row, deep - 1);
        return src[seg] + (TR ? (k0 + f) * ld + r0 : (r0 + f) * ld + k0);
      }
    };
    if (width == (TR ? BR : BK) && (!TR || deep == BK)) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        int row, c;
        const E* at = piece(i, row, c);
        r[i] = *reinterpret_cast<const typename Elem<E>::piece_u*>(at + c);
      }
    } else if (width % P == 0) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        int row, c;
        const E* at = piece(i, row, c);
        const piece_t<E> v = *reinterpret_cast<const typename Elem<E>::piece_u*>(at + min(c, width - P));
        const bool live = c < width && (!TR || row < deep);
#pragma unroll
        for (int e = 0; e < P; ++e) r[i][e] = live ? v[e] : E(0.0f);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        int row, c;
        const E* at = piece(i, row, c);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const E v = at[min(c + e, width - 1)];
          r[i][e] = c + e < width && (!TR || row < deep) ? v : E(0.0f);
        }
      }
    }
  }
  __device__ void store(E* t, int tid) const {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int e = tid + i * THREADS, w = (TR ? BR : BK) / P;
      const int row = e / w, c = (e - row * w) * P;
      *reinterpret_cast<piece_t<E>*>(t + row * LD + c) = r[i];
    }
  }
  // The quads of outer rows row0 + 0..15 over 32 contracted entries from k0.  WHOLE: a lane
  // takes 8 consecutive entries (one 16-byte read), which both operands have to do.
  template <bool WHOLE>
  __device__ static void quads(const E* t, int row0, int k0, int lane, quad_t<E>& q0, quad_t<E>& q1) {
    if constexpr (TR) {
      q0 = lds_quad_t(t, LD, k0, row0, lane);
      q1 = lds_quad_t(t, LD, k0 + 16, row0, lane);
    } else if constexpr (WHOLE && sizeof(E) == 2) {
      const piece_t<E> v = *reinterpret_cast<const piece_t<E>*>(t + (row0 + (lane & 15)) * LD + k0 + 8 * (lane >> 4));
      q0 = __builtin_shufflevector(v, v, 0, 1, 2, 3);
      q1 = __builtin_shufflevector(v, v, 4, 5, 6, 7);
    } else {
      q0 = lds_quad(t, LD, row0, k0, lane);
      q1 = lds_quad(t, LD, row0, k0 + 16, lane);
    }
  }
};

// A wave's results: TM x TN tiles from row m0 and column tile j0 of the block's n0; a lane
// has row i * 16 + lo, 4 consecutive columns.
template <typename E, int EPI, int ACT, int TM, int TN>
__device__ inline void gemm_epilogue(const GemmArgs<E>& p, const f32x4 (&acc)[TM][TN], int which, int64_t m0, int64_t n0,
                                     int j0, int lo, int hi) {
  constexpr bool DUAL = EPI == EPI_GATE || EPI == EPI_GATE_SAVE;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t m = m0 + i * 16 + lo;
    if (m >= p.M) continue;
    if constexpr (DUAL) {
      static_assert(TN % 2 == 0, "a wave holds both projections of its features");
#pragma unroll
      for (int j = 0; j < TN; j += 2) {
        const int64_t c = n0 + (j0 + j) * 8 + 4 * hi;
        f32x4 hv;
#pragma unroll
        for (int r = 0; r < 4; ++r) hv[r] = act_only<ACT>(acc[i][j][r]) * acc[i][j + 1][r];
        if (c >= p.N) continue;
        store_quad(p.o0 + m * p.ldo, (int)c, p.N, hv);
        if constexpr (EPI == EPI_GATE_SAVE) {
          store_quad(p.g + m * p.ldg, (int)c, p.N, acc[i][j]);
          store_quad(p.u + m * p.ldg, (int)c, p.N, acc[i][j + 1]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int64_t c = n0 + (j0 + j) * 16 + 4 * hi;
        if (c >= p.N) continue;
        if constexpr (EPI == EPI_STORE) {
          store_quad((which ? p.o1 : p.o0) + m * p.ldo, (int)c, p.N, acc[i][j]);
        } else if constexpr (EPI == EPI_PART) {
          store_quad(p.part + ((int64_t)(blockIdx.z * (1 + p.pair) + which) * p.M + m) * p.N, (int)c, p.N, acc[i][j]);
        } else {
          const f32x4 gv = load_quad_f32(p.g + m * p.ldg, (int)c, p.N), uv = load_quad_f32(p.u + m * p.ldg, (int)c, p.N);
          f32x4 dg, du, hv;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float a, d;
            act_both<ACT>(gv[r], a, d);
            dg[r] = acc[i][j][r] * uv[r] * d, du[r] = acc[i][j][r] * a, hv[r] = a * uv[r];
          }
          store_quad(p.o0 + m * p.ldo, (int)c, p.N, dg);
          store_quad(p.o1 + m * p.ldo, (int)c, p.N, du);
          store_quad(p.o2 + m * p.ldo, (int)c, p.N, hv);
        }
      }
    }
  }
}

// BM x BN tile by WM x WN waves; BN counts both projections' columns with DUAL.
template <typename E, int BM, int BN, int WM, int WN, bool AT, bool BT, int EPI, int ACT>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_kernel(GemmArgs<E> p) {
  constexpr bool DUAL = EPI == EPI_GATE || EPI == EPI_GATE_SAVE;
  constexpr int THREADS = 64 * WM * WN, BK = kGemmBK<E>;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr bool WHOLE = !AT && !BT;
  constexpr int BF = DUAL ? BN / 2 : BN;  // output columns of the tile
  using SA = Stage<E, BM, BK, THREADS, AT, false>;
  using SB = Stage<E, BN, BK, THREADS, BT, DUAL>;
  extern __shared__ __align__(16) char smem[];
  E* ta = reinterpret_cast<E*>(smem);
  E* tb = ta + 2 * SA::ELEMS;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4;
  const int wm = wave / WN, wn = wave - wm * WN;
  const int which = p.pair && blockIdx.x >= gridDim.x / 2;
  const int64_t m0 = (int64_t)(blockIdx.x - which * (gridDim.x / 2)) * BM;
  const int64_t n0 = (int64_t)blockIdx.y * BF;
  const int64_t kb = (int64_t)blockIdx.z * p.k_split;
  const int64_t ke = EPI == EPI_PART ? (kb + p.k_split < p.K ? kb + p.k_split : p.K) : p.K;
  const int tiles = (int)((ke - kb + BK - 1) / BK), total = tiles * (DUAL ? 1 : p.nseg);

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  SA sa;
  SB sb;
  int seg = 0;
  int64_t k = kb;
  if (total > 0) {
    sa.load(p.A, which, p.lda, m0, p.M, k, ke, tid);
    sb.load(p.B, 0, p.ldb, n0, p.N, k, ke, tid);
    sa.store(ta, tid);
    sb.store(tb, tid);
  }
  __syncthreads();
  for (int it = 0; it < total; ++it) {
    const E* ca = ta + (it & 1) * SA::ELEMS;
    const E* cb = tb + (it & 1) * SB::ELEMS;
    const bool more = it + 1 < total;
    if (more) {
      k += BK;
      if (k >= ke) k = kb, ++seg;
      sa.load(p.A, seg + which, p.lda, m0, p.M, k, ke, tid);
      sb.load(p.B, seg, p.ldb, n0, p.N, k, ke, tid);
    }
#pragma unroll
    for (int kk = 0; kk < BK; kk += 32) {
      quad_t<E> a0[TM], a1[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) SA::template quads<WHOLE>(ca, (wm * TM + i) * 16, kk, lane, a0[i], a1[i]);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        quad_t<E> b0, b1;
        SB::template quads<WHOLE>(cb, (wn * TN + j) * 16, kk, lane, b0, b1);
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[i][j] = mma2(b0, b1, a0[i], a1[i], acc[i][j]);
      }
    }
    if (more) {  // the other buffer was last read before the previous barrier
      sa.store(ta + ((it + 1) & 1) * SA::ELEMS, tid);
      sb.store(tb + ((it + 1) & 1) * SB::ELEMS, tid);
    }
    __syncthreads();
  }

  gemm_epilogue<E, EPI, ACT, TM, TN>(p, acc, which, m0 + wm * TM * 16, n0, wn * TN, lo, hi);
}

// The partial sums over the splits, in order: (splits, outputs, n) -> o0 and, of two
// outputs, o1.  A thread 4 entries.
template <typename E>
__global__ __launch_bounds__(256) void gemm_reduce_kernel(const float* __restrict__ part, int64_t n, int outputs,
                                                          int splits, E* __restrict__ o0, E* __restrict__ o1) {
  const int64_t all = n * outputs;
  for (int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; e < all; e += (int64_t)gridDim.x * 1024) {
    f32x4 v = {0, 0, 0, 0};
    if (e + 4 <= all) {
      for (int s = 0; s < splits; ++s) v += load_quad_f32(part + (int64_t)s * all + e, 0, 4);
    } else {
      for (int s = 0; s < splits; ++s) v += load_quad_f32(part + (int64_t)s * all + e, 0, (int)(all - e));
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t i = e + r;
      if (i < n) o0[i] = (E)v[r];
      else if (i < all) o1[i - n] = (E)v[r];
    }
  }
}

// Few rows (M <= 16 MT): bound by reading the weights, and below that by latency.  A
// workgroup has one tile of 16 output columns; its eight waves share the contracted
// index, each reading its own 32-entry steps straight into operands, and meet in LDS.
template <typename E, int MT, int EPI, int ACT>
__global__ __launch_bounds__(512) void gemm_rows_kernel(GemmArgs<E> p) {
  constexpr bool DUAL = EPI == EPI_GATE || EPI == EPI_GATE_SAVE;
  constexpr int NB = DUAL ? 2 : 1, P = Elem<E>::PIECE, STEP = 4 * P;  // contracted entries of a step
  __shared__ f32x4 red[8][MT * NB][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + lo < p.N ? n0 + lo : p.N - 1;  // past the edge: results not stored
  const E* b[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) b[i] = p.B[i] + n * p.ldb;
  const E* a[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = 16 * i + lo < p.M ? 16 * i + lo : p.M - 1;
    a[i] = p.A[0] + m * p.lda;
  }
  f32x4 acc[MT][NB];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  auto mul = [&](const piece_t<E>(&pa)[MT], const piece_t<E>(&pb)[NB]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if constexpr (sizeof(E) == 2) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pb[j], pa[i], acc[i][j], 0, 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(pb[j][e], pa[i][e], acc[i][j], 0, 0, 0);
        }
      }
  };
  // whole steps, U at a time so that their loads are in flight together
  constexpr int U = 4;
  const int64_t steps = p.K / STEP;
  int64_t s = wave;
  for (; s + 8 * (U - 1) < steps; s += 8 * U) {
    piece_t<E> pa[U][MT], pb[U][NB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = (s + 8 * u) * STEP + P * hi;
#pragma unroll
      for (int j = 0; j < NB; ++j) pb[u][j] = *reinterpret_cast<const typename Elem<E>::piece_u*>(b[j] + k);
#pragma unroll
      for (int i = 0; i < MT; ++i) pa[u][i] = *reinterpret_cast<const typename Elem<E>::piece_u*>(a[i] + k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) mul(pa[u], pb[u]);
  }
  for (; s * STEP < p.K; s += 8) {
    const int64_t k = s * STEP;
    piece_t<E> pa[MT], pb[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) pb[j] = load_piece(b[j] + k, P * hi, (int)(p.K - k < STEP ? p.K - k : STEP), true);
#pragma unroll
    for (int i = 0; i < MT; ++i) pa[i] = load_piece(a[i] + k, P * hi, (int)(p.K - k < STEP ? p.K - k : STEP), true);
    mul(pa, pb);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) red[wave][i * NB + j][lane] = acc[i][j];
  __syncthreads();
  if (wave >= MT) return;
  f32x4 sum[1][NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    sum[0][j] = red[0][wave * NB + j][lane];
#pragma unroll
    for (int w = 1; w < 8; ++w) sum[0][j] += red[w][wave * NB + j][lane];
  }
  gemm_epilogue<E, EPI, ACT, 1, NB>(p, sum, 0, 16 * wave, n0, 0, lo, hi);
}

template <typename E, int BM, int BN, bool AT, bool BT, int THREADS, bool DUAL>
constexpr size_t gemm_lds() {
  constexpr int BK = kGemmBK<E>;
  return 2 * sizeof(E) * (size_t)(Stage<E, BM, BK, THREADS, AT, false>::ELEMS + Stage<E, BN, BK, THREADS, BT, DUAL>::ELEMS);
}

}  // namespace tmpc
