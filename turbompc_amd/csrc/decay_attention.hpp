// Linear attention with a decay for each head.  Problem b, head h, g = log_decay[h]:
//   S_t = e^g S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t        (S fp32, DK x DV).
//
// Chunked form.  Over C steps from the state S_in,
//   O = (Q K^T o Gamma) V + diag(e^{g (i+1)}) Q S_in,  Gamma_ij = e^{g (i-j)} for i >= j, else 0
//   S_out = e^{g L} S_in + K^T diag(e^{g (L-1-j)}) V,  L the chunk's live steps;
// every exponent's factor of g is >= 0, so a strong decay underflows to zero and
// nothing overflows.  Gamma's zeros hold for finite values alone: runs with others are made
// again step by step (attn_by_step).
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

// Steps of a chunk: 64 rows of 128 bf16 values are 16 KiB, 32 of as many fp32 ones the same.
template <typename E>
struct AttnTile {
  static constexpr int C = sizeof(E) == 2 ? 64 : 32;
  static constexpr int PAD = 16 / sizeof(E);          // of an LDS row: its quads spread over the banks
};

__device__ inline float decay_pow(float g, int n) { return n == 0 ? 1.0f : __expf(g * (float)n); }

// By its bytes (q, k, v read and o written once) the operator is bound by memory; what the
// kernels meet first is the latency of the chain inside a chunk, two waves a SIMD, with
// vector and matrix instructions each issuing about a third of the time (64 x 64 heads:
// 413 and 58 a wave and chunk).  One launch over 512 heads of 1024 steps, 64 wide, bf16: 74
// us, 3.6 TB/s of the 4.9 that a copy reaches; 50001 steps of 16 heads, 128 wide, in 32 runs
// a head: 254 us, and 121 and 16 us for the runs' sums and their scan.
//
// A workgroup carries one (problem, head) through its chunks.  Wave w owns NV
// 16-column tiles of the values and all of the scores: S, the scores and O stay in
// its registers (each product's accumulator is the next one's operand) and waves meet
// only where a chunk's rows change in LDS.  Every wave forms the scores again: cheaper than
// an exchange through LDS and the barrier that it needs, up to 128 x 128.
template <typename E, int DA, int DC>
struct AttnShape {
  static constexpr int W = DC / 16 < 4 ? DC / 16 : 4;  // waves
  static constexpr int NV = DC / 16 / W;               // value tiles of a wave
  static constexpr int THREADS = 64 * W;
  static constexpr int C = AttnTile<E>::C;
  static constexpr int LDA = DA + AttnTile<E>::PAD, LDC = DC + AttnTile<E>::PAD;
  // 128 x 128: the registers do not hold the operands of all scores beside S, so the waves
  // share the scores out and exchange them in LDS
  static constexpr bool SHARE = DA == 128 && DC == 128;
  static constexpr int LDP = C + AttnTile<E>::PAD;
  // Registers that a lane holds through a whole chunk: S and the next chunk's rows on their way (a
  // row of `d` elements takes d / P threads).  Where they are many, no operand is kept from one row
  // tile to the next, or they spill: 64 x 512 x 8 heads, bf16, 128 x 32 (104 held) 78 us against
  // 116, 128 x 128 (112) no difference, 128 x 64 (72) 66 against 62, 64 x 128 and 64 x 64 (64, 40) none.
  static constexpr int rows_held(int d) {
    constexpr int P = Elem<E>::PIECE;
    return 4 * C / (THREADS / (d / P) < C ? THREADS / (d / P) : C);
  }
  static constexpr int HELD = DA / 16 * NV * 4 + 2 * rows_held(DA) + rows_held(DC);
  static constexpr bool FENCE = HELD > 96;
  // elements of a chunk's rows in LDS: b and c, and a (and the scores) with outputs
  static constexpr int TILE_STATE = C * LDA + C * LDC, TILE = TILE_STATE + C * LDA + (SHARE ? C * LDP : 0);
  // workgroups of a CU, by their registers; the tiles twice (one barrier a chunk instead of
  // two) where they still fit
  static constexpr int PER_CU = 2;
  static constexpr int BUFS = 2 * sizeof(E) * TILE <= 160 * 1024 / PER_CU ? 2 : 1;
  static constexpr size_t LDS_STATE = sizeof(E) * (size_t)BUFS * TILE_STATE;
  static constexpr size_t LDS = sizeof(E) * (size_t)BUFS * TILE;
};

// Buffer descriptors let a load or store name a place past the end: the load gives zero,
// the store is dropped, and no branch stands between the memory operations of a chunk.
constexpr unsigned kBufferEnd = 0x80000000u, kNowhere = 0xfffffff0u;  // bytes from a descriptor's base
__device__ inline __amdgpu_buffer_rsrc_t buffer_at(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, kBufferEnd, 0x00027000);
}
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// A chunk's rows of one operand on their way from memory through registers to LDS: the
// next chunk's are in flight while this one's are multiplied.  A thread moves N pieces
// of one column, RS rows apart.  VEC: rows of whole pieces at 4-byte addresses; else any
// width and alignment, element by element.
template <typename E, int C, int D, int THREADS, bool VEC>
struct AttnRows {
  static constexpr int P = Elem<E>::PIECE, W = D / P, RS = THREADS / W < C ? THREADS / W : C, N = C / RS;
  static constexpr int LD = D + AttnTile<E>::PAD;
  static_assert(THREADS % W == 0 && C % RS == 0, "whole rows a pass");
  piece_t<E> r[N];
  const E* base;    // the first step of the next chunk
  int64_t step;     // elements between steps, negative where they are walked backwards
  unsigned off[N];  // bytes from the chunk's lowest address
  int row, c;

  __device__ void init(const E* b, int64_t stride, int t0, int width, int tid) {
    row = tid / W, c = (tid - row * W) * P, step = stride;
    base = b + t0 * stride;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t s = stride < 0 ? -stride * (C - 1 - row - i * RS) : stride * (row + i * RS);
      off[i] = c < width && row < RS ? (unsigned)((s + c) * (int64_t)sizeof(E)) : kNowhere;
    }
  }
  // the next chunk's rows, n of them live
  __device__ void load(int n, int width) {
    const __amdgpu_buffer_rsrc_t rs = buffer_at(step < 0 ? base + (C - 1) * step : base);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned at = row + i * RS < n ? off[i] : kNowhere;
      if constexpr (VEC) {
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
    base += C * step;
  }
  __device__ void store(E* tile) const {
    if (RS * W < THREADS && row >= RS) return;
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<piece_t<E>*>(tile + (row + i * RS) * LD + c) = r[i];
  }
};

__device__ inline float uniform(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}

// a b, and 0 where either is zero, an infinity's factor or not: what overflows above the
// diagonal has no part in a score
extern "C" __device__ float mul_zero(float a, float b) __asm("llvm.amdgcn.fmul.legacy");

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

// One chunk of one recurrence for a wave's NV value tiles (columns col0 ..): the outputs
// through store(tile it, x, values of row 16 it + lo, columns 4 hi ..), and the state.
// n live steps; ta, tb (C x DA, pitch LDA) and tc (pitch LDC) hold zeros after them.
template <typename E, typename S, int KA, int NV, int CT, bool FULL, typename Store>
__device__ inline void attn_chunk(const E* ta, const E* tb, const E* tc, E* tp, int col0, f32x4 (&s)[KA][NV],
                                  const AttnPowers<CT>& pw, float g, float su, int rev, int n, int lane, Store store) {
  constexpr int C = S::C, LDA = S::LDA, LDC = S::LDC, LDP = S::LDP;
  const int lo = lane & 15, hi = lane >> 4;
  // A tile (it, jt <= it) of the scores as its transpose: a lane holds 4 consecutive j of one
  // i, the operand of the product with V; rounded to E, as the output is.  a: row tile it's quads.
  auto score = [&](int jt, const quad_t<E>(&a)[KA]) {
    f32x4 t = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < KA; k += 2)
      t = mma2(lds_quad(tb, LDA, 16 * jt, 16 * k, lane), lds_quad(tb, LDA, 16 * jt, 16 * k + 16, lane), a[k], a[k + 1], t);
    return t;
  };
  if constexpr (FULL && S::SHARE) {
    for (int q = S::W - 1 - (col0 / (16 * NV)); q < CT * (CT + 1) / 2; q += S::W) {
      int it = 0, jt = q;
      while (jt > it) jt -= ++it;
      float far = 1.0f;
#pragma unroll
      for (int d = 1; d < CT - 1; ++d) far *= it - jt - 1 >= d ? pw.tile[1] : 1.0f;
      quad_t<E> a[KA];
#pragma unroll
      for (int k = 0; k < KA; ++k) a[k] = lds_quad(ta, LDA, 16 * it, 16 * k, lane);
      f32x4 t = score(jt, a);
#pragma unroll
      for (int r = 0; r < 4; ++r) t[r] = mul_zero(t[r], it == jt ? pw.diag[r] : far * pw.near[r]);
      *reinterpret_cast<quad_t<E>*>(tp + (16 * it + lo) * LDP + 16 * jt + 4 * hi) = to_quad<E>(t);
    }
    __syncthreads();
  }
  // the wave's values, contracted over the steps
  quad_t<E> v[CT][NV];
#pragma unroll
  for (int j = 0; j < CT; ++j)
#pragma unroll
    for (int x = 0; x < NV; ++x) v[j][x] = lds_quad_t(tc, LDC, 16 * j, col0 + 16 * x, lane);

  if constexpr (FULL) {
    quad_t<E> sq[KA][NV];  // the state rounds to E as this product's operand only
#pragma unroll
    for (int k = 0; k < KA; ++k)
#pragma unroll
      for (int x = 0; x < NV; ++x) sq[k][x] = to_quad<E>(s[k][x]);
#pragma unroll
    for (int it = 0; it < CT; ++it) {
      // Past the last live step.  With the scores shared the branch costs registers, which spill: 64 x
      // 512 x 8 heads 97.5 us against 87.9; ragged batches of 512 x 4 heads of up to 512, 200 and 70
      // steps 286, 142 and 80 against 268, 138 and 82.
      if (!S::SHARE && 16 * it >= n) break;
      if constexpr (S::FENCE) asm volatile("" ::: "memory");
      quad_t<E> a[KA];
#pragma unroll
      for (int k = 0; k < KA; ++k) a[k] = lds_quad(ta, LDA, 16 * it, 16 * k, lane);
      // O^T tiles: columns i, rows the values
      f32x4 acc[NV];
#pragma unroll
      for (int x = 0; x < NV; ++x) acc[x] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KA; k += 2)
#pragma unroll
        for (int x = 0; x < NV; ++x) acc[x] = mma2(sq[k][x], sq[k + 1][x], a[k], a[k + 1], acc[x]);
      const float f = pw.rowf * pw.tile[it];
#pragma unroll
      for (int x = 0; x < NV; ++x) acc[x] *= f;
#pragma unroll
      for (int j = 0; j <= it; j += 2) {
        quad_t<E> p[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int jt = j + e;
          if (jt > it) {
            p[e] = to_quad<E>(f32x4{0, 0, 0, 0});
          } else if constexpr (S::SHARE) {
            p[e] = lds_quad(tp, LDP, 16 * it, 16 * jt, lane);
          } else {
            f32x4 t = score(jt, a);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              t[r] = mul_zero(t[r], jt == it ? pw.diag[r] : pw.tile[it > jt ? it - jt - 1 : 0] * pw.near[r]);
            p[e] = to_quad<E>(t);
          }
        }
#pragma unroll
        for (int x = 0; x < NV; ++x) acc[x] = mma2(v[j][x], v[j + 1][x], p[0], p[1], acc[x]);
      }
#pragma unroll
      for (int x = 0; x < NV; ++x) store(it, x, acc[x]);
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
    if (16 * j >= n) break;  // (128 x 128, the same cases: 88, 268, 138 and 82 us against 99, 335, 168 and 98 without)
    f32x4 d0, d1;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (whole) {
        d0[r] = pw.tile[CT - 1 - j] * pw.tail[r], d1[r] = pw.tile[CT - 2 - j] * pw.tail[r];
      } else {
        const int j0 = 16 * j + 4 * hi + r;
        d0[r] = su * decay_pow(g, max(n - 1 - j0, 0) + rev);
        d1[r] = su * decay_pow(g, max(n - 17 - j0, 0) + rev);
      }
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
}

// The state's rows 16 m + 4 hi + r, columns col0 + 16 x + lo of a (da, dc) matrix, or of
// the transpose of a (dc, da) one; zeros where src is NULL and outside.
template <int KA, int NV>
__device__ inline void load_state(f32x4 (&s)[KA][NV], const float* src, bool transposed, int da, int dc, int col0, int lo,
                                  int hi) {
  const __amdgpu_buffer_rsrc_t rs = buffer_at(src);
  const int rp = transposed ? 1 : dc, cp = transposed ? da : 1;
#pragma unroll
  for (int m = 0; m < KA; ++m)
#pragma unroll
    for (int x = 0; x < NV; ++x)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * m + 4 * hi + r, col = col0 + 16 * x + lo;
        const unsigned at = src && row < da && col < dc ? (row * rp + col * cp) * 4u : kNowhere;
        s[m][x][r] = __builtin_bit_cast(float, (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 0));
      }
}
template <int KA, int NV>
__device__ inline void store_state(const f32x4 (&s)[KA][NV], float* dst, int da, int dc, int col0, int lo, int hi) {
  const __amdgpu_buffer_rsrc_t rs = buffer_at(dst);
#pragma unroll
  for (int m = 0; m < KA; ++m)
#pragma unroll
    for (int x = 0; x < NV; ++x)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * m + 4 * hi + r, col = col0 + 16 * x + lo;
        const float v = s[m][x][r];
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), rs,
                                              row < da && col < dc ? (row * dc + col) * 4u : kNowhere, 0, 0);
      }
}

// Zero rows [z0, z1) of an output (T, H, d) of one head from `base`.
__device__ inline void zero_rows(void* o, bool f32, int elem, int64_t base, int64_t pitch, int d, int64_t z0, int64_t z1,
                                 int tid, int threads) {
  for (int64_t e = z0 * d + tid; e < z1 * d; e += threads) {
    const int64_t t = e / d, at = base + t * pitch + (e - t * d);
    if (f32 || elem == 4)
      reinterpret_cast<float*>(o)[at] = 0.0f;
    else
      reinterpret_cast<uint16_t*>(o)[at] = 0;
  }
}

// A wave's columns of a run whose keys or values are not all finite, by the definition, a step
// at a time: in a chunk they meet the earlier steps' outputs with a factor of zero, which
// makes those NaN.  Rare, so simple and in few registers.
template <typename E, int KA, int NV>
__device__ __attribute__((always_inline)) inline void attn_by_step(const AttnArgs<E>& p, int block, int tid) {
  const int lo = tid & 15, hi = (tid & 63) >> 4, col0 = (tid >> 6) * NV * 16;
  const int bh = block / p.segs, seg = block - bh * p.segs, b = bh / p.H, h = bh - b * p.H;
  const float g = p.log_decay[h];
  const int L = attn_length(p, b), begin = seg * p.seg_len, end = min(L, begin + p.seg_len);
  const int64_t first = p.rev ? L - 1 : 0, dir = p.rev ? -1 : 1;
  const E* pa = p.a + b * p.as[0] + (h / p.ga) * p.as[2] + first * p.as[1];
  const E* pb = p.b + b * p.bs[0] + (h / p.gb) * p.bs[2] + first * p.bs[1];
  const E* pc = p.c + b * p.cs[0] + (h / p.gc) * p.cs[2] + first * p.cs[1];
  const int64_t orow = (int64_t)p.H * p.dc, o = ((int64_t)b * p.T * p.H + h) * p.dc + first * orow;
  const int64_t size = (int64_t)p.da * p.dc, sbase = bh * size;
  f32x4 s[KA][NV];
  if (p.segs > 1) load_state(s, p.seg_state + block * size, false, p.da, p.dc, col0, lo, hi);
  else load_state(s, p.s_in ? p.s_in + sbase : nullptr, p.s_in_t, p.da, p.dc, col0, lo, hi);
  const float gamma = decay_pow(g, 1), before = p.rev ? 1.0f : gamma, after = p.rev ? gamma : 1.0f;
  for (int t = begin; t < end; ++t) {
    const E *at = pa + dir * t * p.as[1], *bt = pb + dir * t * p.bs[1], *ct = pc + dir * t * p.cs[1];
    float cv[NV], sum[NV];
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      const int col = col0 + 16 * x + lo;
      cv[x] = col < p.dc ? p.su * (float)ct[col] : 0.0f, sum[x] = 0.0f;
    }
#pragma unroll
    for (int m = 0; m < KA; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * m + 4 * hi + r;
        if (row >= p.da) continue;
        const float av = (float)at[row], bv = (float)bt[row];
#pragma unroll
        for (int x = 0; x < NV; ++x) {
          s[m][x][r] = s[m][x][r] * before + bv * cv[x];
          sum[x] += av * s[m][x][r];
          s[m][x][r] *= after;
        }
      }
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      const int col = col0 + 16 * x + lo;
      sum[x] += __shfl_xor(sum[x], 16, 64);
      sum[x] += __shfl_xor(sum[x], 32, 64);
      if (hi == 0 && col < p.dc) {
        if (p.o_f32) reinterpret_cast<float*>(p.o)[o + dir * t * orow + col] = p.si * sum[x];
        else reinterpret_cast<E*>(p.o)[o + dir * t * orow + col] = (E)(p.si * sum[x]);
      }
    }
  }
  if (p.s_out && seg == (L - 1) / p.seg_len) store_state(s, p.s_out + sbase, p.da, p.dc, col0, lo, hi);
}

// FULL: outputs and the carried state; else the run's own sum alone, into seg_state.
template <typename E, int DA, int DC, bool FULL, bool VEC>
__global__ __launch_bounds__((AttnShape<E, DA, DC>::THREADS), 2) void attn_chunk_kernel(AttnArgs<E> p) {
  using S = AttnShape<E, DA, DC>;
  constexpr int C = S::C, NV = S::NV, LDA = S::LDA, LDC = S::LDC, CT = C / 16, KA = DA / 16;
  constexpr int TILE = FULL ? S::TILE : S::TILE_STATE;
  extern __shared__ __align__(16) char smem[];
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

  AttnRows<E, C, DA, S::THREADS, VEC> ra, rb;
  AttnRows<E, C, DC, S::THREADS, VEC> rc;
  rb.init(pb, dir * p.bs[1], begin, p.da, tid);
  rc.init(pc, dir * p.cs[1], begin, p.dc, tid);
  if constexpr (FULL) ra.init(pa, dir * p.as[1], begin, p.da, tid);
  auto fetch = [&](int n) {
    rb.load(n, p.da);
    rc.load(n, p.dc);
    if constexpr (FULL) ra.load(n, p.da);
  };
  if (begin < end) fetch(end - begin);
  f32x4 s[KA][NV];
  if constexpr (FULL)
    load_state(s, seg_state ? seg_state : p.s_in ? p.s_in + sbase : nullptr, !seg_state && p.s_in_t, p.da, p.dc, col0, lo, hi);
  else
    load_state(s, nullptr, false, p.da, p.dc, col0, lo, hi);
  AttnPowers<CT> pw;
  pw.init(g, p.rev, p.ss, p.si, p.su, lo, hi);
  const int osize = p.o_f32 ? 4 : (int)sizeof(E);
  // the output chunk's lowest row, and this lane's place in it
  char* obuf = reinterpret_cast<char*>(p.o) + (obase + (first + dir * begin - (p.rev ? C - 1 : 0)) * orow) * osize;
  unsigned ooff[NV];
#pragma unroll
  for (int x = 0; x < NV; ++x) {
    const int c = col0 + 16 * x + 4 * hi;
    ooff[x] = c < p.dc ? (unsigned)(((p.rev ? C - 1 - lo : lo) * orow + c) * osize) : kNowhere;
  }
  const int otile = (int)(dir * 16 * orow * osize);
  int buf = 0;
  for (int t0 = begin; t0 < end; t0 += C) {
    const int n = min(C, end - t0);  // live steps
    E* tb = reinterpret_cast<E*>(smem) + buf * TILE;
    E* tc = tb + C * LDA;
    E* ta = tc + C * LDC;
    rb.store(tb);
    rc.store(tc);
    if constexpr (FULL) ra.store(ta);
    __syncthreads();
    if (t0 + C < end) fetch(end - t0 - C);
    attn_chunk<E, S, KA, NV, CT, FULL>(ta, tb, tc, ta + C * LDA, col0, s, pw, g, p.su, p.rev, n, lane,
                                              [&](int it, int x, f32x4 v) {
      const __amdgpu_buffer_rsrc_t rs = buffer_at(obuf);
      const unsigned at = 16 * it + lo < n && ooff[x] != kNowhere ? ooff[x] + it * otile : kNowhere;
      if constexpr (VEC) {
        if (sizeof(E) == 4 || p.o_f32)
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rs, at, 0, 0);
        else
          __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, to_bf16(v)), rs, at, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned ae = col0 + 16 * x + 4 * hi + e < p.dc && at != kNowhere ? at + e * osize : kNowhere;
          const float f = v[e];
          if (sizeof(E) == 4 || p.o_f32)
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, f), rs, ae, 0, 0);
          else
            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (bf16)f), rs, ae, 0, 0);
        }
      }
    });
    obuf += dir * C * orow * osize;
    if constexpr (S::BUFS == 2)
      buf ^= 1;  // the other tiles' readers passed this chunk's barrier
    else
      __syncthreads();
  }

  // What follows makes its indexes again from one that the compiler does not see through: its
  // addresses and load_state's would be kept through every chunk (64 x 1024 x 8 heads, 64 x 64, with
  // gradients 267 us against 271, 2048 x 101 x 4, 64 x 128, 918 against 975).
  int end_tid = tid;
  asm volatile("" : "+v"(end_tid));
  const int end_lo = end_tid & 15, end_hi = (end_tid & 63) >> 4, end_col = (end_tid >> 6) * NV * 16;
  if constexpr (FULL) {  // this run's steps past the end
    zero_rows(p.o, p.o_f32, sizeof(E), obase, orow, p.dc, max(L, begin), min((int64_t)p.T, (int64_t)begin + p.seg_len), tid,
              S::THREADS);
    // An infinite or NaN key or value leaves the state so, to the end: in all columns, or in its own.
    f32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int m = 0; m < KA; ++m)
#pragma unroll
      for (int x = 0; x < NV; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) zero[r] = fmaf(s[m][x][r], 0.0f, zero[r]);
    if (begin < end && __ballot(!(zero[0] + zero[1] + zero[2] + zero[3] == 0.0f))) {
      __threadfence_block();  // the rows written above are written again; the state is not written yet
      // The arguments are read again too, for the same reason.  (In a function that is called their
      // address is null: it is taken in the kernel.)
      auto* args = __builtin_amdgcn_kernarg_segment_ptr();
      int block = blockIdx.x;
      asm volatile("" : "+s"(args), "+s"(block));
      attn_by_step<E, KA, NV>(*(const AttnArgs<E>*)args, block, end_tid);
    } else if (p.s_out && seg == (L > 0 ? (L - 1) / p.seg_len : 0)) {  // the run that holds the last live step
      store_state(s, p.s_out + sbase, p.da, p.dc, end_col, end_lo, end_hi);
    }
  } else {
    store_state(s, seg_state, p.da, p.dc, end_col, end_lo, end_hi);
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
// A thread 4 columns of a row; q = ceil(d / 4).
template <typename E>
__global__ __launch_bounds__(256) void attn_head_sum_kernel(const float* __restrict__ in, int64_t rows, int G, int d, int q,
                                                            E* __restrict__ out) {
  const int per = 256 / q;  // rows a block at a time
  const int r = threadIdx.x / q, c = (threadIdx.x - r * q) * 4;
  if (r >= per) return;
  for (int64_t row = (int64_t)blockIdx.x * per + r; row < rows; row += (int64_t)gridDim.x * per) {
    const float* src = in + row * G * d;
    f32x4 v = {0, 0, 0, 0};
    for (int i = 0; i < G; ++i) v += load_quad_f32(src + (int64_t)i * d, c, d);
    store_quad(out + row * d, c, d, v);
  }
}

// One step: S := e^g S + k^T v, o = scale q S in place, a (problem, head) a workgroup.
// Bound by the state's read and write: 4096 problems of 8 heads of 64 x 64, a quarter of
// them idle, 155 us, 5.2 TB/s.  Thread (row group, 4 columns): the rows of S
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
