// The block's bf16 products on large shapes: 256 x 256 tiles by eight waves (128 x 64
// each), K steps of 64, operands moved from memory straight into LDS.  A step takes 2048
// cycles of the matrix units against about 1536 of LDS reads, which is why the tile is no
// smaller; two tiles of each operand (128 KiB) leave one workgroup a CU.  16384 x 2048 x
// 5504: both projections 763 us, the down projection 369 us alone, 1150 TFLOP/s over the
// block, where 128 x 128 tiles through registers (gemm_kernel) reach 590 and a library's plain
// product of the first shape 1060.
#pragma once
#include "gated_ff.hpp"

namespace tmpc {

// 16 bytes a lane from base + off (bytes) to LDS at lds + 16 * lane: the data never pass
// through registers.  Waited for with dma_wait, before a barrier.
__device__ inline void dma_to_lds(const void* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ inline void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// One operand's tile: 256 outer entries x 64 contracted ones, 32 KiB.
//   !TR: rows of 64 contracted entries (8 pieces of 16 bytes); piece p of row r lies in
//        slot p ^ (r % 8), so 16 rows of one piece column spread over the banks.
//   TR:  64 rows of 256 outer entries (32 pieces); piece p of row k lies in slot
//        p ^ 2 (k % 4 + 4 (k / 8 % 4)): a transposed read takes 32 bytes of the 16 rows
//        8 g + r (g, r < 4), which then meet every bank twice.
template <bool TR, bool DUAL>
struct WideTile {
  static constexpr int BK = 64, R = 256, BYTES = R * BK * 2;
  unsigned off[4];  // bytes from the tile's base, of the four pieces this lane moves

  __device__ static int tr_swizzle(int k) { return 2 * ((k & 3) + 4 * ((k >> 3) & 3)); }

  __device__ void init(int64_t ld, int64_t r0, int64_t rows, int tid) {
    const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (!TR) {
        int row = (wave * 4 + i) * 8 + (lane >> 3);
        if constexpr (DUAL) row = (row >> 5) * 16 + (row & 15);
        const int64_t last = rows - 1 - r0;  // past the edge: any row, its results are not stored
        row = row < last ? row : (int)last;
        off[i] = (unsigned)(((int64_t)row * ld + (((lane & 7) ^ (lane >> 3)) * 8)) * 2);
      } else {
        const int k = (wave * 4 + i) * 2 + (lane >> 5);
        int c = ((lane & 31) ^ tr_swizzle(k)) * 8;
        const int64_t last = ((rows - r0 + 7) & ~int64_t(7)) - 8;
        c = c < last ? c : (int)last;
        off[i] = (unsigned)(((int64_t)k * ld + c) * 2);
      }
    }
  }
  // which of the two projections' rows piece i of this wave comes from
  __device__ static int matrix(int i, int tid) { return DUAL ? (((tid >> 6) * 4 + i) >> 1) & 1 : 0; }

  __device__ static const bf16* base(const bf16* src, int64_t ld, int64_t r0, int64_t k) {
    return TR ? src + k * ld + r0 : src + r0 * ld + k;
  }
  // a whole K step
  __device__ void move(const bf16* b0, const bf16* b1, unsigned lds, int tid) const {
    const unsigned at = lds + __builtin_amdgcn_readfirstlane(tid >> 6) * 4096;
#pragma unroll
    for (int i = 0; i < 4; ++i) dma_to_lds(matrix(i, __builtin_amdgcn_readfirstlane(tid)) ? b1 : b0, off[i], at + i * 1024);
  }
  // the last K step of `left` < 64 entries, zeros after them, through registers
  __device__ void move_tail(const bf16* b0, const bf16* b1, char* tile, int left, int tid) const {
    const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const char* src = reinterpret_cast<const char*>(matrix(i, tid) ? b1 : b0) + off[i];
      bf16x8 v;
      if constexpr (!TR) {
        const int c = ((lane & 7) ^ (lane >> 3)) * 8;
        v = load_piece(reinterpret_cast<const bf16*>(src) - c, c, left, true);
      } else {
        const int k = (wave * 4 + i) * 2 + (lane >> 5);
        v = load_piece(reinterpret_cast<const bf16*>(src), 0, 8, k < left);
      }
      *reinterpret_cast<bf16x8*>(tile + (wave * 4 + i) * 1024 + lane * 16) = v;
    }
  }
  // 8 contracted entries kk + 8 (lane / 16) .. of outer entry row0 + lane % 16
  __device__ static bf16x8 frag(const char* tile, int row0, int kk, int lane) {
    if constexpr (!TR) {
      const int row = row0 + (lane & 15), p = (kk >> 3) + (lane >> 4);
      return *reinterpret_cast<const bf16x8*>(tile + row * 128 + ((p ^ (row & 7)) << 4));
    } else {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      bf16x4 q[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = kk + 8 * (lane >> 4) + 4 * j + ((lane & 15) >> 2);
        const int c = row0 + 4 * (lane & 3);
        const char* at = tile + k * 512 + (((c >> 3) ^ tr_swizzle(k)) << 4) + (c & 4) * 2;
        q[j] = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at));
      }
      return __builtin_shufflevector(q[0], q[1], 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

constexpr int kWidePitch = 256 + 4;  // fp32 columns of the results' rows in LDS

// EPI_DGATE by way of LDS, 128 rows at a time, so that memory is read and written in whole rows
// of 256 columns: lane by lane they are 32- and 64-byte pieces of 16 rows (20705 x 512 x 1408:
// 198 us that way, 130 this; the products that only store are no faster for it, 1152 us
// against 1132 of 16384 x 2048 x 5504).  A thread has 8 columns.
template <int ACT>
__device__ inline void wide_dgate(const GemmArgs<bf16>& p, const f32x4 (&acc)[8][4], char* smem, int64_t m0, int64_t n0,
                                  int tid) {
  float* t = reinterpret_cast<float*>(smem);
  const int lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4, wm = wave >> 2, wn = wave & 3;
  const int c = (tid & 31) * 8, r0 = tid >> 5;
  const int64_t col = n0 + c;
  const int width = (int)(p.N - col < 8 ? p.N - col : 8);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half) __syncthreads();
    if (wm == half) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f32x4*>(t + (16 * i + lo) * kWidePitch + (wn * 4 + j) * 16 + 4 * hi) = acc[i][j];
    }
    __syncthreads();
    if (width <= 0) continue;
#pragma unroll 4
    for (int r = r0; r < 128; r += 16) {
      const int64_t m = m0 + 128 * half + r;
      if (m >= p.M) break;
      const float* v = t + r * kWidePitch + c;
      const float *gp = p.g + m * p.ldg + col, *up = p.u + m * p.ldg + col;
      const f32x4 g0 = load_quad_f32(gp, 0, width), g1 = load_quad_f32(gp, 4, width);
      const f32x4 u0 = load_quad_f32(up, 0, width), u1 = load_quad_f32(up, 4, width);
      bf16x8 dg, du, h;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float ge = e < 4 ? g0[e & 3] : g1[e & 3], ue = e < 4 ? u0[e & 3] : u1[e & 3];
        float a, d;
        act_both<ACT>(ge, a, d);
        dg[e] = (bf16)(v[e] * ue * d), du[e] = (bf16)(v[e] * a), h[e] = (bf16)(a * ue);
      }
      store_piece(p.o0 + m * p.ldo + col, 0, width, dg);
      store_piece(p.o1 + m * p.ldo + col, 0, width, du);
      store_piece(p.o2 + m * p.ldo + col, 0, width, h);
    }
  }
}

template <bool AT, bool BT, int EPI, int ACT>
__global__ __launch_bounds__(512, 2) void gemm_wide_kernel(GemmArgs<bf16> p) {
  constexpr bool DUAL = EPI == EPI_GATE || EPI == EPI_GATE_SAVE;
  constexpr int BM = 256, BN = 256, BK = 64, WN = 4, TM = 8, TN = 4;
  constexpr int BF = DUAL ? BN / 2 : BN;
  using TA = WideTile<AT, false>;
  using TB = WideTile<BT, DUAL>;
  extern __shared__ __align__(16) char smem[];
  typedef __attribute__((address_space(3))) char lds_char;
  const unsigned lds0 = (unsigned)(uintptr_t)(lds_char*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lo = lane & 15, hi = lane >> 4;
  const int wm = wave / WN, wn = wave - wm * WN;
  const int which = p.pair && blockIdx.x >= gridDim.x / 2;
  const int64_t m0 = (int64_t)(blockIdx.x - which * (gridDim.x / 2)) * BM, n0 = (int64_t)blockIdx.y * BF;
  const int64_t kb = (int64_t)blockIdx.z * p.k_split;
  const int64_t ke = EPI == EPI_PART ? (kb + p.k_split < p.K ? kb + p.k_split : p.K) : p.K;
  const int tiles = (int)((ke - kb + BK - 1) / BK), total = tiles * (DUAL ? 1 : p.nseg);

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  TA ta;
  TB tb;
  ta.init(p.lda, m0, p.M, tid);
  tb.init(p.ldb, n0, p.N, tid);
  int seg = 0;
  int64_t k = kb;
  auto stage = [&](int buf) {
    const int at = buf * (TA::BYTES + TB::BYTES);
    const bf16* a = TA::base(p.A[seg + which], p.lda, m0, k);
    const bf16* b = TB::base(DUAL ? p.B[0] : p.B[seg], p.ldb, n0, k);
    const bf16* b1 = DUAL ? TB::base(p.B[1], p.ldb, n0, k) : b;
    if (k + BK <= ke) {
      ta.move(a, a, lds0 + at, tid);
      tb.move(b, b1, lds0 + at + TA::BYTES, tid);
    } else {
      ta.move_tail(a, a, smem + at, (int)(ke - k), tid);
      tb.move_tail(b, b1, smem + at + TA::BYTES, (int)(ke - k), tid);
    }
    k += BK;
    if (k >= ke) k = kb, ++seg;
  };
  if (total > 0) stage(0);
  dma_wait();
  __syncthreads();
  for (int it = 0; it < total; ++it) {
    const char* ca = smem + (it & 1) * (TA::BYTES + TB::BYTES);
    const char* cb = ca + TA::BYTES;
    if (it + 1 < total) stage((it + 1) & 1);  // last read before the previous barrier
#pragma unroll
    for (int kk = 0; kk < BK; kk += 32) {
      bf16x8 a[TM], b[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) b[j] = TB::frag(cb, (wn * TN + j) * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < TM; ++i) a[i] = TA::frag(ca, (wm * TM + i) * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], a[i], acc[i][j], 0, 0, 0);
    }
    dma_wait();
    __syncthreads();
  }
  if constexpr (EPI == EPI_DGATE)
    wide_dgate<ACT>(p, acc, smem, m0, n0, tid);
  else
    gemm_epilogue<bf16, EPI, ACT, TM, TN>(p, acc, which, m0 + wm * TM * 16, n0, wn * TN, lo, hi);
}

// two tiles of each operand; EPI_DGATE's 128 rows of results are a little more
constexpr size_t wide_lds(int epi) { return epi == EPI_DGATE ? 128 * kWidePitch * 4 : 2 * 2 * 256 * 64 * 2; }

}  // namespace tmpc
