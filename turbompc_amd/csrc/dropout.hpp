// Dropout whose mask is made again wherever it is needed and never stored:
//   y = x / (share kept) where kept, else 0.
// Element (row, column) is kept where its 16 random bits are at least p 65536 (rounded to a whole
// number, so the share kept is exactly (65536 - that) / 65536).  The bits are half word
// column % 8 of Philox-4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", 2011) at the counter (column / 8, row, call, step) under a 64-bit key: any thread can
// make any element's bits, and the 16 bytes of 8 bf16 elements take one evaluation.  Bound by memory, the
// generator's 80 instructions an evaluation behind it: 206848 x 512, bf16: 75 to 78 us a direction, 5.5 TB/s.
#pragma once
#include "learn_common.hpp"

namespace tmpc {

struct DropKey {
  const int64_t* key;  // (seed, step), on the device; NULL: nothing is dropped
  uint32_t call, least;
  float factor;
};

struct Philox {
  uint32_t k0, k1, call, step;
  __device__ Philox(const DropKey& d) : k0(0), k1(0), call(d.call), step(0) {
    if (d.key) {
      const uint64_t seed = (uint64_t)d.key[0];
      k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32), step = (uint32_t)d.key[1];
    }
  }
  __device__ inline uint4 operator()(uint32_t piece, uint32_t row) const {
    uint32_t c0 = piece, c1 = row, c2 = call, c3 = step, a = k0, b = k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      const uint64_t m0 = (uint64_t)0xD2511F53u * c0, m1 = (uint64_t)0xCD9E8D57u * c2;
      c0 = (uint32_t)(m1 >> 32) ^ c1 ^ a, c1 = (uint32_t)m1;
      c2 = (uint32_t)(m0 >> 32) ^ c3 ^ b, c3 = (uint32_t)m0;
      a += 0x9E3779B9u, b += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
  }
};

// the piece of a row from column c on (a multiple of the piece): a bit an element, set where it is kept
template <int P>
__device__ inline uint32_t drop_mask(const Philox& rng, const DropKey& d, uint32_t row, int c) {
  const uint4 w = rng((uint32_t)c / 8, row);
  const bool second = P == 4 && (c & 4);
  const uint32_t bits[4] = {second ? w.z : w.x, second ? w.w : w.y, w.z, w.w};
  uint32_t kept = 0;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    const uint32_t h = e & 1 ? bits[e / 2] >> 16 : bits[e / 2] & 0xffffu;
    kept |= (h >= d.least ? 1u : 0u) << e;
  }
  return kept;
}
// what is kept, times the factor
template <int P>
__device__ inline void drop_piece(uint32_t kept, const DropKey& d, float (&v)[P]) {
#pragma unroll
  for (int e = 0; e < P; ++e) v[e] = kept >> e & 1 ? v[e] * d.factor : 0.0f;
}

// A thread a piece, `pieces` a row.
template <typename E>
__global__ __launch_bounds__(256) void dropout_kernel(uint32_t n, int width, uint32_t pieces, uint32_t row0, const E* x,
                                                      int64_t ldx, DropKey d, E* y) {
  constexpr int P = Elem<E>::PIECE;
  const Philox rng(d);
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) {
    const uint32_t r = i / pieces, row = row0 + r;
    const int c = (int)(i - r * pieces) * P;
    const piece_t<E> in = load_piece(x + row * ldx, c, width, true);
    float v[P];
#pragma unroll
    for (int e = 0; e < P; ++e) v[e] = (float)in[e];
    drop_piece(drop_mask<P>(rng, d, row, c), d, v);
    piece_t<E> out;
#pragma unroll
    for (int e = 0; e < P; ++e) out[e] = (E)v[e];
    store_piece(y + (int64_t)row * width, c, width, out);
  }
}

}  // namespace tmpc
