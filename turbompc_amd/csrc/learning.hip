// C ABI of the history model's operators (include/tmpc.h): argument checks, the
// choice of tile and workspace, launches.
#include <algorithm>

#include "../../include/tmpc.h"
#include "decay_attention.hpp"
#include "gated_ff.hpp"
#include "gemm_wide.hpp"
#include "rms_norm.hpp"

namespace tmpc {
namespace {

constexpr int kCUs = 256;

inline size_t align_up(size_t n) { return (n + 255) & ~size_t(255); }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int launch_status() { return hipGetLastError() == hipSuccess ? TMPC_OK : TMPC_ELAUNCH; }

// Dynamic LDS above the 64 KiB default needs an explicit opt-in per kernel.
template <typename K>
void lds_optin(K kernel, size_t bytes) {
  if (bytes > 65536)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)bytes);
}

// ---------------------------------------------------------------- rms norm --
constexpr int kMaxWidth = 8192;
// Blocks of the backward pass, whose rows meet in the blocks' partial sums.  bf16, forward and backward,
// with 512, 1024 and 2048: 206848 rows of 512 349, 330 and 373 us; 4096 of 8192 130, 148 and 187.
constexpr int kRmsBlocks = 1024;

// f(threads per row, pieces per thread) of the smallest form that holds `width`
template <typename E, typename F>
void with_row(int width, F f) {
  const int pieces = (width + Elem<E>::PIECE - 1) / Elem<E>::PIECE;
  using std::integral_constant;
  if (pieces <= 16) f(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (pieces <= 64) f(integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (pieces <= 128) f(integral_constant<int, 64>(), integral_constant<int, 2>());
  else if (pieces <= 256) f(integral_constant<int, 256>(), integral_constant<int, 1>());
  else if (pieces <= 512) f(integral_constant<int, 256>(), integral_constant<int, 2>());
  else if (pieces <= 1024) f(integral_constant<int, 256>(), integral_constant<int, 4>());
  else f(integral_constant<int, 256>(), integral_constant<int, 8>());
}

inline int64_t rms_rows_per_block(int width, int elem_bytes) {
  const int pieces = (width * elem_bytes + 15) / 16;
  return pieces <= 16 ? 16 : pieces <= 128 ? 4 : 1;
}
inline int64_t rms_backward_blocks(int64_t rows, int width, int elem_bytes) {
  return std::min<int64_t>(ceil_div(rows, rms_rows_per_block(width, elem_bytes)), kRmsBlocks);
}

bool rms_shape_ok(int64_t rows, int width) { return rows >= 0 && width >= 1 && width <= kMaxWidth; }

template <typename E>
int rms_forward_impl(hipStream_t st, int64_t rows, int32_t width, const void* x, int64_t ldx, const void* r,
                     int64_t ldr, const void* w, double eps, void* y, void* s, float* rstd) {
  if (!rms_shape_ok(rows, width)) return TMPC_EBADSHAPE;
  if (rows == 0) return TMPC_OK;
  if (!x || !w || !y || !(eps >= 0.0) || ldx < 0 || ldr < 0) return TMPC_EBADARG;
  const RmsArgs<E> a{rows, width, (const E*)x, (const E*)r, (const E*)w, ldx, ldr, (float)eps, (E*)y, (E*)s, rstd};
  with_row<E>(width, [&](auto tpr, auto np) {
    const int64_t blocks = ceil_div(rows, 256 / tpr());
    hipLaunchKernelGGL((rms_forward_kernel<E, tpr(), np()>), dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)),
                       dim3(256), 0, st, a);
  });
  return launch_status();
}

template <typename E>
int rms_backward_impl(hipStream_t st, int64_t rows, int32_t width, const void* dy, int64_t lddy, const void* ds,
                      int64_t ldds, const void* s, int64_t lds, const void* w, const float* rstd, void* dx, void* dw,
                      void* ws, size_t wsb) {
  if (!rms_shape_ok(rows, width)) return TMPC_EBADSHAPE;
  if (!dw || (rows > 0 && (!dy || !s || !w || !rstd || !dx)) || lddy < 0 || ldds < 0 || lds < 0) return TMPC_EBADARG;
  const int64_t blocks = rms_backward_blocks(rows, width, sizeof(E));
  const size_t need = (size_t)blocks * width * sizeof(float);
  if (wsb < need) return TMPC_EWORKSPACE;
  if (need > 0 && !ws) return TMPC_EBADARG;
  float* part = (float*)ws;
  if (rows > 0) {
    const RmsBwdArgs<E> a{rows, width, (const E*)dy, (const E*)ds, (const E*)s, (const E*)w, lddy, ldds, lds, rstd, (E*)dx, part};
    with_row<E>(width, [&](auto tpr, auto np) {
      hipLaunchKernelGGL((rms_backward_kernel<E, tpr(), np()>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    });
  }
  hipLaunchKernelGGL((rms_dweight_kernel<E>), dim3((unsigned)ceil_div(width, 16)), dim3(256), 0, st, part, (int)blocks,
                     width, (E*)dw);
  return launch_status();
}

// --------------------------------------------------------- decay attention --
constexpr int kMaxHeads = 32768;            // a chunk of contiguous output rows, 64 x H x 128 fp32, within 31 bits
constexpr int64_t kMaxStep = (1 << 23) - 1; // elements between steps: 64 fp32 steps within 31 bits
constexpr int kMaxSteps = 1 << 30;          // the last run's end, less than T + a run, and t0 + C within 31 bits

bool attn_shape_ok(const tmpc_decay_attention* a) {
  return a && a->B >= 0 && a->T >= 0 && a->T <= kMaxSteps && a->H >= 1 && a->Hk >= 1 && a->H % a->Hk == 0 && a->dk >= 1 && a->dk <= 128 &&
         a->dv >= 1 && a->dv <= 128 && (int64_t)a->B * a->H <= 1 << 23 && a->H <= kMaxHeads;  // threads of a launch within 32 bits
}
// a chunk's steps lie within the 31 bits of a descriptor
bool step_ok(const int64_t* stride) { return stride[1] >= 0 && stride[1] <= kMaxStep; }

// One long history of few heads does not fill the chip, its chunks following one another:
// it is cut into runs of whole chunks.  A first pass sums each run on its own (keys and
// values alone), a scan carries the states through, and the outputs start from those.
// As many runs as are resident together, two workgroups a CU (one more round of them costs more:
// 96 heads of 2048 steps, 64 wide, bf16, 48 us in 5 runs a head, 58 in 6); two runs a head do not pay
// for reading keys and values twice (192 heads, 1024 steps: 53 us against 44 whole; 160 heads in
// three: 45 against 43, and 71 against 91 with 2048 steps).  A run has four chunks at least (16
// heads, 1024 steps: 25 us against 35 with eight), a history that is cut 16 (512 steps whole 22
// us, in two runs 25).
struct AttnSplit {
  int segs, len;
};
template <typename E>
AttnSplit attn_split(int64_t bh, int T) {
  constexpr int C = AttnTile<E>::C;
  const int64_t chunks = std::max<int64_t>(1, ceil_div(T, C));
  const int64_t runs = 2 * kCUs / std::max<int64_t>(bh, 1);
  const int64_t want = runs < 3 || chunks < 16 ? 1 : std::min(runs, chunks / 4);
  const int64_t len = ceil_div(chunks, want);
  return {(int)ceil_div(chunks, len), (int)(len * C)};
}
template <typename E>
size_t attn_split_bytes(const tmpc_decay_attention* x) {
  const int64_t bh = (int64_t)x->B * x->H;
  const int segs = bh > 0 ? attn_split<E>(bh, x->T).segs : 1;
  return segs > 1 ? align_up((size_t)bh * segs * x->dk * x->dv * sizeof(float)) : 0;
}

// Rows of whole 16-byte pieces at 4-byte addresses: moved a piece at a time.
template <typename E>
bool attn_vec_ok(const AttnArgs<E>& p) {
  constexpr int P = Elem<E>::PIECE;
  bool ok = p.da % P == 0 && p.dc % P == 0 && ((uintptr_t)p.o & 3) == 0;
  auto operand = [&](const E* x, const int64_t* s) {
    if (((uintptr_t)x & 3) != 0) ok = false;
    for (int i = 0; i < 3; ++i)
      if (s[i] * (int64_t)sizeof(E) % 4 != 0) ok = false;
  };
  operand(p.a, p.as), operand(p.b, p.bs), operand(p.c, p.cs);
  return ok;
}

template <typename E>
void launch_attn(hipStream_t st, AttnArgs<E> p, float* seg_state) {
  const AttnSplit split = attn_split<E>((int64_t)p.B * p.H, p.T);
  p.segs = split.segs, p.seg_len = split.len, p.seg_state = seg_state;
  const bool vec = attn_vec_ok(p);
  auto run = [&](auto da, auto dc, auto v) {
    using S = AttnShape<E, da(), dc()>;
    const dim3 grid((unsigned)(p.B * p.H * p.segs));
    if (p.segs > 1) {
      auto k = attn_chunk_kernel<E, da(), dc(), false, v()>;
      lds_optin(k, S::LDS_STATE);
      hipLaunchKernelGGL(k, grid, dim3(S::THREADS), S::LDS_STATE, st, p);
      hipLaunchKernelGGL((attn_scan_kernel<E>), dim3((unsigned)(p.B * p.H * ceil_div(p.da * p.dc, 256))), dim3(256), 0,
                         st, p);
    }
    auto k = attn_chunk_kernel<E, da(), dc(), true, v()>;
    lds_optin(k, S::LDS);
    hipLaunchKernelGGL(k, grid, dim3(S::THREADS), S::LDS, st, p);
  };
  auto go = [&](auto da, auto dc) {
    if (vec) run(da, dc, std::true_type());
    else run(da, dc, std::false_type());
  };
  using std::integral_constant;
  auto with_c = [&](auto da) {
    if (p.dc <= 32) go(da, integral_constant<int, 32>());
    else if (p.dc <= 64) go(da, integral_constant<int, 64>());
    else go(da, integral_constant<int, 128>());
  };
  if (p.da <= 32) with_c(integral_constant<int, 32>());
  else if (p.da <= 64) with_c(integral_constant<int, 64>());
  else with_c(integral_constant<int, 128>());
}

template <typename E>
AttnArgs<E> attn_args(const tmpc_decay_attention* x) {
  AttnArgs<E> p{};
  p.B = x->B, p.T = x->T, p.H = x->H, p.da = x->dk, p.dc = x->dv;
  p.log_decay = x->log_decay, p.lengths = x->lengths;
  p.ga = p.gb = p.gc = 1;
  return p;
}

template <typename E>
size_t attn_ws_bytes(const tmpc_decay_attention* x, bool backward) {
  const size_t split = attn_split_bytes<E>(x);
  if (!backward || x->H == x->Hk) return split;
  const size_t tok = (size_t)x->B * x->T * x->H * sizeof(float);
  return split + align_up(tok * x->dk) + align_up(tok * x->dv);
}

template <typename E>
int attn_forward_impl(hipStream_t st, const tmpc_decay_attention* x, void* o, float* state_out, void* ws, size_t wsb) {
  if (!attn_shape_ok(x)) return TMPC_EBADSHAPE;
  if (x->B == 0) return TMPC_OK;
  if (!step_ok(x->q_stride) || !step_ok(x->k_stride) || !step_ok(x->v_stride)) return TMPC_EBADSHAPE;
  if (!x->log_decay || (x->T > 0 && (!x->q || !x->k || !x->v || !o))) return TMPC_EBADARG;
  const size_t need = attn_ws_bytes<E>(x, false);
  if (wsb < need) return TMPC_EWORKSPACE;
  if (need > 0 && !ws) return TMPC_EBADARG;
  AttnArgs<E> p = attn_args<E>(x);
  p.a = (const E*)x->q, p.b = (const E*)x->k, p.c = (const E*)x->v;
  std::copy_n(x->q_stride, 3, p.as), std::copy_n(x->k_stride, 3, p.bs), std::copy_n(x->v_stride, 3, p.cs);
  p.gb = p.gc = x->H / x->Hk;
  p.ss = p.si = (float)x->scale, p.su = 1.0f;
  p.s_in = x->state_in, p.s_out = state_out, p.o = o;
  launch_attn(st, p, (float*)ws);
  return launch_status();
}

template <typename E>
int attn_backward_impl(hipStream_t st, const tmpc_decay_attention* x, const void* d_o, const int64_t* dos,
                       const float* d_state_out, void* dq, void* dk, void* dv, float* d_state_in, void* ws,
                       size_t wsb) {
  if (!attn_shape_ok(x)) return TMPC_EBADSHAPE;
  if (x->B == 0) return TMPC_OK;
  if (!step_ok(x->q_stride) || !step_ok(x->k_stride) || !step_ok(x->v_stride) || (dos && !step_ok(dos)))
    return TMPC_EBADSHAPE;
  if (!x->log_decay || !dos || (x->T > 0 && (!x->q || !x->k || !x->v || !d_o || !dq || !dk || !dv)))
    return TMPC_EBADARG;
  if (wsb < attn_ws_bytes<E>(x, true)) return TMPC_EWORKSPACE;
  if (attn_ws_bytes<E>(x, true) > 0 && !ws) return TMPC_EBADARG;
  float* seg_state = (float*)ws;
  char* rest = (char*)ws + attn_split_bytes<E>(x);
  const int G = x->H / x->Hk;
  const float scale = (float)x->scale;
  {  // dq: (do, v, k) from the transposed state
    AttnArgs<E> p = attn_args<E>(x);
    p.da = x->dv, p.dc = x->dk;
    p.a = (const E*)d_o, p.b = (const E*)x->v, p.c = (const E*)x->k;
    std::copy_n(dos, 3, p.as), std::copy_n(x->v_stride, 3, p.bs), std::copy_n(x->k_stride, 3, p.cs);
    p.gb = p.gc = G;
    p.ss = p.si = scale, p.su = 1.0f;
    p.s_in = x->state_in, p.s_in_t = 1, p.o = dq;
    launch_attn(st, p, seg_state);
  }
  // shared heads' gradients: every head's part in fp32, then their sum.  (Taking a group's heads
  // in turn in one workgroup needs no such parts, but its registers spill: 1755 us against 1088.)
  const size_t tok = (size_t)x->B * x->T * x->H * sizeof(float);
  float* gk = G > 1 ? (float*)rest : nullptr;
  float* gv = G > 1 ? (float*)(rest + align_up(tok * x->dk)) : nullptr;
  {  // dk: backwards, (v, do, q) from the transposed gradient of the state
    AttnArgs<E> p = attn_args<E>(x);
    p.da = x->dv, p.dc = x->dk, p.rev = 1;
    p.a = (const E*)x->v, p.b = (const E*)d_o, p.c = (const E*)x->q;
    std::copy_n(x->v_stride, 3, p.as), std::copy_n(dos, 3, p.bs), std::copy_n(x->q_stride, 3, p.cs);
    p.ga = G;
    p.ss = p.su = scale, p.si = 1.0f;
    p.s_in = d_state_out, p.s_in_t = 1;
    p.o = gk ? (void*)gk : dk, p.o_f32 = gk != nullptr;
    launch_attn(st, p, seg_state);
  }
  {  // dv: backwards, (k, q, do)
    AttnArgs<E> p = attn_args<E>(x);
    p.rev = 1;
    p.a = (const E*)x->k, p.b = (const E*)x->q, p.c = (const E*)d_o;
    std::copy_n(x->k_stride, 3, p.as), std::copy_n(x->q_stride, 3, p.bs), std::copy_n(dos, 3, p.cs);
    p.ga = G;
    p.ss = p.su = scale, p.si = 1.0f;
    p.s_in = d_state_out, p.s_out = d_state_in;
    p.o = gv ? (void*)gv : dv, p.o_f32 = gv != nullptr;
    launch_attn(st, p, seg_state);
  }
  if (G > 1 && x->T > 0) {
    auto sum = [&](const float* in, int d, void* out) {
      const int64_t rows = (int64_t)x->B * x->T * x->Hk;
      const int q = (d + 3) / 4;
      hipLaunchKernelGGL((attn_head_sum_kernel<E>), dim3((unsigned)std::min<int64_t>(ceil_div(rows, 256 / q), 16 * kCUs)),
                         dim3(256), 0, st, in, rows, G, d, q, (E*)out);
    };
    sum(gk, x->dk, dk);
    sum(gv, x->dv, dv);
  }
  return launch_status();
}

template <typename E>
int attn_step_impl(hipStream_t st, const tmpc_decay_attention* x, const uint8_t* active, float* state, void* o) {
  if (!attn_shape_ok(x) || x->T != 1) return TMPC_EBADSHAPE;
  if (x->B == 0) return TMPC_OK;
  if (!x->q || !x->k || !x->v || !x->log_decay || !state || !o) return TMPC_EBADARG;
  AttnStepArgs<E> p{x->B, x->H, x->H / x->Hk, x->dk, x->dv, (const E*)x->q, (const E*)x->k, (const E*)x->v};
  p.qs[0] = x->q_stride[0], p.qs[1] = x->q_stride[2];
  p.ks[0] = x->k_stride[0], p.ks[1] = x->k_stride[2];
  p.vs[0] = x->v_stride[0], p.vs[1] = x->v_stride[2];
  p.log_decay = x->log_decay, p.active = active, p.scale = (float)x->scale, p.state = state, p.o = (E*)o;
  hipLaunchKernelGGL((attn_step_kernel<E>), dim3((unsigned)(x->B * x->H)), dim3(256), 0, st, p);
  return launch_status();
}

// ------------------------------------------------------ gated feed-forward --
constexpr int64_t kMaxPitch = 1 << 20;  // elements: 256 rows of a tile within 31 bits, 65535 tiles of 32 columns

bool ff_shape_ok(const tmpc_gated_ff* a) {
  return a && a->M >= 0 && a->M <= 1 << 30 && a->D >= 1 && a->D <= kMaxPitch && a->F >= 1 && a->F <= kMaxPitch &&
         a->Dout >= 1 && a->Dout <= kMaxPitch && a->ldx <= kMaxPitch;
}
// pitch of the block's own (M, F) arrays: rows of whole 16-byte pieces
template <typename E>
int64_t ff_pitch(const tmpc_gated_ff* a) {
  return ceil_div(a->F, Elem<E>::PIECE) * Elem<E>::PIECE;
}

// How a product runs: few rows (gemm_rows_kernel), the wide kernel, or tiles of 128, 64
// or 32 rows; splits of the contracted index.
enum GemmForm { FORM_ROWS, FORM_WIDE, FORM_128, FORM_64, FORM_32 };
struct GemmPlan {
  GemmForm form;
  int splits;
};

inline int64_t tiles_of(int64_t rows, int64_t cols, int bm, int bf) { return ceil_div(rows, bm) * ceil_div(cols, bf); }

// The wide kernel moves 16-byte pieces between memory and LDS: rows of whole pieces.
template <typename E>
bool wide_ok(const GemmArgs<E>& p, bool at, bool bt, bool own_a, bool own_b) {
  if (sizeof(E) != 2) return false;
  auto aligned = [](const void* q) { return ((uintptr_t)q & 15) == 0; };
  for (int i = 0; i < 2; ++i)
    if (!aligned(p.A[i]) || !aligned(p.B[i])) return false;
  // a transposed operand's last piece reaches past its columns, within the pitch of the
  // block's own arrays alone
  return p.lda % 8 == 0 && p.ldb % 8 == 0 && (!at || own_a || p.M % 8 == 0) && (!bt || own_b || p.N % 8 == 0);
}

template <typename E, bool AT, bool BT, int EPI, int ACT = 0>
void launch_gemm(hipStream_t st, GemmArgs<E> p, GemmPlan plan) {
  constexpr bool DUAL = EPI == EPI_GATE || EPI == EPI_GATE_SAVE;
  if (plan.splits == 1) p.k_split = std::max<int64_t>(p.K, 1);
  auto grid = [&](int bm, int bf) {
    return dim3((unsigned)(ceil_div(p.M, bm) * (1 + p.pair)), (unsigned)ceil_div(p.N, bf), (unsigned)plan.splits);
  };
  auto go = [&](auto bm, auto bn) {
    constexpr int BM = bm(), BN = bn();
    constexpr size_t lds = gemm_lds<E, BM, BN, AT, BT, 256, DUAL>();
    auto k = gemm_kernel<E, BM, BN, 2, 2, AT, BT, EPI, ACT>;
    lds_optin(k, lds);
    hipLaunchKernelGGL(k, grid(BM, DUAL ? BN / 2 : BN), dim3(256), lds, st, p);
  };
  using std::integral_constant;
  switch (plan.form) {
    case FORM_ROWS:
      if constexpr (!AT && !BT && EPI != EPI_PART) {
        auto rows = [&](auto mt) {
          hipLaunchKernelGGL((gemm_rows_kernel<E, mt(), EPI, ACT>), dim3((unsigned)ceil_div(p.N, 16)), dim3(512), 0, st, p);
        };
        if (p.M <= 16) rows(integral_constant<int, 1>());
        else if (p.M <= 32) rows(integral_constant<int, 2>());
        else rows(integral_constant<int, 4>());
      }
      break;
    case FORM_WIDE:
      if constexpr (sizeof(E) == 2) {
        auto k = gemm_wide_kernel<AT, BT, EPI, ACT>;
        lds_optin(k, wide_lds(EPI));
        hipLaunchKernelGGL(k, grid(256, DUAL ? 128 : 256), dim3(512), wide_lds(EPI), st, p);
      }
      break;
    case FORM_128: go(integral_constant<int, 128>(), integral_constant<int, 128>()); break;
    case FORM_64: go(integral_constant<int, 64>(), integral_constant<int, 64>()); break;
    case FORM_32: go(integral_constant<int, 32>(), integral_constant<int, 64>()); break;
  }
}

// Small products have few tiles, each a chain of K steps whose loads' latency (about 1.3 us a
// step) nothing hides: the contracted index is split until four workgroups a CU hide it
// (fp32, 2091 x 200 from 2 x 520: 44 us in one, 29 in three with their sum).
template <typename E>
int store_splits(int64_t M, int64_t N, int64_t K, GemmForm form) {
  if (M == 0 || (form != FORM_64 && form != FORM_32)) return 1;
  const int64_t tiles = tiles_of(M, N, form == FORM_64 ? 64 : 32, 64);
  return (int)std::max<int64_t>(1, std::min(4 * kCUs / tiles, ceil_div(K, kGemmBK<E>) / 4));
}
// workspace for it: no form makes more splits of more rows than this
template <typename E>
size_t store_part_bytes(int64_t M, int64_t N, int64_t K) {
  int most = 1;
  for (GemmForm f : {FORM_64, FORM_32}) most = std::max(most, store_splits<E>(M, N, K, f));
  return most > 1 ? align_up((size_t)most * M * N * sizeof(float)) : 0;
}

// The form of a product, where both were measured (us of one product; bf16 unless it says fp32):
//   up to 64 rows, as many as gemm_rows_kernel's registers hold: 64 rows of 512 x 1408 14.2
//     against 15.2 in tiles, 16 rows 9.0 against 15.1; 64 of 2048 x 5504 51 and 55, fp32 108 and 100;
//   wide tiles once the 128s, four for each, take more than the one round of two workgroups a CU
//     that 128 wide tiles make: K = 512, 128 tiles 4.5 slower, 144 to 160 5.3 to 5.9 faster; K =
//     1408, 128 tiles 3.8 slower, 144 22 faster;
//   tiles of 128 once they are more than the CUs: K = 512, 256 tiles 2.6 slower than in 64s, 264 2.3
//     faster; K = 1408, 188 11 slower; fp32, 192 10 slower, 440 5.7 faster;
//   tiles of 64 from three for four CUs on: under it 32s are up to 1.6 faster (fp32 3.4), from 700
//     on up to 5 slower, in between the two are within 1.4 (fp32 4.3).
template <typename E, bool AT, bool BT, int EPI>
GemmPlan gemm_plan(const GemmArgs<E>& p, bool own_a, bool own_b) {
  constexpr int D = EPI == EPI_GATE || EPI == EPI_GATE_SAVE ? 2 : 1;
  if (!AT && !BT && p.nseg == 1 && p.M <= 64) return {FORM_ROWS, 1};
  if (wide_ok(p, AT, BT, own_a, own_b) && tiles_of(p.M, p.N, 256, 256 / D) > kCUs / 2) return {FORM_WIDE, 1};
  if (tiles_of(p.M, p.N, 128, 128 / D) > kCUs) return {FORM_128, 1};
  const GemmForm form = tiles_of(p.M, p.N, 64, 64 / D) >= 3 * kCUs / 4 ? FORM_64 : FORM_32;
  return {form, EPI == EPI_STORE ? store_splits<E>(p.M, p.N, p.K, form) : 1};
}

// launch_gemm, with the sum over the plan's splits through `part`
template <typename E, bool AT, bool BT>
void launch_store(hipStream_t st, GemmArgs<E> p, GemmPlan plan, float* part) {
  if (plan.splits == 1) {
    launch_gemm<E, AT, BT, EPI_STORE>(st, p, plan);
    return;
  }
  p.part = part;
  p.k_split = ceil_div(ceil_div(p.K, kGemmBK<E>), plan.splits) * kGemmBK<E>;
  launch_gemm<E, AT, BT, EPI_PART>(st, p, plan);
  const int64_t n = p.M * p.N;
  hipLaunchKernelGGL((gemm_reduce_kernel<E>), dim3((unsigned)std::min<int64_t>(ceil_div(n * (1 + p.pair), 1024), 8 * kCUs)),
                     dim3(256), 0, st, part, n, 1 + p.pair, plan.splits, p.o0, p.o1);
}

// The weight gradients' rows are few and their contracted index is every row of the batch:
// it is split until the tiles fill the chip (of the `pair` products together), with at
// least 8 K steps a split.  The same for every alignment, since it sizes the workspace.
// A training step's us, bf16: with 4, 8 and 16 steps a split 160, 156 and 170 (8000 rows of 512 x
// 512), 65, 84 and 83 (1000 of 200 x 520), 125, 112 and 114 (20000 of 64 x 256); with one, two and
// four tiles a CU (of 128 and 64) 361, 273 and 254 (20000 of 200 x 520), 152, 122 and 119 (3000 of 264
// x 1040), fp32 180, 188 and 194 (20000 of 64 x 256).
template <typename E>
int grad_splits(int64_t rows, int64_t cols, int64_t K, int pair, int tile) {
  const int64_t tiles = tiles_of(rows, cols, tile, tile) * (1 + pair);
  return (int)std::max<int64_t>(1, std::min((tile == 256 ? 1 : 2) * kCUs / tiles, K / (8 * kGemmBK<E>)));
}
// the tile of a weight gradient: 256 where it wastes little of its edges, 128 where those are
// many (fp32, 520 x 200 over 2091 rows: 42 us in 128s, 25 splits of 20 tiles, 20 us in 64s).
// Without the 256s a bf16 training step of 20705 rows of 512 x 1408 takes 730 us, not 542 (500 rows 77,
// not 95); with up to twice the work in them, not 3/2, 20000 rows of 200 x 520 223, not 273, and 2091
// 94, not 83.  128s from half as many and twice as many tiles on: within 2% but for fp32, 500 rows
// of 512 x 1408 (164 us, 190 and 143) and 8000 of 512 x 512 (432, 415 and 432).
template <typename E>
int grad_tile(int64_t rows, int64_t cols, int pair) {
  if (sizeof(E) == 2 && rows >= 192 && cols >= 192 && tiles_of(rows, cols, 256, 256) * 256 * 256 <= rows * cols * 3 / 2)
    return 256;
  return tiles_of(rows, cols, 128, 128) * (1 + pair) >= kCUs / 4 ? 128 : 64;
}
template <typename E>
size_t grad_part_bytes(int64_t rows, int64_t cols, int64_t K, int pair) {
  // the wide kernel's tile and the one that stands in for it where the operands are not aligned
  int most = 1;
  for (int tile : {grad_tile<E>(rows, cols, pair), 128})
    most = std::max(most, grad_splits<E>(rows, cols, K, pair, tile));
  return most > 1 ? align_up((size_t)most * (1 + pair) * rows * cols * sizeof(float)) : 0;
}

template <typename E>
size_t ff_ws_bytes(const tmpc_gated_ff* a, bool backward) {
  const size_t act = align_up((size_t)a->M * ff_pitch<E>(a) * sizeof(E));
  if (!backward) return act + store_part_bytes<E>(a->M, a->Dout, a->F);
  return 3 * act + std::max(store_part_bytes<E>(a->M, a->D, a->F), std::max(grad_part_bytes<E>(a->F, a->D, a->M, 1), grad_part_bytes<E>(a->Dout, a->F, a->M, 0)));
}

// dW (rows, cols) = P^T X over the batch's M rows, and with out1 a second one, P1^T X, beside it
template <typename E>
void launch_weight_grad(hipStream_t st, int64_t M, int rows, int cols, const E* P, const E* P1, int64_t ldp, bool own_p,
                        const E* X, int64_t ldx, bool own_x, E* out, E* out1, float* part) {
  GemmArgs<E> p{};
  p.M = rows, p.N = cols, p.nseg = 1, p.K = M, p.pair = out1 != nullptr;
  p.A[0] = P, p.A[1] = P1, p.lda = ldp, p.B[0] = X, p.ldb = ldx;
  p.o0 = out, p.o1 = out1, p.ldo = cols;
  int tile = grad_tile<E>(rows, cols, p.pair);
  if (tile == 256 && !wide_ok(p, true, true, own_p, own_x)) tile = 128;
  launch_store<E, true, true>(st, p, {tile == 256 ? FORM_WIDE : tile == 128 ? FORM_128 : FORM_64,
                                      grad_splits<E>(rows, cols, M, p.pair, tile)}, part);
}

template <typename E>
int ff_forward_impl(hipStream_t st, const tmpc_gated_ff* a, void* y, float* gate, float* up, void* ws, size_t wsb) {
  if (!ff_shape_ok(a)) return TMPC_EBADSHAPE;
  if (a->M == 0) return TMPC_OK;
  if (!a->x || !a->w_gate || !a->w_up || !a->w_down || !y || !gate != !up || a->ldx < 0 ||
      (a->activation != ACT_SILU && a->activation != ACT_GELU))
    return TMPC_EBADARG;
  if (wsb < ff_ws_bytes<E>(a, false)) return TMPC_EWORKSPACE;
  if (!ws) return TMPC_EBADARG;
  const int64_t ldh = ff_pitch<E>(a);
  E* h = (E*)ws;
  GemmArgs<E> p{};
  p.M = a->M, p.N = a->F, p.nseg = 1, p.K = a->D;
  p.A[0] = (const E*)a->x, p.lda = a->ldx;
  p.B[0] = (const E*)a->w_gate, p.B[1] = (const E*)a->w_up, p.ldb = a->D;
  p.o0 = h, p.ldo = ldh, p.g = gate, p.u = up, p.ldg = a->F;
  const GemmPlan plan = gemm_plan<E, false, false, EPI_GATE>(p, false, false);
  if (a->activation == ACT_SILU) {
    if (gate) launch_gemm<E, false, false, EPI_GATE_SAVE, ACT_SILU>(st, p, plan);
    else launch_gemm<E, false, false, EPI_GATE, ACT_SILU>(st, p, plan);
  } else {
    if (gate) launch_gemm<E, false, false, EPI_GATE_SAVE, ACT_GELU>(st, p, plan);
    else launch_gemm<E, false, false, EPI_GATE, ACT_GELU>(st, p, plan);
  }
  GemmArgs<E> d{};
  d.M = a->M, d.N = a->Dout, d.nseg = 1, d.K = a->F;
  d.A[0] = h, d.lda = ldh, d.B[0] = (const E*)a->w_down, d.ldb = a->F, d.o0 = (E*)y, d.ldo = a->Dout;
  launch_store<E, false, false>(st, d, gemm_plan<E, false, false, EPI_STORE>(d, true, false),
                                 (float*)((char*)ws + align_up((size_t)a->M * ldh * sizeof(E))));
  return launch_status();
}

template <typename E>
int ff_backward_impl(hipStream_t st, const tmpc_gated_ff* a, const float* gate, const float* up, const void* dy,
                     int64_t lddy, void* dx, void* dwg, void* dwu, void* dwd, void* ws, size_t wsb) {
  if (!ff_shape_ok(a) || lddy > kMaxPitch) return TMPC_EBADSHAPE;
  if (!a->w_gate || !a->w_up || !a->w_down || !dwg || !dwu || !dwd || a->ldx < 0 || lddy < 0 ||
      (a->M > 0 && (!a->x || !gate || !up || !dy || !dx)) ||
      (a->activation != ACT_SILU && a->activation != ACT_GELU))
    return TMPC_EBADARG;
  const size_t need = ff_ws_bytes<E>(a, true);
  if (wsb < need) return TMPC_EWORKSPACE;
  if (need > 0 && !ws) return TMPC_EBADARG;
  const int64_t ldh = ff_pitch<E>(a);
  const size_t act = align_up((size_t)a->M * ldh * sizeof(E));
  E* dg = (E*)ws;
  E* du = (E*)((char*)ws + act);
  E* h = (E*)((char*)ws + 2 * act);
  float* part = (float*)((char*)ws + 3 * act);
  if (a->M > 0) {
    GemmArgs<E> p{};
    p.M = a->M, p.N = a->F, p.nseg = 1, p.K = a->Dout;
    p.A[0] = (const E*)dy, p.lda = lddy, p.B[0] = (const E*)a->w_down, p.ldb = a->F;
    p.o0 = dg, p.o1 = du, p.o2 = h, p.ldo = ldh, p.g = const_cast<float*>(gate), p.u = const_cast<float*>(up), p.ldg = a->F;
    const GemmPlan plan = gemm_plan<E, false, true, EPI_DGATE>(p, false, false);
    if (a->activation == ACT_SILU) launch_gemm<E, false, true, EPI_DGATE, ACT_SILU>(st, p, plan);
    else launch_gemm<E, false, true, EPI_DGATE, ACT_GELU>(st, p, plan);
    GemmArgs<E> d{};
    d.M = a->M, d.N = a->D, d.nseg = 2, d.K = a->F;
    d.A[0] = dg, d.A[1] = du, d.lda = ldh;
    d.B[0] = (const E*)a->w_gate, d.B[1] = (const E*)a->w_up, d.ldb = a->D;
    d.o0 = (E*)dx, d.ldo = a->D;
    launch_store<E, false, true>(st, d, gemm_plan<E, false, true, EPI_STORE>(d, true, false), part);
  }
  launch_weight_grad<E>(st, a->M, a->F, a->D, dg, du, ldh, true, (const E*)a->x, a->ldx, false, (E*)dwg, (E*)dwu, part);
  launch_weight_grad<E>(st, a->M, a->Dout, a->F, (const E*)dy, nullptr, lddy, false, h, ldh, true, (E*)dwd, nullptr, part);
  return launch_status();
}

}  // namespace
}  // namespace tmpc

using namespace tmpc;

extern "C" {

size_t tmpc_rms_norm_backward_workspace_bytes(int elem_bytes, int64_t rows, int32_t width) {
  if (!rms_shape_ok(rows, width) || (elem_bytes != 2 && elem_bytes != 4)) return 0;
  return align_up((size_t)rms_backward_blocks(rows, width, elem_bytes) * width * sizeof(float));
}
size_t tmpc_decay_attention_workspace_bytes(int elem_bytes, const tmpc_decay_attention* a, int backward) {
  if (!attn_shape_ok(a) || (elem_bytes != 2 && elem_bytes != 4)) return 0;
  return elem_bytes == 2 ? attn_ws_bytes<bf16>(a, backward != 0) : attn_ws_bytes<float>(a, backward != 0);
}
size_t tmpc_gated_ff_workspace_bytes(int elem_bytes, const tmpc_gated_ff* a, int backward) {
  if (!ff_shape_ok(a) || (elem_bytes != 2 && elem_bytes != 4)) return 0;
  return elem_bytes == 2 ? ff_ws_bytes<bf16>(a, backward != 0) : ff_ws_bytes<float>(a, backward != 0);
}

#define TMPC_LEARNING(SFX, E)                                                                                          \
  int tmpc_rms_norm_forward_##SFX(hipStream_t s, int64_t rows, int32_t width, const void* x, int64_t ldx,              \
                                  const void* r, int64_t ldr, const void* w, double eps, void* y, void* sum,           \
                                  float* rstd) {                                                                       \
    return rms_forward_impl<E>(s, rows, width, x, ldx, r, ldr, w, eps, y, sum, rstd);                                  \
  }                                                                                                                    \
  int tmpc_rms_norm_backward_##SFX(hipStream_t s, int64_t rows, int32_t width, const void* dy, int64_t lddy,           \
                                   const void* ds, int64_t ldds, const void* sum, int64_t lds, const void* w,          \
                                   const float* rstd, void* dx, void* dw, void* ws, size_t wsb) {                      \
    return rms_backward_impl<E>(s, rows, width, dy, lddy, ds, ldds, sum, lds, w, rstd, dx, dw, ws, wsb);               \
  }                                                                                                                    \
  int tmpc_decay_attention_forward_##SFX(hipStream_t s, const tmpc_decay_attention* a, void* o, float* state_out,      \
                                         void* ws, size_t wsb) {                                                       \
    return attn_forward_impl<E>(s, a, o, state_out, ws, wsb);                                                          \
  }                                                                                                                    \
  int tmpc_decay_attention_backward_##SFX(hipStream_t s, const tmpc_decay_attention* a, const void* d_o,               \
                                          const int64_t* d_o_stride, const float* d_state_out, void* dq, void* dk,     \
                                          void* dv, float* d_state_in, void* ws, size_t wsb) {                         \
    return attn_backward_impl<E>(s, a, d_o, d_o_stride, d_state_out, dq, dk, dv, d_state_in, ws, wsb);                 \
  }                                                                                                                    \
  int tmpc_decay_attention_step_##SFX(hipStream_t s, const tmpc_decay_attention* a, const uint8_t* active,             \
                                      float* state, void* o) {                                                         \
    return attn_step_impl<E>(s, a, active, state, o);                                                                  \
  }                                                                                                                    \
  int tmpc_gated_ff_forward_##SFX(hipStream_t s, const tmpc_gated_ff* a, void* y, float* gate, float* up, void* ws,      \
                                  size_t wsb) {                                                                        \
    return ff_forward_impl<E>(s, a, y, gate, up, ws, wsb);                                                             \
  }                                                                                                                    \
  int tmpc_gated_ff_backward_##SFX(hipStream_t s, const tmpc_gated_ff* a, const float* gate, const float* up,            \
                                   const void* dy, int64_t lddy, void* dx, void* dwg, void* dwu, void* dwd, void* ws,  \
                                   size_t wsb) {                                                                       \
    return ff_backward_impl<E>(s, a, gate, up, dy, lddy, dx, dwg, dwu, dwd, ws, wsb);                                  \
  }
TMPC_LEARNING(f32, float)
TMPC_LEARNING(bf16, bf16)

}  // extern "C"
