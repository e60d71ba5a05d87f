// The gated delta rule's C entry points (include/tmpc.h) for an element type: argument checks,
// workspace, launches.  Each type is a translation unit of its own (learning_delta_*.hip): they are
// the library's longest to compile.
#pragma once
#include <algorithm>

#include "delta_attention.hpp"
#include "learn_host.hpp"

namespace tmpc {
namespace {

constexpr int64_t kMaxStep = (1 << 23) - 1;  // elements between steps: 64 fp32 steps within 31 bits
constexpr int kMaxHeads = 32768, kMaxSteps = 1 << 30;
constexpr int64_t kMaxBatchHeads = 1 << 22;  // workgroups of a walk, of up to 704 threads: a launch has less than 2^32

bool shape_ok(const tmpc_delta_attention* a) {
  auto heads = [&](int n) { return n >= 1 && a->H % n == 0; };
  return a && a->B >= 0 && a->T >= 0 && a->T <= kMaxSteps && a->H >= 1 && a->H <= kMaxHeads && heads(a->Hq) &&
         heads(a->Hk) && heads(a->Hv) && a->dk >= 1 && a->dk <= 128 && a->dv >= 1 && a->dv <= 128 &&
         (int64_t)a->B * a->H <= kMaxBatchHeads;
}
// the backward pass' chunks, counted in 31 bits
bool chunks_ok(const tmpc_delta_attention* a) {
  return (int64_t)a->B * a->H * ceil_div(a->T, 32) < int64_t(1) << 31;
}
bool steps_ok(const tmpc_delta_attention* a) {
  for (const int64_t* s : {a->q_stride, a->k_stride, a->v_stride, a->log_decay_stride, a->beta_stride})
    if (s[1] < 0 || s[1] > kMaxStep) return false;
  return true;
}

template <typename E>
DeltaArgs<E> delta_args(const tmpc_delta_attention* x) {
  DeltaArgs<E> p{};
  p.B = x->B, p.T = x->T, p.H = x->H, p.dk = x->dk, p.dv = x->dv;
  p.gq = x->H / x->Hq, p.gk = x->H / x->Hk, p.gv = x->H / x->Hv;
  p.q = (const E*)x->q, p.k = (const E*)x->k, p.v = (const E*)x->v, p.beta = (const E*)x->beta, p.g = x->log_decay;
  std::copy_n(x->q_stride, 3, p.qs), std::copy_n(x->k_stride, 3, p.ks), std::copy_n(x->v_stride, 3, p.vs);
  std::copy_n(x->beta_stride, 3, p.bs), std::copy_n(x->log_decay_stride, 3, p.gs);
  p.lengths = x->lengths, p.scale = (float)x->scale, p.s_in = x->state_in;
  return p;
}

// f(widths of the keys' and the values' tiles)
template <typename F>
void with_widths(int dk, int dv, F f) {
  using std::integral_constant;
  auto with_v = [&](auto k) {
    if (dv <= 32) f(k, integral_constant<int, 32>());
    else if (dv <= 64) f(k, integral_constant<int, 64>());
    else f(k, integral_constant<int, 128>());
  };
  if (dk <= 32) with_v(integral_constant<int, 32>());
  else if (dk <= 64) with_v(integral_constant<int, 64>());
  else with_v(integral_constant<int, 128>());
}

// Rows of whole 16-byte pieces at 4-byte addresses: moved a piece at a time.
template <typename E>
bool rows_ok(const E* x, const int64_t* s, int width) {
  if (width % Elem<E>::PIECE != 0 || ((uintptr_t)x & 3) != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (s[i] * (int64_t)sizeof(E) % 4 != 0) return false;
  return true;
}
template <typename E>
bool vec_ok(const DeltaArgs<E>& p) {
  return rows_ok(p.q, p.qs, p.dk) && rows_ok(p.k, p.ks, p.dk) && rows_ok(p.v, p.vs, p.dv) && ((uintptr_t)p.o & 15) == 0;
}

// How a history is cut into runs, and their arrays in the workspace.  A run costs its columns of the unit matrix
// beside its own, twice the work and more, so a history is cut only where its heads leave CUs empty, into as many
// runs as workgroups fill the CUs once: one a CU where the values are wider than 64 (eleven waves), else two.  (Two
// histories of 200000 steps, 8 heads of 128: 3.9 ms with two a CU, 3.4 with one; 4 of 4096, 8 heads of 64,
// with gradients: 327 us with one a CU, 315 with two.)  The runs' states are joined one after another, so
// the best number goes by the root of the length, that of 40 times its stretches (10, 40, 160: 113, 97, 106 us for
// 20000 steps of 4 heads of 64, 211, 199, 271 for 2 of 128, 66, 47, 47 for 4096 steps of 4 of 64).
// Fewer than four runs are not worth their maps and not asked for: two cost 447 us where whole histories take
// 261 (16 of 4096, 16 heads of 64) and 551 where they take 408 (8 of 4096, 16 of 128); three 421 and 402 (5 of
// 4096), but 1.43 ms and 1.58 at 16384 steps.  Runs are whole stretches, so four of five, six or
// nine stretches come out as three: forwards 93 and 92 us where whole histories take 76 and 90 (16 of 1280 and 1536, 8
// heads of 64, bf16), with gradients 390 and 414 against 373 and 441; 128 wide, 8 of 1280 and 1500, 168 and 168
// against 139 and 163, with gradients 667 and 685 against 712 and 840.
struct RunPlan {
  int segs, len;
  size_t state, map;  // bytes of a head's states and maps of all runs, of all heads
};
inline int tile_width(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }
inline RunPlan run_plan(const tmpc_delta_attention* x) {
  const int64_t bh = std::max<int64_t>(1, (int64_t)x->B * x->H), stretches = std::max<int64_t>(1, ceil_div(x->T, kDeltaSeg));
  const int64_t fill = (x->dv > 64 ? 1 : 2) * kCUs / bh;
  int64_t want = std::min(fill, stretches);
  while (want > 8 && want * want > 40 * stretches) --want;
  if (want < 4) want = 1;
  const int64_t len = ceil_div(stretches, want);
  RunPlan p{(int)ceil_div(stretches, len), (int)(len * kDeltaSeg), 0, 0};
  if (p.segs > 1) {
    const size_t DK = tile_width(x->dk), DV = tile_width(x->dv), n = (size_t)x->B * x->H * p.segs * sizeof(float);
    p.state = align_up(n * DK * DV), p.map = align_up(n * DK * DK);
  }
  return p;
}
template <typename K, typename... A>
void launch(hipStream_t st, K k, dim3 grid, int threads, size_t lds, A... args) {
  lds_optin(k, lds);
  hipLaunchKernelGGL(k, grid, dim3(threads), lds, st, args...);
}
template <typename E, int DK, int DV, int MODE>
void launch_walk(hipStream_t st, const DeltaBwdArgs<E>& a, int columns, int run_width) {
  const dim3 grid((unsigned)((int64_t)a.f.B * a.f.H * a.f.segs), (unsigned)ceil_div(columns, DV));
  launch(st, delta_walk_kernel<E, DK, DV, MODE>, grid, DeltaShape<E, DK, DV>::THREADS, DeltaWalkLds<E, DK, DV, MODE>::all, a, run_width);
}
template <typename E, int DK, int DV, bool RUN>
void launch_reverse(hipStream_t st, const DeltaBwdArgs<E>& a, int columns, int run_width) {
  const dim3 grid((unsigned)((int64_t)a.f.B * a.f.H * a.f.segs), (unsigned)ceil_div(columns, DV));
  launch(st, delta_reverse_kernel<E, DK, DV, RUN>, grid, DeltaShape<E, DK, DV>::THREADS, DeltaReverseLds<E, DK, DV, RUN>::all, a, run_width);
}
// A launch of n workgroups: the kernel's `flat_block()` tells them.
inline dim3 flat_grid(int64_t n) { return dim3((unsigned)std::min(n, kFlatGrid), (unsigned)ceil_div(n, kFlatGrid)); }
// the runs' starts, from the pass before the outputs'
template <typename E, int DK>
void launch_runs(hipStream_t st, const DeltaBwdArgs<E>& a, int DV) {
  const DeltaArgs<E>& p = a.f;
  // 128 wide keys: one set of helpers a CU in place of two (16 heads of 128 / 128, 50001 steps: 1.00 ms against 1.02)
  launch_walk<E, DK, DK == 128 ? 128 : 64, WALK_RUN>(st, a, DV + DK, DV);
  launch(st, delta_scan_kernel<DK, false>, dim3((unsigned)((int64_t)p.B * p.H * (DV / 16))), 256, 0, (const float*)p.seg_map, p.seg_state,
         p.segs, DV, p.s_in, p.dk, p.dv);
}

bool data_ok(const tmpc_delta_attention* x) {
  return x->T == 0 || (x->q && x->k && x->v && x->log_decay && x->beta);
}

template <typename E>
int forward_impl(hipStream_t st, const tmpc_delta_attention* x, void* o, float* state_out, void* ws, size_t wsb) {
  if (!shape_ok(x)) return TMPC_EBADSHAPE;
  if (x->B == 0) return TMPC_OK;
  if (!steps_ok(x)) return TMPC_EBADSHAPE;
  if (!data_ok(x) || (x->T > 0 && !o)) return TMPC_EBADARG;
  DeltaBwdArgs<E> a{};
  a.f = delta_args<E>(x);
  DeltaArgs<E>& p = a.f;
  p.s_out = state_out, p.o = (E*)o;
  p.vec = vec_ok(p);
  const RunPlan runs = run_plan(x);
  if (wsb < runs.state + runs.map) return TMPC_EWORKSPACE;
  if (runs.segs > 1 && !ws) return TMPC_EBADARG;
  p.segs = runs.segs, p.seg_len = runs.len, p.seg_state = (float*)ws, p.seg_map = (float*)((char*)ws + runs.state);
  with_widths(x->dk, x->dv, [&](auto dk, auto dv) {
    if (p.segs > 1) launch_runs<E, dk()>(st, a, dv());
    launch_walk<E, dk(), dv(), WALK_OUT>(st, a, dv(), 0);
  });
  return launch_status();
}

// The backward pass' arrays in the workspace, one after another.
struct BackwardPlan {
  int chunks, stretches, DK, DV;
  size_t x, x_low, y_low, s, s_low, r, r_low, w, z, s_seg, dot, dot0, y, y_part, q_part, k_part, run_state, run_map, run_grad, bytes;
  RunPlan runs;
};
template <typename E>
BackwardPlan backward_plan(const tmpc_delta_attention* x) {
  constexpr int C = AttnTile<E>::C;
  BackwardPlan p{};
  p.chunks = (int)ceil_div(x->T, C), p.stretches = (int)ceil_div(x->T, kDeltaSeg);
  p.DK = tile_width(x->dk), p.DV = tile_width(x->dv);
  const size_t bh = (size_t)x->B * x->H, state = (size_t)p.DK * p.DV, rows = bh * p.chunks * C;
  const size_t tok = (size_t)x->B * x->T * x->H * sizeof(float);
  auto take = [&](size_t bytes) {
    const size_t at = p.bytes;
    p.bytes += align_up(bytes);
    return at;
  };
  p.x = take(rows * p.DV * sizeof(E));
  p.s = take(bh * p.chunks * state * sizeof(E)), p.r = take(bh * p.chunks * state * sizeof(E));
  if (sizeof(E) == 2) {
    p.x_low = take(rows * p.DV * sizeof(E)), p.y_low = take(rows * p.DV * sizeof(E));
    p.s_low = take(bh * p.chunks * state), p.r_low = take(bh * p.chunks * state);
  }
  p.w = take(rows * sizeof(float)), p.z = take(rows * sizeof(float));
  p.s_seg = take(bh * p.stretches * state * sizeof(float)), p.dot = take(bh * p.stretches * sizeof(float));
  if (x->T > 0) p.dot0 = take(bh * 8 * sizeof(float));
  if (x->Hv != x->H) p.y = take(rows * p.DV * sizeof(E)), p.y_part = take(tok * x->dv);
  if (x->Hq != x->H) p.q_part = take(tok * x->dk);
  if (x->Hk != x->H) p.k_part = take(tok * x->dk);
  p.runs = run_plan(x);
  p.run_state = take(p.runs.state), p.run_map = take(p.runs.map), p.run_grad = take(p.runs.state);
  return p;
}

template <typename E>
int backward_impl(hipStream_t st, const tmpc_delta_attention* x, const void* d_o, const int64_t* dos,
                  const float* d_out, void* dq, void* dk, void* dv, float* dg, void* dbeta, float* d_in, void* ws,
                  size_t wsb) {
  if (!shape_ok(x) || !chunks_ok(x)) return TMPC_EBADSHAPE;
  if (x->B == 0) return TMPC_OK;
  if (!steps_ok(x) || (dos && (dos[1] < 0 || dos[1] > kMaxStep))) return TMPC_EBADSHAPE;
  if (!dos || !data_ok(x) || (x->T > 0 && (!d_o || !dq || !dk || !dv || !dg || !dbeta))) return TMPC_EBADARG;
  const BackwardPlan w = backward_plan<E>(x);
  if (wsb < w.bytes) return TMPC_EWORKSPACE;
  if (w.bytes > 0 && !ws) return TMPC_EBADARG;
  char* base = (char*)ws;
  DeltaBwdArgs<E> a{};
  a.f = delta_args<E>(x);
  a.d_o = (const E*)d_o, a.d_out = d_out;
  std::copy_n(dos, 3, a.dos);
  a.chunks = w.chunks, a.stretches = w.stretches;
  a.x = (E*)(base + w.x), a.x_low = (E*)(base + w.x_low), a.s = (E*)(base + w.s), a.r = (E*)(base + w.r), a.w = (float*)(base + w.w);
  a.y_low = (E*)(base + w.y_low), a.s_low = (uint8_t*)(base + w.s_low), a.r_low = (uint8_t*)(base + w.r_low);
  a.z = (float*)(base + w.z), a.s_seg = (float*)(base + w.s_seg), a.dot = (float*)(base + w.dot), a.dot0 = (float*)(base + w.dot0);
  if (x->Hv != x->H) {
    a.y = (E*)(base + w.y), a.y_part = (float*)(base + w.y_part), a.y_width = w.DV;
    a.ys[0] = (int64_t)w.chunks * AttnTile<E>::C * w.DV, a.ys[1] = w.DV;
  } else {
    a.y = (E*)dv, a.y_width = x->dv, a.ys[0] = (int64_t)x->T * x->H * x->dv, a.ys[1] = (int64_t)x->H * x->dv;
  }
  a.q_part = x->Hq != x->H, a.k_part = x->Hk != x->H;
  a.dq = a.q_part ? base + w.q_part : dq, a.dk = a.k_part ? base + w.k_part : dk;
  a.dbeta = (E*)dbeta, a.dg = dg, a.d_in = d_in;
  a.f.segs = w.runs.segs, a.f.seg_len = w.runs.len, a.f.seg_state = (float*)(base + w.run_state);
  a.f.seg_map = (float*)(base + w.run_map), a.r_seg = (float*)(base + w.run_grad);
  const int64_t bh = (int64_t)x->B * x->H;
  a.f.vec = rows_ok(a.f.q, a.f.qs, x->dk) && rows_ok(a.f.k, a.f.ks, x->dk) && rows_ok(a.f.v, a.f.vs, x->dv) &&
            rows_ok(a.d_o, a.dos, x->dv) && ((uintptr_t)dv & 3) == 0;
  with_widths(x->dk, x->dv, [&](auto dkw, auto dvw) {
    if (a.f.segs > 1) {
      launch_runs<E, dkw()>(st, a, dvw());
      launch_reverse<E, dkw(), dvw(), true>(st, a, dvw(), dvw());
      launch(st, delta_scan_kernel<dkw(), true>, dim3((unsigned)(bh * (dvw() / 16))), 256, 0, (const float*)a.f.seg_map, a.r_seg,
             a.f.segs, (int)dvw(), d_out, x->dk, x->dv);
    }
    if (x->T > 0) launch_walk<E, dkw(), dvw(), WALK_STATES>(st, a, dvw(), 0);
    launch_reverse<E, dkw(), dvw(), false>(st, a, dvw(), 0);
    if (x->T > 0)
      launch(st, delta_dqk_kernel<E, dkw(), dvw()>, flat_grid(bh * w.chunks), DeltaDqkShape<E, dkw(), dvw()>::THREADS,
             DeltaDqkShape<E, dkw(), dvw()>::LDS, a);
  });
  if (x->T > 0) {
    hipLaunchKernelGGL((delta_dgate_kernel<E>), flat_grid(bh * w.stretches), dim3(64), 0, st, a, w.chunks * AttnTile<E>::C, w.DV / 16);
    auto sum = [&](const void* in, int heads, int d, void* out) {
      const int64_t rows = (int64_t)x->B * x->T * heads;
      const int q = (d + 3) / 4;
      hipLaunchKernelGGL((attn_head_sum_kernel<E>), dim3((unsigned)std::min<int64_t>(ceil_div(rows, 256 / q), 16 * kCUs)),
                         dim3(256), 0, st, (const float*)in, rows, x->H / heads, d, q, (E*)out);
    };
    if (x->Hq != x->H) sum(a.dq, x->Hq, x->dk, dq);
    if (x->Hk != x->H) sum(a.dk, x->Hk, x->dk, dk);
    if (x->Hv != x->H) sum(a.y_part, x->Hv, x->dv, dv);
  }
  return launch_status();
}

template <typename E>
int step_impl(hipStream_t st, const tmpc_delta_attention* x, const uint8_t* active, float* state, void* o) {
  if (!shape_ok(x) || x->T != 1) return TMPC_EBADSHAPE;
  if (x->B == 0) return TMPC_OK;
  if (!data_ok(x) || !state || !o) return TMPC_EBADARG;
  DeltaStepArgs<E> p{x->B, x->H, x->H / x->Hq, x->H / x->Hk, x->H / x->Hv, x->dk, x->dv};
  p.q = (const E*)x->q, p.k = (const E*)x->k, p.v = (const E*)x->v, p.beta = (const E*)x->beta, p.g = x->log_decay;
  auto two = [](const int64_t* s, int64_t* d) { d[0] = s[0], d[1] = s[2]; };
  two(x->q_stride, p.qs), two(x->k_stride, p.ks), two(x->v_stride, p.vs), two(x->beta_stride, p.bs);
  two(x->log_decay_stride, p.gs);
  p.active = active, p.scale = (float)x->scale, p.state = state, p.o = (E*)o;
  const int rg = 256 / ((x->dv + 3) / 4), rows = (x->dk + rg - 1) / rg;
  auto go = [&](auto nr) {
    hipLaunchKernelGGL((delta_step_kernel<E, nr()>), dim3((unsigned)(x->B * x->H)), dim3(256), 0, st, p);
  };
  using std::integral_constant;
  if (rows <= 2) go(integral_constant<int, 2>());
  else if (rows <= 4) go(integral_constant<int, 4>());
  else if (rows <= 8) go(integral_constant<int, 8>());
  else go(integral_constant<int, 16>());
  return launch_status();
}

}  // namespace
}  // namespace tmpc

#define TMPC_LEARNING_DELTA(SFX, E)                                                                                    \
  int tmpc_delta_attention_forward_##SFX(hipStream_t s, const tmpc_delta_attention* a, void* o, float* state_out,      \
                                         void* ws, size_t wsb) {                                                       \
    return forward_impl<E>(s, a, o, state_out, ws, wsb);                                                               \
  }                                                                                                                    \
  int tmpc_delta_attention_backward_##SFX(hipStream_t s, const tmpc_delta_attention* a, const void* d_o,               \
                                          const int64_t* d_o_stride, const float* d_state_out, void* dq, void* dk,     \
                                          void* dv, float* dlog_decay, void* dbeta, float* d_state_in, void* ws,       \
                                          size_t wsb) {                                                                \
    return backward_impl<E>(s, a, d_o, d_o_stride, d_state_out, dq, dk, dv, dlog_decay, dbeta, d_state_in, ws, wsb);   \
  }                                                                                                                    \
  int tmpc_delta_attention_step_##SFX(hipStream_t s, const tmpc_delta_attention* a, const uint8_t* active,             \
                                      float* state, void* o) {                                                         \
    return step_impl<E>(s, a, active, state, o);                                                                       \
  }
