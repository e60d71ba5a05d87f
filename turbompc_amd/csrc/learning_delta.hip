// C ABI of the gated delta rule (include/tmpc.h): argument checks, workspace, launches.
#include <algorithm>

#include "delta_attention.hpp"
#include "learn_host.hpp"

namespace tmpc {
namespace {

constexpr int64_t kMaxStep = (1 << 23) - 1;  // elements between steps: 64 fp32 steps within 31 bits
constexpr int kMaxHeads = 32768, kMaxSteps = 1 << 30;

bool shape_ok(const tmpc_delta_attention* a) {
  auto heads = [&](int n) { return n >= 1 && a->H % n == 0; };
  return a && a->B >= 0 && a->T >= 0 && a->T <= kMaxSteps && a->H >= 1 && a->H <= kMaxHeads && heads(a->Hq) &&
         heads(a->Hk) && heads(a->Hv) && a->dk >= 1 && a->dk <= 128 && a->dv >= 1 && a->dv <= 128 &&
         (int64_t)a->B * a->H <= 1 << 23;
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

bool data_ok(const tmpc_delta_attention* x) {
  return x->T == 0 || (x->q && x->k && x->v && x->log_decay && x->beta);
}

template <typename E>
int forward_impl(hipStream_t st, const tmpc_delta_attention* x, void* o, float* state_out, void* ws, size_t wsb) {
  if (!shape_ok(x)) return TMPC_EBADSHAPE;
  if (x->B == 0) return TMPC_OK;
  if (!steps_ok(x)) return TMPC_EBADSHAPE;
  if (!data_ok(x) || (x->T > 0 && !o)) return TMPC_EBADARG;
  DeltaArgs<E> p = delta_args<E>(x);
  p.s_out = state_out, p.o = (E*)o;
  with_widths(x->dk, x->dv, [&](auto dk, auto dv) {
    auto go = [&](auto vec) {
      constexpr size_t lds = delta_forward_lds<E, dk(), dv()>();
      auto k = delta_forward_kernel<E, dk(), dv(), vec()>;
      lds_optin(k, lds);
      hipLaunchKernelGGL(k, dim3((unsigned)(x->B * x->H)), dim3(DeltaShape<E, dk(), dv()>::THREADS), lds, st, p);
    };
    if (vec_ok(p)) go(std::true_type());
    else go(std::false_type());
  });
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

using namespace tmpc;

extern "C" {

size_t tmpc_delta_attention_workspace_bytes(int elem_bytes, const tmpc_delta_attention* a, int backward) {
  if (!a || !shape_ok(a) || (elem_bytes != 2 && elem_bytes != 4)) return 0;
  (void)backward;
  return 0;
}

#define TMPC_LEARNING_DELTA(SFX, E)                                                                                    \
  int tmpc_delta_attention_forward_##SFX(hipStream_t s, const tmpc_delta_attention* a, void* o, float* state_out,      \
                                         void* ws, size_t wsb) {                                                       \
    return forward_impl<E>(s, a, o, state_out, ws, wsb);                                                               \
  }                                                                                                                    \
  int tmpc_delta_attention_step_##SFX(hipStream_t s, const tmpc_delta_attention* a, const uint8_t* active,             \
                                      float* state, void* o) {                                                         \
    return step_impl<E>(s, a, active, state, o);                                                                       \
  }
TMPC_LEARNING_DELTA(f32, float)
TMPC_LEARNING_DELTA(bf16, bf16)

}  // extern "C"
