// The gated delta rule in fp32, and its workspace query.
#include "delta_api.hpp"

using namespace tmpc;

extern "C" {

size_t tmpc_delta_attention_workspace_bytes(int elem_bytes, const tmpc_delta_attention* a, int backward) {
  if (!a || !shape_ok(a) || (elem_bytes != 2 && elem_bytes != 4)) return 0;
  if (!backward) {
    const RunPlan runs = run_plan(a);
    return runs.state + runs.map;
  }
  if (!chunks_ok(a)) return 0;
  return elem_bytes == 2 ? backward_plan<bf16>(a).bytes : backward_plan<float>(a).bytes;
}

TMPC_LEARNING_DELTA(f32, float)

}  // extern "C"
