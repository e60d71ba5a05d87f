// The gated delta rule in bf16.
#include "delta_api.hpp"

using namespace tmpc;

extern "C" {

TMPC_LEARNING_DELTA(bf16, bf16)

}  // extern "C"
