// fcmoe_expanded.hip -- expanded latent attention, plain form.
#include "fcmoe_expanded_kernel.h"

using namespace fcmoe;

extern "C" size_t fcmoe_expanded_attention_workspace_bytes(const fcmoe_expanded_args* a) {
  return expanded_sizes_known(a) ? expanded_plan(a, nullptr).bytes : 0;
}

extern "C" int fcmoe_expanded_attention(const fcmoe_expanded_args* a, hipStream_t stream) {
  return expanded_run<false>(a, nullptr, stream);
}
