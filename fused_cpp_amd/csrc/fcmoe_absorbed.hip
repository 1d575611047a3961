// fcmoe_absorbed.hip -- absorbed latent attention, plain causal form.
#include "fcmoe_absorbed_kernel.h"

using namespace fcmoe;

extern "C" size_t fcmoe_absorbed_attention_workspace_bytes(const fcmoe_absorbed_args* a) {
  if (check_absorbed(a) != FCMOE_OK || a->tokens == 0) return 0;
  return absorbed_plan(a, nullptr).bytes;
}

extern "C" int fcmoe_absorbed_attention(const fcmoe_absorbed_args* a, hipStream_t stream) {
  return absorbed_run<false>(a, nullptr, stream);
}
