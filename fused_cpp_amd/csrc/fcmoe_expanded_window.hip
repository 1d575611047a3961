// fcmoe_expanded_window.hip -- expanded latent attention over a sliding window
// and the sequence's first tokens.
#include "fcmoe_expanded_kernel.h"

using namespace fcmoe;

extern "C" size_t fcmoe_expanded_attention_masked_workspace_bytes(const fcmoe_expanded_args* a, const fcmoe_key_mask* m) {
  if (!expanded_sizes_known(a) || !m || m->window < 0 || m->sinks < 0) return 0;
  const fcmoe_key_mask mask = bounded(*m);
  return expanded_plan(a, &mask).bytes;
}

extern "C" int fcmoe_expanded_attention_masked(const fcmoe_expanded_args* a, const fcmoe_key_mask* m, hipStream_t stream) {
  if (!a || !m) return fail(FCMOE_EINVAL, "expanded_attention_masked: NULL args");
  if (m->window < 0 || m->sinks < 0) return fail(FCMOE_EINVAL, "expanded_attention_masked: window and sinks must not be negative");
  if (m->tree_masks) return fail(FCMOE_EINVAL, "expanded_attention_masked: trees are read in the absorbed form");
  if (!a->causal) return fail(FCMOE_EINVAL, "expanded_attention_masked: a window needs causal");
  const fcmoe_key_mask mask = bounded(*m);
  return expanded_run<true>(a, &mask, stream);
}
