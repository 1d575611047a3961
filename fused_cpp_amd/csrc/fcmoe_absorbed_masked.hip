// fcmoe_absorbed_masked.hip -- absorbed latent attention over a part of the
// context: a sliding window with the sequence's first tokens, and trees of
// drafted tokens behind it.
#include "fcmoe_absorbed_kernel.h"
#include "fcmoe_absorbed_tall.h"

namespace fcmoe {

namespace {

int check_mask(const fcmoe_absorbed_args* a, const fcmoe_key_mask* m) {
  const char* what = "absorbed_attention_masked: ";
  if (const int rc = check_absorbed(a)) return rc;
  if (!m) return fail(FCMOE_EINVAL, std::string(what) + "NULL mask");
  if (m->window < 0 || m->sinks < 0) return fail(FCMOE_EINVAL, std::string(what) + "window and sinks must not be negative");
  if (!m->tree_masks) return FCMOE_OK;
  if (!m->tree_depths || !a->query_starts) return fail(FCMOE_EINVAL, std::string(what) + "a tree needs depths and query_starts");
  if (m->mask_words < 1 || m->mask_words > 16 || m->mask_stride < 0 || (uintptr_t)m->tree_masks % 8 || (uintptr_t)m->tree_depths % 4)
    return fail(FCMOE_EINVAL, std::string(what) + "tree masks must have 1 to 16 aligned words a token");
  // masks and depths are addressed by 32-bit offsets
  if (m->mask_stride > (1 << 24) || a->tokens * (m->mask_stride + m->mask_words) * 8 > INT32_MAX)
    return fail(FCMOE_EINVAL, std::string(what) + "tree masks of 2 GiB and more");
  return FCMOE_OK;
}

}  // namespace

}  // namespace fcmoe

using namespace fcmoe;

extern "C" size_t fcmoe_absorbed_attention_masked_workspace_bytes(const fcmoe_absorbed_args* a, const fcmoe_key_mask* m) {
  if (check_mask(a, m) != FCMOE_OK || a->tokens == 0) return 0;
  const fcmoe_key_mask mask = bounded(*m);
  return absorbed_plan(a, &mask).bytes;
}

extern "C" int fcmoe_absorbed_attention_masked(const fcmoe_absorbed_args* a, const fcmoe_key_mask* m, hipStream_t stream) {
  if (const int rc = check_mask(a, m)) return rc;
  const fcmoe_key_mask mask = bounded(*m);
  return absorbed_run<true>(a, &mask, stream);
}
