// Attention over a paged cache of binary32.
#include "mmnb_paged_attn.h"

namespace mmnb {

int paged_attention_f32(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t) {
  return paged_attention<float>(ctx, a, t);
}

}  // namespace mmnb
