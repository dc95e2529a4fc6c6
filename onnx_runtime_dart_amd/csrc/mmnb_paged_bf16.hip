// Attention over a paged cache of bf16.
#include "mmnb_paged_attn.h"

namespace mmnb {

int paged_attention_bf16(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t) {
  return paged_attention<__bf16>(ctx, a, t);
}

}  // namespace mmnb
