// Attention over a paged cache of fp16.
#include "mmnb_paged_attn.h"

namespace mmnb {

int paged_attention_f16(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t) {
  return paged_attention<_Float16>(ctx, a, t);
}

}  // namespace mmnb
