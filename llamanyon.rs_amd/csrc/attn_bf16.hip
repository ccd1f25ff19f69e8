// attn_bf16.hip -- the paged attention (attn_core.hpp) over a bf16 cache.
#include "attn_core.hpp"

int swamp_attn_bf16(const swamp_attn::Work &w, int parts, hipStream_t s) {
  return launch_dim<__bf16>(w, parts, s);
}
