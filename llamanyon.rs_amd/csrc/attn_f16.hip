// attn_f16.hip -- the paged attention (attn_core.hpp) over a fp16 cache.
#include "attn_core.hpp"

int swamp_attn_f16(const swamp_attn::Work &w, int parts, hipStream_t s) {
  return launch_dim<_Float16>(w, parts, s);
}
