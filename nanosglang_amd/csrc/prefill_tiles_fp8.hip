// Attention tiles over the 8-bit pool, whole and as partials (prefill_tiles.hpp).
#include "prefill_tiles.hpp"

namespace nsg {

int32_t launch_prefill_attn_fp8(int head_dim, int waves, int num_work, const AttnParams& prm,
                                hipStream_t stream) {
  return launch_tiles<true, false>(head_dim, waves, num_work, prm, stream);
}

int32_t launch_tiles_part_fp8(int head_dim, int waves, int num_work, const AttnParams& prm,
                              hipStream_t stream) {
  return launch_tiles<true, true>(head_dim, waves, num_work, prm, stream);
}

}  // namespace nsg
