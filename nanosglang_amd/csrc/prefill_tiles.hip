// Attention tiles that leave partials over the bf16 pool (prefill_tiles.hpp).
#include "prefill_tiles.hpp"

namespace nsg {

int32_t launch_tiles_part(int head_dim, int waves, int num_work, const AttnParams& prm,
                          hipStream_t stream) {
  return launch_tiles<false, true>(head_dim, waves, num_work, prm, stream);
}

}  // namespace nsg
