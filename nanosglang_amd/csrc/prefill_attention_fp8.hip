// Prefill attention over the 8-bit pool (prefill_attention.hpp).  A file of its
// own because a row of that pool may stand for NaN: it is compiled with NaNs
// honoured, the bf16 one is not.
#include "prefill_attention.hpp"

namespace nsg {

int32_t launch_prefill_attn_fp8(int head_dim, int waves, int num_work, const AttnParams& prm,
                                hipStream_t stream) {
  return launch_prefill<true, false>(head_dim, waves, num_work, prm, stream);
}
int32_t launch_prefill_part_fp8(int head_dim, int waves, int num_work, const AttnParams& prm,
                                 hipStream_t stream) {
  return launch_prefill<true, true>(head_dim, waves, num_work, prm, stream);
}

}  // namespace nsg
