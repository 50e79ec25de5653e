// Prefill attention over the bf16 pool; the kernel is in prefill_attention.hpp.
#include "prefill_attention.hpp"

namespace nsg {

int32_t launch_prefill_attn(int head_dim, int waves, int num_work, const AttnParams& prm,
                            hipStream_t stream) {
  return launch_prefill<false, false>(head_dim, waves, num_work, prm, stream);
}
int32_t launch_prefill_part(int head_dim, int waves, int num_work, const AttnParams& prm,
                                 hipStream_t stream) {
  return launch_prefill<false, true>(head_dim, waves, num_work, prm, stream);
}

}  // namespace nsg
