// D = 256 instantiations of the attention over the paged cache (lvsa_paged_attn.h).
#include "lvsa_paged_attn.h"

namespace lvsa {

int paged_attn_d256(const PagedAttnParams& p, int bits, int rows, bool bf16, hipStream_t stream) {
  return paged_launch<256>(p, bits, rows, bf16, stream);
}

}  // namespace lvsa
