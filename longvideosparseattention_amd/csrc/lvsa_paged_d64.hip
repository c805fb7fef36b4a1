// D = 64 instantiations of the attention over the paged cache (lvsa_paged_attn.h).
#include "lvsa_paged_attn.h"

namespace lvsa {

int paged_attn_d64(const PagedAttnParams& p, int bits, int rows, bool bf16, hipStream_t stream) {
  return paged_launch<64>(p, bits, rows, bf16, stream);
}

}  // namespace lvsa
