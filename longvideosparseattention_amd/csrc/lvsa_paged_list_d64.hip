// D = 64 instantiations of the attention over lists of blocks and of the accumulated
// weights (lvsa_paged_list.h, lvsa_paged_weights.h).
#include "lvsa_paged_list.h"
#include "lvsa_paged_weights.h"

namespace lvsa {

int paged_block_attn_d64(const PagedAttnParams& p, const BlockAttnParams& l, int bits, int rows, bool bf16, hipStream_t stream) {
  return paged_block_launch<64>(p, l, bits, rows, bf16, stream);
}
int paged_weights_d64(const PagedAttnParams& p, const WeightsParams& w, int bits, bool bf16, hipStream_t stream) {
  return paged_weights_launch<64>(p, w, bits, bf16, stream);
}

}  // namespace lvsa
