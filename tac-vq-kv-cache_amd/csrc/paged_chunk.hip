// Attention of chunks of new tokens over a paged K/V cache, and the weights that
// its entries receive: plain scores.  (The kernels, their reasons and what they
// measure are in chunk_attn.h.)
#include "chunk_attn.h"

namespace jkv {

int paged_launch_chunk(const PagedAttnArgs& a, int32_t dtype, int64_t D, hipStream_t stream) {
  if (dtype == JKV_F16) return D == 128 ? launch_chunk<JKV_F16, 128, kFormPlain>(a, stream) : launch_chunk<JKV_F16, 64, kFormPlain>(a, stream);
  return D == 128 ? launch_chunk<JKV_BF16, 128, kFormPlain>(a, stream) : launch_chunk<JKV_BF16, 64, kFormPlain>(a, stream);
}

}  // namespace jkv
