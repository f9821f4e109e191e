// Gradients of the attention of packed sequences, bf16.  The kernels are in packed_grad.h.
#include "packed_grad.h"

namespace jkv {

int packed_grad_launch_bf16(const PackedGradArgs& a, int form, int64_t D, hipStream_t stream) {
  return launch_grad_form<JKV_BF16>(a, form, D, stream);
}

}  // namespace jkv
