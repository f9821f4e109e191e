// Attention over a paged K/V cache with shaped scores (caps, distance biases,
// prefixes), fp16.  The kernels are in few_attn.h and chunk_attn.h.
#include "chunk_attn.h"
#include "few_attn.h"

namespace jkv {

template <int FORM>
static int launch_form(const PagedAttnArgs& a, bool few, int64_t D, hipStream_t stream) {
  if (few) return D == 128 ? launch_few<JKV_F16, 128, FORM>(a, stream) : launch_few<JKV_F16, 64, FORM>(a, stream);
  return D == 128 ? launch_chunk<JKV_F16, 128, FORM>(a, stream) : launch_chunk<JKV_F16, 64, FORM>(a, stream);
}

int paged_launch_form_f16(const PagedAttnArgs& a, int form, bool few, int64_t D, hipStream_t stream) {
  switch (form) {
    case kFormShaped: return launch_form<kFormShaped>(a, few, D, stream);
    case kFormShaped | kFormCap: return launch_form<kFormShaped | kFormCap>(a, few, D, stream);
    case kFormShaped | kFormBias: return launch_form<kFormShaped | kFormBias>(a, few, D, stream);
    default: return launch_form<kFormShaped | kFormCap | kFormBias>(a, few, D, stream);
  }
}

}  // namespace jkv
