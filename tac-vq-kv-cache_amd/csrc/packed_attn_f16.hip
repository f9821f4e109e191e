// Attention of packed sequences without pages, fp16.  The kernel is in chunk_attn.h.
#include "chunk_attn.h"
#include "packed.h"

namespace jkv {

template <int D, int FORM>
static void launch_packed(const PagedAttnArgs& a, hipStream_t stream) {
  const dim3 grid((uint32_t)((int64_t)a.items * a.KVH));
  if (a.lse != nullptr) hipLaunchKernelGGL((paged_chunk_kernel<JKV_F16, D, false, 4, FORM, true, true>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((paged_chunk_kernel<JKV_F16, D, false, 4, FORM, true, false>), grid, dim3(256), 0, stream, a);
}

void packed_launch_f16(const PagedAttnArgs& a, int form, int64_t D, hipStream_t stream) {
  switch (form) {
    case kFormShaped: return D == 128 ? launch_packed<128, kFormShaped>(a, stream) : launch_packed<64, kFormShaped>(a, stream);
    case kFormShaped | kFormCap:
      return D == 128 ? launch_packed<128, kFormShaped | kFormCap>(a, stream) : launch_packed<64, kFormShaped | kFormCap>(a, stream);
    case kFormShaped | kFormBias:
      return D == 128 ? launch_packed<128, kFormShaped | kFormBias>(a, stream) : launch_packed<64, kFormShaped | kFormBias>(a, stream);
    default:
      return D == 128 ? launch_packed<128, kFormShaped | kFormCap | kFormBias>(a, stream)
                      : launch_packed<64, kFormShaped | kFormCap | kFormBias>(a, stream);
  }
}

}  // namespace jkv
