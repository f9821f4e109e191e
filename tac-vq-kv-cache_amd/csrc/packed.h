// What the kernels over packed sequences without pages share.
#pragma once

#include "paged.h"

namespace jkv {

// What the kernels of the attention's gradients share.  Strides in bytes; dq, dk
// and dv are contiguous.
struct PackedGradArgs {
  const uint8_t *q, *k, *v, *o, *d, *rest;  // rest: what o's rounding took off, contiguous, or null
  int64_t qst, qsh, kst, ksh, vst, vsh, ost, osh, dst, dsh;
  uint8_t *dq, *dk, *dv;  // null: not wanted
  const int32_t *starts, *prefixes;
  const float* lse;
  int32_t N, B, QH, KVH, per, window, sinks;
  float scale, scale2, cap_mul, cap2;
  const float* slopes;
  float *bases, *minus_delta;  // [QH][N]: 10 and the cap (base 2) less the base-2 log-sum-exp, -rowsum(do o)
  // dk and dv: 32 keys a workgroup instead of 128; or the group's heads in splits
  // of heads_each, whose sums a last launch adds up
  int32_t alone, splits, heads_each;
  float* part;  // [splits][dk, dv][N][KVH][D]
};
static const int kGradBlocks = 512;  // workgroups of the rows' pass

// How dk and dv are divided.
struct PackedGradPlan {
  int32_t alone, splits, heads_each;
  int64_t stats_bytes, part_at, bytes;
};
PackedGradPlan packed_grad_plan(int64_t N, int64_t B, int64_t QH, int64_t KVH, int64_t D, int64_t window);

// launches of the gradients: the rows' sums, then dk and dv, then dq
int packed_grad_launch_f16(const PackedGradArgs& a, int form, int64_t D, hipStream_t stream);
int packed_grad_launch_bf16(const PackedGradArgs& a, int form, int64_t D, hipStream_t stream);

// launches of the attention; all but the type is in the arguments
void packed_launch_f16(const PagedAttnArgs& a, int form, int64_t D, hipStream_t stream);
void packed_launch_bf16(const PagedAttnArgs& a, int form, int64_t D, hipStream_t stream);

}  // namespace jkv
