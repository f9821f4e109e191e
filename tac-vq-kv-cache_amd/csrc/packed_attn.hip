// Attention inside sequences that lie packed one behind another, keys and values
// beside the queries: prompts without a cache, and training.
//
// Sequence b owns rows starts[b] to starts[b+1]; its row i sees its row j where
// (j <= i or j < prefix) and (j > i - window or j < sinks):
//   x_ij = cap tanh(scale q_i k_j / cap) - slope |i - j|,  p = softmax_j(x),  o_i = sum_j p_ij v_j
// Here: a call's checks and the division of its work.  The kernel is the paged
// chunks' one (chunk_attn.h) over rows in place of pages.
#include <math.h>

#include <algorithm>

#include "packed.h"

namespace jkv {

static int packed_checks(int32_t dtype, int64_t N, int64_t B, int64_t QH, int64_t KVH, int64_t D, int64_t window, int64_t sinks,
                         float scale) {
  JKV_CHECK_ARG(dtype == JKV_F16 || dtype == JKV_BF16, "packed attention takes fp16 or bf16, got dtype %d", dtype);
  JKV_CHECK_ARG(D == 64 || D == 128, "packed attention supports head_dim 64 and 128, got %lld", (long long)D);
  JKV_CHECK_ARG(QH > 0 && KVH > 0 && QH % KVH == 0 && QH < 65536, "query heads must be a multiple of kv heads");
  JKV_CHECK_ARG(N >= 0 && N < ((int64_t)1 << 30) && B >= 0 && B < ((int64_t)1 << 24), "too many rows or sequences");
  JKV_CHECK_ARG(N * QH < ((int64_t)1 << 31) - 256, "too many rows");
  JKV_CHECK_ARG(window >= 0 && sinks >= 0, "window and sinks must not be negative");
  JKV_CHECK_ARG(fabsf(scale) < 1e30f, "the softmax scale must be finite and below 1e30");
  return JKV_OK;
}

// token and head strides of 16-bit rows
static int packed_strides(const int64_t* strides, int count) {
  for (int i = 0; i < count; ++i)
    JKV_CHECK_ARG(strides[i] % 8 == 0 && strides[i] >= 0 && strides[i] < (i % 2 ? (int64_t)1 << 40 : (int64_t)1 << 22),
                  "token and head strides must be multiples of 8 elements, a token's below 2^22");
  return JKV_OK;
}

// dk and dv: 128 keys a workgroup that walks all heads of the group (two a CU), the
// same with the heads in splits whose sums are joined, or 32 keys a workgroup whose
// waves share out the walk (one a CU at 128 dims, two at 64, and four times the rows'
// traffic).  In steps of one head's 32 rows: the CUs' share of all walks, half the
// longest walk for the end where not all CUs have one, and the join.  us of the
// gradients of k and v with 1, 2 and 4 splits and with 32 keys, 32/8 heads of 128,
// bf16: one sequence of 8,192 2,609, 2,370, 2,300 and 2,633; of 2,048 440, 282, 222
// and 230; of 512 125, 87, 83 and 73; four of 2,048 742, 714, 723 and 808; eight of
// 1,000 416, 423, 452 and 485; one of 4,096 with 8/8 heads 316 and (32 keys) 291; 48
// texts of up to 511, 28/4 heads of 64, fp16, 275, 286, 300 and 248; 16/16 heads 191
// and (32 keys) 258.  The choice is within 1 % of the least in 25 of 26 such, and 5 %
// off it for two sequences of 8,192 with a window of 256 and heads of 64.
PackedGradPlan packed_grad_plan(int64_t N, int64_t B, int64_t QH, int64_t KVH, int64_t D, int64_t window) {
  PackedGradPlan p = {};
  const int64_t per = QH / KVH;
  const double mean = (double)N / (double)std::max<int64_t>(B, 1);  // rows of a sequence
  const double seen = window > 0 ? std::min((double)window, mean) : mean;
  const double walk = ceil(std::min(mean, seen + 128.0) / 32.0) * (double)per, all =
      ((double)N / 128.0 + 0.5 * (double)B) * (double)KVH * walk * (1.0 - 0.5 * seen / mean);
  const double step_us = D == 128 ? 2.4 : 1.5;
  double least = 1e300;
  for (int64_t each = per; each >= 1; each = each / 2) {
    const int64_t splits = ceil_div(per, each);
    const double join = splits > 1 ? 6.0 + 16.0 * (double)splits * (double)(N * KVH * D) / 4.5e6 : 0.0;
    const double t = all / 512.0 + 0.5 * walk / (double)splits + join / step_us;
    if (t < 0.95 * least) {
      least = t;
      p.heads_each = (int32_t)each;
      p.splits = (int32_t)splits;
    }
  }
  if ((D == 128 ? 2.0 : 1.2) * all / 512.0 + 0.125 * walk < least) {
    p.alone = 1;
    p.heads_each = (int32_t)per;
    p.splits = 1;
  }
  p.stats_bytes = ceil_div(N * QH * 4, 256) * 256;
  p.part_at = 2 * p.stats_bytes;
  p.bytes = p.part_at + (p.splits > 1 ? 2 * p.splits * N * KVH * D * 4 : 0);
  return p;
}

}  // namespace jkv

extern "C" {

int jkv_packed_attention(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_stride_t,
                         int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h, int32_t dtype,
                         const int32_t* starts, const int32_t* prefixes, int64_t N, int64_t B, int64_t QH, int64_t KVH,
                         int64_t D, int64_t window, int64_t sinks, float scale, float softcap, const float* slopes,
                         void* out, int64_t out_stride_t, int64_t out_stride_h, float* lse, void* rest,
                         jkv_stream_t stream_) {
  using namespace jkv;
  int rc = packed_checks(dtype, N, B, QH, KVH, D, window, sinks, scale);
  if (rc != JKV_OK) return rc;
  const int64_t strides[8] = {q_stride_t, q_stride_h, k_stride_t, k_stride_h, v_stride_t, v_stride_h, out_stride_t, out_stride_h};
  rc = packed_strides(strides, 8);
  if (rc != JKV_OK) return rc;
  PagedAttnArgs a = {};
  int form;
  rc = paged_form_args(&a, &form, scale, softcap, slopes, prefixes);
  if (rc != JKV_OK) return rc;
  if (form == kFormPlain) {
    form = kFormShaped;
    paged_scale_args(&a, scale);
  }
  if (N == 0) return JKV_OK;
  JKV_CHECK_ARG(q && k && v && out && starts, "null buffer");
  JKV_CHECK_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)rest) % 16 == 0, "packed rows must be 16-byte aligned");
  a.c.k = (uint8_t*)k; a.c.v = (uint8_t*)v;
  a.c.head_bytes = 2 * k_stride_h; a.c.slot_bytes = 2 * k_stride_t;
  a.v_head_bytes = 2 * v_stride_h; a.v_slot_bytes = 2 * v_stride_t;
  a.c.starts = starts;
  a.c.N = (int32_t)N; a.c.B = (int32_t)B;
  a.q = (const uint8_t*)q; a.qst = 2 * q_stride_t; a.qsh = 2 * q_stride_h;
  a.out = (uint8_t*)out; a.ost = 2 * out_stride_t; a.osh = 2 * out_stride_h;
  a.lse = lse; a.rest = (uint8_t*)rest;
  a.QH = (int32_t)QH; a.KVH = (int32_t)KVH; a.per = (int32_t)(QH / KVH);
  a.window = (int32_t)(window > 0 && window < kPagedMost ? window : kPagedMost);
  a.sinks = (int32_t)(sinks < kPagedMost ? sinks : kPagedMost);
  a.max_new = (int32_t)N;
  a.splits = 1;
  // Blocks of 128 rows: vector instructions bound shaped scores, and two
  // workgroups a CU, which meet apart, overlap them with products better than one
  // of eight waves does (1.55 -> 1.46 ms for 21,760 bf16 tokens with a window of
  // 4,096, 198 -> 180 us for four biased prompts; 1.44 and 175 now).  At most those of
  // all sequences, and one that clears unowned rows.
  a.item_rows = 128;
  const int64_t items = std::min<int64_t>(B * ceil_div(N * a.per, 128), N * a.per / 128 + B) + 1;
  JKV_CHECK_GRID(items * KVH, 2 * a.item_rows);
  a.items = (int32_t)items;
  // (where all blocks are resident at once, two a CU, long ones share a CU with short ones)
  a.fold = items * KVH > 256 && items * KVH <= 512 ? (int32_t)(256 / KVH) : 0x7fffffff;
  hipStream_t stream = (hipStream_t)stream_;
  if (dtype == JKV_F16) packed_launch_f16(a, form, D, stream);
  else packed_launch_bf16(a, form, D, stream);
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

int64_t jkv_packed_backward_workspace_bytes(int64_t N, int64_t B, int64_t QH, int64_t KVH, int64_t D, int64_t window) {
  // sizes that the call refuses need none
  if (N <= 0 || B < 0 || QH <= 0 || KVH <= 0 || QH % KVH || QH >= 65536 || N >= ((int64_t)1 << 30) || B >= ((int64_t)1 << 24) ||
      N * QH >= ((int64_t)1 << 31) || (D != 64 && D != 128) || window < 0)
    return 0;
  return jkv::packed_grad_plan(N, B, QH, KVH, D, window).bytes;
}

int jkv_packed_attention_backward(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_stride_t,
                                  int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h,
                                  const void* o, int64_t o_stride_t, int64_t o_stride_h, const void* rest,
                                  const void* d_out, int64_t d_stride_t, int64_t d_stride_h, const float* lse, int32_t dtype,
                                  const int32_t* starts, const int32_t* prefixes, int64_t N, int64_t B, int64_t QH,
                                  int64_t KVH, int64_t D, int64_t window, int64_t sinks, float scale, float softcap,
                                  const float* slopes, void* d_q, void* d_k, void* d_v, void* workspace,
                                  int64_t workspace_bytes, jkv_stream_t stream_) {
  using namespace jkv;
  int rc = packed_checks(dtype, N, B, QH, KVH, D, window, sinks, scale);
  if (rc != JKV_OK) return rc;
  const int64_t strides[10] = {q_stride_t, q_stride_h, k_stride_t, k_stride_h, v_stride_t,
                               v_stride_h, o_stride_t, o_stride_h, d_stride_t, d_stride_h};
  rc = packed_strides(strides, 10);
  if (rc != JKV_OK) return rc;
  PagedAttnArgs shape = {};
  int form;
  rc = paged_form_args(&shape, &form, scale, softcap, slopes, prefixes);
  if (rc != JKV_OK) return rc;
  if (N == 0) return JKV_OK;
  JKV_CHECK_ARG(q && k && v && o && d_out && lse && starts, "null buffer");
  JKV_CHECK_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)rest | (uintptr_t)d_out | (uintptr_t)d_q | (uintptr_t)d_k |
                 (uintptr_t)d_v) % 16 == 0, "packed rows must be 16-byte aligned");
  const PackedGradPlan plan = packed_grad_plan(N, B, QH, KVH, D, window);
  const int64_t need = plan.bytes;
  JKV_CHECK_ARG(workspace != nullptr && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need,
                "packed gradients need an aligned workspace of %lld bytes, got %lld", (long long)need, (long long)workspace_bytes);
  PackedGradArgs a = {};
  a.q = (const uint8_t*)q; a.k = (const uint8_t*)k; a.v = (const uint8_t*)v; a.o = (const uint8_t*)o; a.d = (const uint8_t*)d_out;
  a.rest = (const uint8_t*)rest;
  a.qst = 2 * q_stride_t; a.qsh = 2 * q_stride_h; a.kst = 2 * k_stride_t; a.ksh = 2 * k_stride_h;
  a.vst = 2 * v_stride_t; a.vsh = 2 * v_stride_h; a.ost = 2 * o_stride_t; a.osh = 2 * o_stride_h;
  a.dst = 2 * d_stride_t; a.dsh = 2 * d_stride_h;
  a.dq = (uint8_t*)d_q; a.dk = (uint8_t*)d_k; a.dv = (uint8_t*)d_v;
  a.starts = starts; a.prefixes = prefixes; a.lse = lse;
  a.N = (int32_t)N; a.B = (int32_t)B; a.QH = (int32_t)QH; a.KVH = (int32_t)KVH; a.per = (int32_t)(QH / KVH);
  a.window = (int32_t)(window > 0 && window < kPagedMost ? window : kPagedMost);
  a.sinks = (int32_t)(sinks < kPagedMost ? sinks : kPagedMost);
  a.scale = scale; a.scale2 = scale * 1.4426950408889634f;
  a.cap_mul = softcap > 0.f ? 2.f * a.scale2 / softcap : 0.f; a.cap2 = shape.cap2; a.slopes = slopes;
  a.bases = (float*)workspace;
  a.minus_delta = (float*)((uint8_t*)workspace + plan.stats_bytes);
  a.part = (float*)((uint8_t*)workspace + plan.part_at);
  a.alone = plan.alone; a.splits = plan.splits; a.heads_each = plan.heads_each;
  if (form == kFormPlain) form = kFormShaped;
  return dtype == JKV_F16 ? packed_grad_launch_f16(a, form, D, (hipStream_t)stream_)
                          : packed_grad_launch_bf16(a, form, D, (hipStream_t)stream_);
}

}  // extern "C"
