// Attention of a batch's new tokens over a paged K/V cache, with a sliding
// window and a few first entries that stay visible, and the weight that every
// cached entry receives.
//
// Token t of a sequence with T new tokens and L entries sits at entry
// i = L - T + t and sees the entries j <= i with j > i - window or j < sinks:
//   o_t = sum_j p_tj v_j,  p_tj = softmax_j(scale q_t k_j),  w_j = sum_t,h p_tj
// A row that sees nothing (or only scores of -infinity) gives 0.
// Here: a call's checks, the division of its work and its workspace.  Sequences
// of few rows (paged_few.hip) and chunks (paged_chunk.hip) have kernels of
// their own.
#include <math.h>

#include <algorithm>

#include "paged.h"

namespace jkv {

// How a call's work is divided and what of the workspace it takes.
struct PagedPlan {
  bool few;  // at most 32 rows a sequence and kv head
  int64_t items, item_rows, waves, splits, split_tiles, score_width;
  int64_t ml_at, o_at, lse2_at, scores_at, q_at, bytes;
};

static PagedPlan paged_plan(int64_t N, int64_t B, int64_t QH, int64_t KVH, int64_t D, int64_t max_new, int64_t max_length,
                            int64_t window, int64_t sinks, bool weights) {
  PagedPlan p = {};
  const int64_t per = QH / KVH;
  p.few = max_new * per <= 32;
  p.splits = 1;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += ceil_div(bytes, 256) * 256;
    return from;
  };
  if (p.few) {
    // the most tiles a sequence can have
    int64_t tiles = ceil_div(max_length, 32);
    const int64_t bound = ceil_div(window + max_new, 32) + 1 + ceil_div(sinks, 32);
    if (bound < tiles) tiles = bound;
    if (tiles < 1) tiles = 1;
    // A wave's tile takes about 1.7 us (its loads), a join 5: up to four tiles
    // stay with one wave.  More waves of a workgroup that join in LDS save the
    // join where each has at most two tiles, or eight where the sequences alone
    // fill half the CUs, and where one round of workgroups holds all (a CU holds
    // one at 128 dims, two at 64).  us with splits and with eight waves, 32/8
    // heads of 128: 16 x 128 entries 13.1 and 9.9, 16 x 500 18.4 and 16.7, 16 x
    // 1,000 23.5 and 21.1; 4 x 1,000 16.4 and 18.7, 64 x 500 36.8 and 40.7.
    const int64_t bh = B * KVH, many = D == 128 && max_new * per > 16 ? 4 : 8;
    p.waves = 1;
    if (tiles <= 4) {
      p.split_tiles = tiles;
    } else if (bh <= 256 * (128 / D) && (tiles <= 2 * many || (bh >= 128 && tiles <= 8 * many))) {
      p.waves = many;
      p.split_tiles = tiles;
    } else {
      // a wave a SIMD of every CU, two at 64 dims: 64 KiB of loads in flight a CU
      // carry the memory's rate, and more splits are more to join.  us with 1,024
      // waves and with 2,048: 4 ragged sequences to 65,536 entries 122 and 133, 1
      // x 60,000 59 and 65, 16 x 4,096 60 and 62; at 64 dims 24 windows of 4,096
      // 29 and 27.
      const int64_t want = std::max<int64_t>(1, 1024 * (128 / D) / std::max<int64_t>(1, bh));
      p.split_tiles = std::max<int64_t>(2, ceil_div(tiles, want));
    }
    p.splits = ceil_div(tiles, p.split_tiles);
    if (p.splits > 1) {
      p.ml_at = take(p.splits * N * QH * 8);
      p.o_at = take(p.splits * N * QH * D * 4);
    }
    if (weights) {
      p.lse2_at = take(N * QH * 4);
      p.score_width = ceil_div(max_length, 32) * 32;
      if ((double)(B * KVH) * (double)(max_new * per) * (double)p.score_width > 1e14) {  // no memory holds them
        p.bytes = INT64_MAX;
        return p;
      }
      p.scores_at = take(B * KVH * max_new * per * p.score_width * 4);
    }
  } else {
    // Eight-wave blocks of 256 rows where one a CU goes round: their tiles serve
    // twice the rows.  Where most of what is seen is the chunk itself, blocks
    // differ in length, and it takes two a CU to even them out.  us with four and
    // with eight waves, 32/8 heads of 128: 2 x 2,048 tokens over 16,384 entries
    // 917 and 852, 2 x 1,024 over 4,096 135 and 129; prompts of 1 x 2,000 57 and
    // 63, 16 x 2,048 the same; at 64 dims, where three workgroups share a CU, 4 x
    // 1,024 over 4,096 150 and 168.
    auto blocks_of = [&](int64_t rows) { return std::min<int64_t>(B * ceil_div(max_new * per, rows), N * per / rows + B); };
    const int64_t rounds = blocks_of(256) * KVH / 256;
    p.item_rows = D == 128 && rounds >= (max_length >= 2 * max_new ? 1 : 2) ? 256 : 128;
    p.items = blocks_of(p.item_rows);
    int64_t tiles = ceil_div(max_length, 64);
    const int64_t bound = ceil_div(window + std::min<int64_t>(max_new, p.item_rows / per + 1), 64) + 1 + ceil_div(sinks, 64);
    if (bound < tiles) tiles = bound;
    if (tiles < 1) tiles = 1;
    // Splits save (1 - 1/s) of a block's tiles, about 1 us each at 128 dims, and
    // cost a join of 6 us and its parts' way through memory, N QH D 8 bytes each
    // at 4 TB/s: the best s is the root of the two's ratio.  us with two splits
    // and without, 32/8 heads: 1 x 1,000 tokens 44 and 36; with four and
    // without, 1 x 512 over 4,096 entries 59 and 75.
    const double save = (double)tiles * (D == 128 ? 1.0 : 0.6), part = (double)(N * QH) * (double)D * 8.0 / 4.0e6;
    const int64_t most = std::min<int64_t>(512 / (p.items * KVH), tiles / 4);
    const int64_t best = std::min<int64_t>(most, (int64_t)(sqrt(save / part) + 0.5));
    p.splits = best > 1 && save * (1.0 - 1.0 / (double)best) > 6.0 + part * (double)best ? best : 1;
    // Between one and two workgroups a CU some CUs have two and the others wait
    // for them: two splits even that out where long chains pay for the join.  us
    // with two and without: 1 x 1,200 tokens over 16,384 entries 392 and 404, 1 x
    // 1,500 over 32,000 765 and 812, four ragged of 500 over 16,384 273 and 309,
    // 1 x 1,500 over 16,384 at 64 dims 240 and 275; below the line 1 x 1,100 over
    // 6,000 156 and 146, 1 x 1,600 over 16,384 480 and 445.
    const int64_t groups = p.items * KVH;
    if (groups > 256 && groups < 512 && 0.45 * (double)tiles * (1.0 - (double)groups / 512.0) > 6.0 + 2.0 * part) p.splits = 2;
    if (p.splits > 1) {
      p.ml_at = take(p.splits * N * QH * 8);
      p.o_at = take(p.splits * N * QH * D * 4);
    }
    if (weights) {
      p.lse2_at = take(N * QH * 4);
      p.q_at = take(N * QH * D * 4);
    }
  }
  p.bytes = at;
  return p;
}

// A shaped score's scale, above 0: a negative one turns the queries round, and one
// of 0 is near it (a masked score is -infinity times it).
void paged_scale_args(PagedAttnArgs* a, float scale) {
  a->q_mul = a->rope.on ? 0.5f : 1.f;  // a rotated fp16 query reaches sqrt 2 of its size
  a->scale2 = fmaxf(fabsf(scale) * 1.4426950408889634f / a->q_mul, 1e-37f);
  if (scale < 0.f) a->q_mul = -a->q_mul;
}

// what becomes of a score: the form's bits and what its kernels take
int paged_form_args(PagedAttnArgs* a, int* form, float scale, float softcap, const float* slopes, const int32_t* prefixes) {
  *form = kFormPlain;
  // (a capped score is within 2e-7 of the cap)
  JKV_CHECK_ARG(softcap == 0.f || (softcap >= 1e-3f && softcap <= 1024.f), "a cap must be from 0.001 to 1024, or 0 for none");
  if (softcap == 0.f && slopes == nullptr && prefixes == nullptr) return JKV_OK;
  *form = kFormShaped | (softcap > 0.f ? kFormCap : 0) | (slopes != nullptr ? kFormBias : 0);
  a->slopes = slopes;
  a->prefixes = prefixes;
  paged_scale_args(a, scale);
  if (softcap > 0.f) {
    a->cap_mul = 2.f * a->scale2 / softcap;
    a->cap2 = softcap * 1.4426950408889634f;
  }
  return JKV_OK;
}

}  // namespace jkv

extern "C" {

int64_t jkv_paged_attention_workspace_bytes(int64_t N, int64_t B, int64_t QH, int64_t KVH, int64_t D, int64_t max_new,
                                            int64_t max_length, int64_t window, int64_t sinks, int32_t with_weights) {
  if (N <= 0 || B <= 0 || QH <= 0 || KVH <= 0 || QH % KVH != 0) return 0;
  // sizes that the call refuses need none
  if ((D != 64 && D != 128) || N >= ((int64_t)1 << 30) || B >= ((int64_t)1 << 24) || QH >= 65536 || max_length < 0 ||
      window < 0 || sinks < 0)
    return 0;
  const int64_t most = jkv::kPagedMost;
  return jkv::paged_plan(N, B, QH, KVH, D, std::max<int64_t>(1, std::min(max_new, N)), std::min(max_length, most),
                         window > 0 && window < most ? window : most, std::min(sinks, most), with_weights != 0).bytes;
}

int jkv_paged_attention_shaped(const void* q, int64_t q_stride_t, int64_t q_stride_h, int32_t dtype, const void* key_pages,
                        const void* value_pages, int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                        int64_t n_pages, int64_t page_size, const int32_t* block_tables, int64_t table_stride,
                        int64_t table_width, const int32_t* lengths, const int32_t* starts, const int32_t* positions,
                        int64_t N, int64_t B, int64_t QH, int64_t KVH, int64_t D, int64_t max_new, int64_t max_length,
                        int64_t window, int64_t sinks, double rope_theta, float scale, void* out, int64_t out_stride_t,
                        int64_t out_stride_h, float* lse, float* weights, int64_t weight_stride_b,
                        int64_t weight_stride_h, int64_t weight_width, int32_t accumulate, float softcap,
                        const float* slopes, const int32_t* prefixes, void* workspace, int64_t workspace_bytes,
                        jkv_stream_t stream_) {
  using namespace jkv;
  hipStream_t stream = (hipStream_t)stream_;
  PagedAttnArgs a = {};
  JKV_CHECK_ARG(QH > 0 && KVH > 0 && QH % KVH == 0 && QH < 65536, "query heads must be a multiple of kv heads");
  JKV_CHECK_ARG(max_new >= 0 && max_length >= 0, "max_new and max_length must not be negative");
  int rc = paged_cache_args(&a.c, key_pages, value_pages, page_stride, head_stride, slot_stride, n_pages, page_size,
                            block_tables, table_stride, table_width, lengths, starts, positions, N, B, KVH, D, max_length,
                            dtype);
  if (rc != JKV_OK) return rc;
  rc = paged_rope_args(&a.rope, rope_theta, D);
  if (rc != JKV_OK) return rc;
  JKV_CHECK_ARG(window >= 0 && sinks >= 0, "window and sinks must not be negative");
  // (its powers of two have to fit 32 bits below)
  JKV_CHECK_ARG(fabsf(scale) < 1e30f, "the softmax scale must be finite and below 1e30");
  const int64_t strides[4] = {q_stride_t, q_stride_h, out_stride_t, out_stride_h};
  for (int i = 0; i < 4; ++i)
    JKV_CHECK_ARG(strides[i] % 8 == 0, "token and head strides must be multiples of 8 elements");
  JKV_CHECK_ARG(((uintptr_t)q | (uintptr_t)out) % 16 == 0, "queries and outputs must be 16-byte aligned");
  max_length = a.c.top;
  JKV_CHECK_ARG(weights == nullptr || weight_width >= max_length, "weights have fewer entries than max_length");
  int form;
  rc = paged_form_args(&a, &form, scale, softcap, slopes, prefixes);
  if (rc != JKV_OK) return rc;
  if (B == 0) return JKV_OK;
  a.QH = (int32_t)QH; a.KVH = (int32_t)KVH; a.per = (int32_t)(QH / KVH);
  a.weights = weights; a.wsb = weight_stride_b; a.wsh = weight_stride_h; a.accumulate = accumulate;
  if (N == 0) {  // nobody attends: the entries received nothing
    if (weights == nullptr || accumulate) return JKV_OK;
    JKV_CHECK_ARG(lengths, "null buffer");
    return paged_launch_few_weights(a, stream);
  }
  JKV_CHECK_ARG(q && out, "null buffer");
  JKV_CHECK_ARG(N * QH < ((int64_t)1 << 31) - 256, "too many rows");
  max_new = std::max<int64_t>(1, std::min(max_new, N));
  a.window = (int32_t)(window > 0 && window < kPagedMost ? window : kPagedMost);
  a.sinks = (int32_t)(sinks < kPagedMost ? sinks : kPagedMost);
  PagedPlan p = paged_plan(N, B, QH, KVH, D, max_new, max_length, a.window, a.sinks, weights != nullptr);
  JKV_CHECK_ARG(workspace_bytes >= p.bytes && (p.bytes == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0)),
                "paged attention needs an aligned workspace of %lld bytes, got %lld", (long long)p.bytes,
                (long long)workspace_bytes);
  if (form != kFormPlain && p.item_rows == 256) {
    // Shaped scores are bound by vector instructions, and four-wave blocks, two a CU,
    // overlap those with products where the blocks of 256 rows are few or part full.  us
    // with 128 rows and with 256, capped bf16, 32/8 heads of 128: 2,048 tokens over 8,192
    // entries 304 and 319, with one token over 3,436 beside them 332 and 326, 2 x 2,048
    // over 8,192 584 and 565, 40 x 10 over 4,096 157 and 195, 60 x 10 over 16,384 694 and
    // 764.  Without the two splits that the plan may have made for blocks of 256, and
    // with them: 2,048 over 8,192 304 and 338, 40 x 10 over 16,384 590 and 573.
    p.item_rows = 128;
    p.items = std::min<int64_t>(B * ceil_div(max_new * (QH / KVH), 128), N * (QH / KVH) / 128 + B);
    p.splits = 1;
  }
  uint8_t* ws = (uint8_t*)workspace;
  a.q = (const uint8_t*)q; a.qst = 2 * q_stride_t; a.qsh = 2 * q_stride_h;
  a.out = (uint8_t*)out; a.ost = 2 * out_stride_t; a.osh = 2 * out_stride_h;
  a.lse = lse;
  a.max_new = (int32_t)max_new;
  if (form == kFormPlain) {
    a.q_mul = scale * 1.4426950408889634f;
    a.scale2 = 1.f;
    while (fabsf(a.q_mul) > 0.5f) {
      a.q_mul *= 0.5f;
      a.scale2 *= 2.f;
    }
  }
  a.splits = (int32_t)p.splits; a.split_tiles = (int32_t)p.split_tiles;
  a.items = (int32_t)p.items;
  a.item_rows = (int32_t)p.item_rows;
  const bool resident = p.item_rows == 128 && p.splits == 1 && p.items * KVH > 256 && p.items * KVH <= 512;
  a.fold = resident ? (int32_t)(256 / KVH) : 0x7fffffff;
  a.waves = (int32_t)p.waves;
  a.part_ml = (float2*)(ws + p.ml_at);
  a.part_o = (float*)(ws + p.o_at);
  if (weights != nullptr) {
    a.lse2 = (float*)(ws + p.lse2_at);
    a.score_width = p.score_width;
    if (p.few) a.scores = (float*)(ws + p.scores_at);
    else a.q_parts = ws + p.q_at;
  }
  if (form != kFormPlain)
    return dtype == JKV_F16 ? paged_launch_form_f16(a, form, p.few, D, stream) : paged_launch_form_bf16(a, form, p.few, D, stream);
  return p.few ? paged_launch_few(a, dtype, D, stream) : paged_launch_chunk(a, dtype, D, stream);
}

int jkv_paged_attention(const void* q, int64_t q_stride_t, int64_t q_stride_h, int32_t dtype, const void* key_pages,
                        const void* value_pages, int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                        int64_t n_pages, int64_t page_size, const int32_t* block_tables, int64_t table_stride,
                        int64_t table_width, const int32_t* lengths, const int32_t* starts, const int32_t* positions,
                        int64_t N, int64_t B, int64_t QH, int64_t KVH, int64_t D, int64_t max_new, int64_t max_length,
                        int64_t window, int64_t sinks, double rope_theta, float scale, void* out, int64_t out_stride_t,
                        int64_t out_stride_h, float* lse, float* weights, int64_t weight_stride_b,
                        int64_t weight_stride_h, int64_t weight_width, int32_t accumulate, void* workspace,
                        int64_t workspace_bytes, jkv_stream_t stream) {
  return jkv_paged_attention_shaped(q, q_stride_t, q_stride_h, dtype, key_pages, value_pages, page_stride, head_stride,
                                    slot_stride, n_pages, page_size, block_tables, table_stride, table_width, lengths,
                                    starts, positions, N, B, QH, KVH, D, max_new, max_length, window, sinks, rope_theta,
                                    scale, out, out_stride_t, out_stride_h, lse, weights, weight_stride_b,
                                    weight_stride_h, weight_width, accumulate, 0.f, nullptr, nullptr, workspace,
                                    workspace_bytes, stream);
}

}  // extern "C"
