// Attention of a batch's new tokens over a paged K/V cache, with a sliding
// window and a few first entries that stay visible, and the weight that every
// cached entry receives.
//
// Token t of a sequence with T new tokens and L entries sits at entry
// i = L - T + t and sees the entries j <= i with j > i - window or j < sinks:
//   o_t = sum_j p_tj v_j,  p_tj = softmax_j(scale q_t k_j),  w_j = sum_t,h p_tj
// One wave per (token, query head); lanes share out the entries for the
// products with the keys, and the dims for those with the values.
#include <math.h>

#include <algorithm>

#include "paged.h"

namespace jkv {

// the row of a packed token, or -1
__device__ __forceinline__ int32_t paged_seq_of(const PagedCache& c, int32_t n) {
  if (c.starts == nullptr) return n < c.B ? n : -1;
  if (c.B == 0 || n < c.starts[0] || n >= c.starts[c.B]) return -1;
  int32_t lo = 0, hi = c.B;
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (c.starts[mid] <= n) lo = mid; else hi = mid;
  }
  return lo;
}

template <int DT, int D>
__global__ __launch_bounds__(64) void paged_row_kernel(PagedAttnArgs a) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V8 V8;
  __shared__ float qs[D];
  __shared__ float ps[64];
  const int lane = threadIdx.x;
  const int32_t n = (int32_t)blockIdx.x, head = (int32_t)blockIdx.y;
  const int32_t b = paged_seq_of(a.c, n);
  if (b < 0) return;
  const PagedSeq s = paged_seq(a.c, b);
  const int32_t t = n - s.row0;
  if (t < 0 || t >= s.tokens) return;
  const int32_t kvh = head / a.per;
  const T* qp = (const T*)(a.q + n * a.qst + head * a.qsh);
  if (lane < D / 2) {
    float u = (float)qp[lane], w = (float)qp[lane + D / 2];
    if (a.rope.on) {
      float c, sn;
      rope_trig(a.rope.turns[lane], s.pos0 + t, &c, &sn);
      const float r = u * c - w * sn;
      w = w * c + u * sn;
      u = r;
    }
    qs[lane] = u;
    qs[lane + D / 2] = w;
  }
  __syncthreads();
  const int32_t self = s.length - s.tokens + t;
  auto row_of = [&](const uint8_t* pool, int32_t j) -> const uint8_t* {
    const int32_t page = a.c.tables[b * a.c.table_stride + (j >> a.c.page_shift)];
    if ((uint32_t)page >= (uint32_t)a.c.n_pages) return nullptr;
    return pool + page * a.c.page_bytes + kvh * a.c.head_bytes +
           (int64_t)(j & ((1 << a.c.page_shift) - 1)) * a.c.slot_bytes;
  };
  float m = -INFINITY, l = 0.f, o[D / 64];
#pragma unroll
  for (int i = 0; i < D / 64; ++i) o[i] = 0.f;
  const int64_t low = (int64_t)self - a.window;  // entries at or below it are sinks or unseen
  for (int32_t j0 = 0; j0 <= self; j0 += 64) {
    if (j0 >= a.sinks && j0 + 63 <= low) {
      j0 = (int32_t)((low + 1) & ~63) - 64;
      continue;
    }
    const int32_t j = j0 + lane;
    const bool seen = j <= self && (j > low || j < a.sinks);
    float v = -INFINITY;
    if (seen) {
      const uint8_t* kr = row_of(a.c.k, j);
      v = 0.f;
      if (kr != nullptr)
        for (int d = 0; d < D; d += 8) {
          const V8 x = *(const V8*)(kr + 2 * d);
#pragma unroll
          for (int e = 0; e < 8; ++e) v = fmaf((float)x[e], qs[d + e], v);
        }
      v *= a.q_mul * a.scale2 * 0.6931471805599453f;
    }
    float mx = v;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
    const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.f : mn;
    const float alpha = expf(m - mu), p = seen ? expf(v - mu) : 0.f;
    m = mn;
    l = l * alpha + p;
    ps[lane] = p;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < D / 64; ++i) o[i] *= alpha;
    for (int k = 0; k < 64; ++k) {
      const int32_t jj = j0 + k;
      if (!(jj <= self && (jj > low || jj < a.sinks))) continue;
      const uint8_t* vr = row_of(a.c.v, jj);
      if (vr == nullptr) continue;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) o[i] = fmaf(ps[k], (float)((const T*)vr)[lane + 64 * i], o[i]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) l += __shfl_xor(l, off, 64);
  T* op = (T*)(a.out + n * a.ost + head * a.osh);
  const bool none = self < 0;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) op[lane + 64 * i] = (T)(none ? 0.f : o[i] / l);
  if (a.lse != nullptr && lane == 0) a.lse[(int64_t)n * a.QH + head] = none ? -INFINITY : m + logf(l);
}

// one thread per entry: the weights of every token and head of the group
template <int DT, int D>
__global__ __launch_bounds__(256) void paged_weights_kernel(PagedAttnArgs a) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V8 V8;
  __shared__ float qs[D];
  const int32_t b = (int32_t)blockIdx.z, kvh = (int32_t)blockIdx.y, j = (int32_t)(blockIdx.x * 256 + threadIdx.x);
  const PagedSeq s = paged_seq(a.c, b);
  if ((int32_t)(blockIdx.x * 256) >= s.length) return;
  float k[D];
  const int32_t page = j < s.length ? a.c.tables[b * a.c.table_stride + (j >> a.c.page_shift)] : -1;
  const bool ok = (uint32_t)page < (uint32_t)a.c.n_pages;
  const uint8_t* kr = a.c.k + (ok ? page * a.c.page_bytes + kvh * a.c.head_bytes +
                                        (int64_t)(j & ((1 << a.c.page_shift) - 1)) * a.c.slot_bytes : 0);
#pragma unroll
  for (int d = 0; d < D; d += 8) {
    V8 x = {};
    if (ok) x = *(const V8*)(kr + 2 * d);
#pragma unroll
    for (int e = 0; e < 8; ++e) k[d + e] = (float)x[e];
  }
  float sum = 0.f;
  for (int32_t t = 0; t < s.tokens; ++t)
    for (int32_t g = 0; g < a.per; ++g) {
      const int32_t head = kvh * a.per + g, n = s.row0 + t;
      const T* qp = (const T*)(a.q + n * a.qst + head * a.qsh);
      __syncthreads();
      if (threadIdx.x < D / 2) {
        const int i = threadIdx.x;
        float u = (float)qp[i], w = (float)qp[i + D / 2];
        if (a.rope.on) {
          float c, sn;
          rope_trig(a.rope.turns[i], s.pos0 + t, &c, &sn);
          const float r = u * c - w * sn;
          w = w * c + u * sn;
          u = r;
        }
        qs[i] = u;
        qs[i + D / 2] = w;
      }
      __syncthreads();
      const int32_t self = s.length - s.tokens + t;
      if (!(j <= self && (j > (int64_t)self - a.window || j < a.sinks))) continue;
      float v = 0.f;
#pragma unroll
      for (int d = 0; d < D; ++d) v = fmaf(k[d], qs[d], v);
      sum += expf(v * a.q_mul * a.scale2 * 0.6931471805599453f - a.lse[(int64_t)n * a.QH + head]);
    }
  if (j < s.length) {
    float* w = a.weights + b * a.wsb + kvh * a.wsh + j;
    *w = a.accumulate ? *w + sum : sum;
  }
}

template <int DT, int D>
static void launch_paged(const PagedAttnArgs& a, int64_t max_length, hipStream_t stream) {
  hipLaunchKernelGGL((paged_row_kernel<DT, D>), dim3(a.c.N, a.QH), dim3(64), 0, stream, a);
  if (a.weights != nullptr)
    hipLaunchKernelGGL((paged_weights_kernel<DT, D>), dim3((uint32_t)ceil_div(std::max<int64_t>(max_length, 1), 256), a.KVH, a.c.B), dim3(256),
                       0, stream, a);
}

// How a call's work is divided and what of the workspace it takes.
struct PagedPlan {
  bool few;  // at most 32 rows a sequence and kv head
  int64_t splits, split_tiles, score_width;
  int64_t ml_at, o_at, lse_at, lse2_at, scores_at, bytes;
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
    // two waves a SIMD of every CU
    const int64_t want = std::max<int64_t>(1, 2048 / std::max<int64_t>(1, B * KVH));
    p.split_tiles = std::max<int64_t>(2, ceil_div(tiles, want));
    p.splits = ceil_div(tiles, p.split_tiles);
    if (p.splits > 1) {
      p.ml_at = take(p.splits * N * QH * 8);
      p.o_at = take(p.splits * N * QH * D * 4);
    }
    if (weights) {
      p.lse2_at = take(N * QH * 4);
      p.score_width = ceil_div(max_length, 32) * 32;
      p.scores_at = take(B * KVH * max_new * per * p.score_width * 4);
    }
  } else if (weights) {
    p.lse_at = take(N * QH * 4);
  }
  p.bytes = at;
  return p;
}

}  // namespace jkv

extern "C" {

int64_t jkv_paged_attention_workspace_bytes(int64_t N, int64_t B, int64_t QH, int64_t KVH, int64_t D, int64_t max_new,
                                            int64_t max_length, int64_t window, int64_t sinks, int32_t with_weights) {
  if (N <= 0 || B <= 0 || QH <= 0 || KVH <= 0 || QH % KVH != 0) return 0;
  const int64_t most = jkv::kPagedMost;
  return jkv::paged_plan(N, B, QH, KVH, D, std::min(max_new, N), std::min(max_length, most),
                         window > 0 && window < most ? window : most, std::min(sinks, most), with_weights != 0).bytes;
}

int jkv_paged_attention(const void* q, int64_t q_stride_t, int64_t q_stride_h, int32_t dtype, const void* key_pages,
                        const void* value_pages, int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                        int64_t n_pages, int64_t page_size, const int32_t* block_tables, int64_t table_stride,
                        int64_t table_width, const int32_t* lengths, const int32_t* starts, const int32_t* positions,
                        int64_t N, int64_t B, int64_t QH, int64_t KVH, int64_t D, int64_t max_new, int64_t max_length,
                        int64_t window, int64_t sinks, double rope_theta, float scale, void* out, int64_t out_stride_t,
                        int64_t out_stride_h, float* lse, float* weights, int64_t weight_stride_b,
                        int64_t weight_stride_h, int64_t weight_width, int32_t accumulate, void* workspace,
                        int64_t workspace_bytes, jkv_stream_t stream_) {
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
  JKV_CHECK_ARG(isfinite(scale), "the softmax scale must be finite");
  const int64_t strides[4] = {q_stride_t, q_stride_h, out_stride_t, out_stride_h};
  for (int i = 0; i < 4; ++i)
    JKV_CHECK_ARG(strides[i] % 8 == 0, "token and head strides must be multiples of 8 elements");
  JKV_CHECK_ARG(((uintptr_t)q | (uintptr_t)out) % 16 == 0, "queries and outputs must be 16-byte aligned");
  max_length = a.c.top;
  JKV_CHECK_ARG(weights == nullptr || weight_width >= max_length, "weights have fewer entries than max_length");
  if (N == 0 || B == 0) return JKV_OK;
  JKV_CHECK_ARG(q && out, "null buffer");
  if (max_new > N) max_new = N;
  a.window = (int32_t)(window > 0 && window < kPagedMost ? window : kPagedMost);
  a.sinks = (int32_t)(sinks < kPagedMost ? sinks : kPagedMost);
  const PagedPlan p = paged_plan(N, B, QH, KVH, D, max_new, max_length, a.window, a.sinks, weights != nullptr);
  JKV_CHECK_ARG(workspace_bytes >= p.bytes && (p.bytes == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0)),
                "paged attention needs an aligned workspace of %lld bytes, got %lld", (long long)p.bytes,
                (long long)workspace_bytes);
  uint8_t* ws = (uint8_t*)workspace;
  a.q = (const uint8_t*)q; a.qst = 2 * q_stride_t; a.qsh = 2 * q_stride_h;
  a.out = (uint8_t*)out; a.ost = 2 * out_stride_t; a.osh = 2 * out_stride_h;
  a.lse = lse;
  a.weights = weights; a.wsb = weight_stride_b; a.wsh = weight_stride_h; a.accumulate = accumulate;
  a.QH = (int32_t)QH; a.KVH = (int32_t)KVH; a.per = (int32_t)(QH / KVH);
  a.max_new = (int32_t)max_new;
  a.q_mul = scale == 0.f ? 0.f : scale < 0.f ? -0.5f : 0.5f;
  a.scale2 = scale == 0.f ? 1.f : fabsf(scale) * 2.f * 1.4426950408889634f;
  a.splits = (int32_t)p.splits; a.split_tiles = (int32_t)p.split_tiles;
  if (p.few) {
    a.part_ml = (float2*)(ws + p.ml_at);
    a.part_o = (float*)(ws + p.o_at);
    if (weights != nullptr) {
      a.lse2 = (float*)(ws + p.lse2_at);
      a.scores = (float*)(ws + p.scores_at);
      a.score_width = p.score_width;
    }
    return paged_launch_few(a, dtype, D, stream);
  }
  if (lse == nullptr && weights != nullptr) a.lse = (float*)(ws + p.lse_at);
  if (dtype == JKV_F16 && D == 128) launch_paged<JKV_F16, 128>(a, max_length, stream);
  else if (dtype == JKV_F16) launch_paged<JKV_F16, 64>(a, max_length, stream);
  else if (D == 128) launch_paged<JKV_BF16, 128>(a, max_length, stream);
  else launch_paged<JKV_BF16, 64>(a, max_length, stream);
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

}  // extern "C"
