// Attention over a paged K/V cache for sequences with few rows: plain scores, the
// weights that entries receive, and the join of the splits' parts.  (The kernel,
// its reasons and what it measures are in few_attn.h.)
#include "few_attn.h"

namespace jkv {

// The weights of few rows, from the scores that the attention left: one thread
// an entry, its rows' sum in their order.
__global__ __launch_bounds__(256) void paged_few_weights_kernel(PagedAttnArgs a) {
  const uint32_t bh = blockIdx.y + blockIdx.z * 32768u;
  const int32_t b = (int32_t)(bh / (uint32_t)a.KVH), kvh = (int32_t)(bh - (uint32_t)b * (uint32_t)a.KVH);
  if (b >= a.c.B) return;
  const PagedSeq s = paged_seq(a.c, b);
  const int32_t j = (int32_t)(blockIdx.x * 256 + threadIdx.x);
  if (j >= s.length) return;
  const int32_t tokens = s.tokens < a.max_new ? s.tokens : a.max_new, first = s.length - s.tokens;
  const float* sc = a.scores + ((int64_t)b * a.KVH + kvh) * (a.max_new * a.per) * a.score_width + j;
  float sum = 0.f;
  const int32_t prefix = paged_prefix(a.prefixes, b, s.length);
  for (int32_t t = 0; t < tokens; ++t) {
    const int32_t self = first + t;
    if (!((j <= self || (j < prefix && self >= 0)) && (j > self - a.window || j < a.sinks))) continue;
    const float* norm = a.lse2 + ((int64_t)kvh * a.c.N + s.row0 + t) * a.per;
    for (int32_t g = 0; g < a.per; ++g) {
      const float p = __builtin_amdgcn_exp2f(sc[(int64_t)(t * a.per + g) * a.score_width] - norm[g]);
      sum += norm[g] == -INFINITY ? 0.f : p;  // (a row of only -infinities saw nothing)
    }
  }
  float* w = a.weights + b * a.wsb + kvh * a.wsh + j;
  *w = a.accumulate ? *w + sum : sum;
}

// Joins the splits' parts of a row by their maxima and sums.  D/4 lanes hold a
// row; GROUPS of them share out its splits, several loads in flight each, and
// meet in LDS, always in the same order.
struct JoinArgs {
  const float2* part_ml;
  const float* part_o;
  const int32_t* starts;
  uint8_t* out;
  int64_t ost, osh;
  float *lse, *lse2;
  int32_t N, B, QH, per, splits;
};

template <int DT, int D, int GROUPS>
__global__ __launch_bounds__(8 * D) void paged_join_kernel(JoinArgs a) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V4 V4;
  constexpr int kLanes = D / 4, kRows = 32 / GROUPS;
  __shared__ __align__(16) float o_lds[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? kRows : 1][D];
  __shared__ float2 ml_lds[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? kRows : 1];
  const int tid = threadIdx.x, part = tid % kLanes, g = tid / kLanes % GROUPS, r = tid / (kLanes * GROUPS);
  const int64_t rows = (int64_t)a.N * a.QH;
  int64_t row = (int64_t)blockIdx.x * kRows + r;
  bool on = row < rows;
  if (!on) row = rows - 1;
  const int32_t n = (int32_t)((uint32_t)row / (uint32_t)a.QH), head = (int32_t)(row - (int64_t)n * a.QH);
  if (a.starts != nullptr) on = on && n >= a.starts[0] && n < a.starts[a.B];  // nobody's rows stay as they are
  float m = -INFINITY, l = 0.f;
  float4v o = {0.f, 0.f, 0.f, 0.f};
  {
    for (int32_t i0 = g; i0 < a.splits; i0 += 8 * GROUPS) {
      float2 ml[8];
      float4v p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int32_t i = i0 + j * GROUPS < a.splits ? i0 + j * GROUPS : i0;
        ml[j] = a.part_ml[i * rows + row];
        p[j] = *(const float4v*)(a.part_o + (i * rows + row) * D + 4 * part);
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (i0 + j * GROUPS >= a.splits) ml[j] = float2{-INFINITY, 0.f};
        top = fmaxf(top, ml[j].x);
      }
      const float f0 = m == top ? 1.f : part_factor(m, top);
      l *= f0;
      o *= f0;
      m = top;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (ml[j].y != 0.f) {  // a split that saw nothing may have written no sums
          const float f = part_factor(ml[j].x, top);
          l = fmaf(ml[j].y, f, l);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = fmaf(p[j][e], f, o[e]);
        }
    }
  }
  if constexpr (GROUPS > 1) {
    *(float4v*)&o_lds[g][r][4 * part] = o;
    if (part == 0) ml_lds[g][r] = float2{m, l};
    __syncthreads();
    if (g != 0) return;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) top = fmaxf(top, ml_lds[j][r].x);
    l = 0.f;
    o = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      const float2 ml = ml_lds[j][r];
      if (ml.y == 0.f) continue;
      const float f = part_factor(ml.x, top);
      l = fmaf(ml.y, f, l);
      const float4v p = *(const float4v*)&o_lds[j][r][4 * part];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(p[e], f, o[e]);
    }
    m = top;
  }
  if (!on) return;
  const bool none = l == 0.f;
  if (part == 0) {
    const float l2 = none ? -INFINITY : (m == -INFINITY ? 0.f : m) + log2f(l);
    if (a.lse != nullptr) a.lse[row] = l2 * 0.6931471805599453f;
    if (a.lse2 != nullptr) a.lse2[paged_lse2_at(a.N, a.per, row, a.QH)] = l2;
  }
  V4 h;
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = (T)(none ? 0.f : o[e] / l);
  *(V4*)(a.out + n * a.ost + head * a.osh + 8 * part) = h;
}

template <int DT, int D>
static void launch_join(const PagedAttnArgs& x, hipStream_t stream) {
  const JoinArgs a = {x.part_ml, x.part_o, x.c.starts, x.out, x.ost, x.osh, x.lse, x.lse2, x.c.N, x.c.B, x.QH, x.per, x.splits};
  const int64_t rows = (int64_t)a.N * a.QH;
  const dim3 block(8 * D);
  if (a.splits > 8)
    hipLaunchKernelGGL((paged_join_kernel<DT, D, 8>), dim3((uint32_t)ceil_div(rows, 4)), block, 0, stream, a);
  else
    hipLaunchKernelGGL((paged_join_kernel<DT, D, 1>), dim3((uint32_t)ceil_div(rows, 32)), block, 0, stream, a);
}

int paged_launch_join(const PagedAttnArgs& a, int32_t dtype, int64_t D, hipStream_t stream) {
  JKV_CHECK_GRID(ceil_div((int64_t)a.c.N * a.QH, a.splits > 8 ? 4 : 32), 1024);
  if (dtype == JKV_F16) D == 128 ? launch_join<JKV_F16, 128>(a, stream) : launch_join<JKV_F16, 64>(a, stream);
  else D == 128 ? launch_join<JKV_BF16, 128>(a, stream) : launch_join<JKV_BF16, 64>(a, stream);
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

int paged_launch_few_weights(const PagedAttnArgs& a, hipStream_t stream) {
  const int64_t bh = (int64_t)a.c.B * a.KVH;
  if (a.c.top > 0)
    hipLaunchKernelGGL(paged_few_weights_kernel, dim3((uint32_t)ceil_div(a.c.top, 256), (uint32_t)(bh < 32768 ? bh : 32768),
                       (uint32_t)ceil_div(bh, 32768)), dim3(256), 0, stream, a);
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

int paged_launch_few(const PagedAttnArgs& a, int32_t dtype, int64_t D, hipStream_t stream) {
  if (dtype == JKV_F16) return D == 128 ? launch_few<JKV_F16, 128, kFormPlain>(a, stream) : launch_few<JKV_F16, 64, kFormPlain>(a, stream);
  return D == 128 ? launch_few<JKV_BF16, 128, kFormPlain>(a, stream) : launch_few<JKV_BF16, 64, kFormPlain>(a, stream);
}

}  // namespace jkv
