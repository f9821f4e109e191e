// Queries and keys turned at their positions, in one launch.
//
// Pair i of a head's first R dims, (i, i + R/2) or (2i, 2i + 1), turns by the
// angle a = position * rate_i:
//   (x, y) -> m (x cos a - y sin a, y cos a + x sin a),
// the gradient by -a.  Dims from R on are copied.  Position and rate multiply
// in 64 bits and lose whole turns and quarters there (32 bits lose the angle of
// far positions); sine and cosine of what is left and the products are 32-bit,
// rounded once to the tensors' type.
//
// Memory bounds it, or the launch where there are few tokens.  A workgroup
// takes a few tokens: their angles' functions are computed once for all heads
// and lie in LDS, threads share out the heads' units of 2 x VEC dims.  32/8 heads of
// 128 of 10,430 bf16 tokens, 213 MB in and out, 44 us, 4.8 TB/s (a large copy reaches
// 4.97; stores that the caches need not keep take 55); 16 single tokens 5 us.
#include <math.h>

#include "paged.h"

namespace jkv {

static const int kRotaryThreads = 256;
static const int kRotaryMost = 256;  // dims of a head

struct RotaryArgs {
  const uint8_t *q, *k;
  uint8_t *q_out, *k_out;
  int64_t qst, qsh, kst, ksh, qost, qosh, kost, kosh;  // byte strides
  int32_t QH, KVH, N, B, dims, units, turned;  // units of a head, and how many of them turn
  int32_t tokens;                              // of a workgroup
  const int32_t *starts, *positions;
  float magnitude, sign;
  double turns[kRotaryMost / 2];  // of a position
};

// cos and sin of rate * position turns: whole turns and quarters taken off in 64
// bits.  (No contraction, here and in the rotation: all vector widths agree.)
#pragma clang fp contract(off)
__device__ __forceinline__ float2 turn_trig(double rate, int32_t position) {
  const double turns = rate * (double)position;
  const double part = 4.0 * (turns - rint(turns));  // quarters, in [-2, 2]
  const double quarter = rint(part);
  float s, c;
  sincospif(0.5f * (float)(part - quarter), &s, &c);
  const int n = (int)quarter & 3;
  if (n & 1) {
    const float t = c;
    c = -s;
    s = t;
  }
  return n & 2 ? float2{-c, -s} : float2{c, s};
}
#pragma clang fp contract(on)

template <int DT, int VEC, bool PAIRS_SIDE_BY_SIDE>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
  typedef typename Elem<DT>::T T;
  struct alignas(sizeof(T) * VEC) Vec { T x[VEC]; };
  extern __shared__ float2 trig[];  // [tokens][dims / 2]
  __shared__ int32_t at[8];
  __shared__ int32_t owned[8];
  const int tid = threadIdx.x, lane = tid & 63, half = a.dims / 2;
  const int32_t n0 = (int32_t)blockIdx.x * a.tokens;
  const int32_t tokens = a.N - n0 < a.tokens ? a.N - n0 : a.tokens;
  // a wave finds a token's position
  for (int t = tid >> 6; t < tokens; t += kRotaryThreads / 64) {
    const int32_t n = n0 + t;
    int32_t pos = n;
    bool mine = true;
    if (a.starts != nullptr) {
      // the last sequence that starts at or before it
      int32_t upto = 0;
      for (int32_t b0 = 0; b0 < a.B; b0 += 64)
        upto += __popcll(__ballot(b0 + lane < a.B && a.starts[b0 + lane < a.B ? b0 + lane : 0] <= n));
      mine = upto > 0 && n < a.starts[a.B];
      if (mine) pos = n - a.starts[upto - 1] + (a.positions != nullptr ? a.positions[upto - 1] : 0);
    } else if (a.positions != nullptr) {
      pos = a.positions[n];
    }
    if (lane == 0) {
      at[t] = pos;
      owned[t] = mine;
    }
  }
  __syncthreads();
  for (int i = tid; i < tokens * half; i += kRotaryThreads) {
    const int t = i / half;
    float2 cs = turn_trig(a.turns[i - t * half], at[t]);
    cs.x *= a.magnitude;
    cs.y *= a.magnitude * a.sign;
    trig[i] = owned[t] ? cs : float2{1.f, 0.f};
  }
  __syncthreads();
  const int32_t per_token = (a.QH + a.KVH) * a.units;
  for (int32_t i = tid; i < tokens * per_token; i += kRotaryThreads) {
    const int32_t t = i / per_token, of = i - t * per_token, hh = of / a.units, u = of - hh * a.units;
    const bool key = hh >= a.QH;
    const int32_t h = key ? hh - a.QH : hh;
    const int64_t n = n0 + t;
    const uint8_t* from = key ? a.k + n * a.kst + h * a.ksh : a.q + n * a.qst + h * a.qsh;
    uint8_t* to = key ? a.k_out + n * a.kost + h * a.kosh : a.q_out + n * a.qost + h * a.qosh;
    // the unit's two vectors
    const bool turn = u < a.turned;
    const bool apart = !PAIRS_SIDE_BY_SIDE && turn;
    const int32_t d0 = apart ? u * VEC : 2 * u * VEC, d1 = apart ? d0 + half : d0 + VEC;
    Vec x = *(const Vec*)(from + d0 * (int)sizeof(T)), y = *(const Vec*)(from + d1 * (int)sizeof(T));
    if (turn) {
      const float2* cs = trig + t * half + u * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        // element 2e of the two vectors in turn, or element e of each
        T* p0 = PAIRS_SIDE_BY_SIDE ? (2 * e < VEC ? &x.x[2 * e < VEC ? 2 * e : 0] : &y.x[2 * e < VEC ? 0 : 2 * e - VEC]) : &x.x[e];
        T* p1 = PAIRS_SIDE_BY_SIDE ? (2 * e + 1 < VEC ? &x.x[2 * e + 1 < VEC ? 2 * e + 1 : 0] : &y.x[2 * e + 1 < VEC ? 0 : 2 * e + 1 - VEC])
                                   : &y.x[e];
        const float c = cs[e].x, s = cs[e].y;
        const float v = Elem<DT>::load(p0, 0), w = Elem<DT>::load(p1, 0);
        // (the empty asm keeps the 32-bit rounding: some widths' code would fuse the
        // product into the conversion)
        float lo = fmaf(v, c, -(w * s)), hi = fmaf(w, c, v * s);
        asm volatile("" : "+v"(lo), "+v"(hi));
        Elem<DT>::store(p0, 0, lo);
        Elem<DT>::store(p1, 0, hi);
      }
    }
    *(Vec*)(to + d0 * (int)sizeof(T)) = x;
    *(Vec*)(to + d1 * (int)sizeof(T)) = y;
  }
}

template <int DT, int VEC>
static void launch_rotary(const RotaryArgs& a, bool side_by_side, uint32_t lds, hipStream_t stream) {
  const dim3 grid((uint32_t)ceil_div(a.N, a.tokens)), block(kRotaryThreads);
  if (side_by_side) hipLaunchKernelGGL((rotary_kernel<DT, VEC, true>), grid, block, lds, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<DT, VEC, false>), grid, block, lds, stream, a);
}

}  // namespace jkv

extern "C" {

int jkv_rotary(const void* q, int64_t q_stride_t, int64_t q_stride_h, void* q_out, int64_t q_out_stride_t,
               int64_t q_out_stride_h, int64_t QH, const void* k, int64_t k_stride_t, int64_t k_stride_h, void* k_out,
               int64_t k_out_stride_t, int64_t k_out_stride_h, int64_t KVH, int32_t dtype, int64_t N, int64_t D,
               int64_t dims, int32_t side_by_side, const double* rates, double magnitude, int32_t inverse,
               const int32_t* starts, int64_t B, const int32_t* positions, jkv_stream_t stream_) {
  using namespace jkv;
  JKV_CHECK_ARG(dtype == JKV_F16 || dtype == JKV_BF16 || dtype == JKV_F32, "rotary takes fp16, bf16 or fp32, got dtype %d", dtype);
  JKV_CHECK_ARG(D > 0 && D <= kRotaryMost && D % 2 == 0, "rotary supports even head dims up to 256, got %lld", (long long)D);
  JKV_CHECK_ARG(dims > 0 && dims <= D && dims % 2 == 0, "the turned dims must be even and at most the head's, got %lld",
                (long long)dims);
  JKV_CHECK_ARG(N >= 0 && N < ((int64_t)1 << 30) && B >= 0 && B < ((int64_t)1 << 24), "too many rows or sequences");
  JKV_CHECK_ARG(QH >= 0 && KVH >= 0 && QH + KVH > 0 && QH + KVH < 65536, "invalid rotary heads");
  JKV_CHECK_ARG(rates, "null buffer");
  JKV_CHECK_ARG(isfinite(magnitude), "the magnitude must be finite");
  const int64_t size = dtype == JKV_F32 ? 4 : 2;
  const int64_t strides[8] = {q_stride_t, q_stride_h, q_out_stride_t, q_out_stride_h,
                              k_stride_t, k_stride_h, k_out_stride_t, k_out_stride_h};
  if (N == 0) return JKV_OK;
  JKV_CHECK_ARG((QH == 0 || (q && q_out)) && (KVH == 0 || (k && k_out)), "null buffer");
  RotaryArgs a = {};
  for (int64_t i = 0; i < dims / 2; ++i) {
    JKV_CHECK_ARG(isfinite(rates[i]), "rotary rates must be finite");
    a.turns[i] = rates[i] / 6.283185307179586476925286766559;
  }
  // the widest vectors that pairs, rows and strides allow, at most 16 bytes
  uintptr_t odd = 0;
  if (QH) odd |= (uintptr_t)q | (uintptr_t)q_out;
  if (KVH) odd |= (uintptr_t)k | (uintptr_t)k_out;
  for (int i = QH ? 0 : 4; i < (KVH ? 8 : 4); ++i) odd |= (uintptr_t)(strides[i] * size);
  JKV_CHECK_ARG(odd % size == 0, "rotary buffers must be aligned to their elements");
  int64_t vec = 16 / size;
  while (vec > 1 && (odd % (vec * size) || dims / 2 % vec || (D - dims) % (2 * vec))) vec /= 2;
  a.q = (const uint8_t*)q; a.q_out = (uint8_t*)q_out; a.k = (const uint8_t*)k; a.k_out = (uint8_t*)k_out;
  a.qst = q_stride_t * size; a.qsh = q_stride_h * size; a.qost = q_out_stride_t * size; a.qosh = q_out_stride_h * size;
  a.kst = k_stride_t * size; a.ksh = k_stride_h * size; a.kost = k_out_stride_t * size; a.kosh = k_out_stride_h * size;
  a.QH = (int32_t)QH; a.KVH = (int32_t)KVH; a.N = (int32_t)N; a.B = (int32_t)B; a.dims = (int32_t)dims;
  a.units = (int32_t)(D / (2 * vec)); a.turned = (int32_t)(dims / (2 * vec));
  a.starts = starts; a.positions = positions;
  a.magnitude = (float)magnitude; a.sign = inverse ? -1.f : 1.f;
  // a token's threads that work at once
  a.tokens = 1;
  while (a.tokens < 8 && a.tokens * (QH + KVH) * a.units < 2 * kRotaryThreads && ceil_div(N, 2 * a.tokens) >= 1024) a.tokens *= 2;
  const uint32_t lds = (uint32_t)(a.tokens * dims / 2 * sizeof(float2));
  JKV_CHECK_GRID(ceil_div(N, a.tokens), kRotaryThreads);
  hipStream_t stream = (hipStream_t)stream_;
  const bool side = side_by_side != 0;
  if (dtype == JKV_F32) {
    if (vec == 4) launch_rotary<JKV_F32, 4>(a, side, lds, stream);
    else if (vec == 2) launch_rotary<JKV_F32, 2>(a, side, lds, stream);
    else launch_rotary<JKV_F32, 1>(a, side, lds, stream);
  } else if (dtype == JKV_F16) {
    if (vec == 8) launch_rotary<JKV_F16, 8>(a, side, lds, stream);
    else if (vec == 4) launch_rotary<JKV_F16, 4>(a, side, lds, stream);
    else if (vec == 2) launch_rotary<JKV_F16, 2>(a, side, lds, stream);
    else launch_rotary<JKV_F16, 1>(a, side, lds, stream);
  } else {
    if (vec == 8) launch_rotary<JKV_BF16, 8>(a, side, lds, stream);
    else if (vec == 4) launch_rotary<JKV_BF16, 4>(a, side, lds, stream);
    else if (vec == 2) launch_rotary<JKV_BF16, 2>(a, side, lds, stream);
    else launch_rotary<JKV_BF16, 1>(a, side, lds, stream);
  }
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

}  // extern "C"
