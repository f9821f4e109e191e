// Gradients of the attention of packed sequences.
//
// With x the shaped score, p = exp(x - lse), delta_i = do_i o_i and s' the cap's
// slope at a score (1 without a cap):
//   dv_j = sum_i p_ij do_i        ds_ij = p_ij (do_i v_j - delta_i) s'_ij scale
//   dq_i = sum_j ds_ij k_j        dk_j = sum_i ds_ij q_i
// Three launches: the rows' delta and base-2 log-sum-exps; dk and dv, a workgroup
// a block of keys that walks the rows that see it, of all heads of the group in
// turn; dq, a workgroup a block of (token, head) rows that walks the keys.  Scores
// are formed in both walks: seven products in place of five, and no sum waits on
// another workgroup or on the order of atomics.
//
// p and ds enter their products rounded once to the inputs' type, p as 2^10 of
// itself (fp16 holds 2^-34 of it then), ds in fp16 times a power of two that keeps
// the largest that inputs of their sizes could give below 2^15.
//
// A masked weight is 0, but 0 times an infinite or NaN row is not: in tiles with
// masked places the second operands are read with such elements as 0.  Where they
// are seen, p or delta are not finite and carry it.
#pragma once

#include "chunk_attn.h"
#include "packed.h"

namespace jkv {

// max of |x| over the finite halves of w, 0 if there are none
template <int DT>
__device__ __forceinline__ float largest_finite(uint4v w, float most) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V8 V8;
  const V8 v = finite_part<DT>(__builtin_bit_cast(V8, w));
#pragma unroll
  for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf((float)v[e]));
  return most;
}

// Per row: delta, and the log-sum-exp as the walks take it.  Rows that no sequence
// owns get gradients of 0 here.
template <int DT, int D>
__global__ __launch_bounds__(256) void packed_rows_kernel(PackedGradArgs a) {
  typedef typename Half16<DT>::V8 V8;
  constexpr int kLanes = D / 8, kRows = 256 / kLanes;
  const int tid = threadIdx.x, part = tid % kLanes, r = tid / kLanes;
  int32_t lead = clamp_i32(a.starts[0], 0, a.N), from = clamp_i32(a.starts[a.B], 0, a.N);
  if (from < lead) from = lead;
  float most_d = 0.f, most_v = 0.f;
  const int64_t rows = (int64_t)a.N * a.QH, stride = (int64_t)gridDim.x * kRows;
  for (int64_t row = (int64_t)blockIdx.x * kRows + r; row < rows; row += stride) {
    const int32_t n = (int32_t)((uint32_t)row / (uint32_t)a.QH), head = (int32_t)(row - (int64_t)n * a.QH);
    if (n < lead || n >= from) {
      if (a.dq != nullptr) *(uint4v*)(a.dq + row * (2 * D) + 16 * part) = uint4v{0u, 0u, 0u, 0u};
      continue;
    }
    const uint4v dw = *(const uint4v*)(a.d + n * a.dst + head * a.dsh + 16 * part);
    const V8 d = __builtin_bit_cast(V8, dw), o = *(const V8*)(a.o + n * a.ost + head * a.osh + 16 * part);
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf((float)d[e], (float)o[e], sum);
    // (where one place holds most of a row's weight, do v and delta are near each
    // other: without the rest the gradients of bf16 rows are 3.6e-3 off, with it 2.5e-3)
    if (a.rest != nullptr) {
      const V8 rest = *(const V8*)(a.rest + row * (2 * D) + 16 * part);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf((float)d[e], (float)rest[e], sum);
    }
    if constexpr (DT == JKV_F16) most_d = largest_finite<DT>(dw, most_d);
#pragma unroll
    for (int off = kLanes / 2; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (part == 0) {
      const float lse = a.lse[row];
      // (a row that saw nothing weighs nothing)
      const int64_t at = (int64_t)head * a.N + n;
      a.lse2[at] = lse == -INFINITY ? INFINITY : fmaf(lse, 1.4426950408889634f, -10.f);
      a.minus_delta[at] = -sum;
    }
  }
  const int64_t kv_rows = (int64_t)a.N * a.KVH;
  if (DT == JKV_F16 || a.dk != nullptr || a.dv != nullptr)
    for (int64_t row = (int64_t)blockIdx.x * kRows + r; row < kv_rows; row += stride) {
      const int32_t n = (int32_t)((uint32_t)row / (uint32_t)a.KVH), head = (int32_t)(row - (int64_t)n * a.KVH);
      if (n < lead || n >= from) {
        if (a.dk != nullptr) *(uint4v*)(a.dk + row * (2 * D) + 16 * part) = uint4v{0u, 0u, 0u, 0u};
        if (a.dv != nullptr) *(uint4v*)(a.dv + row * (2 * D) + 16 * part) = uint4v{0u, 0u, 0u, 0u};
      } else if constexpr (DT == JKV_F16) {
        most_v = largest_finite<DT>(*(const uint4v*)(a.v + n * a.vst + head * a.vsh + 16 * part), most_v);
      }
    }
  if constexpr (DT == JKV_F16) {
    __shared__ float2 waves[4];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      most_d = fmaxf(most_d, __shfl_xor(most_d, off, 64));
      most_v = fmaxf(most_v, __shfl_xor(most_v, off, 64));
    }
    if ((tid & 63) == 0) waves[tid >> 6] = float2{most_d, most_v};
    __syncthreads();
    if (tid == 0)
      a.maxima[blockIdx.x] = float2{fmaxf(fmaxf(waves[0].x, waves[1].x), fmaxf(waves[2].x, waves[3].x)),
                                    fmaxf(fmaxf(waves[0].y, waves[1].y), fmaxf(waves[2].y, waves[3].y))};
  }
}

// The power of two that ds takes (with p's 2^10) so that it stays below 2^15:
// |do v - delta| is at most 2 D max|do| max|v|.
template <int DT, int D>
__device__ __forceinline__ float ds_factor(const PackedGradArgs& a) {
  if constexpr (DT != JKV_F16) return 1.f;
  const int lane = threadIdx.x & 63;
  float most_d = 0.f, most_v = 0.f;
#pragma unroll
  for (int i = 0; i < kGradBlocks / 64; ++i) {
    const float2 m = a.maxima[64 * i + lane];
    most_d = fmaxf(most_d, m.x);
    most_v = fmaxf(most_v, m.y);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    most_d = fmaxf(most_d, __shfl_xor(most_d, off, 64));
    most_v = fmaxf(most_v, __shfl_xor(most_v, off, 64));
  }
  const float most = 2.f * D * most_d * most_v;
  if (!(most > 0.f)) return 1.f;
  // (fp16 values: 2^-48 to 2^32 times 2^8)
  int e;
  frexpf(most, &e);  // most < 2^e
  return __uint_as_float((uint32_t)(127 + 5 - e) << 23);
}

// Blocks of `rows` of the sequences' rows times `per`: the sequence and block of
// an item, blocks in their order.
__device__ __forceinline__ bool packed_block(const PackedGradArgs& a, int32_t per, int32_t rows, int32_t item, int32_t* b, int32_t* block) {
  const int lane = threadIdx.x & 63;
  int32_t before = 0;
  for (int32_t b0 = 0; b0 < a.B; b0 += 64) {
    int32_t upto = 0;
    if (b0 + lane < a.B) {
      const int32_t row0 = clamp_i32(a.starts[b0 + lane], 0, a.N), tokens = clamp_i32(a.starts[b0 + lane + 1], row0, a.N) - row0;
      upto = (tokens * per + rows - 1) / rows;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int32_t up = __shfl_up(upto, off, 64);
      if (lane >= off) upto += up;
    }
    const int32_t all = __builtin_amdgcn_readlane(upto, 63);
    if (item < before + all) {
      const int at = __builtin_ctzll(__ballot(item < before + upto));
      *b = b0 + at;
      *block = item - before - (at > 0 ? __builtin_amdgcn_readlane(upto, at > 0 ? at - 1 : 0) : 0);
      return true;
    }
    before += all;
  }
  return false;
}

// A score's weight exponent and the cap's slope there.
template <int FORM>
__device__ __forceinline__ float shape_and_slant(const ScoreShape& s, float x, float distance, float* slant) {
  x *= s.mul;
  if constexpr (FORM & kFormCap) {
    const float r = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x));  // tanh = 1 - 2r
    *slant = 4.f * fmaf(-r, r, r);
    x = fmaf(s.twice, r, s.cap2);
  }
  if constexpr (FORM & kFormBias) x = fmaf(-s.slope2, fabsf(distance), x);
  return x;
}

// 32 rows of D elements into LDS, a wave's share of 8: row r's chunk j in slot
// chunk_both_slot(r, j).  Rows at or behind `left` land as zeros.
template <int D>
__device__ __forceinline__ void load_rows32(const uint8_t* base, int32_t left, uint32_t stride, uint32_t to, int wave, int lane) {
  constexpr int kRowBytes = 2 * D, kRowsPerLoad = 1024 / kRowBytes, kLoads = 8 / kRowsPerLoad;
  const uint32_t bytes = left > 0 ? (uint32_t)((left < 32 ? left : 32) - 1) * stride + kRowBytes : 0u;
  const uint64_t at = (uint64_t)base;
  const uint4v rsrc = {(uint32_t)__builtin_amdgcn_readfirstlane((int32_t)at), (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)(at >> 32)) & 0xffffu,
                       (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)bytes), 0x00020000u};
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int r = 8 * wave + j * kRowsPerLoad + lane / (64 / kRowsPerLoad), slot = lane % (64 / kRowsPerLoad);
    load_to_lds<16>(to + (uint32_t)(8 * wave * kRowBytes) + 1024u * j, (uint32_t)r * stride + 16u * (uint32_t)chunk_both_slot<D>(r, slot), rsrc);
  }
}

// dk and dv of 128 keys: a wave's 32 are columns of S = Q K^T and dP = dO V^T
// (v_mfma_f32_32x32x16; 16 of 32 rows a lane), and rows of dv += P^T dO and dk +=
// dS^T Q, which take P and dS from those registers and dO and Q by transposing
// reads in the same order.  Keys stay in registers, values in LDS, 32 rows of q and
// do of one head come a step ahead.
template <int DT, int D, int FORM>
__global__ __launch_bounds__(256, 2) void packed_kv_grad_kernel(PackedGradArgs a) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V8 V8;
  typedef typename Half16<DT>::V4 V4;
  typedef __attribute__((address_space(3))) const V8 lds_v8;
  typedef __attribute__((address_space(3))) const float4v lds_f4;
  constexpr int kSteps = D / 16, kDims = D / 32, kRowBytes = 2 * D, kTile = 32 * kRowBytes, kStage = 2 * kTile + 512;
  __shared__ __align__(1024) uint8_t lds[4 * kTile + 2 * kStage];  // values; twice rows of q, rows of do, their stats
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t at_item = blockIdx.x / (uint32_t)a.KVH;  // (kv heads fastest: each XCD has its own)
  const int32_t kvh = (int32_t)(blockIdx.x - at_item * (uint32_t)a.KVH);
  int32_t b, block;
  if (!packed_block(a, 1, 128, (int32_t)at_item, &b, &block)) return;
  b = __builtin_amdgcn_readfirstlane(b);
  block = __builtin_amdgcn_readfirstlane(block);
  const int32_t row0 = clamp_i32(a.starts[b], 0, a.N), T0 = clamp_i32(a.starts[b + 1], row0, a.N) - row0;
  const int32_t prefix = paged_prefix(a.prefixes, b, T0);
  const int32_t j0 = 128 * block, wj0 = j0 + 32 * wave;
  const uint32_t lds_base = lds_address(lds);

  // values into LDS, the wave's keys into registers (B operand: 8 dims of key ln)
#pragma unroll
  for (int w = 0; w < 4; ++w)
    load_rows32<D>(a.v + (int64_t)(row0 + j0 + 32 * w) * a.vst + (int64_t)kvh * a.vsh, T0 - j0 - 32 * w, (uint32_t)a.vst,
                   lds_base + w * kTile, wave, lane);
  V8 kf[kSteps];
  {
    const bool ok = wj0 + ln < T0;
    const uint8_t* kp = a.k + (int64_t)(row0 + (ok ? wj0 + ln : 0)) * a.kst + (int64_t)kvh * a.ksh + 16 * lh;
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      kf[c] = V8{};
      if (ok) kf[c] = *(const V8*)(kp + 32 * c);
    }
#pragma unroll
    for (int c = 0; c < kSteps; ++c) asm volatile("" : "+v"(kf[c]));  // waited for here
  }
  const float factor = ds_factor<DT, D>(a);

  // the rows that see some key of the block
  const int32_t i0 = prefix > j0 ? 0 : j0;
  int32_t i1 = T0;
  if (j0 >= a.sinks && (int64_t)j0 + 127 + a.window < i1) i1 = j0 + 127 + a.window;
  const int32_t tile0 = i0 / 32, tile1 = (i1 + 31) / 32;
  // steps: (row tile, head of the group), heads fastest
  auto load_step = [&](int32_t tile, int32_t g, int stage) {
    const int32_t head = kvh * a.per + g, left = T0 - 32 * tile;
    const int64_t n = row0 + 32 * tile;
    const uint32_t to = lds_base + 4 * kTile + stage * kStage;
    load_rows32<D>(a.q + n * a.qst + (int64_t)head * a.qsh, left, (uint32_t)a.qst, to, wave, lane);
    load_rows32<D>(a.d + n * a.dst + (int64_t)head * a.dsh, left, (uint32_t)a.dst, to + kTile, wave, lane);
    if (wave < 2) {
      const uint64_t at = (uint64_t)((wave == 0 ? a.lse2 : a.minus_delta) + (int64_t)head * a.N + n);
      const int32_t bytes = 4 * (left < 32 ? (left > 0 ? left : 0) : 32);
      const uint4v rsrc = {(uint32_t)__builtin_amdgcn_readfirstlane((int32_t)at), (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)(at >> 32)) & 0xffffu,
                           (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
      load_to_lds<4>(to + 2 * kTile + 256 * wave, 4u * (uint32_t)lane, rsrc);
    }
  };
  float16v dk[kDims], dv[kDims];
#pragma unroll
  for (int d = 0; d < kDims; ++d) {
    dk[d] = float16v{};
    dv[d] = float16v{};
  }
  // LDS addresses: rows as A operand (8 dims of row ln), transposed (4 of each of
  // two groups of 8 rows, dim ln); the rest are offsets known at compile time
  uint32_t row_at[kSteps], lo_at[kDims], hi_at[kDims];
#pragma unroll
  for (int c = 0; c < kSteps; ++c) row_at[c] = lds_base + (uint32_t)(ln * kRowBytes + 16 * chunk_both_slot<D>(ln, 2 * c + lh));
  const uint32_t v_wave = (uint32_t)(wave * kTile);
  const int tr_row = 4 * lh + ((lane & 15) >> 2), tr_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
  for (int d = 0; d < kDims; ++d) {
    lo_at[d] = lds_base + (uint32_t)(tr_row * kRowBytes + 16 * chunk_both_slot<D>(tr_row, 4 * d + tr_chunk) + 8 * (lane & 1));
    hi_at[d] = lds_base + (uint32_t)((tr_row + 8) * kRowBytes + 16 * chunk_both_slot<D>(tr_row + 8, 4 * d + tr_chunk) + 8 * (lane & 1));
  }
  auto transposed = [&](int d, uint32_t off) -> V8 {
    const V4 lo = lds_read_tr<V4>(lo_at[d] + off), hi = lds_read_tr<V4>(hi_at[d] + off);
    return V8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  const int32_t key = wj0 + ln;

  auto work = [&](int32_t tile, int32_t g, auto stage, auto masked) {
    constexpr bool MASKED = decltype(masked)::value;
    const uint32_t stage_at = 4 * kTile + (uint32_t)(stage * kStage);
    const int32_t head = kvh * a.per + g, t0 = 32 * tile;
    const ScoreShape shape = score_shape<FORM>(a, head);
    // row 8 q4 + 4 lh + e's statistics: of 16 rows a lane
    const uint32_t stats_at = lds_base + 16u * (uint32_t)lh + stage_at + 2 * kTile;
    float16v sc = {}, dp;  // dp starts from -delta
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const float4v d = *(lds_f4*)(size_t)(stats_at + 256 + 32 * q4);
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[4 * q4 + e] = d[e];
    }
#pragma unroll
    for (int c = 0; c < kSteps; ++c) sc = mfma32<DT>(*(lds_v8*)(size_t)(row_at[c] + stage_at), kf[c], sc);
#pragma unroll
    for (int c = 0; c < kSteps; ++c)
      dp = mfma32<DT>(*(lds_v8*)(size_t)(row_at[c] + stage_at + kTile), *(lds_v8*)(size_t)(row_at[c] + v_wave), dp);
    __builtin_amdgcn_sched_barrier(0);
    V8 pf[2], df[2];
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const float4v lse = *(lds_f4*)(size_t)(stats_at + 32 * q4);
      float4v poison;
      if constexpr (MASKED) poison = *(lds_f4*)(size_t)(stats_at + 256 + 32 * q4) * 0.f;
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int e = 4 * q4 + e4;
        const int32_t i = t0 + 8 * q4 + 4 * lh + e4;
        float slant = 1.f;
        float x = shape_and_slant<FORM>(shape, sc[e], (float)(i - key), &slant) - lse[e4];
        bool seen = true;
        if constexpr (MASKED) {
          seen = (key <= i || key < prefix) && (key > i - a.window || key < a.sinks) && i < T0;
          x = seen ? x : -INFINITY;
        }
        float p = __builtin_amdgcn_exp2f(x);
        float ds = p * dp[e];
        if constexpr (FORM & kFormCap) ds *= slant;
        if constexpr (DT == JKV_F16) ds *= factor;
        if constexpr (MASKED) {
          ds = seen ? ds : 0.f;
          p = seen ? p + poison[e4] : 0.f;  // (NaN where do is not finite)
        }
        pf[e >> 3][e & 7] = (T)p;
        df[e >> 3][e & 7] = (T)ds;
      }
      if (q4 == 1) __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        V8 dot = transposed(d, stage_at + kTile + 16 * st * kRowBytes), qt = transposed(d, stage_at + 16 * st * kRowBytes);
        if constexpr (MASKED) {
          dot = finite_part<DT>(dot);
          qt = finite_part<DT>(qt);
        }
        dv[d] = mfma32<DT>(pf[st], dot, dv[d]);
        dk[d] = mfma32<DT>(df[st], qt, dk[d]);
      }
    JKV_SG(0x100, 4);
    for (int x = 0; x < 2 * kDims - 1; ++x) { JKV_SG(0x100, 4); JKV_SG(0x8, 2); }
    JKV_SG(0x8, 2);
    __builtin_amdgcn_sched_barrier(0);
  };

  // Row tiles that all of the block's keys are seen by, [full0, full1), come last and
  // have code without masks (in one loop with the masked tiles' code, the compiler
  // keeps the sums in two places: 214 registers spilled).
  int32_t full0 = j0 + 128 <= prefix ? tile0 : j0 / 32 + 4, full1 = T0 / 32;
  if (j0 + 128 > a.sinks && (j0 + a.window) / 32 < full1) full1 = (j0 + a.window) / 32;
  if (full0 < tile0) full0 = tile0;
  if (full1 > tile1) full1 = tile1;
  if (j0 + 128 > T0 || full1 <= full0) full0 = full1 = tile1;
  const int32_t plain = (full1 - full0) * a.per, edge = tile1 > tile0 ? (tile1 - tile0) * a.per - plain : 0;
  struct Step { int32_t tile, g; };
  Step now = {tile0 == full0 ? full1 : tile0, 0};
  if (now.tile >= tile1) now.tile = full0;
  Step next = now;
  // heads of a tile in turn; tiles before the full ones, behind them, then those
  auto advance = [&](Step& s) {
    if (++s.g < a.per) return;
    s.g = 0;
    const bool in_full = s.tile >= full0 && s.tile < full1;
    ++s.tile;
    if (in_full) return;
    if (s.tile == full0) s.tile = full1;
    if (s.tile >= tile1) s.tile = full0;
  };
  int32_t left = edge + plain;  // steps not yet loaded
  // the step ahead into the other stage, once every load has landed and every LDS
  // access of the step before is done, in all waves
  auto turn_over = [&](int other) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (left > 0) {
      load_step(next.tile, next.g, other);
      advance(next);
      --left;
    }
  };
  if (left > 0) {
    load_step(next.tile, next.g, edge & 1);  // (so that the full tiles start in stage 0)
    advance(next);
    --left;
  }
  for (int32_t n = edge; n > 0; --n) {
    turn_over((n & 1) ^ 1);
    const int32_t t0 = 32 * now.tile;
    if (wj0 < T0 && (wj0 <= t0 + 31 || wj0 < prefix) && (wj0 + 31 > t0 - a.window || wj0 < a.sinks))
      work(now.tile, now.g, n & 1, std::true_type());
    advance(now);
  }
  for (int32_t n = 0; n < plain; n += 2) {
    turn_over(1);
    work(now.tile, now.g, std::integral_constant<int, 0>(), std::false_type());
    advance(now);
    if (n + 1 >= plain) break;
    turn_over(0);
    work(now.tile, now.g, std::integral_constant<int, 1>(), std::false_type());
    advance(now);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // lane holds dim 32d + ln of keys 8(e/4) + 4lh + e%4
  const float dv_mul = 0x1p-10f, dk_mul = a.scale * 0x1p-10f / factor;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int32_t j = wj0 + 8 * (e >> 2) + 4 * lh + (e & 3);
    if (j >= T0) continue;
    const int64_t at = ((int64_t)(row0 + j) * a.KVH + kvh) * D + ln;
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      if (a.dk != nullptr) ((T*)a.dk)[at + 32 * d] = (T)(dk[d][e] * dk_mul);
      if (a.dv != nullptr) ((T*)a.dv)[at + 32 * d] = (T)(dv[d][e] * dv_mul);
    }
  }
}

// dq of 128 (token, head) rows of a sequence and kv head, 32 a wave, as in the
// attention: S^T = K Q^T and dP^T = V dO^T leave a lane one row's places, dq^T +=
// K^T dS^T takes dS from those registers and K by transposing reads.
template <int DT, int D, int FORM>
__global__ __launch_bounds__(256, 2) void packed_q_grad_kernel(PackedGradArgs a) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V8 V8;
  typedef typename Half16<DT>::V4 V4;
  typedef __attribute__((address_space(3))) const V8 lds_v8;
  constexpr int kSteps = D / 16, kDims = D / 32, kRowBytes = 2 * D, kTile = 32 * kRowBytes;
  __shared__ __align__(1024) uint8_t lds[4 * kTile];  // twice 32 keys and values
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t at_item = blockIdx.x / (uint32_t)a.KVH;
  const int32_t kvh = (int32_t)(blockIdx.x - at_item * (uint32_t)a.KVH);
  int32_t b, block;
  if (!packed_block(a, a.per, 128, (int32_t)at_item, &b, &block)) return;
  b = __builtin_amdgcn_readfirstlane(b);
  block = __builtin_amdgcn_readfirstlane(block);
  const int32_t row0 = clamp_i32(a.starts[b], 0, a.N), T0 = clamp_i32(a.starts[b + 1], row0, a.N) - row0;
  const int32_t prefix = paged_prefix(a.prefixes, b, T0);
  const uint32_t per = (uint32_t)a.per;
  const int32_t R = T0 * a.per;
  block = (R + 127) / 128 - 1 - block;  // a sequence's last block first: it sees most
  const int32_t r0 = 128 * block, r1 = R - r0 > 128 ? r0 + 128 : R;
  const int32_t first = (int32_t)((uint32_t)r0 / per), last = (int32_t)((uint32_t)(r1 - 1) / per);
  const int32_t wr0 = r0 + 32 * wave, wr1 = wr0 + 32 < r1 ? wr0 + 32 : r1;
  const bool wave_on = wr0 < r1;
  const int32_t wfirst = wave_on ? (int32_t)((uint32_t)wr0 / per) : kPagedMost, wlast = wave_on ? (int32_t)((uint32_t)(wr1 - 1) / per) : -1;
  const bool row_ok = wr0 + ln < r1;
  const int32_t self = row_ok ? (int32_t)((uint32_t)(wr0 + ln) / per) : 0;
  const int32_t head = kvh * a.per + (row_ok ? wr0 + ln - self * a.per : 0);
  const int32_t reach = row_ok ? row_reach<FORM>(self, prefix) : -1;
  const uint32_t lds_base = lds_address(lds);

  const PagedTiles pt = paged_tiles(first, row_reach<FORM>(last, prefix), a.window, a.sinks, 32);
  auto entry_of = [&](int32_t i) { return (i < pt.lead ? i : pt.main + i - pt.lead) * 32; };
  auto load_step = [&](int32_t i, int stage) {
    const int32_t e0 = entry_of(i);
    const int64_t n = row0 + e0;
    load_rows32<D>(a.k + n * a.kst + (int64_t)kvh * a.ksh, T0 - e0, (uint32_t)a.kst, lds_base + 2 * stage * kTile, wave, lane);
    load_rows32<D>(a.v + n * a.vst + (int64_t)kvh * a.vsh, T0 - e0, (uint32_t)a.vst, lds_base + (2 * stage + 1) * kTile, wave, lane);
  };

  // the wave's queries and output gradients (B operands: 8 dims of row ln)
  V8 qf[kSteps], dof[kSteps];
  {
    const uint8_t* qp = a.q + (int64_t)(row0 + self) * a.qst + (int64_t)head * a.qsh + 16 * lh;
    const uint8_t* dp = a.d + (int64_t)(row0 + self) * a.dst + (int64_t)head * a.dsh + 16 * lh;
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      qf[c] = *(const V8*)(qp + 32 * c);
      dof[c] = *(const V8*)(dp + 32 * c);
    }
  }
  const float lse = a.lse2[(int64_t)head * a.N + row0 + self], minus_delta = a.minus_delta[(int64_t)head * a.N + row0 + self];
  const float factor = ds_factor<DT, D>(a);
  const ScoreShape shape = score_shape<FORM>(a, head);

  float16v dq[kDims];
#pragma unroll
  for (int d = 0; d < kDims; ++d) dq[d] = float16v{};
  uint32_t row_at[kSteps], lo_at[kDims], hi_at[kDims];
#pragma unroll
  for (int c = 0; c < kSteps; ++c) row_at[c] = lds_base + (uint32_t)(ln * kRowBytes + 16 * chunk_both_slot<D>(ln, 2 * c + lh));
  const int tr_row = 4 * lh + ((lane & 15) >> 2), tr_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
  for (int d = 0; d < kDims; ++d) {
    lo_at[d] = lds_base + (uint32_t)(tr_row * kRowBytes + 16 * chunk_both_slot<D>(tr_row, 4 * d + tr_chunk) + 8 * (lane & 1));
    hi_at[d] = lds_base + (uint32_t)((tr_row + 8) * kRowBytes + 16 * chunk_both_slot<D>(tr_row + 8, 4 * d + tr_chunk) + 8 * (lane & 1));
  }
  auto transposed = [&](int d, uint32_t off) -> V8 {
    const V4 lo = lds_read_tr<V4>(lo_at[d] + off), hi = lds_read_tr<V4>(hi_at[d] + off);
    return V8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto work = [&](int32_t e0, auto stage, auto masked) {
    constexpr bool MASKED = decltype(masked)::value;
    const uint32_t stage_at = (uint32_t)(stage * 2 * kTile);
    float16v sc = {}, dp = {};
#pragma unroll
    for (int c = 0; c < kSteps; ++c) sc = mfma32<DT>(*(lds_v8*)(size_t)(row_at[c] + stage_at), qf[c], sc);
#pragma unroll
    for (int c = 0; c < kSteps; ++c) dp = mfma32<DT>(*(lds_v8*)(size_t)(row_at[c] + stage_at + kTile), dof[c], dp);
    V8 df[2];
    const float at = (float)(e0 + 4 * lh - self);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float slant = 1.f;
      float x = shape_and_slant<FORM>(shape, sc[e], at + (float)(8 * (e >> 2) + (e & 3)), &slant) - lse;
      bool seen = true;
      if constexpr (MASKED) {
        const int32_t j = e0 + 8 * (e >> 2) + 4 * lh + (e & 3);
        seen = j <= reach && (j > self - a.window || j < a.sinks);
        x = seen ? x : -INFINITY;
      }
      float ds = __builtin_amdgcn_exp2f(x) * (dp[e] + minus_delta);
      if constexpr (FORM & kFormCap) ds *= slant;
      if constexpr (DT == JKV_F16) ds *= factor;
      if constexpr (MASKED) ds = seen ? ds : 0.f;
      df[e >> 3][e & 7] = (T)ds;
    }
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        V8 kt = transposed(d, stage_at + 16 * st * kRowBytes);
        if constexpr (MASKED) kt = finite_part<DT>(kt);
        dq[d] = mfma32<DT>(kt, df[st], dq[d]);
      }
  };
  // as above: the tiles that all rows see, [full0, full1), come last
  int32_t full1 = pt.lead + (row_reach<FORM>(first, prefix) + 1) / 32 - pt.main, full0 = pt.lead;
  if (last >= a.window && (last - a.window) / 32 + 1 > pt.main) full0 += (last - a.window) / 32 + 1 - pt.main;
  if (full1 > pt.count) full1 = pt.count;
  if (full1 <= full0) full0 = full1 = pt.count;
  const int32_t plain = full1 - full0, edge = pt.count - plain;
  int32_t now = full0 == 0 ? full1 : 0;
  if (now >= pt.count) now = full0;
  int32_t next = now, left = pt.count;
  auto advance = [&](int32_t& i) {
    const bool in_full = i >= full0 && i < full1;
    ++i;
    if (in_full) return;
    if (i == full0) i = full1;
    if (i >= pt.count) i = full0;
  };
  auto turn_over = [&](int other) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (left > 0) {
      load_step(next, other);
      advance(next);
      --left;
    }
  };
  if (left > 0) {
    load_step(next, edge & 1);
    advance(next);
    --left;
  }
  for (int32_t n = edge; n > 0; --n) {
    turn_over((n & 1) ^ 1);
    const int32_t e0 = entry_of(now);
    if (e0 <= row_reach<FORM>(wlast, prefix) && (e0 + 31 > wfirst - a.window || e0 < a.sinks)) work(e0, n & 1, std::true_type());
    advance(now);
  }
  for (int32_t n = 0; n < plain; n += 2) {
    turn_over(1);
    work(entry_of(now), std::integral_constant<int, 0>(), std::false_type());
    advance(now);
    if (n + 1 >= plain) break;
    turn_over(0);
    work(entry_of(now), std::integral_constant<int, 1>(), std::false_type());
    advance(now);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (!row_ok) return;
  // lane holds dims 32d + 8(e/4) + 4lh + e%4 of row ln
  const float mul = a.scale * 0x1p-10f / factor;
  uint8_t* to = a.dq + ((int64_t)(row0 + self) * a.QH + head) * kRowBytes;
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      V4 h;
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = (T)(dq[d][4 * q4 + e] * mul);
      *(V4*)(to + 2 * (32 * d + 8 * q4 + 4 * lh)) = h;
    }
}

template <int DT, int D, int FORM>
static int launch_grad(PackedGradArgs a, hipStream_t stream) {
  hipLaunchKernelGGL((packed_rows_kernel<DT, D>), dim3(kGradBlocks), dim3(256), 0, stream, a);
  auto blocks_of = [&](int64_t per) -> int64_t {
    const int64_t a1 = a.B * ceil_div((int64_t)a.N * per, 128), a2 = (int64_t)a.N * per / 128 + a.B;
    return (a1 < a2 ? a1 : a2) * a.KVH;
  };
  if ((a.dk != nullptr || a.dv != nullptr) && a.B > 0) {
    JKV_CHECK_GRID(blocks_of(1), 256);
    hipLaunchKernelGGL((packed_kv_grad_kernel<DT, D, FORM>), dim3((uint32_t)blocks_of(1)), dim3(256), 0, stream, a);
  }
  if (a.dq != nullptr && a.B > 0) {
    JKV_CHECK_GRID(blocks_of(a.per), 256);
    hipLaunchKernelGGL((packed_q_grad_kernel<DT, D, FORM>), dim3((uint32_t)blocks_of(a.per)), dim3(256), 0, stream, a);
  }
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

template <int DT>
static int launch_grad_form(const PackedGradArgs& a, int form, int64_t D, hipStream_t stream) {
  switch (form) {
    case kFormShaped: return D == 128 ? launch_grad<DT, 128, kFormShaped>(a, stream) : launch_grad<DT, 64, kFormShaped>(a, stream);
    case kFormShaped | kFormCap:
      return D == 128 ? launch_grad<DT, 128, kFormShaped | kFormCap>(a, stream) : launch_grad<DT, 64, kFormShaped | kFormCap>(a, stream);
    case kFormShaped | kFormBias:
      return D == 128 ? launch_grad<DT, 128, kFormShaped | kFormBias>(a, stream) : launch_grad<DT, 64, kFormShaped | kFormBias>(a, stream);
    default:
      return D == 128 ? launch_grad<DT, 128, kFormShaped | kFormCap | kFormBias>(a, stream)
                      : launch_grad<DT, 64, kFormShaped | kFormCap | kFormBias>(a, stream);
  }
}

}  // namespace jkv
