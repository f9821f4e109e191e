// Gradients of the attention of packed sequences.
//
// With x the shaped score, p = exp(x - lse), delta_i = do_i o_i and s' the cap's
// slope at a score (1 without a cap):
//   dv_j = sum_i p_ij do_i        ds_ij = p_ij (do_i v_j - delta_i) s'_ij scale
//   dq_i = sum_j ds_ij k_j        dk_j = sum_i ds_ij q_i
// Three launches: the rows' delta and base-2 log-sum-exps; dk and dv, a workgroup
// a block of keys that walks the rows that see it, of all heads of the group in
// turn; dq, a workgroup a block of (token, head) rows that walks the keys.  A fourth
// joins the heads' sums where they were split.  Scores are formed in both walks, and ds
// has two parts: nine products in place of five, and no sum waits on another workgroup
// or on the order of atomics.
//
// 21,760 bf16 tokens of three texts, 32/8 heads of 128, capped scores, window 4,096
// (5.2e11 flops a product): rows 115 us (560 MB, 4.9 TB/s), dk and dv 2,510 (five
// products, 1,035 TFLOP/s), dq 1,945 (four, 1,070).  Products fill 57 and 59 % of their
// cycles, vector instructions 62 and 75, both at once 26 and 34; the clock falls to
// 1.77 GHz, so more of either at once brings less than it seems.  dk and dv read 5.8
// GB; walks that start at one place of the window for all blocks read 2.3 GB and took
// as long.  48 texts of up to 511 fp16 tokens, 28/4 heads of 64: 40, 128 and 123 us,
// vector instructions, and masked tiles at both ends of short walks.
//
// p enters its product rounded once to the inputs' type, as 2^10 of itself (fp16
// holds 2^-34 of it then): dv is 1.35 to 1.45 times as far off as its own rounding.  ds
// enters as a sum of two parts: a row's ds cancel, and one part's rounding left dq of
// sharp heads 1.5 to 1.9 times its own off and dk 1.4 to 1.55; with two 1.0 to 1.4 and
// 1.1 (the rest is delta's, from the rounded weights of the forward), for a product
// more in each walk.  In fp16 ds takes a power of two of its row (dq) or key (dk): from
// 2^64 on it falls as the largest ds passes 2^15, which then is 2^7 to 2^8, and the sums
// with it.  So it follows from what a row sees, or what sees a key, alone, and holds
// 2^-32 of the largest.
//
// A masked weight is 0, but 0 times an infinite or NaN row is not: whatever is not
// finite in a tile, seen or not, makes the sums so.  A walk that ends in finite sums
// needs no second; after another, the walk is made again with the masked p and ds
// selected, all tiles alike, the last products' operands with such elements as 0, and
// what they are added where they are seen: do's to dv with their sign, NaN for those of q
// and k (their scores are not finite: their ds is 0 or NaN).
#pragma once

#include <utility>

#include "chunk_attn.h"
#include "packed.h"

namespace jkv {

// f(0), f(1), .. f(N - 1), each with its number as a constant.
template <typename F, int... I> __device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F> __device__ __forceinline__ void each_to(F&& f) {
  each_of(f, std::make_integer_sequence<int, N>());
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
  const int64_t rows = (int64_t)a.N * a.QH, stride = (int64_t)gridDim.x * kRows;
  // (four rows' loads in flight)
  for (int64_t row0 = (int64_t)blockIdx.x * kRows + r; row0 < rows; row0 += 4 * stride) {
    V8 d[4], o[4], rest[4];
    int32_t n[4], head[4];
    bool on[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = row0 + i * stride;
      n[i] = (int32_t)((uint32_t)row / (uint32_t)a.QH);
      head[i] = (int32_t)(row - (int64_t)n[i] * a.QH);
      on[i] = row < rows && n[i] >= lead && n[i] < from;
      if (row < rows && !on[i] && a.dq != nullptr) *(uint4v*)(a.dq + row * (2 * D) + 16 * part) = uint4v{0u, 0u, 0u, 0u};
      d[i] = V8{};
      o[i] = V8{};
      rest[i] = V8{};
      if (!on[i]) continue;
      d[i] = *(const V8*)(a.d + n[i] * a.dst + head[i] * a.dsh + 16 * part);
      o[i] = __builtin_nontemporal_load((const V8*)(a.o + n[i] * a.ost + head[i] * a.osh + 16 * part));
      if (a.rest != nullptr) rest[i] = __builtin_nontemporal_load((const V8*)(a.rest + row * (2 * D) + 16 * part));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (where one place holds most of a row's weight, do v and delta are near each
      // other: without the rest the gradients of bf16 rows are 3.6e-3 off, with it 2.5e-3)
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf((float)d[i][e], (float)o[i][e], sum);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf((float)d[i][e], (float)rest[i][e], sum);
#pragma unroll
      for (int off = kLanes / 2; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
      if (on[i] && part == 0) {
        const float lse = a.lse[(int64_t)n[i] * a.QH + head[i]];
        // (a row that saw nothing weighs nothing)
        const int64_t at = (int64_t)head[i] * a.N + n[i];
        a.bases[at] = lse == -INFINITY ? -INFINITY : fmaf(lse, -1.4426950408889634f, 10.f + a.cap2);
        a.minus_delta[at] = -sum;
      }
    }
  }
  if (a.dk == nullptr && a.dv == nullptr) return;
  const int64_t kv_rows = (int64_t)a.N * a.KVH;
  for (int64_t row = (int64_t)blockIdx.x * kRows + r; row < kv_rows; row += stride) {
    const int32_t n = (int32_t)((uint32_t)row / (uint32_t)a.KVH);
    if (n >= lead && n < from) continue;
    if (a.dk != nullptr) *(uint4v*)(a.dk + row * (2 * D) + 16 * part) = uint4v{0u, 0u, 0u, 0u};
    if (a.dv != nullptr) *(uint4v*)(a.dv + row * (2 * D) + 16 * part) = uint4v{0u, 0u, 0u, 0u};
  }
}

// What ds takes in fp16 at first (with p's 2^10, 2^64: |do v - delta| of finite rows is
// below 2^41), and what brings it, `most` at the largest, to 2^7 to 2^8 once it has
// passed 2^15 (1 before, and where it is not finite).
static constexpr float kMostDs = 0x1p15f, kFirstDs = 0x1p54f;
__device__ __forceinline__ float ds_shrink(float most) {
  return most > kMostDs && most < INFINITY ? __builtin_amdgcn_ldexpf(1.f, 8 - __builtin_amdgcn_frexp_expf(most)) : 1.f;
}

// Of 64 sequences with `own` blocks in a lane's (`upto` of it and those before), the
// lane and rank (from a sequence's last block on) of the `item`-th (below their sum):
// all sequences' highest ranks first, as key blocks that are seen by many rows and
// start last are waited for by all CUs; where a sequence has more than 64, one sequence
// after another.  dk and dv of 48 texts of up to 511, 28/4 heads of 64, 131 -> 115 us,
// of three of up to 8,192, 32/8 of 128, window 4,096, 2,470 -> 2,350.  Row blocks (the
// attention's and dq's) are shorter and gain nothing, and prompts that see a prefix
// lose what they share of it in the caches (180 -> 214 us).
__device__ __forceinline__ int ranked_block(int32_t own, int32_t upto, int32_t item, int32_t* rank) {
  const int lane = threadIdx.x & 63;
  int32_t most = own;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const int32_t other = __shfl_xor(most, off, 64);
    most = other > most ? other : most;
  }
  most = __builtin_amdgcn_readfirstlane(most);
  if (most > 64) {
    const int at = __builtin_ctzll(__ballot(item < upto));
    *rank = __builtin_amdgcn_readlane(upto, at) - 1 - item;
    return at;
  }
  uint64_t have = 0;
  int32_t r = most;
  while (r > 0) {
    have = __ballot(own >= r);
    const int32_t count = __builtin_popcountll(have);
    --r;
    if (item < count) break;
    item -= count;
  }
  *rank = r;
  // the item-th of those that have one
  const bool is = (have >> lane & 1) && __builtin_popcountll(have & ((uint64_t{1} << lane) - 1)) == item;
  return __builtin_ctzll(__ballot(is));
}

// Blocks of `rows` of the sequences' rows times `per`: the sequence and block of
// an item, blocks in their order (RANKED: in that of ranked_block).
template <bool RANKED>
__device__ __forceinline__ bool packed_block(const PackedGradArgs& a, int32_t per, int32_t rows, int32_t item, int32_t* b, int32_t* block) {
  const int lane = threadIdx.x & 63;
  int32_t before = 0;
  for (int32_t b0 = 0; b0 < a.B; b0 += 64) {
    int32_t own = 0;
    if (b0 + lane < a.B) {
      const int32_t row0 = clamp_i32(a.starts[b0 + lane], 0, a.N), tokens = clamp_i32(a.starts[b0 + lane + 1], row0, a.N) - row0;
      own = (tokens * per + rows - 1) / rows;
    }
    int32_t upto = own;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int32_t up = __shfl_up(upto, off, 64);
      if (lane >= off) upto += up;
    }
    const int32_t all = __builtin_amdgcn_readlane(upto, 63);
    if (item < before + all) {
      if constexpr (RANKED) {
        int32_t rank;
        const int at = ranked_block(own, upto, item - before, &rank);
        *b = b0 + at;
        *block = __builtin_amdgcn_readlane(own, at) - 1 - rank;
      } else {
        const int at = __builtin_ctzll(__ballot(item < before + upto));
        *b = b0 + at;
        *block = item - before - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(own, at));
      }
      return true;
    }
    before += all;
  }
  return false;
}

// Of what shape_first left of a score: its weight's exponent, and a quarter of the
// cap's slope.  `base` is cap2 less the log-sum-exp.
template <int FORM>
__device__ __forceinline__ float shape_and_slant(const ScoreShape& s, float x, float distance, float base, float* slant) {
  if constexpr (FORM & kFormCap) {
    const float r = __builtin_amdgcn_rcpf(x);  // tanh = 1 - 2r
    *slant = fmaf(-r, r, r);
    x = fmaf(s.twice, r, base);
  } else {
    x = fmaf(x, s.mul, base);
  }
  if constexpr (FORM & kFormBias) x = fmaf(-s.slope2, fabsf(distance), x);
  return x;
}

// A resource of up to `most` rows of D elements, those at or behind `left` outside it.
// (One for all of a tile's loads: one a load is a hundred scalar instructions a step.)
template <int D>
__device__ __forceinline__ uint4v rows_resource(const uint8_t* base, int32_t left, int32_t most, uint32_t stride) {
  const int32_t rows = left < most ? left : most;
  const uint32_t bytes = rows > 0 ? (uint32_t)(rows - 1) * stride + 2 * D : 0u;
  const uint64_t at = (uint64_t)base;
  return uint4v{(uint32_t)__builtin_amdgcn_readfirstlane((int32_t)at), (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)(at >> 32)) & 0xffffu,
                (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)bytes), 0x00020000u};
}

// ROWS rows into LDS, row r's chunk j in slot chunk_both_slot(r, j), 16 rows (D = 128)
// or 32 a load of the four waves.  Rows at or behind `left` land as zeros.  Two groups
// of 16 rows share their slots, so one offset a lane serves both.
template <int D>
__device__ __forceinline__ uint32_t rows32_offset(uint32_t stride, int wave, int lane) {
  constexpr int kRowsPerLoad = 1024 / (2 * D);
  const int r = kRowsPerLoad * wave + lane / (64 / kRowsPerLoad), slot = lane % (64 / kRowsPerLoad);
  return (uint32_t)r * stride + 16u * (uint32_t)chunk_both_slot<D>(r, slot);
}
template <int D, int ROWS>
__device__ __forceinline__ void load_rows(const uint8_t* base, int32_t left, uint32_t stride, uint32_t offset, uint32_t to, int wave) {
  constexpr int kEach = 4096 / (2 * D);
  const uint4v rsrc = rows_resource<D>(base, left, ROWS, stride);
  asm volatile("" : "+v"(offset));  // (what is made from it is not kept)
#pragma unroll
  for (int j = 0; j < ROWS / kEach; ++j) load_to_lds<16>(to + 4096u * j + 1024u * (uint32_t)wave, offset + (uint32_t)(j * kEach) * stride, rsrc);
}

// 32 rows by one wave.
template <int D>
__device__ __forceinline__ void load_rows32_alone(const uint8_t* base, int32_t left, uint32_t stride, uint32_t to, int lane) {
  constexpr int kRowBytes = 2 * D, kEach = 1024 / kRowBytes;
  const int r = lane / (64 / kEach), slot = lane % (64 / kEach);
  uint32_t row = (uint32_t)r * stride, part = 16u * (uint32_t)chunk_both_slot<D>(r, slot);
  const uint4v rsrc = rows_resource<D>(base, left, 32, stride);
  asm volatile("" : "+v"(row), "+v"(part));
  // (row r + 4 or 8's slots)
#pragma unroll
  for (int j = 0; j < 32 / kEach; ++j)
    load_to_lds<16>(to + 1024u * j, row + (uint32_t)(j * kEach) * stride + (part ^ (D == 128 ? 16u * (j & 3) : 32u * (j & 1))), rsrc);
}

// A lane's LDS addresses in a tile of 32 rows.  Row ln's 16-byte chunk 2c + lh (an
// operand's 8 contracted places) is at rows ^ 32c; 4 elements of each of two groups
// of 8 rows, dim 32d + ln (transposing reads), at cols ^ 64d and, 8 rows on, at
// (cols ^ 64d ^ 32) + 8 rows.  Two registers held in place of sixteen: the others
// are made anew in every step.
struct TileAt {
  uint32_t rows, cols;
};
template <int D>
__device__ __forceinline__ TileAt tile_at(uint32_t lds_base, int lane) {
  constexpr int kRowBytes = 2 * D;
  const int ln = lane & 31, lh = lane >> 5, r = 4 * lh + ((lane & 15) >> 2), chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  return TileAt{lds_base + (uint32_t)(ln * kRowBytes + 16 * chunk_both_slot<D>(ln, lh)),
                lds_base + (uint32_t)(r * kRowBytes + 16 * chunk_both_slot<D>(r, chunk) + 8 * (lane & 1))};
}
template <int DT, int D>
__device__ __forceinline__ typename Half16<DT>::V8 read_rows(uint32_t rows, int c, uint32_t off) {
  typedef __attribute__((address_space(3))) const typename Half16<DT>::V8 lds_v8;
  return *(lds_v8*)(size_t)((rows ^ (uint32_t)(32 * c)) + off);
}
template <int DT, int D>
__device__ __forceinline__ typename Half16<DT>::V8 read_cols(uint32_t cols, int d, uint32_t off) {
  typedef typename Half16<DT>::V8 V8;
  typedef typename Half16<DT>::V4 V4;
  const V4 lo = lds_read_tr<V4>((cols ^ (uint32_t)(64 * d)) + off), hi = lds_read_tr<V4>((cols ^ (uint32_t)(64 * d + 32)) + (off + 16u * D));
  return V8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// How a walk takes a tile.
enum { kSeenInPart, kSeenWhole, kWalkedAgain };

// dk and dv of 128 keys: a wave's 32 are columns of S = Q K^T and dP = dO V^T
// (v_mfma_f32_32x32x16; 16 of 32 rows a lane), and rows of dv += P^T dO and dk +=
// dS^T Q, which take P and dS from those registers and dO and Q by transposing
// reads in the same order.  Keys stay in registers, values in LDS, 32 rows of q and
// do of one head come a step ahead.
//
// ALONE: 32 keys a workgroup, whose waves share out the steps, each with rows of
// its own, and add their sums up in LDS in the waves' order: a quarter of the chain
// where there are few keys or short texts.
template <int DT, int D, int FORM, bool ALONE>
__global__ __launch_bounds__(256, ALONE && D == 128 ? 1 : 2) void packed_kv_grad_kernel(PackedGradArgs a) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V8 V8;
  typedef __attribute__((address_space(3))) const float4v lds_f4;
  constexpr int kSteps = D / 16, kDims = D / 32, kRowBytes = 2 * D, kTile = 32 * kRowBytes, kStage = 2 * kTile + 512;
  constexpr int kKeys = ALONE ? 32 : 128, kValues = (kKeys / 32) * kTile, kStride = ALONE ? 4 : 1;
  // values; (each wave's) twice rows of q, rows of do, their stats
  __shared__ __align__(1024) uint8_t lds[kValues + (ALONE ? 4 : 1) * 2 * kStage];
  static_assert(2 * kStage >= 2 * 32 * D * 4, "a wave's sums fit its rows' room");
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t at_split = blockIdx.x / (uint32_t)a.KVH;  // (kv heads fastest: each XCD has its own)
  const int32_t kvh = (int32_t)(blockIdx.x - at_split * (uint32_t)a.KVH);
  const uint32_t at_item = ALONE ? at_split : at_split / (uint32_t)a.splits;
  const int32_t split = ALONE ? 0 : (int32_t)(at_split - at_item * (uint32_t)a.splits);
  // the heads of the group that it walks
  const int32_t g0 = split * a.heads_each, heads = a.per - g0 < a.heads_each ? a.per - g0 : a.heads_each;
  int32_t b, block;
  if (!packed_block<true>(a, 1, kKeys, (int32_t)at_item, &b, &block)) return;
  b = __builtin_amdgcn_readfirstlane(b);
  block = __builtin_amdgcn_readfirstlane(block);
  const int32_t row0 = clamp_i32(a.starts[b], 0, a.N), T0 = clamp_i32(a.starts[b + 1], row0, a.N) - row0;
  const int32_t prefix = paged_prefix(a.prefixes, b, T0);
  const int32_t j0 = kKeys * block, wj0 = ALONE ? j0 : j0 + 32 * wave;
  const uint32_t lds_base = lds_address(lds), stages_at = kValues + (ALONE ? (uint32_t)(wave * 2 * kStage) : 0u);

  // values into LDS, the wave's keys into registers (B operand: 8 dims of key ln)
#pragma unroll
  for (int w = 0; w < kKeys / 32; ++w)
    load_rows<D, 32>(a.v + (int64_t)(row0 + j0 + 32 * w) * a.vst + (int64_t)kvh * a.vsh, T0 - j0 - 32 * w, (uint32_t)a.vst,
                   rows32_offset<D>((uint32_t)a.vst, wave, lane), lds_base + w * kTile, wave);
  V8 kf[kSteps];
  {
    const bool ok = wj0 + ln < T0;
    const uint8_t* kp = a.k + (int64_t)(row0 + (ok ? wj0 + ln : 0)) * a.kst + (int64_t)kvh * a.ksh + 16 * lh;
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      kf[c] = V8{};
      if (ok) kf[c] = *(const V8*)(kp + 32 * c);
    }
  }

  // the rows that see some key of the block
  const int32_t i0 = prefix > j0 ? 0 : j0;
  int32_t i1 = T0;
  if (j0 >= a.sinks && (int64_t)j0 + kKeys - 1 + a.window < i1) i1 = j0 + kKeys - 1 + a.window;
  const int32_t tile0 = i0 / 32, tile1 = (i1 + 31) / 32;
  // steps: (row tile, head of the group), heads fastest
  const uint32_t q_off = rows32_offset<D>((uint32_t)a.qst, wave, lane), d_off = rows32_offset<D>((uint32_t)a.dst, wave, lane);
  auto load_step = [&](int32_t tile, int32_t g, int stage) {
    const int32_t head = kvh * a.per + g0 + g, left = T0 - 32 * tile;
    const int64_t n = row0 + 32 * tile;
    const uint32_t to = lds_base + stages_at + stage * kStage;
    const uint8_t* q_at = a.q + n * a.qst + (int64_t)head * a.qsh;
    const uint8_t* d_at = a.d + n * a.dst + (int64_t)head * a.dsh;
    if constexpr (ALONE) {
      load_rows32_alone<D>(q_at, left, (uint32_t)a.qst, to, lane);
      load_rows32_alone<D>(d_at, left, (uint32_t)a.dst, to + kTile, lane);
    } else {
      load_rows<D, 32>(q_at, left, (uint32_t)a.qst, q_off, to, wave);
      load_rows<D, 32>(d_at, left, (uint32_t)a.dst, d_off, to + kTile, wave);
    }
    const uint32_t bytes = 4u * (uint32_t)(left < 32 ? (left > 0 ? left : 0) : 32);
    auto load_stats = [&](const float* from, uint32_t at_to) {
      const uint64_t at = (uint64_t)(from + (int64_t)head * a.N + n);
      const uint4v rsrc = {(uint32_t)__builtin_amdgcn_readfirstlane((int32_t)at), (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)(at >> 32)) & 0xffffu,
                           (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)bytes), 0x00020000u};
      load_to_lds<4>(at_to, 4u * (uint32_t)lane, rsrc);
    };
    if (ALONE || wave == 0) load_stats(a.bases, to + 2 * kTile);
    if (ALONE || wave == 1) load_stats(a.minus_delta, to + 2 * kTile + 256);
  };
  float16v dk[kDims], dv[kDims];
#pragma unroll
  for (int d = 0; d < kDims; ++d) {
    dk[d] = float16v{};
    dv[d] = float16v{};
  }
  float factor = DT == JKV_F16 ? kFirstDs : 1.f;  // of the lane's key
  const TileAt tile_lane = tile_at<D>(lds_base, lane);
  const int32_t key = wj0 + ln;
  // rows [key_from, key_from + key_rows) see the lane's key
  const int32_t key_from = key < prefix ? 0 : key;
  int32_t key_upto = key >= a.sinks && key + a.window < T0 ? key + a.window : T0;
  const uint32_t key_rows = key_upto > key_from ? (uint32_t)(key_upto - key_from) : 0u;

  // dk times what the keys' lanes hold: sums are of key 8(e/4) + 4lh + e%4
  auto scale_keys = [&](float by) {
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
#pragma unroll
      for (int e = 4 * q4; e < 4 * q4 + 4; ++e) {
        const float of = __uint_as_float((uint32_t)__builtin_amdgcn_ds_bpermute(16 * lh + 4 * (8 * q4 + (e & 3)), (int)__float_as_uint(by)));
#pragma unroll
        for (int d = 0; d < kDims; ++d) dk[d][e] *= of;
      }
      __builtin_amdgcn_sched_barrier(0);  // (four at a time: all would take 16 registers)
    }
  };

  // A step's products in turn: S, dP, dv, dk, and beside each a few places' vector
  // instructions, fenced (the compiler else gathers each kind, and they overlap
  // little).  Operands are read two products ahead.
  auto work = [&](int32_t tile, int32_t g, auto stage, auto kind) {
    constexpr bool MASKED = decltype(kind)::value != kSeenWhole, AGAIN = decltype(kind)::value == kWalkedAgain;
    constexpr int kOps = 2 * kSteps + 4 * kDims;
    const uint32_t stage_at = stages_at + (uint32_t)(stage * kStage);
    const int32_t t0 = 32 * tile;
    const ScoreShape shape = score_shape<FORM>(a, kvh * a.per + g0 + g);
    const float at = (float)(t0 + 4 * lh - key);  // (distances below 2^24 are exact)
    uint32_t rows = tile_lane.rows, cols = tile_lane.cols;
    asm volatile("" : "+v"(rows), "+v"(cols));  // (what is made from them is not kept)
    const uint32_t v_rows = ALONE ? rows : rows + (uint32_t)(wave * kTile);
    // row 8 q4 + 4 lh + e's statistics: of 16 rows a lane
    const uint32_t stats_at = lds_base + 16u * (uint32_t)lh + stage_at + 2 * kTile;
    float16v sc = {}, dp;
    float4v bases[4];
    V8 pf[2], df[2], dl[2], ring[3], values[3];
    auto read = [&](int n) {
      if (n < kSteps) ring[n % 3] = read_rows<DT, D>(rows, n, stage_at);
      else if (n < 2 * kSteps) {
        ring[n % 3] = read_rows<DT, D>(rows, n - kSteps, stage_at + kTile);
        values[n % 3] = read_rows<DT, D>(v_rows, n - kSteps, 0);
      } else if (n < kOps) {
        const int m = (n - 2 * kSteps) % (2 * kDims);
        ring[n % 3] = read_cols<DT, D>(cols, m % kDims, stage_at + (n < 2 * kSteps + 2 * kDims ? kTile : 0) + 16 * (m / kDims) * kRowBytes);
      }
    };
    auto operand = [&](int n) -> V8 {
      if constexpr (AGAIN) return finite_part<DT>(ring[n % 3]);
      return ring[n % 3];
    };
    const uint32_t seen_at = (uint32_t)(t0 + 4 * lh - key_from);
    auto is_seen = [&](int e) { return seen_at + (uint32_t)(8 * (e >> 2) + (e & 3)) < key_rows; };
    auto read_bases = [&](int q4) { bases[q4] = *(lds_f4*)(size_t)(stats_at + 32 * q4); };
    auto first = [&](int e) { sc[e] = shape_first<FORM>(shape, sc[e]); };
    // p, and what ds takes of it (in sc)
    auto weigh = [&](int e) {
      float slant = 1.f;
      const float x = shape_and_slant<FORM>(shape, sc[e], at + (float)(8 * (e >> 2) + (e & 3)), bases[e >> 2][e & 3], &slant);
      float p = __builtin_amdgcn_exp2f(x);
      if constexpr (MASKED) p = is_seen(e) ? p : 0.f;
      pf[e >> 3][e & 7] = (T)p;
      if constexpr (FORM & kFormCap) p *= slant;
      if constexpr (DT == JKV_F16) p *= factor;
      sc[e] = p;
    };
    // ds (in dp), and its two parts
    auto lean = [&](int e) {
      dp[e] *= sc[e];
      if constexpr (AGAIN) dp[e] = is_seen(e) ? dp[e] : 0.f;
    };
    auto part = [&](int e) {
#pragma clang fp contract(off)  // (fused with ds's product in one kind of tile, it would differ in another)
      const T lead = (T)dp[e];
      df[e >> 3][e & 7] = lead;
      dl[e >> 3][e & 7] = (T)(dp[e] - (float)lead);
    };
    // the keys' factors less where a ds is too large for them
    auto fit = [&]() {
      float most = 0.f, other = 0.f;
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        most = fmaxf(fmaxf(most, fabsf(dp[e])), fabsf(dp[e + 1]));
        other = fmaxf(fmaxf(other, fabsf(dp[e + 2])), fabsf(dp[e + 3]));
      }
      most = fmaxf(most, other);
      if (__any(most > kMostDs)) {
        const float by = ds_shrink(lanes2_max(most));
        factor *= by;
        dp *= by;
        scale_keys(by);
      }
    };
    read(0);
    read(1);
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {  // dp starts from -delta
      const float4v d = *(lds_f4*)(size_t)(stats_at + 256 + 32 * q4);
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[4 * q4 + e] = d[e];
    }
    each_to<kOps>([&](auto number) {
      constexpr int n = decltype(number)::value;
      read(n + 2);
      if (n < kSteps) {
        sc = mfma32<DT>(ring[n % 3], kf[n], sc);
        if (n == kSteps - 2) { read_bases(0); read_bases(1); }
      } else if (n < 2 * kSteps) {
        constexpr int kFirst = 16 / kSteps, kWeigh = 8 / kSteps;
        const int c = n - kSteps;
        dp = mfma32<DT>(ring[n % 3], values[n % 3], dp);
#pragma unroll
        for (int e = c * kFirst; e < (c + 1) * kFirst; ++e) first(e);
        if (c > 0)
#pragma unroll
          for (int e = (c - 1) * kWeigh; e < c * kWeigh; ++e) weigh(e);
        if (c == kSteps - 1) {
#pragma unroll
          for (int e = c * kWeigh; e < 8; ++e) weigh(e);
          read_bases(2);
          read_bases(3);
        }
      } else {
        constexpr int kEach = 8 / kDims;
        constexpr int m = (n - 2 * kSteps) % (2 * kDims), d = m % kDims, st = m / kDims;
        if (n < 2 * kSteps + 2 * kDims) {
          dv[d] = mfma32<DT>(pf[st], operand(n), dv[d]);
#pragma unroll
          for (int e = d * kEach; e < (d + 1) * kEach; ++e) {
            if (st == 0) {
              weigh(8 + e);
            } else {
              lean(e);
              if constexpr (DT == JKV_F16) lean(8 + e);
              else part(e);
            }
          }
          if constexpr (DT == JKV_F16 && m == 2 * kDims - 1) {
            fit();
#pragma unroll
            for (int e = 0; e < 8; ++e) part(e);
          }
        } else {
          dk[d] = mfma32<DT>(df[st], operand(n), dk[d]);
          dk[d] = mfma32<DT>(dl[st], operand(n), dk[d]);
          if (st == 0)
#pragma unroll
            for (int e = d * kEach; e < (d + 1) * kEach; ++e) {
              if constexpr (DT != JKV_F16) lean(8 + e);
              part(8 + e);
            }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (AGAIN) {
      V8 seen[2];
#pragma unroll
      for (int e = 0; e < 16; ++e) seen[e >> 3][e & 7] = is_seen(e) ? (T)1.f : (T)0.f;
#pragma unroll
      for (int n = 0; n < 2 * kDims; ++n) {  // rows of do, then of q
        const int d = n % kDims;
        float16v up = {}, down = {};
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          V8 vu, vd;
          non_finite_marks<DT>(read_cols<DT, D>(cols, d, stage_at + (n < kDims ? kTile : 0) + 16 * st * kRowBytes), &vu, &vd);
          up = mfma32<DT>(seen[st], vu, up);
          down = mfma32<DT>(seen[st], vd, down);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (n < kDims) dv[d][e] = marked(dv[d][e], up[e], down[e]);
          else dk[d][e] = up[e] + down[e] > 0.f ? NAN : dk[d][e];
        }
      }
    }
  };

  // Row tiles that all of the block's keys are seen by, [full0, full1), come last and
  // have code without masks (in one loop with the masked tiles' code, the compiler
  // keeps the sums in two places: 214 registers spilled).
  int32_t full0 = j0 + kKeys <= prefix ? tile0 : (j0 + kKeys) / 32, full1 = T0 / 32;
  if (j0 + kKeys > a.sinks && (j0 + a.window) / 32 < full1) full1 = (j0 + a.window) / 32;
  if (full0 < tile0) full0 = tile0;
  if (full1 > tile1) full1 = tile1;
  if (j0 + kKeys > T0 || full1 <= full0) full0 = full1 = tile1;
  int32_t plain = (full1 - full0) * heads, edge = tile1 > tile0 ? (tile1 - tile0) * heads - plain : 0;
  struct Step { int32_t tile, g; };
  // heads of a tile in turn; tiles before the full ones and those behind them; full
  // ones from the last on, which all of a sequence's blocks see, so that they read
  // it at about the same time (8,192 causal bf16 tokens in one sequence, 32/8 heads:
  // 2,260 us from the first on)
  auto advance = [&](Step& s, int32_t by) {
    for (s.g += by; s.g >= heads; s.g -= heads)
      if (++s.tile == full0) s.tile = full1;
  };
  auto go_back = [&](Step& s, int32_t by) {
    for (s.g += by; s.g >= heads; s.g -= heads) --s.tile;
  };
  Step now = {tile0 == full0 ? full1 : tile0, 0}, first_plain = {full1 - 1, 0};
  constexpr auto kPart = std::integral_constant<int, kSeenInPart>();
  constexpr auto kWhole = std::integral_constant<int, kSeenWhole>();
  if constexpr (ALONE) {  // a wave's share: every fourth
    advance(now, wave);
    go_back(first_plain, wave);
    edge = (edge - wave + 3) / 4;
    plain = (plain - wave + 3) / 4;
  }
  const Step first_edge = now;
  Step next = now;
  int32_t loaded = 0;
  auto load_next = [&](int stage) {
    if (loaded == edge + plain) return;
    if (loaded == edge) next = first_plain;
    load_step(next.tile, next.g, stage);
    if (loaded < edge) advance(next, kStride);
    else go_back(next, kStride);
    ++loaded;
  };
  // the step ahead into the other stage, once every load has landed and every LDS
  // access of the step before is done, in all waves (that share the rows)
  auto turn_over = [&](int other) {
    if constexpr (ALONE) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    load_next(other);
  };
  load_next(edge & 1);  // (so that the full tiles start in stage 0)
#pragma unroll
  for (int c = 0; c < kSteps; ++c) asm volatile("" : "+v"(kf[c]));  // waited for here, with all loads before
  if constexpr (ALONE) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the values have landed
  auto is_on = [&](int32_t tile) {
    const int32_t t0 = 32 * tile;
    return wj0 < T0 && (wj0 <= t0 + 31 || wj0 < prefix) && (wj0 + 31 > t0 - a.window || wj0 < a.sinks);
  };
  for (int32_t n = edge; n > 0; --n) {
    turn_over((n & 1) ^ 1);
    if (is_on(now.tile)) work(now.tile, now.g, n & 1, kPart);
    advance(now, kStride);
  }
  now = first_plain;
  for (int32_t n = 0; n < plain; n += 2) {
    turn_over(1);
    work(now.tile, now.g, std::integral_constant<int, 0>(), kWhole);
    go_back(now, kStride);
    if (n + 1 >= plain) break;
    turn_over(0);
    work(now.tile, now.g, std::integral_constant<int, 1>(), kWhole);
    go_back(now, kStride);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // (see the head of this file; the same steps in the same order, a stage's loads
  // waited for)
  float odd = 0.f;
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) odd = fmaf(dv[d][e], 0.f, fmaf(dk[d][e], 0.f, odd));
  if (ALONE ? __any(odd != 0.f) : __syncthreads_or(odd != 0.f)) {
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      dk[d] = float16v{};
      dv[d] = float16v{};
    }
    if constexpr (DT == JKV_F16) factor = kFirstDs;
    auto meet = [&]() {
      if constexpr (ALONE) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    now = first_edge;
    for (int32_t n = 0; n < edge + plain; ++n) {
      if (n == edge) now = first_plain;
      meet();
      load_step(now.tile, now.g, 0);
      meet();
      if (is_on(now.tile)) work(now.tile, now.g, std::integral_constant<int, 0>(), std::integral_constant<int, kWalkedAgain>());
      if (n < edge) advance(now, kStride);
      else go_back(now, kStride);
    }
  }

  // lane holds dim 32d + ln of keys 8(e/4) + 4lh + e%4
  const float dv_mul = 0x1p-10f, dk_mul = a.scale * (FORM & kFormCap ? 4.f : 1.f) * 0x1p-10f;
  if constexpr (DT == JKV_F16) {
    scale_keys(1.f / factor);
  }
  if constexpr (ALONE) {
    __syncthreads();
    float* sums = (float*)(lds + kValues);  // [wave][dk, dv][dims / 32][e][lane]
    constexpr int kWave = 2 * kStage / 4;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        sums[wave * kWave + (16 * d + e) * 64 + lane] = dk[d][e];
        sums[wave * kWave + (16 * (kDims + d) + e) * 64 + lane] = dv[d][e];
      }
    __syncthreads();
#pragma unroll 4
    for (int i = wave; i < 32 * kDims; i += 4) {
      const bool value = i >= 16 * kDims;
      const int d = (i >> 4) % kDims, e = i & 15;
      const int32_t j = j0 + 8 * (e >> 2) + 4 * lh + (e & 3);
      const float* at = sums + i * 64 + lane;
      const float sum = (at[0] + at[kWave]) + (at[2 * kWave] + at[3 * kWave]);
      T* to = (T*)(value ? a.dv : a.dk);
      if (j < T0 && to != nullptr) to[((int64_t)(row0 + j) * a.KVH + kvh) * D + 32 * d + ln] = (T)(sum * (value ? dv_mul : dk_mul));
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int32_t j = wj0 + 8 * (e >> 2) + 4 * lh + (e & 3);
    if (j >= T0) continue;
    const int64_t at = ((int64_t)(row0 + j) * a.KVH + kvh) * D + ln;
    if (a.splits > 1) {
      const int64_t all = (int64_t)a.N * a.KVH * D;
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        a.part[2 * split * all + at + 32 * d] = dk[d][e] * dk_mul;
        a.part[(2 * split + 1) * all + at + 32 * d] = dv[d][e] * dv_mul;
      }
      continue;
    }
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      if (a.dk != nullptr) ((T*)a.dk)[at + 32 * d] = (T)(dk[d][e] * dk_mul);
      if (a.dv != nullptr) ((T*)a.dv)[at + 32 * d] = (T)(dv[d][e] * dv_mul);
    }
  }
}

// The splits' sums of dk (blockIdx.y 0) and dv added up, in their order.
template <int DT, int D>
__global__ __launch_bounds__(256) void packed_join_kernel(PackedGradArgs a) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V4 V4;
  const int64_t all = (int64_t)a.N * a.KVH * D, i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  T* to = (T*)(blockIdx.y == 0 ? a.dk : a.dv);
  if (i >= all || to == nullptr) return;
  const int64_t n = i / ((int64_t)a.KVH * D);
  if (n < a.starts[0] || n >= a.starts[a.B]) return;  // nobody's: 0 already
  float4v sum = __builtin_nontemporal_load((const float4v*)(a.part + blockIdx.y * all + i));
  for (int s = 1; s < a.splits; ++s) sum += __builtin_nontemporal_load((const float4v*)(a.part + (2 * s + blockIdx.y) * all + i));
  V4 h;
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = (T)sum[e];
  *(V4*)(to + i) = h;
}

// dq of 128 (token, head) rows of a sequence and kv head, 32 a wave, as in the
// attention: S^T = K Q^T and dP^T = V dO^T leave a lane one row's places, dq^T +=
// K^T dS^T takes dS from those registers and K by transposing reads.
template <int DT, int D, int FORM>
__global__ __launch_bounds__(256, 2) void packed_q_grad_kernel(PackedGradArgs a) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V8 V8;
  typedef typename Half16<DT>::V4 V4;
  constexpr int kSteps = D / 16, kDims = D / 32, kRowBytes = 2 * D, kTile = 64 * kRowBytes;
  __shared__ __align__(1024) uint8_t lds[4 * kTile];  // twice 64 keys and values
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t at_item = blockIdx.x / (uint32_t)a.KVH;
  const int32_t kvh = (int32_t)(blockIdx.x - at_item * (uint32_t)a.KVH);
  int32_t b, block;
  if (!packed_block<false>(a, a.per, 128, (int32_t)at_item, &b, &block)) return;
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

  const PagedTiles pt = paged_tiles(first, row_reach<FORM>(last, prefix), a.window, a.sinks, 64);
  auto entry_of = [&](int32_t i) { return (i < pt.lead ? i : pt.main + i - pt.lead) * 64; };
  const uint32_t k_off = rows32_offset<D>((uint32_t)a.kst, wave, lane), v_off = rows32_offset<D>((uint32_t)a.vst, wave, lane);
  auto load_step = [&](int32_t i, int stage) {
    const int32_t e0 = entry_of(i);
    const int64_t n = row0 + e0;
    const uint32_t to = lds_base + 2 * stage * kTile;
    load_rows<D, 64>(a.k + n * a.kst + (int64_t)kvh * a.ksh, T0 - e0, (uint32_t)a.kst, k_off, to, wave);
    load_rows<D, 64>(a.v + n * a.vst + (int64_t)kvh * a.vsh, T0 - e0, (uint32_t)a.vst, v_off, to + kTile, wave);
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
  // (lanes without a row weigh nothing)
  float base = row_ok ? a.bases[(int64_t)head * a.N + row0 + self] : -INFINITY;
  const float minus_delta = a.minus_delta[(int64_t)head * a.N + row0 + self];
  const float first_base = DT == JKV_F16 ? base + 54.f : base;
  base = first_base;
  float factor = DT == JKV_F16 ? kFirstDs : 1.f;  // what of base is ds's, of the lane's row
  const ScoreShape shape = score_shape<FORM>(a, head);

  // entries [seen_from, seen_from + seen_count) are seen, and those before `sunk`
  // more (counted from seen_from on)
  const int32_t seen_from = self >= a.window ? self - a.window + 1 : 0;
  const uint32_t seen_count = reach >= seen_from ? (uint32_t)(reach - seen_from + 1) : 0u;
  const int32_t sunk = row_ok ? (a.sinks < seen_from ? a.sinks : seen_from) - seen_from : -kPagedMost - 1;

  float16v dq[kDims];
#pragma unroll
  for (int d = 0; d < kDims; ++d) dq[d] = float16v{};
  const TileAt tile_lane = tile_at<D>(lds_base, lane);
  auto work = [&](int32_t e0, auto stage, auto kind) {
    constexpr bool MASKED = decltype(kind)::value != kSeenWhole, AGAIN = decltype(kind)::value == kWalkedAgain;
    const uint32_t stage_at = (uint32_t)(stage * 2 * kTile);
    uint32_t rows = tile_lane.rows, cols = tile_lane.cols;
    asm volatile("" : "+v"(rows), "+v"(cols));
    // S^T and dP^T of each half of 32 entries, then its part of dq; fenced as above
    constexpr int kOps = 4 * kSteps + 4 * kDims, kBoth = 2 * kSteps;
    float16v sc[2] = {}, dp[2] = {};
    V8 df[2][2], dl[2][2], ring[3];
    auto read = [&](int n) {
      if (n < 4 * kSteps) {
        const int half = n / kBoth, m = n % kBoth;
        ring[n % 3] = read_rows<DT, D>(rows, m % kSteps, stage_at + half * (kTile / 2) + (m < kSteps ? 0 : kTile));
      } else if (n < kOps) {
        const int m = n - 4 * kSteps;
        ring[n % 3] = read_cols<DT, D>(cols, m % kDims, stage_at + 16 * (m / kDims) * kRowBytes);
      }
    };
    const uint32_t seen_at = (uint32_t)(e0 + 4 * lh - seen_from);
    auto is_seen = [&](int half, int e) {  // entries of the window, or first ones before it
      const uint32_t from = seen_at + (uint32_t)(32 * half + 8 * (e >> 2) + (e & 3));
      return from < seen_count || (int32_t)from < sunk;
    };
    const float at = (float)(e0 + 4 * lh - self);
    auto first = [&](int half, int e) { sc[half][e] = shape_first<FORM>(shape, sc[half][e]); };
    auto weigh = [&](int half, int e) {
      float slant = 1.f;
      const float x = shape_and_slant<FORM>(shape, sc[half][e], at + (float)(32 * half + 8 * (e >> 2) + (e & 3)), base, &slant);
      float p = __builtin_amdgcn_exp2f(x);
      if constexpr (MASKED) p = is_seen(half, e) ? p : 0.f;
      if constexpr (FORM & kFormCap) p *= slant;
      sc[half][e] = p;
    };
    auto part = [&](int half, int e) {
#pragma clang fp contract(off)
      const T lead = (T)dp[half][e];
      df[half][e >> 3][e & 7] = lead;
      dl[half][e >> 3][e & 7] = (T)(dp[half][e] - (float)lead);
    };
    auto lean = [&](int half, int e) {
      dp[half][e] = sc[half][e] * (dp[half][e] + minus_delta);
      if constexpr (AGAIN) dp[half][e] = is_seen(half, e) ? dp[half][e] : 0.f;
      if constexpr (DT != JKV_F16) part(half, e);
    };
    // 8 places' ds in parts, the rows' factors less where they are too large
    auto fit = [&](int half, int st) {
      float most = 0.f;
#pragma unroll
      for (int e = 8 * st; e < 8 * st + 8; e += 2) most = fmaxf(fmaxf(most, fabsf(dp[half][e])), fabsf(dp[half][e + 1]));
      if (__any(most > kMostDs)) {
        const float by = ds_shrink(lanes2_max(most));
        factor *= by;
        base = first_base + (float)(__builtin_amdgcn_frexp_expf(factor) - 55);
#pragma unroll
        for (int e = 8 * st; e < 8 * st + 8; ++e) dp[half][e] *= by;
        // what was weighed and not leaned yet, and what waits for its product
        if (st == 0)
#pragma unroll
          for (int e = 8; e < 16; ++e) sc[half][e] *= by;
        if (half == 0 && st == 1)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            df[0][0][e] = (T)((float)df[0][0][e] * by);
            dl[0][0][e] = (T)((float)dl[0][0][e] * by);
          }
#pragma unroll
        for (int d = 0; d < kDims; ++d) dq[d] *= by;
      }
#pragma unroll
      for (int e = 8 * st; e < 8 * st + 8; ++e) part(half, e);
    };
    read(0);
    read(1);
    each_to<kOps>([&](auto number) {
      constexpr int n = decltype(number)::value;
      constexpr int kEach = 16 / kSteps, kBeside = 8 / kDims;
      read(n + 2);
      if (n < 4 * kSteps) {
        constexpr int half = n / kBoth, m = n % kBoth, c = m % kSteps;
        if (m < kSteps) sc[half] = mfma32<DT>(ring[n % 3], qf[c], sc[half]);
        else dp[half] = mfma32<DT>(ring[n % 3], dof[c], dp[half]);
#pragma unroll
        for (int e = c * kEach; e < (c + 1) * kEach; ++e) {
          if (m >= kSteps) first(half, e);
          if (half == 1 && m < kSteps) weigh(0, e);
          if (half == 1 && m >= kSteps) lean(0, e);
        }
        if constexpr (DT == JKV_F16 && half == 1 && m >= kSteps && (c + 1) * kEach % 8 == 0) fit(0, (c + 1) * kEach / 8 - 1);
      } else {
        constexpr int m = n - 4 * kSteps, d = m % kDims, st = m / kDims;
        V8 keys = ring[n % 3];
        if constexpr (AGAIN) keys = finite_part<DT>(keys);
        dq[d] = mfma32<DT>(keys, df[st / 2][st % 2], dq[d]);
        dq[d] = mfma32<DT>(keys, dl[st / 2][st % 2], dq[d]);
#pragma unroll
        for (int e = d * kBeside; e < (d + 1) * kBeside; ++e) {
          if (st == 0) weigh(1, e);
          if (st == 1) { weigh(1, 8 + e); lean(1, e); }
          if (st == 2) lean(1, 8 + e);
        }
        if constexpr (DT == JKV_F16 && (st == 1 || st == 2) && d == kDims - 1) fit(1, st - 1);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (AGAIN) {
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        float16v some = {};
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          V8 vu, vd, seen;
#pragma unroll
          for (int e = 0; e < 8; ++e) seen[e] = is_seen(st / 2, 8 * (st % 2) + e) ? (T)1.f : (T)0.f;
          non_finite_marks<DT>(read_cols<DT, D>(cols, d, stage_at + 16 * st * kRowBytes), &vu, &vd);
          some = mfma32<DT>(vu, seen, some);
          some = mfma32<DT>(vd, seen, some);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[d][e] = some[e] > 0.f ? NAN : dq[d][e];
      }
    }
  };
  // as above: the tiles that all rows see, [full0, full1), come last
  int32_t full1 = pt.lead + (row_reach<FORM>(first, prefix) + 1) / 64 - pt.main, full0 = pt.lead;
  if (last >= a.window && (last - a.window) / 64 + 1 > pt.main) full0 += (last - a.window) / 64 + 1 - pt.main;
  if (full1 > pt.count) full1 = pt.count;
  if (full1 <= full0) full0 = full1 = pt.count;
  const int32_t plain = full1 - full0, edge = pt.count - plain;
  int32_t now = full0 == 0 ? full1 : 0;
  if (now >= pt.count) now = full0;
  const int32_t start = now;
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
  auto is_on = [&](int32_t e0) { return e0 <= row_reach<FORM>(wlast, prefix) && (e0 + 63 > wfirst - a.window || e0 < a.sinks); };
  for (int32_t n = edge; n > 0; --n) {
    turn_over((n & 1) ^ 1);
    const int32_t e0 = entry_of(now);
    if (is_on(e0)) work(e0, n & 1, std::integral_constant<int, kSeenInPart>());
    advance(now);
  }
  constexpr auto kWhole = std::integral_constant<int, kSeenWhole>();
  for (int32_t n = 0; n < plain; n += 2) {
    turn_over(1);
    work(entry_of(now), std::integral_constant<int, 0>(), kWhole);
    advance(now);
    if (n + 1 >= plain) break;
    turn_over(0);
    work(entry_of(now), std::integral_constant<int, 1>(), kWhole);
    advance(now);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  float odd = 0.f;  // as above
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) odd = fmaf(dq[d][e], 0.f, odd);
  if (__syncthreads_or(row_ok && odd != 0.f)) {
#pragma unroll
    for (int d = 0; d < kDims; ++d) dq[d] = float16v{};
    base = first_base;
    if constexpr (DT == JKV_F16) factor = kFirstDs;
    auto meet = [&]() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    now = start;
    for (int32_t n = 0; n < pt.count; ++n) {
      const int32_t e0 = entry_of(now);
      meet();
      load_step(now, 0);
      meet();
      if (is_on(e0)) work(e0, std::integral_constant<int, 0>(), std::integral_constant<int, kWalkedAgain>());
      advance(now);
    }
  }
  if (!row_ok) return;
  // lane holds dims 32d + 8(e/4) + 4lh + e%4 of row ln
  const float mul = a.scale * (FORM & kFormCap ? 4.f : 1.f) * 0x1p-10f / factor;
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
  auto blocks_of = [&](int64_t per, int64_t rows) -> int64_t {
    const int64_t a1 = a.B * ceil_div((int64_t)a.N * per, rows), a2 = (int64_t)a.N * per / rows + a.B;
    return (a1 < a2 ? a1 : a2) * a.KVH;
  };
  if ((a.dk != nullptr || a.dv != nullptr) && a.B > 0) {
    const int64_t blocks = blocks_of(1, a.alone ? 32 : 128) * a.splits;
    JKV_CHECK_GRID(blocks, 256);
    const dim3 grid((uint32_t)blocks);
    if (a.alone) hipLaunchKernelGGL((packed_kv_grad_kernel<DT, D, FORM, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((packed_kv_grad_kernel<DT, D, FORM, false>), grid, dim3(256), 0, stream, a);
    if (a.splits > 1) {
      const int64_t joins = ceil_div((int64_t)a.N * a.KVH * D, 1024);
      JKV_CHECK_GRID(joins, 256);
      hipLaunchKernelGGL((packed_join_kernel<DT, D>), dim3((uint32_t)joins, 2), dim3(256), 0, stream, a);
    }
  }
  if (a.dq != nullptr && a.B > 0) {
    JKV_CHECK_GRID(blocks_of(a.per, 128), 256);
    hipLaunchKernelGGL((packed_q_grad_kernel<DT, D, FORM>), dim3((uint32_t)blocks_of(a.per, 128)), dim3(256), 0, stream, a);
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
