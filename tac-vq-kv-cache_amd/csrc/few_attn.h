// Attention over a paged K/V cache for sequences with few rows (tokens times
// query heads of a kv head, at most 32): single tokens above all.  FORM: what
// becomes of a score before its softmax.
//
// The bytes of the cache bound it.  One wave per (sequence, kv head, split of
// the entries): its rows are the columns of every product, so each key and
// value is read once for all heads of the group, whole rows at a time.  A tile
// of 32 entries waits in registers while the one before is worked on from
// 2 x 32 x D x 2 bytes of LDS of the wave's own, so waves share nothing and
// meet no barrier (where eight of them make a workgroup, they meet once, at its
// end), and four of them a CU hold 64 KiB of loads in flight.  16 sequences of
// 4,096 entries, 32/8 heads of 128: 55 us, 4.9 TB/s; four of up to 65,536: 115
// us, 4.8 TB/s (a large copy reaches 5.15).  Caps and biases hide behind the loads:
// 50 and 116 us with capped and with biased scores.
//
// On v_mfma_f32_16x16x32: S^T[entry][row] = K Q^T, O^T[dim][row] += V^T P^T
// (V^T by transposing reads of the row-major tile; the contraction order of
// P's accumulator layout, 4 entries of each of two groups of 16 a lane).  The
// matrix cores have time to spare here, so neither q nor p is rounded to 16
// bits: both enter as a sum of two (q = hi + lo, p = hi + lo), which leaves
// 32-bit scores and sums and the output's own rounding.  (Two bf16 parts hold a
// query to 2^-17: the weights are 2e-6 off, 7e-7 in fp16.  A third part took 1 to
// 3 % longer.)
#pragma once
#include <math.h>

#include <type_traits>

#include "paged.h"

namespace jkv {

static const int kFewTile = 32;

template <int DT>
__device__ __forceinline__ float4v mfma16(typename Half16<DT>::V8 a, typename Half16<DT>::V8 b, float4v c) {
  if constexpr (DT == JKV_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// max / sum over lanes l, l^16, l^32, l^48 by row swaps
__device__ __forceinline__ float lanes4_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float lanes4_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A part's factor against the largest maximum.  Never 0: a part may hold an
// infinite value (2^-149 of the largest finite one is 5e-7).
__device__ __forceinline__ float part_factor(float m, float top) { return fmaxf(__builtin_amdgcn_exp2f(m - top), 0x1p-149f); }

// Slot of 16-byte chunk j of row r in a tile: keys so that 16 rows' equal
// chunks, values so that 8 rows' equal chunk pairs, fall on distinct banks.
template <int D> __device__ __forceinline__ int key_slot(int r, int j) {
  return D == 128 ? j ^ (r & 15) : j ^ ((r >> 1) & 7);
}
template <int D> __device__ __forceinline__ int value_slot(int r, int j) {
  return D == 128 ? j ^ (2 * (r & 7)) : j ^ (2 * ((r >> 1) & 3));
}

template <int DT, int D, int RG, int W, int FORM = kFormPlain>
__global__ __launch_bounds__(64 * W, RG == 2 && D == 128 ? 1 : 2) void paged_few_kernel(PagedAttnArgs a) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V8 V8;
  typedef typename Half16<DT>::V4 V4;
  constexpr int kSteps = D / 32, kDims = D / 16, kRowBytes = 2 * D;
  constexpr int kRowsPerLoad = 1024 / kRowBytes, kLoads = kFewTile / kRowsPerLoad, kHalfLoads = kLoads / 2;
  __shared__ __align__(16) uint8_t lds[W][2 * kFewTile * kRowBytes];
  static_assert(2 * kFewTile * kRowBytes >= 16 * RG * D * 4, "a wave's sums fit its tile's room");
  __shared__ float2 ml_lds[W > 1 ? W : 1][W > 1 ? 16 * RG : 1];

  const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4;
  const int wave = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  uint8_t* const k_lds = lds[wave];
  uint8_t* const v_lds = lds[wave] + kFewTile * kRowBytes;
  const uint32_t bid = blockIdx.x;
  const uint32_t bh = bid / (uint32_t)a.splits;
  const int32_t split = (int32_t)(bid - bh * (uint32_t)a.splits);
  const int32_t b = (int32_t)(bh / (uint32_t)a.KVH), kvh = (int32_t)(bh - (uint32_t)b * (uint32_t)a.KVH);
  const PagedSeq s = paged_seq(a.c, b);
  const int32_t tokens = s.tokens < a.max_new ? s.tokens : a.max_new;
  if (tokens == 0) return;
  const int32_t R = tokens * a.per;  // <= 16 RG, as max_new * per is
  const int32_t first = s.length - s.tokens, last = first + tokens - 1;

  // what the rows see beside the entries up to their own (a row before the first
  // entry sees nothing)
  const int32_t prefix = FORM == kFormPlain ? 0 : paged_prefix(a.prefixes, b, s.length);
  auto reach = [&](int32_t i) { return FORM == kFormPlain || i < 0 || i >= prefix ? i : prefix - 1; };
  const PagedTiles pt = paged_tiles(first, reach(last), a.window, a.sinks, kFewTile);
  int32_t tile0 = split * a.split_tiles;
  int32_t tile1 = split == a.splits - 1 || tile0 + a.split_tiles > pt.count ? pt.count : tile0 + a.split_tiles;
  if constexpr (W > 1) {  // the workgroup's waves share them out
    const int32_t each = tile1 > tile0 ? (tile1 - tile0 + W - 1) / W : 0;
    tile0 += wave * each;
    if (tile0 + each < tile1) tile1 = tile0 + each;
  }

  // the lane's rows, one per row group
  int32_t row_t[RG], self[RG];
  bool row_ok[RG];
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    const int32_t r = 16 * g + ln;
    row_ok[g] = r < R;
    row_t[g] = (int32_t)((uint32_t)(row_ok[g] ? r : 0) / (uint32_t)a.per);
    self[g] = first + row_t[g];
  }
  auto packed_row = [&](int g) -> int64_t {  // n * QH + head
    const int32_t r = row_ok[g] ? 16 * g + ln : 0;
    return (int64_t)(s.row0 + row_t[g]) * a.QH + kvh * a.per + (r - row_t[g] * a.per);
  };

  float m[RG], l[RG];
  float4v o[RG][kDims];
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[g][d] = float4v{0.f, 0.f, 0.f, 0.f};
  }

  if (tile0 < tile1) {
    // ---- the queries as they are: their loads run beside the look-ups below ----
    V8 qx[RG][kSteps];
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      const int32_t r = row_ok[g] ? 16 * g + ln : 0;
      const uint8_t* qp = a.q + (int64_t)(s.row0 + row_t[g]) * a.qst +
                          (int64_t)(kvh * a.per + (r - row_t[g] * a.per)) * a.qsh;
#pragma unroll
      for (int c = 0; c < kSteps; ++c) qx[g][c] = *(const V8*)(qp + 64 * c + 16 * lg);
    }

    // ---- tile loader: 16-entry halves lie in one page (page sizes are multiples
    // of 16).  A page outside the pool and the entries at or behind the length
    // lie beyond the resource's bound and load as zeros. ----
    const int32_t* table = a.c.tables + b * a.c.table_stride;
    const int32_t mask = (1 << a.c.page_shift) - 1;
    const int lrow = lane / (64 / kRowsPerLoad), lchunk = lane % (64 / kRowsPerLoad);
    uint32_t voff[kHalfLoads];
#pragma unroll
    for (int i = 0; i < kHalfLoads; ++i) voff[i] = (uint32_t)(i * kRowsPerLoad + lrow) * (uint32_t)a.c.slot_bytes + 16u * lchunk;
    uint4v ks[kLoads], vs[kLoads];
    const uint8_t* k_head = a.c.k + kvh * a.c.head_bytes;
    const uint8_t* v_head = a.c.v + kvh * a.c.head_bytes;
    auto entry_of = [&](int32_t i) { return (i < pt.lead ? i : pt.main + i - pt.lead) * kFewTile; };
    // lane h holds the page of half h of a run of 32 tiles
    int32_t pages = -1, run0 = -32;
    auto look_up = [&](int32_t i) {
      run0 = i;
      const int32_t e = entry_of(i + (lane >> 1)) + 16 * (lane & 1);
      pages = -1;
      if (i + (lane >> 1) < tile1 && e < s.length) pages = table[e >> a.c.page_shift];
      if ((uint32_t)pages >= (uint32_t)a.c.n_pages) pages = -1;
    };
    auto fetch = [&](int32_t i) {
      const int32_t e0 = entry_of(i);
      if (i - run0 >= 32) look_up(i);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int32_t e = e0 + 16 * hf;
        const int32_t left = s.length - e;  // entries of this half that exist
        const int32_t page = __builtin_amdgcn_readlane(pages, 2 * (i - run0) + hf);
        const int64_t at = page >= 0 ? page * a.c.page_bytes + (int64_t)(e & mask) * a.c.slot_bytes : 0;
        const int32_t bytes = page >= 0 ? ((left < 16 ? left : 16) - 1) * (int32_t)a.c.slot_bytes + kRowBytes : 0;
        const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void*)(k_head + at), (short)0, bytes, 0x00020000);
        const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void*)(v_head + at), (short)0, bytes, 0x00020000);
#pragma unroll
        for (int j = 0; j < kHalfLoads; ++j) {
          ks[hf * kHalfLoads + j] = __builtin_bit_cast(uint4v, __builtin_amdgcn_raw_buffer_load_b128(kr, (int)voff[j], 0, 0));
          vs[hf * kHalfLoads + j] = __builtin_bit_cast(uint4v, __builtin_amdgcn_raw_buffer_load_b128(vr, (int)voff[j], 0, 0));
        }
      }
    };
    // every row sees the whole tile, or some entries are masked
    auto is_full = [&](int32_t e0) {
      return e0 + kFewTile - 1 <= reach(first) && (e0 > last - a.window || e0 + kFewTile <= a.sinks);
    };
    bool found = false;  // an infinite or NaN value in a tile that was staged without them
    auto stage = [&](bool full) {
      if (!full) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) vs[i] = finite_halves<DT>(vs[i], &found);
      }
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int r = i * kRowsPerLoad + lrow;
        *(uint4v*)(k_lds + r * kRowBytes + 16 * key_slot<D>(r, lchunk)) = ks[i];
        *(uint4v*)(v_lds + r * kRowBytes + 16 * value_slot<D>(r, lchunk)) = vs[i];
      }
    };
    fetch(tile0);

    // ---- the rotated queries, in two 16-bit parts (B operand: 8 dims of row ln) ----
    V8 qh[RG][kSteps], ql[RG][kSteps];
#pragma unroll
    for (int g = 0; g < RG; ++g) {
#pragma unroll
      for (int c = 0; c < kSteps / 2; ++c) {
        const int d0 = 32 * c + 8 * lg;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float u = (float)qx[g][c][e], w = (float)qx[g][c + kSteps / 2][e];
          if (a.rope.on) {
            float cs, sn;
            rope_trig(a.rope.turns[d0 + e], s.pos0 + row_t[g], &cs, &sn);
            const float t = u * cs - w * sn;
            w = w * cs + u * sn;
            u = t;
          }
          u = row_ok[g] ? u * a.q_mul : 0.f;
          w = row_ok[g] ? w * a.q_mul : 0.f;
          const T uh = (T)u, wh = (T)w;
          qh[g][c][e] = uh;
          ql[g][c][e] = (T)(u - (float)uh);
          qh[g][c + kSteps / 2][e] = wh;
          ql[g][c + kSteps / 2][e] = (T)(w - (float)wh);
        }
      }
    }

    const uint32_t v_base = lds_address(v_lds);
    const int tr_row = 4 * lg + (ln >> 2);
    auto value_operand = [&](int d) -> V8 {
      const uint32_t at = v_base + (uint32_t)(tr_row * kRowBytes + 16 * value_slot<D>(tr_row, 2 * d + ((ln & 3) >> 1)) + 8 * (ln & 1));
      const V4 lo = lds_read_tr<V4>(at), hi = lds_read_tr<V4>(at + 16u * kRowBytes);
      return V8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    // TRAILING_FINITE: infinite keys meet the queries' leading part alone
    auto scores = [&](float4v (&sc)[RG][2], auto trailing_finite) {
      constexpr bool TRAILING_FINITE = decltype(trailing_finite)::value;
#pragma unroll
      for (int kg = 0; kg < 2; ++kg) {
#pragma unroll
        for (int g = 0; g < RG; ++g) sc[g][kg] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          const int r = 16 * kg + ln;
          const V8 ka = *(const V8*)(k_lds + r * kRowBytes + 16 * key_slot<D>(r, 4 * c + lg));
          V8 kl = ka;
          if constexpr (TRAILING_FINITE) kl = finite_part<DT>(ka);
#pragma unroll
          for (int g = 0; g < RG; ++g) {
            sc[g][kg] = mfma16<DT>(ka, qh[g][c], sc[g][kg]);
            sc[g][kg] = mfma16<DT>(kl, ql[g][c], sc[g][kg]);
          }
        }
      }
    };
    ScoreShape shape[RG];
#pragma unroll
    for (int g = 0; g < RG; ++g)
      shape[g] = score_shape<FORM>(a, kvh * a.per + (row_ok[g] ? 16 * g + ln - row_t[g] * a.per : 0));
    const float scale2 = FORM == kFormPlain ? a.scale2 : 1.f;  // of scores as they are below
    bool again = false;
    for (;; again = true) {
      for (int32_t i = tile0; i < tile1; ++i) {
        const int32_t e0 = entry_of(i);
        const bool full = is_full(e0);
        stage(full && !again);
        if (i + 1 < tile1) fetch(i + 1);

        float4v sc[RG][2];
        scores(sc, std::false_type());
        if (again) scores(sc, std::true_type());
        V8 ph[RG], pl[RG];
#pragma unroll
        for (int g = 0; g < RG; ++g) {
          if constexpr (FORM != kFormPlain) {
            const float at = (float)(e0 + 4 * lg - self[g]);  // (distances below 2^24 are exact)
#pragma unroll
            for (int kg = 0; kg < 2; ++kg)
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[g][kg][e] = shape_score<FORM>(shape[g], sc[g][kg][e], at + (float)(16 * kg + e));
          }
          if (!full) {
#pragma unroll
            for (int kg = 0; kg < 2; ++kg)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int32_t j = e0 + 16 * kg + 4 * lg + e;
                const bool seen = j <= reach(self[g]) && (j > self[g] - a.window || j < a.sinks);
                sc[g][kg][e] = seen ? sc[g][kg][e] : -INFINITY;
              }
          }
          if (a.scores != nullptr && row_ok[g]) {
            float* to = a.scores + (((int64_t)b * a.KVH + kvh) * (a.max_new * a.per) + 16 * g + ln) * a.score_width + e0 + 4 * lg;
#pragma unroll
            for (int kg = 0; kg < 2; ++kg) *(float4v*)(to + 16 * kg) = sc[g][kg] * scale2;
          }
          float mx = -INFINITY;
#pragma unroll
          for (int kg = 0; kg < 2; ++kg)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[g][kg][e]);
          mx = lanes4_max(mx) * scale2;
          // the reference moves only when the maximum passes it by more than 4;
          // p is 2^10 times its weight against the reference, at most 2^14, so
          // that fp16 holds weights of 2^-34
          const float mn = mx > m[g] + 4.f ? mx : m[g], mu = mn == -INFINITY ? 0.f : mn - 10.f;
          const float alpha = m[g] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[g] - mn);
          if (__any(mn != m[g])) {
#pragma unroll
            for (int d = 0; d < kDims; ++d) o[g][d] *= alpha;
            l[g] *= alpha;
          }
          m[g] = mn;
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float p = __builtin_amdgcn_exp2f(fmaf(sc[g][e >> 2][e & 3], scale2, -mu));
            sum += p;
            const T hi = (T)p;
            ph[g][e] = hi;
            pl[g][e] = (T)(p - (float)hi);
          }
          l[g] += sum;
        }
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          const V8 va = value_operand(d);
#pragma unroll
          for (int g = 0; g < RG; ++g) {
            o[g][d] = mfma16<DT>(va, ph[g], o[g][d]);
            o[g][d] = mfma16<DT>(va, pl[g], o[g][d]);
          }
        }
      }
      // An infinite value times a weight's trailing part, or one that rounds to 0,
      // an infinite key times a query's trailing part: 0 times infinity or the other
      // infinity, NaN where there is a result.  What these go into is not finite, so
      // a walk that ends in finite sums needs no second.
      float odd = 0.f;
#pragma unroll
      for (int g = 0; g < RG; ++g) {
        odd = fmaf(l[g], 0.f, odd);
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) odd = fmaf(o[g][d][e], 0.f, odd);
      }
      if (again || !__any(odd != 0.f)) break;
#pragma unroll
      for (int g = 0; g < RG; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.f;
#pragma unroll
        for (int d = 0; d < kDims; ++d) o[g][d] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kSteps; ++c)  // (infinite queries have no trailing part)
#pragma unroll
          for (int e = 0; e < 8; ++e) ql[g][c][e] = __builtin_isfinite((float)qh[g][c][e]) ? ql[g][c][e] : (T)0.f;
      }
      look_up(tile0);
      fetch(tile0);
    }
    if (__any(found)) {
      for (int32_t i = tile0; i < tile1; ++i) {
        const int32_t e0 = entry_of(i);
        if (is_full(e0) && !again) continue;
        look_up(i);
        fetch(i);
        stage(true);  // as they are
        V8 seen[RG];
#pragma unroll
        for (int g = 0; g < RG; ++g)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int32_t j = e0 + 16 * (e >> 2) + 4 * lg + (e & 3);
            seen[g][e] = j <= reach(self[g]) && (j > self[g] - a.window || j < a.sinks) ? (T)1.f : (T)0.f;
          }
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          V8 vu, vd;
          non_finite_marks<DT>(value_operand(d), &vu, &vd);
#pragma unroll
          for (int g = 0; g < RG; ++g) {
            const float4v zero = {0.f, 0.f, 0.f, 0.f};
            const float4v up = mfma16<DT>(vu, seen[g], zero), down = mfma16<DT>(vd, seen[g], zero);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[g][d][e] = marked(o[g][d][e], up[e], down[e]);
          }
        }
      }
    }
  }

  // ---- out, or this split's part of it ----
  if constexpr (W > 1) {
    // the waves' sums meet in LDS, in the waves' order (such sequences are not split)
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      const float lt = lanes4_sum(l[g]);
      if (lg == 0) ml_lds[wave][16 * g + ln] = float2{m[g] == -INFINITY ? m[g] : m[g] - 10.f, lt};
#pragma unroll
      for (int d = 0; d < kDims; ++d)
        *(float4v*)(lds[wave] + ((16 * g + ln) * D + 16 * d + 4 * lg) * 4) = o[g][d];
    }
    __syncthreads();
    for (int32_t i = threadIdx.x; i < R * (D / 4); i += 64 * W) {
      const int32_t r = i / (D / 4), part = i % (D / 4);
      float top = -INFINITY, lt = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, ml_lds[w][r].x);
      float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 ml = ml_lds[w][r];
        if (ml.y == 0.f) continue;
        const float f = part_factor(ml.x, top);
        lt = fmaf(ml.y, f, lt);
        const float4v p = *(const float4v*)(lds[w] + (r * D + 4 * part) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(p[e], f, acc[e]);
      }
      const int32_t t = (int32_t)((uint32_t)r / (uint32_t)a.per), head = kvh * a.per + (r - t * a.per);
      const int64_t row = (int64_t)(s.row0 + t) * a.QH + head;
      const bool none = lt == 0.f;  // sees nothing
      if (part == 0) {
        const float l2 = none ? -INFINITY : (top == -INFINITY ? 0.f : top) + log2f(lt);
        if (a.lse != nullptr) a.lse[row] = l2 * 0.6931471805599453f;
        if (a.lse2 != nullptr) a.lse2[paged_lse2_at(a.c.N, a.per, row, a.QH)] = l2;
      }
      V4 h;
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = (T)(none ? 0.f : acc[e] / lt);
      *(V4*)(a.out + (int64_t)(s.row0 + t) * a.ost + (int64_t)head * a.osh + 8 * part) = h;
    }
    return;
  }
  // lane holds dims 16d + 4lg + e of row ln
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    const float lt = lanes4_sum(l[g]);
    if (!row_ok[g]) continue;
    const int64_t row = packed_row(g);
    if (a.splits > 1) {
      const int64_t at = (int64_t)split * a.c.N * a.QH + row;
      if (lg == 0) a.part_ml[at] = float2{m[g] == -INFINITY ? m[g] : m[g] - 10.f, lt};
      if (tile0 < tile1)
#pragma unroll
        for (int d = 0; d < kDims; ++d) *(float4v*)(a.part_o + at * D + 16 * d + 4 * lg) = o[g][d];
      continue;
    }
    const bool none = lt == 0.f;  // sees nothing
    if (lg == 0) {
      const float l2 = none ? -INFINITY : (m[g] == -INFINITY ? 0.f : m[g] - 10.f) + log2f(lt);
      if (a.lse != nullptr) a.lse[row] = l2 * 0.6931471805599453f;
      if (a.lse2 != nullptr) a.lse2[paged_lse2_at(a.c.N, a.per, row, a.QH)] = l2;
    }
    const float inv = 1.0f / lt;
    uint8_t* op = a.out + (int64_t)(s.row0 + row_t[g]) * a.ost + (row - (int64_t)(s.row0 + row_t[g]) * a.QH) * a.osh;
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      V4 h;
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = (T)(none ? 0.f : o[g][d][e] * inv);
      *(V4*)(op + 2 * (16 * d + 4 * lg)) = h;
    }
  }
}

template <int DT, int D, int FORM>
static int launch_few(const PagedAttnArgs& a, hipStream_t stream) {
  const int64_t blocks = (int64_t)a.c.B * a.KVH * a.splits;
  JKV_CHECK_GRID(blocks, 64 * a.waves);
  const dim3 grid((uint32_t)blocks);
  constexpr int W2 = D == 128 ? 4 : 8;
  if (a.max_new * a.per <= 16) {
    if (a.waves > 1) hipLaunchKernelGGL((paged_few_kernel<DT, D, 1, 8, FORM>), grid, dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((paged_few_kernel<DT, D, 1, 1, FORM>), grid, dim3(64), 0, stream, a);
  } else {
    if (a.waves > 1) hipLaunchKernelGGL((paged_few_kernel<DT, D, 2, W2, FORM>), grid, dim3(64 * W2), 0, stream, a);
    else hipLaunchKernelGGL((paged_few_kernel<DT, D, 2, 1, FORM>), grid, dim3(64), 0, stream, a);
  }
  if (a.splits > 1) {
    const int rc = paged_launch_join(a, DT, D, stream);
    if (rc != JKV_OK) return rc;
  }
  if (a.weights != nullptr) return paged_launch_few_weights(a, stream);
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

}  // namespace jkv
