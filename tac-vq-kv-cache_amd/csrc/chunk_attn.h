// Attention of chunks of new tokens over a paged K/V cache, or of whole
// sequences that lie one behind another without pages.
//
// The matrix products bound it.  The packed (token, query head) rows of a
// sequence and kv head go 128 or 256 to a workgroup, 32 rows a wave, so any
// number of heads shares the keys and values of its group.  Tiles of 64
// entries lie twice in LDS (keys and values 4 x 64 x D x 2 bytes), loaded
// there directly a tile ahead.
//
// On v_mfma_f32_32x32x16, S^T[entry][row] = K Q^T gives a lane one row's
// scores (16 of 32 entries, the other half-wave the rest): a row's maximum and
// sum take one swap.  O^T[dim][row] += V^T P^T takes P from those registers,
// 4 entries of each of two groups of 8 a lane, and V^T by transposing reads of
// the row-major tile in the same order.  Online softmax in 32 bits; p and the
// rotated, scaled q enter the products rounded once to the cache's type: up to
// 2^-8 of a bf16 weight and of a score's terms.  The output is 0.30 % off where
// its own rounding alone is 0.17 % (fp16 0.041 and 0.021).  A second part of q
// would bring 0.23 % for half as many products again: 2 x 2,048 bf16 tokens over
// 16,384 entries 894 -> 1,200 us, ragged fp16 chunks of 777 62 -> 72; one of p
// too, the output's own rounding for twice the products.  With EXACT, where weights
// or log-sum-exps are asked for (they would show it), q is a sum of two parts.
//
// 2 x 2,048 bf16 tokens over 16,384 entries, 32/8 heads of 128: 852 to 892 us on
// different cards, 1.15 to 1.21 PFLOP/s (a large matrix product reaches 1.26 to
// 1.30).  Of its cycles the products fill 61 %, vector instructions 46 %, both at
// once 22 %, and the products' power holds the clock at 1.76 GHz.  Measured
// without gain: three and four stages of tiles, wave priorities around the
// products, the next tile's loads behind the scores (1,720 us: they take a whole
// tile's time to come).
//
// FORM says what becomes of a score (kFormPlain: nothing but its scale, and no
// prefix): kFormShaped allows prefixes that all rows see, kFormCap bends scores by
// a tanh, kFormBias takes a slope times the distance off.  Shaped scores leave the
// products as they are and are scaled, bent and biased in 32 bits, so their queries
// enter the products as they came, or rounded once after their rotation.
#pragma once
#include <math.h>

#include <type_traits>

#include "paged.h"

namespace jkv {

#define JKV_SG(what, n) __builtin_amdgcn_sched_group_barrier(what, n, 0)

static const int kChunkTile = 64;

// sum + a + b in 32 bits (ones times both)
template <int DT>
__device__ __forceinline__ float add_pair(typename Half16<DT>::T a, typename Half16<DT>::T b, float sum) {
  if constexpr (DT == JKV_F16) {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(half2v{a, b}, half2v{(_Float16)1.f, (_Float16)1.f}, sum, false);
  } else {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(bf16x2{a, b}, bf16x2{(__bf16)1.f, (__bf16)1.f}, sum, false);
  }
}

template <int DT>
__device__ __forceinline__ float16v mfma32(typename Half16<DT>::V8 a, typename Half16<DT>::V8 b, float16v c) {
  if constexpr (DT == JKV_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// max / sum over lanes l and l^32
__device__ __forceinline__ float lanes2_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float lanes2_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// BYTES a lane from the resource's `off` into LDS at `to` and on, lane after lane.
// (Asm: for the builtin the compiler holds every LDS read back until all loads
// have landed.  There are no result registers, and the callers' waits count these
// loads.  M0 holds their place in LDS; a register that the compiler reserves
// cannot be declared as changed, so it is left as it was.)
template <int BYTES>
__device__ __forceinline__ void load_to_lds(uint32_t to, uint32_t off, uint4v rsrc) {
  static_assert(BYTES == 4 || BYTES == 16, "one or four words a lane");
  uint32_t m0;
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "s"(to), "v"(off), "s"(rsrc) : "memory");
  else
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dword %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "s"(to), "v"(off), "s"(rsrc) : "memory");
}

// Slot of 16-byte chunk j of row r in a tile: keys so that 16 rows' equal
// chunks, values so that 4 rows' 64-byte groups, fall on distinct banks.
template <int D> __device__ __forceinline__ int chunk_key_slot(int r, int j) {
  return D == 128 ? j ^ (r & 15) : j ^ ((r >> 1) & 7);
}
template <int D> __device__ __forceinline__ int chunk_value_slot(int r, int j) {
  return D == 128 ? j ^ (4 * (r & 3)) : j ^ (4 * ((r >> 1) & 1));
}

// Slot of a chunk in a tile that is read both by rows and transposed.
template <int D> __device__ __forceinline__ int chunk_both_slot(int r, int j) {
  return D == 128 ? j ^ (((r & 3) << 2) | ((r >> 2) & 3)) : j ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
}

// The sequence and row block of an item: items are the row blocks of all
// sequences in turn (SORTED: by length where there are few), a sequence's last one
// first (it sees most).  From item `fold` on the order runs backwards, so that where
// all workgroups are resident at once, two a CU, one that sees much shares a CU with
// one that sees little.
template <bool SORTED>
__device__ __forceinline__ bool paged_item(const PagedAttnArgs& a, int32_t item, int32_t fold, int32_t* b, int32_t* block) {
  const int lane = threadIdx.x & 63;
  // The longest of up to eight sequences first, so that short walks come last (four
  // biased prompts of 670 to 2,047, 179 -> 173 us).  Of more, the last is a small part
  // of all, and finding its place takes an instruction or three a sequence.
  if (SORTED && a.c.B <= 8) {
    int32_t own = 0, mine = 0, total = 0;
    if (lane < a.c.B) {
      int32_t row0, tokens;
      paged_rows(a.c, lane, &row0, &tokens);
      if (tokens > a.max_new) tokens = a.max_new;
      own = (tokens * a.per + a.item_rows - 1) / a.item_rows;
    }
    for (int32_t j = 0; j < a.c.B; ++j) {
      const int32_t other = __builtin_amdgcn_readlane(own, j);
      total += other;
      if (other > own || (other == own && j < lane)) mine += other;
    }
    if (item >= fold && item < total) item = fold + (total - 1 - item);
    const uint64_t is = __ballot(item >= mine && item < mine + own);
    *block = total;
    if (is == 0) return false;
    const int at = __builtin_ctzll(is);
    *b = at;
    *block = __builtin_amdgcn_readlane(mine, at) + __builtin_amdgcn_readlane(own, at) - 1 - item;
    return true;
  }
  auto blocks_upto = [&](int32_t b0) -> int32_t {  // of sequences b0 to b0 + lane
    int32_t upto = 0;
    if (b0 + lane < a.c.B) {
      int32_t row0, tokens;
      paged_rows(a.c, b0 + lane, &row0, &tokens);
      if (tokens > a.max_new) tokens = a.max_new;
      upto = (tokens * a.per + a.item_rows - 1) / a.item_rows;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int32_t up = __shfl_up(upto, off, 64);
      if (lane >= off) upto += up;
    }
    return upto;
  };
  if (item >= fold) {
    int32_t total = 0;
    for (int32_t b0 = 0; b0 < a.c.B; b0 += 64) total += __builtin_amdgcn_readlane(blocks_upto(b0), 63);
    if (item < total) item = fold + (total - 1 - item);
  }
  int32_t before = 0;
  for (int32_t b0 = 0; b0 < a.c.B; b0 += 64) {
    const int32_t upto = blocks_upto(b0), all = __builtin_amdgcn_readlane(upto, 63);
    if (item < before + all) {
      const int at = __builtin_ctzll(__ballot(item < before + upto));
      *b = b0 + at;
      *block = before + __builtin_amdgcn_readlane(upto, at) - 1 - item;
      return true;
    }
    before += all;
  }
  *block = before;  // how many items there are
  return false;
}

template <bool LINEAR> __device__ __forceinline__ PagedSeq chunk_seq(const PagedCache& c, int32_t b) {
  if constexpr (!LINEAR) return paged_seq(c, b);
  PagedSeq s;
  paged_rows(c, b, &s.row0, &s.tokens);
  s.length = s.tokens;
  s.pos0 = 0;
  return s;
}

// Packed rows that no sequence owns, of one kv head's queries: zeros, and an lse
// of -infinity.  Workgroup `part` of `parts`.
template <int DT, int D>
__device__ __forceinline__ void clear_unowned(const PagedAttnArgs& a, int32_t part, int32_t parts, int32_t kvh, int32_t threads) {
  int32_t lead = clamp_i32(a.c.starts[0], 0, a.c.N), from = clamp_i32(a.c.starts[a.c.B], 0, a.c.N);
  if (from < lead) from = lead;
  const int64_t pieces = (int64_t)(lead + a.c.N - from) * a.per * (D / 8);
  for (int64_t i = (int64_t)part * threads + threadIdx.x; i < pieces; i += (int64_t)parts * threads) {
    const int64_t rg = i / (D / 8);
    int64_t n = rg / a.per;
    const int32_t head = kvh * a.per + (int32_t)(rg - n * a.per);
    if (n >= lead) n += from - lead;
    *(uint4*)(a.out + n * a.ost + head * a.osh + 16 * (i - rg * (D / 8))) = uint4{0u, 0u, 0u, 0u};
    if (i == rg * (D / 8) && a.lse != nullptr) a.lse[n * a.QH + head] = -INFINITY;
  }
}

// What a row at entry i sees reaches to here (rows before the first entry see nothing).
template <int FORM> __device__ __forceinline__ int32_t row_reach(int32_t i, int32_t prefix) {
  if constexpr (FORM == kFormPlain) return i;
  else return i < 0 || i >= prefix ? i : prefix - 1;
}

// LINEAR: keys and values lie packed as the queries do, a sequence's rows are its
// entries (the cache's head and slot strides are the keys', v_head_bytes and
// v_slot_bytes the values').  Rows that no sequence owns get zeros.  LSE: the
// logarithms of the rows' sums are wanted.
template <int DT, int D, bool EXACT, int kChunkWaves, int FORM = kFormPlain, bool LINEAR = false, bool LSE = EXACT>
__global__ __launch_bounds__(64 * kChunkWaves, 2) void paged_chunk_kernel(PagedAttnArgs a) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V8 V8;
  typedef typename Half16<DT>::V4 V4;
  constexpr int kSteps = D / 16, kDims = D / 32, kRowBytes = 2 * D, kChunkRows = 32 * kChunkWaves;
  constexpr int kTileBytes = kChunkTile * kRowBytes;
  constexpr int kRowsPerLoad = 1024 / kRowBytes, kWaveRows = kChunkTile / kChunkWaves, kLoads = kWaveRows / kRowsPerLoad;
  __shared__ __align__(1024) uint8_t lds[4 * kTileBytes];  // twice a tile of keys, one of values

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, lh = lane >> 5;
  // kv heads run fastest: with eight of them (or a multiple) each XCD has its
  // own, and a sequence's tiles meet in one L2; items spread evenly in any case
  const uint32_t bid = blockIdx.x, at_item = bid / (uint32_t)a.KVH;
  const int32_t kvh = (int32_t)(bid - at_item * (uint32_t)a.KVH);
  const int32_t item = (int32_t)(at_item / (uint32_t)a.splits), split = (int32_t)(at_item - (uint32_t)item * (uint32_t)a.splits);
  int32_t b, block;
  if (!paged_item<LINEAR>(a, item, a.fold, &b, &block)) {
    if constexpr (LINEAR) clear_unowned<DT, D>(a, item - block, a.items - block, kvh, 64 * kChunkWaves);
    return;
  }
  b = __builtin_amdgcn_readfirstlane(b);
  block = __builtin_amdgcn_readfirstlane(block);
  const PagedSeq s = chunk_seq<LINEAR>(a.c, b);
  const int32_t prefix = FORM == kFormPlain ? 0 : paged_prefix(a.prefixes, b, s.length);
  const int32_t tokens = s.tokens < a.max_new ? s.tokens : a.max_new;
  // (rows, N * QH in all, fit 31 bits: host-checked)
  const uint32_t per = (uint32_t)a.per;
  const int32_t R = tokens * a.per;
  const int32_t r0 = block * kChunkRows, r1 = R - r0 > kChunkRows ? r0 + kChunkRows : R;
  const int32_t before = s.length - s.tokens;
  const int32_t first = before + (int32_t)((uint32_t)r0 / per), last = before + (int32_t)((uint32_t)(r1 - 1) / per);
  // this wave's rows
  const int32_t wr0 = r0 + 32 * wave, wr1 = wr0 + 32 < r1 ? wr0 + 32 : r1;
  const bool wave_on = wr0 < r1;
  const int32_t wfirst = wave_on ? before + (int32_t)((uint32_t)wr0 / per) : kPagedMost;
  const int32_t wlast = wave_on ? before + (int32_t)((uint32_t)(wr1 - 1) / per) : -1;
  const bool row_ok = wr0 + ln < r1;
  const int32_t row_t = row_ok ? (int32_t)((uint32_t)(wr0 + ln) / per) : 0;
  const int32_t head = kvh * a.per + (row_ok ? wr0 + ln - row_t * a.per : 0);
  const int32_t self = row_ok ? before + row_t : -1;
  const int32_t reach = row_reach<FORM>(self, prefix);

  const PagedTiles pt = paged_tiles(first, row_reach<FORM>(last, prefix), a.window, a.sinks, kChunkTile);
  int32_t tile0 = 0, tile1 = pt.count;
  if (a.splits > 1) {
    const int32_t each = (pt.count + a.splits - 1) / a.splits;
    tile0 = split * each < pt.count ? split * each : pt.count;
    tile1 = tile0 + each < pt.count ? tile0 + each : pt.count;
  }

  // ---- tile loader: a wave's 8 or 16 entries lie in one page, and go from global
  // memory into LDS directly.  A page outside the pool and the entries at or
  // behind the length lie beyond the resource's bound and land as zeros. ----
  const int32_t* table = a.c.tables + b * a.c.table_stride;
  const int32_t mask = (1 << a.c.page_shift) - 1;
  const int lrow = lane / (64 / kRowsPerLoad), lslot = lane % (64 / kRowsPerLoad);
  const int64_t v_head_bytes = LINEAR ? a.v_head_bytes : a.c.head_bytes, v_slot_bytes = LINEAR ? a.v_slot_bytes : a.c.slot_bytes;
  const uint64_t k_head = (uint64_t)(a.c.k + kvh * a.c.head_bytes), v_head = (uint64_t)(a.c.v + kvh * v_head_bytes);
  const uint32_t lds_base = lds_address(lds);
  // lane -> row lrow of each load, slot lslot: the chunk that belongs there
  uint32_t k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int r = j * kRowsPerLoad + lrow, tile_r = kWaveRows * wave + r;
    k_off[j] = (uint32_t)r * (uint32_t)a.c.slot_bytes + 16u * (uint32_t)chunk_key_slot<D>(tile_r, lslot);
    v_off[j] = (uint32_t)r * (uint32_t)v_slot_bytes + 16u * (uint32_t)chunk_value_slot<D>(tile_r, lslot);
  }
  auto entry_of = [&](int32_t i) { return (i < pt.lead ? i : pt.main + i - pt.lead) * kChunkTile; };
  // What a tile needs is found 64 tiles at a time, a lane each, and read from
  // there: the place of this wave's entries in the pools, the bytes that may
  // be read there (none past the last tile), and
  enum { kBlockFull = 1 << 28, kWaveFull = 2 << 28, kWaveSees = 4 << 28, kBytes = kBlockFull - 1 };
  // all rows of the workgroup, or of the wave, see the whole tile; some row of
  // the wave sees some of it.
  uint32_t at_lo = 0, at_hi = 0;
  int32_t what = 0, run0 = tile0 - 64;  // bytes (below 2^27: host-checked strides) and flags
  auto look_up = [&](int32_t i) {
    if (i - run0 < 64) return;
    run0 = i;
    const int32_t e0 = entry_of(i + lane), e = e0 + kWaveRows * wave, left = s.length - e;
    if constexpr (LINEAR) {
      what = i + lane < tile1 && left > 0 ? (left < kWaveRows ? left : kWaveRows) : 0;  // rows
    } else {
      int32_t page = -1;
      if (i + lane < tile1 && left > 0) page = table[e >> a.c.page_shift];
      const bool ok = (uint32_t)page < (uint32_t)a.c.n_pages;
      const uint64_t at = ok ? page * a.c.page_bytes + (int64_t)(e & mask) * a.c.slot_bytes : 0;
      at_lo = (uint32_t)at;
      at_hi = (uint32_t)(at >> 32);
      what = ok ? ((left < kWaveRows ? left : kWaveRows) - 1) * (int32_t)a.c.slot_bytes + kRowBytes : 0;
    }
    const bool sunk = e0 + kChunkTile <= a.sinks;
    what |= (e0 + kChunkTile - 1 <= row_reach<FORM>(first, prefix) && (e0 > last - a.window || sunk) ? kBlockFull : 0) |
             (e0 + kChunkTile - 1 <= row_reach<FORM>(wfirst, prefix) && (e0 > wlast - a.window || sunk) ? kWaveFull : 0) |
             (e0 <= row_reach<FORM>(wlast, prefix) && (e0 + kChunkTile - 1 > wfirst - a.window || e0 < a.sinks) ? kWaveSees : 0);
    if constexpr (!LINEAR) asm volatile("" : "+v"(at_lo));  // waited for here, not at every tile's use
  };
  auto resource = [&](int32_t i, uint64_t pool, int64_t slot_bytes) -> uint4v {
    if constexpr (LINEAR) {
      const int32_t rows = __builtin_amdgcn_readlane(what, i - run0) & kBytes;
      const uint64_t at = pool + (uint64_t)((int64_t)(s.row0 + entry_of(i) + kWaveRows * wave) * slot_bytes);
      const uint32_t bytes = rows > 0 ? (uint32_t)(rows - 1) * (uint32_t)slot_bytes + kRowBytes : 0u;
      return uint4v{(uint32_t)__builtin_amdgcn_readfirstlane((int32_t)at), (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)(at >> 32)) & 0xffffu,
                    (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)bytes), 0x00020000u};
    }
    const uint32_t lo = __builtin_amdgcn_readlane(at_lo, i - run0), hi = __builtin_amdgcn_readlane(at_hi, i - run0);
    const uint64_t at = pool + (((uint64_t)hi << 32) | lo);
    return uint4v{(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, (uint32_t)__builtin_amdgcn_readlane(what, i - run0) & kBytes, 0x00020000u};
  };
  auto load_tile = [&](uint4v rsrc, const uint32_t (&off)[kLoads], uint32_t to) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      load_to_lds<16>(to + (uint32_t)(kWaveRows * kRowBytes) * (uint32_t)wave + 1024u * j, off[j], rsrc);
  };
  auto load_values = [&](int32_t i, int stage) {
    load_tile(resource(i, v_head, v_slot_bytes), v_off, lds_base + (2 * stage + 1) * kTileBytes);
  };
  auto load_stage = [&](int32_t i, int stage) {
    look_up(i);
    load_tile(resource(i, k_head, a.c.slot_bytes), k_off, lds_base + 2 * stage * kTileBytes);
    load_values(i, stage);
  };
  // every load has landed and every LDS access is done, in all waves
  auto meet = [&]() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  const bool any = tile0 < tile1;
  if (any) load_stage(tile0, 0);

  // ---- the wave's rotated queries times the scale (B operand: 8 dims of row ln) ----
  V8 qf[kSteps], ql[EXACT ? kSteps : 1];
  {
    const uint8_t* qp = a.q + (int64_t)(s.row0 + row_t) * a.qst + (int64_t)head * a.qsh;
    V8 x[kSteps];
#pragma unroll
    for (int c = 0; c < kSteps; ++c) x[c] = *(const V8*)(qp + 32 * c + 16 * lh);
    auto put = [&](int c, int e, float v) {
      v = row_ok ? v * a.q_mul : 0.f;
      qf[c][e] = (T)v;
      if constexpr (EXACT) ql[c][e] = __builtin_isfinite((float)(T)v) ? (T)(v - (float)(T)v) : (T)0.f;
    };
    if constexpr (LINEAR) {  // as they are, or their negatives
      const uint32_t kept_bits = row_ok ? 0xffffffffu : 0u, flip = a.q_mul < 0.f ? 0x80008000u : 0u;
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        uint4v w = __builtin_bit_cast(uint4v, x[c]);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (w[e] ^ flip) & kept_bits;
        qf[c] = __builtin_bit_cast(V8, w);
      }
    } else if (a.rope.on) {
#pragma unroll
      for (int c = 0; c < kSteps / 2; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float cs, sn;
          rope_trig(a.rope.turns[16 * c + 8 * lh + e], s.pos0 + row_t, &cs, &sn);
          const float u = (float)x[c][e], w = (float)x[c + kSteps / 2][e];
          put(c, e, u * cs - w * sn);
          put(c + kSteps / 2, e, w * cs + u * sn);
        }
    } else {
#pragma unroll
      for (int c = 0; c < kSteps; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) put(c, e, (float)x[c][e]);
    }
  }
  if constexpr (EXACT) {
    if (a.q_parts != nullptr && split == 0 && row_ok) {
      uint8_t* to = a.q_parts + (((int64_t)kvh * a.c.N + s.row0) * a.per + wr0 + ln) * (4 * D) + 16 * lh;
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        *(V8*)(to + 32 * c) = qf[c];
        *(V8*)(to + 2 * D + 32 * c) = ql[c];
      }
    }
  }

  // `shift` is minus the reference maximum plus 10 in all elements: the products
  // start from it, so that a score leaves them as the exponent of its p.  p is
  // 2^10 times the weight against the reference, which moves when a maximum
  // passes it by more than 4 (at first: at once): p stays below 2^14, and fp16
  // holds weights of 2^-34.  (In units of scale2, a power of two that only
  // large scales need.)
  float16v shift = {}, o[kDims];
  float l = 0.f, kept = 0.f, limit = -INFINITY;
  // Shaped scores are moved by `from` instead, the reference less kHeld, which
  // moves when a maximum passes it by kRoom: sharp heads move it often, and each
  // time costs a rescaling (with 10 and 4, a quarter of the vector instructions of
  // capped 8,192-token texts).  fp16 p stay below 2^15 and hold weights of 2^-30,
  // bf16 ones below 2^34 (values past 2^93 over the number of entries can pass 32
  // bits).  Their outputs are divided by `kept`, the sum of the p as rounded for the
  // products, not by `l`, which only a row's lse takes (LSE): where one entry holds
  // most of a row its rounding cancels, in the output and in the do out that gradients
  // subtract (queries four times a unit normal, bf16: outputs 1.9e-3 off instead of
  // 2.4e-3, dq 2.6e-3 instead of 3.5e-3).  Both sums are 6 % of a training chunk.
  constexpr float kHeld = DT == JKV_F16 ? 6.f : 10.f, kRoom = DT == JKV_F16 ? 9.f : 24.f;
  float from = 0.f;
  const ScoreShape shape = score_shape<FORM>(a, head);
  // a shaped row sees entries [seen_from, seen_from + seen_count), and those before
  // `sunk` more (counted from seen_from on)
  const int32_t seen_from = self >= a.window ? self - a.window + 1 : 0;
  const uint32_t seen_count = reach >= seen_from ? (uint32_t)(reach - seen_from + 1) : 0u;
  const int32_t sunk = reach >= 0 ? (a.sinks < seen_from ? a.sinks : seen_from) - seen_from : -kPagedMost - 1;
#pragma unroll
  for (int d = 0; d < kDims; ++d) o[d] = float16v{};
  // LDS addresses: a few per lane, the rest are offsets known at compile time
  uint32_t k_at[kSteps], v_at[kDims];
#pragma unroll
  for (int c = 0; c < kSteps; ++c) k_at[c] = lds_base + (uint32_t)(ln * kRowBytes + 16 * chunk_key_slot<D>(ln, 2 * c + lh));
  const int tr_row = 4 * lh + ((lane & 15) >> 2), tr_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
  for (int d = 0; d < kDims; ++d)
    v_at[d] = lds_base + (uint32_t)(kTileBytes + tr_row * kRowBytes + 16 * chunk_value_slot<D>(tr_row, 4 * d + tr_chunk) + 8 * (lane & 1));
  auto value_operand = [&](int d, int st, int buf) -> V8 {
    const uint32_t at = v_at[d] + (uint32_t)(2 * buf * kTileBytes + 16 * st * kRowBytes);
    const V4 lo = lds_read_tr<V4>(at), hi = lds_read_tr<V4>(at + 8 * kRowBytes);
    return V8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  typedef __attribute__((address_space(3))) const V8 lds_v8;
  // AGAIN: infinite keys meet the queries' leading part alone
  auto scores = [&](int buf, float16v (&sc)[2], auto again) {
    constexpr bool AGAIN = decltype(again)::value;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      if constexpr (FORM == kFormPlain) sc[kb] = shift;
      else sc[kb] = float16v{};
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        const V8 ka = *(lds_v8*)(size_t)(k_at[c] + (uint32_t)(2 * buf * kTileBytes + 32 * kb * kRowBytes));
        sc[kb] = mfma32<DT>(ka, qf[c], sc[kb]);
        if constexpr (EXACT && AGAIN) sc[kb] = mfma32<DT>(finite_part<DT>(ka), ql[c], sc[kb]);
        else if constexpr (EXACT) sc[kb] = mfma32<DT>(ka, ql[c], sc[kb]);
      }
    }
  };
  auto hide = [&](int32_t e0, float16v (&sc)[2]) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int32_t j = e0 + 32 * kb + 8 * (e >> 2) + 4 * lh + (e & 3);
        const bool seen = j <= reach && (j > self - a.window || j < a.sinks);
        sc[kb][e] = seen ? sc[kb][e] : -INFINITY;
      }
  };
  auto largest = [&](const float16v (&sc)[2]) -> float {
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; e += 2) mx = fmaxf(fmaxf(mx, sc[kb][e]), sc[kb][e + 1]);
    return lanes2_max(mx);
  };
  auto move_reference = [&](float mx, float16v (&sc)[2]) {
    const bool need = mx > limit;
    if (!__any(need)) return;
    const float d = need ? mx - 10.f : 0.f, by = d / a.scale2;
    const float alpha = limit == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(-d);
    limit = need ? 14.f : limit;
    shift -= by;
    l *= alpha;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) sc[kb] -= d;
#pragma unroll
    for (int x = 0; x < kDims; ++x) o[x] *= alpha;
  };
  // p of 32 of a tile's scores
  auto weigh = [&](const float16v& sc, V8* pf) {
    float t4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float p = __builtin_amdgcn_exp2f(sc[e]);
      t4[e & 3] += p;
      pf[e >> 3][e & 7] = (T)p;
    }
    l += (t4[0] + t4[1]) + (t4[2] + t4[3]);
  };
  const bool unit = a.scale2 == 1.f;

  bool found = false;  // an infinite or NaN value in a tile that was cleaned of them
  auto clean = [&](int buf) {
    for (int at = 16 * tid; at < kTileBytes; at += 16 * 64 * kChunkWaves) {
      uint4v* w = (uint4v*)(lds + (2 * buf + 1) * kTileBytes + at);
      *w = finite_halves<DT>(*w, &found);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  auto work = [&](int32_t i, int32_t is, auto parity, auto again) {
    constexpr int buf = decltype(parity)::value;
    float16v sc[2];
    scores(buf, sc, again);
    JKV_SG(0x100, kSteps);
    for (int x = 0; x < kSteps; ++x) { JKV_SG(0x8, EXACT ? 2 : 1); JKV_SG(0x100, 1); }
    JKV_SG(0x8, EXACT ? 2 * kSteps : kSteps);
    if (!unit || !(is & kWaveFull)) {
      for (int kb = 0; kb < 2; ++kb) sc[kb] *= a.scale2;
      hide(entry_of(i), sc);
    }
    V8 va[2][kDims];
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int d = 0; d < kDims; ++d) va[st][d] = value_operand(d, st, buf);
    const float mx = largest(sc);
    move_reference(mx, sc);
    V8 pf[4];
    weigh(sc[0], pf);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int d = 0; d < kDims; ++d) o[d] = mfma32<DT>(va[st][d], pf[st], o[d]);
    weigh(sc[1], pf + 2);
#pragma unroll
    for (int st = 2; st < 4; ++st)
#pragma unroll
      for (int d = 0; d < kDims; ++d) o[d] = mfma32<DT>(value_operand(d, st, buf), pf[st], o[d]);
    // the second half's exponentials beside the first half's products
    for (int x = 0; x < 2 * kDims; ++x) { JKV_SG(0x8, 1); JKV_SG(0x100, 2); JKV_SG(0x2, 40 / (2 * kDims)); }
    JKV_SG(0x8, 2 * kDims);
  };
  // The same with shaped scores, whose vector instructions take longer than the
  // products (13 and 1 a score, 64 cycles of issue and 32): a half's shaping goes
  // beside the products of the other half's scores or of the values, a product
  // and a few scores at a time, fenced, as the compiler else gathers each kind.
  // Three capped texts of 21,760 bf16 tokens in all, window 4,096, 32/8 heads of 128:
  // 1,440 to 1,480 us, 705 to 725 TFLOP/s, vector instructions 69 % of the cycles,
  // products 37 %, both at once 18 %, 1.85 GHz; in pages 2,048 capped tokens over 8,192
  // entries and one over 3,436 353 us, 680.
  auto work_shaped = [&](int32_t i, int32_t is, auto parity, auto again) {
    constexpr int buf = decltype(parity)::value;
    constexpr bool AGAIN = decltype(again)::value;
    constexpr int kEach = 16 / kSteps, kValues = 2 * kDims, kBeside = 16 / kValues;
    const int32_t e0 = entry_of(i);
    const float at = (float)(e0 + 4 * lh - self);  // (distances below 2^24 are exact)
    float16v sc[2] = {};
    V8 ring[3];
    auto key_operand = [&](int n) -> V8 {
      return *(lds_v8*)(size_t)(k_at[n % kSteps] + (uint32_t)(2 * buf * kTileBytes + 32 * (n / kSteps) * kRowBytes));
    };
    auto first = [&](int kb, int e) { sc[kb][e] = shape_first<FORM>(shape, sc[kb][e]); };
    // Without a bias the first step's maximum is the scores', and the second step
    // subtracts the reference too; with one, the second step comes before the maximum.
    constexpr bool kLate = !(FORM & kFormBias);
    auto second = [&](int kb, int e) {
      sc[kb][e] = shape_second<FORM>(shape, sc[kb][e], at + (float)(32 * kb + 8 * (e >> 2) + (e & 3)), shape.cap2);
    };
    V8 pf[4];
    float sums[4] = {0.f, 0.f, 0.f, 0.f}, keeps[2] = {0.f, 0.f};
    auto keep = [&](int kb, int e) {
      const V8& p8 = pf[2 * kb + (e >> 3)];
      keeps[e >> 1 & 1] = add_pair<DT>(p8[e & 7], p8[(e & 7) + 1], keeps[e >> 1 & 1]);
    };
    auto third = [&](int kb, int e) {
      const float p = __builtin_amdgcn_exp2f(kLate ? shape_second<FORM>(shape, sc[kb][e], 0.f, shape.cap2 - from) : sc[kb][e] - from);
      if constexpr (LSE) sums[e & 3] += p;
      pf[2 * kb + (e >> 3)][e & 7] = (T)p;
      if (e & 1) keep(kb, e - 1);
    };
    auto reference = [&](int kb) {
      if (!(is & kWaveFull)) {
        const uint32_t seen_at = (uint32_t)(e0 + 32 * kb + 4 * lh - seen_from);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t n = seen_at + (uint32_t)(8 * (e >> 2) + (e & 3));
          const bool seen = n < seen_count || (int32_t)n < sunk;
          sc[kb][e] = seen ? sc[kb][e] : kLate ? shape_masked<FORM>() : -INFINITY;
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; e += 2) mx = fmaxf(fmaxf(mx, sc[kb][e]), sc[kb][e + 1]);
      mx = lanes2_max(mx);
      if constexpr (kLate) mx = shape_second<FORM>(shape, mx, 0.f, shape.cap2);
      const bool need = mx > limit;
      if (__any(need)) {
        const float to = need ? mx - kHeld : from;
        const float alpha = limit == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(from - to);
        limit = need ? mx + kRoom : limit;
        from = to;
        if constexpr (LSE) l *= alpha;
        kept *= alpha;
        if constexpr (LSE)
#pragma unroll
          for (int t = 0; t < 4; ++t) sums[t] *= alpha;
#pragma unroll
        for (int t = 0; t < 2; ++t) keeps[t] *= alpha;
#pragma unroll
        for (int x = 0; x < kDims; ++x) o[x] *= alpha;
      }
    };
    ring[0] = key_operand(0);
    ring[1] = key_operand(1);
#pragma unroll
    for (int n = 0; n < 2 * kSteps; ++n) {
      const int kb = n / kSteps, c = n % kSteps;
      if (n + 2 < 2 * kSteps) ring[(n + 2) % 3] = key_operand(n + 2);
      sc[kb] = mfma32<DT>(ring[n % 3], qf[c], sc[kb]);
      if constexpr (EXACT) sc[kb] = mfma32<DT>(AGAIN ? finite_part<DT>(ring[n % 3]) : ring[n % 3], ql[c], sc[kb]);
      if (kb == 1) {
#pragma unroll
        for (int e = c * kEach; e < (c + 1) * kEach; ++e) first(0, e);
        if (c > 0 && !kLate)
#pragma unroll
          for (int e = (c - 1) * kEach; e < c * kEach; ++e) second(0, e);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    ring[0] = value_operand(0, 0, buf);
    ring[1] = value_operand(1, 0, buf);
    if constexpr (!kLate)
#pragma unroll
      for (int e = 16 - kEach; e < 16; ++e) second(0, e);
    reference(0);
#pragma unroll
    for (int e = 0; e < 8; ++e) third(0, e);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int n = 0; n < kValues; ++n) {
        if (n + 2 < kValues) ring[(n + 2) % 3] = value_operand((n + 2) % kDims, 2 * kb + (n + 2) / kDims, buf);
        o[n % kDims] = mfma32<DT>(ring[n % 3], pf[2 * kb + n / kDims], o[n % kDims]);
        if (n < kDims)
#pragma unroll
          for (int e = 8 + n * (8 / kDims); e < 8 + (n + 1) * (8 / kDims); ++e) third(kb, e);
        if (kb == 0) {
#pragma unroll
          for (int e = n * kBeside; e < (n + 1) * kBeside; ++e) first(1, e);
          if (n > 0 && !kLate)
#pragma unroll
            for (int e = (n - 1) * kBeside; e < n * kBeside; ++e) second(1, e);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (kb == 0) {
        ring[0] = value_operand(0, 2, buf);
        ring[1] = value_operand(1, 2, buf);
        if constexpr (!kLate)
#pragma unroll
          for (int e = 16 - kBeside; e < 16; ++e) second(1, e);
        reference(1);
#pragma unroll
        for (int e = 0; e < 8; ++e) third(1, e);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (LSE) l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
    kept += keeps[0] + keeps[1];
  };
  auto step = [&](int32_t i, auto parity) {
    constexpr int buf = decltype(parity)::value;
    const int32_t is = __builtin_amdgcn_readlane(what, i - run0);
    meet();
    load_stage(i + 1, buf ^ 1);
    // (shaped scores: a value that is not finite, seen or not, makes the sums so, and
    // the walk is made again with all tiles cleaned)
    if (FORM == kFormPlain && !(is & kBlockFull)) clean(buf);
    if (is & kWaveSees) {
      if constexpr (FORM == kFormPlain) work(i, is, parity, std::false_type());
      else work_shaped(i, is, parity, std::false_type());
    }
  };
  for (int32_t i = tile0; i < tile1; i += 2) {
    step(i, std::integral_constant<int, 0>());
    if (i + 1 < tile1) step(i + 1, std::integral_constant<int, 1>());
  }

  // An infinite value times a weight that rounds to 0, an infinite key times a
  // query's trailing part: 0 times infinity or the other infinity, NaN where
  // there is a result.  What these go into is not finite, so a walk that ends in
  // finite sums needs no second.
  float odd = (FORM == kFormPlain ? l : kept) * 0.f;
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) odd = fmaf(o[d][e], 0.f, odd);
  const bool again = __syncthreads_or(odd != 0.f);
  if (again) {
    shift = float16v{};
    l = kept = 0.f;
    limit = -INFINITY;
    from = 0.f;
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[d] = float16v{};
    run0 = tile0 - 64;
    for (int32_t i = tile0; i < tile1; ++i) {
      meet();
      load_stage(i, 0);
      const int32_t is = __builtin_amdgcn_readlane(what, i - run0);
      meet();
      clean(0);
      if (is & kWaveSees) {
        if constexpr (FORM == kFormPlain) work(i, is, std::integral_constant<int, 0>(), std::true_type());
        else work_shaped(i, is, std::integral_constant<int, 0>(), std::true_type());
      }
    }
  }

  if (__syncthreads_or(found)) {
    for (int32_t i = tile0; i < tile1; ++i) {
      const int32_t e0 = entry_of(i);
      run0 = i - 64;  // the tile's place anew
      look_up(i);
      if ((__builtin_amdgcn_readlane(what, 0) & kBlockFull) && !again) continue;
      meet();
      load_values(i, 0);
      meet();
      V8 seen[4];
#pragma unroll
      for (int st = 0; st < 4; ++st)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int32_t j = e0 + 16 * st + 8 * (e >> 2) + 4 * lh + (e & 3);
          seen[st][e] = j <= reach && (j > self - a.window || j < a.sinks) ? (T)1.f : (T)0.f;
        }
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        float16v up = {}, down = {};
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          V8 vu, vd;
          non_finite_marks<DT>(value_operand(d, st, 0), &vu, &vd);
          up = mfma32<DT>(vu, seen[st], up);
          down = mfma32<DT>(vd, seen[st], down);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = marked(o[d][e], up[e], down[e]);
      }
    }
  }
  meet();  // (loads ahead of the last tile land before the LDS is given back)

  // ---- out, or this split's part of it: lane holds dims 32d + 8(e/4) + 4lh + e%4 of row ln ----
  const float kt = lanes2_sum(FORM == kFormPlain ? l : kept), lt = FORM == kFormPlain || !LSE ? kt : lanes2_sum(l);
  if (!row_ok) return;
  const int64_t n = s.row0 + row_t, row = n * a.QH + head;
  const float moved = FORM == kFormPlain ? -shift[0] * a.scale2 : from;
  if (a.splits > 1) {
    const int64_t at = (int64_t)split * a.c.N * a.QH + row;
    if (lh == 0) a.part_ml[at] = float2{limit == -INFINITY ? -INFINITY : moved, lt};
    if (tile0 < tile1) {
      // (the join divides by the sum of the splits' lt)
      if constexpr (FORM != kFormPlain && LSE) {
        const float to = lt == 0.f ? 0.f : lt / kt;
#pragma unroll
        for (int d = 0; d < kDims; ++d) o[d] *= to;
      }
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          *(float4v*)(a.part_o + at * D + 32 * d + 8 * q4 + 4 * lh) =
              float4v{o[d][4 * q4], o[d][4 * q4 + 1], o[d][4 * q4 + 2], o[d][4 * q4 + 3]};
    }
    return;
  }
  const bool none = lt == 0.f;  // sees nothing
  if (lh == 0) {
    const float l2 = none ? -INFINITY : log2f(lt) + moved;
    if (a.lse != nullptr) a.lse[row] = l2 * 0.6931471805599453f;
    if (a.lse2 != nullptr) a.lse2[((int64_t)kvh * a.c.N + s.row0) * a.per + wr0 + ln] = l2;
  }
  const float inv = 1.0f / kt;
  uint8_t* op = a.out + n * a.ost + (int64_t)head * a.osh;
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      V4 h;
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = (T)(none ? 0.f : o[d][4 * q4 + e] * inv);
      *(V4*)(op + 2 * (32 * d + 8 * q4 + 4 * lh)) = h;
      if constexpr (LINEAR) {
        if (a.rest != nullptr) {  // what the rounding took off
          V4 r;
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] = (T)(none ? 0.f : o[d][4 * q4 + e] * inv - (float)h[e]);
          *(V4*)(a.rest + row * (2 * D) + 2 * (32 * d + 8 * q4 + 4 * lh)) = r;
        }
      }
    }
}

// The weights of chunks.  A wave holds 32 entries' keys in registers, walks the
// rows that may see them (their rotated queries in two parts) and adds
// exp2(score - lse) up: S^T[entry][row] leaves 16 entries of one row with a
// lane, the sum over the rows' lanes comes last.  Eight waves a workgroup are
// ENTRIES times ROWS of 32, and STAGES of the rows lie in LDS or are on their
// way: a stage's products (0.5 us) are over before its successor's loads have
// come, so what LDS holds goes into stages.  A kv head's rows of a sequence lie one behind another, so a stage is one
// stretch of memory.  Every sum has one order.
template <int DT, int D, int ENTRIES, int ROWS, int STAGES, int FORM = kFormPlain>
__global__ __launch_bounds__(512, 2) void paged_chunk_weights_kernel(PagedAttnArgs a, int32_t blocks) {
  typedef typename Half16<DT>::V8 V8;
  constexpr int kSteps = D / 16, kRowBytes = 4 * D, kChunks = kRowBytes / 16, kRowsPerLoad = 1024 / kRowBytes;
  constexpr int kWeightEntries = 32 * ENTRIES, kWeightRows = 32 * ROWS, kWeightStages = STAGES;
  static_assert(ENTRIES * ROWS == 8, "eight waves");
  constexpr int kLoads = kWeightRows / kRowsPerLoad / 8, kStageBytes = kWeightRows * kRowBytes;
  __shared__ __align__(1024) uint8_t q_lds[kWeightStages * kStageBytes];
  __shared__ __align__(16) float norm_lds[kWeightStages][8][64];  // each wave its own
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t at_block = blockIdx.x / (uint32_t)a.KVH;  // (kv heads fastest, as above)
  const int32_t kvh = (int32_t)(blockIdx.x - at_block * (uint32_t)a.KVH);
  const int32_t b = (int32_t)(at_block / (uint32_t)blocks), blk = (int32_t)(at_block - (uint32_t)b * (uint32_t)blocks);
  const PagedSeq s = paged_seq(a.c, b);
  const int32_t j0 = blk * kWeightEntries;
  if (j0 >= s.length) return;
  const int32_t prefix = FORM == kFormPlain ? 0 : paged_prefix(a.prefixes, b, s.length);
  const int32_t tokens = s.tokens < a.max_new ? s.tokens : a.max_new, before = s.length - s.tokens;
  const int32_t wj0 = j0 + 32 * (wave % ENTRIES);

  // the wave's keys (A operand: 8 dims of entry ln)
  V8 kf[kSteps];
  {
    const int32_t j = wj0 + ln;
    int32_t page = -1;
    if (j < s.length) page = a.c.tables[b * a.c.table_stride + (j >> a.c.page_shift)];
    const bool ok = (uint32_t)page < (uint32_t)a.c.n_pages;
    const uint8_t* kp = a.c.k + (ok ? page * a.c.page_bytes + kvh * a.c.head_bytes +
                                          (int64_t)(j & ((1 << a.c.page_shift) - 1)) * a.c.slot_bytes : 0) + 16 * lh;
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      kf[c] = V8{};
      if (ok) kf[c] = *(const V8*)(kp + 32 * c);
    }
#pragma unroll
    for (int c = 0; c < kSteps; ++c) asm volatile("" : "+v"(kf[c]));  // waited for here, not beside the loads below
  }
  // (infinite keys meet the queries' leading part alone, as in the attention)
  V8 kl[kSteps];
#pragma unroll
  for (int c = 0; c < kSteps; ++c) kl[c] = finite_part<DT>(kf[c]);

  // the rows that may see one of the workgroup's entries
  int32_t t0 = j0 - before, t1 = tokens;
  if (t0 < 0 || (FORM != kFormPlain && j0 < prefix)) t0 = 0;
  if (j0 >= a.sinks) {
    // the last entry's window ends here: far before the new tokens (or 2^31 on),
    // whose product with the heads below would wrap
    const int64_t end = (int64_t)j0 + kWeightEntries - 1 + a.window - before;
    if (end < t1) t1 = end > 0 ? (int32_t)end : 0;
  }
  const uint32_t per = (uint32_t)a.per;
  // (rows fit 31 bits: host-checked)
  const int32_t r0 = __builtin_amdgcn_readfirstlane(t0 * a.per), r1 = __builtin_amdgcn_readfirstlane(t1 * a.per);
  float acc[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;

  const uint32_t lds_base = lds_address(q_lds);
  // (rows at or behind r1 land as zeros and take no part)
  const int64_t row_base = ((int64_t)kvh * a.c.N + __builtin_amdgcn_readfirstlane(s.row0)) * a.per;
  uint32_t off[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int rr = (wave * kLoads + j) * kRowsPerLoad + lane / kChunks;
    off[j] = (uint32_t)(rr * kRowBytes + 16 * ((lane % kChunks) ^ (rr & 15)));
  }
  auto load_stage = [&](int32_t r, int stage) {
    const int32_t some = r1 - r < 0 ? 0 : (r1 - r < 2 * kWeightRows ? r1 - r : 2 * kWeightRows);
    const int32_t left = __builtin_amdgcn_readfirstlane(some);  // (the compiler takes the minimum in a vector register)
    const uint64_t at = (uint64_t)a.q_parts + (uint64_t)(row_base + r) * kRowBytes, norm_at = (uint64_t)(a.lse2 + row_base + r);
    const uint4v rsrc = {(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, (uint32_t)(left * kRowBytes), 0x00020000u};
    const uint4v norm_rsrc = {(uint32_t)norm_at, (uint32_t)(norm_at >> 32) & 0xffffu, 4u * (uint32_t)left, 0x00020000u};
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      load_to_lds<16>(lds_base + (uint32_t)(stage * kStageBytes + 1024 * (wave * kLoads + j)), off[j], rsrc);
    load_to_lds<4>(lds_address(norm_lds[stage][wave]), 4u * (uint32_t)(32 * (wave / ENTRIES) + lane), norm_rsrc);
  };
  typedef __attribute__((address_space(3))) const V8 lds_v8;
  uint32_t q_at[kSteps];
#pragma unroll
  for (int c = 0; c < kSteps; ++c)
    q_at[c] = lds_base + (uint32_t)((32 * (wave / ENTRIES) + ln) * kRowBytes + 16 * ((2 * c + lh) ^ (ln & 15)));

  if (r0 < r1) {
#pragma unroll
    for (int st = 0; st < kWeightStages - 1; ++st) load_stage(r0 + kWeightRows * st, st);
    int stage = 0;
    for (int32_t rs = r0; rs < r1; rs += kWeightRows, stage = (stage + 1) % kWeightStages) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"((kWeightStages - 2) * (kLoads + 1)) : "memory");
      load_stage(rs + kWeightRows * (kWeightStages - 1), (stage + kWeightStages - 1) % kWeightStages);
      const int32_t r = rs + 32 * (wave / ENTRIES);
      if (r >= r1) continue;
      const int32_t row = r + ln;
      const bool row_ok = row < r1;
      float norm = norm_lds[stage][wave][ln];
      if (!row_ok || norm == -INFINITY) norm = INFINITY;  // (it saw nothing)
      float16v sc = {};
      V8 part[2 * kSteps];
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        part[c] = *(lds_v8*)(size_t)(q_at[c] + (uint32_t)(stage * kStageBytes));
        part[kSteps + c] = *(lds_v8*)(size_t)((q_at[c] + (uint32_t)(stage * kStageBytes)) ^ (uint32_t)(2 * D));
      }
#pragma unroll
      for (int c = 0; c < 2 * kSteps; ++c) sc = mfma32<DT>(c < kSteps ? kf[c] : kl[c - kSteps], part[c], sc);
      const int32_t tf = before + (int32_t)((uint32_t)r / per);
      const int32_t tl = before + (int32_t)((uint32_t)(r + 31 < r1 ? r + 31 : r1 - 1) / per);
      // (rows behind the last are zeros, which an infinite key turns into NaN)
      const bool full = r + 31 < r1 && wj0 + 31 <= row_reach<FORM>(tf, prefix) && (wj0 > tl - a.window || wj0 + 32 <= a.sinks);
      if constexpr (FORM != kFormPlain) {
        const int32_t t = row_ok ? (int32_t)((uint32_t)row / per) : 0;
        const ScoreShape shape = score_shape<FORM>(a, kvh * a.per + (row_ok ? row - t * a.per : 0));
        const float at = (float)(wj0 + 4 * lh - (before + t));
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = shape_score<FORM>(shape, sc[e], at + (float)(8 * (e >> 2) + (e & 3)));
      }
      if (!full) {
        const int32_t self = row_ok ? before + (int32_t)((uint32_t)row / per) : -1;
        const int32_t reach = row_reach<FORM>(self, prefix);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int32_t j = wj0 + 8 * (e >> 2) + 4 * lh + (e & 3);
          const bool seen = j <= reach && (j > self - a.window || j < a.sinks);
          sc[e] = seen ? sc[e] : -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] += __builtin_amdgcn_exp2f(FORM == kFormPlain ? fmaf(sc[e], a.scale2, -norm) : sc[e] - norm);
    }
  }
  // the last loads land before their room is used for the row groups' sums
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  float* sums = (float*)q_lds;  // [ROWS][32 ENTRIES]
#pragma unroll
  for (int e = 0; e < 16; ++e) {
#pragma unroll
    for (int off2 = 16; off2 >= 1; off2 >>= 1) acc[e] += __shfl_xor(acc[e], off2, 64);
    if (ln == e) sums[kWeightEntries * (wave / ENTRIES) + 32 * (wave % ENTRIES) + 8 * (e >> 2) + 4 * lh + (e & 3)] = acc[e];
  }
  __syncthreads();
  const int32_t j = j0 + tid;
  if (tid < kWeightEntries && j < s.length) {
    float v = 0.f;
#pragma unroll
    for (int g = 0; g < ROWS; ++g) v += sums[kWeightEntries * g + tid];
    float* w = a.weights + b * a.wsb + kvh * a.wsh + j;
    *w = a.accumulate ? *w + v : v;
  }
}

template <int DT, int D, int FORM>
static int launch_chunk(const PagedAttnArgs& a, hipStream_t stream) {
  const int64_t blocks = (int64_t)a.items * a.KVH * a.splits;
  JKV_CHECK_GRID(blocks, 2 * a.item_rows);
  const dim3 grid((uint32_t)blocks), block((uint32_t)(2 * a.item_rows));
  const bool exact = a.lse != nullptr || a.lse2 != nullptr;
  if constexpr (D == 128 && FORM == kFormPlain) {
    if (a.item_rows == 256) {
      if (exact) hipLaunchKernelGGL((paged_chunk_kernel<DT, D, true, 8, FORM>), grid, block, 0, stream, a);
      else hipLaunchKernelGGL((paged_chunk_kernel<DT, D, false, 8, FORM>), grid, block, 0, stream, a);
    }
  }
  if (a.item_rows == 128) {
    if (exact) hipLaunchKernelGGL((paged_chunk_kernel<DT, D, true, 4, FORM>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((paged_chunk_kernel<DT, D, false, 4, FORM>), grid, block, 0, stream, a);
  }
  if (a.splits > 1) {
    const int rc = paged_launch_join(a, DT, D, stream);
    if (rc != JKV_OK) return rc;
  }
  if (a.weights != nullptr && a.c.top > 0) {
    // 128 entries a workgroup where that fills the CUs, 64 elsewhere.  us of the
    // attention and its weights with 64 and with 128, 32/8 heads of 128: 2 x 1,024
    // tokens over 4,096 entries 386 and 343, 1 x 256 over 8,000 143 and 126, 1 x
    // 2,000 161 and 204 (128 workgroups).
    const int64_t each = ceil_div(a.c.top, 128), all = each * a.c.B * a.KVH;
    JKV_CHECK_GRID(2 * all, 512);
    if (all >= 256)
      hipLaunchKernelGGL((paged_chunk_weights_kernel<DT, D, 4, 2, 4, FORM>), dim3((uint32_t)all), dim3(512), 0, stream, a, (int32_t)each);
    else
      hipLaunchKernelGGL((paged_chunk_weights_kernel<DT, D, 2, 4, 2, FORM>), dim3((uint32_t)(2 * all)), dim3(512), 0, stream, a,
                         (int32_t)(2 * each));
  }
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

}  // namespace jkv
