// Eviction from a paged K/V cache: which entries of each (sequence, kv head)
// stay, and their rows into new pages.
//
// Selection: the first `sinks` and last `recent` entries stay, and of those
// between the ones with the largest weights, the lower index first among
// equals, `budget` in all.  One workgroup per (sequence, kv head) finds the
// weight of the last one that stays by three histograms over 11, 11 and 10
// bits of the weights' order-preserving words, then lists the entries that
// stay in their order, placed by the waves' ballots and one scan a round.  Every
// sum is of integers, so a call repeats exactly.  Barriers and the scans between
// them are most of its time: 15 us for 3,000 entries a head, 18 for 16,384, 110
// for 100,000 (one workgroup reads them four times).  The copy of the rows that
// stay is bound by memory: 54 us for 260 MB, 4.8 TB/s.
#include "paged.h"

namespace jkv {

static const int kSelectThreads = 1024;
static const int kRound = 16 * kSelectThreads;

// Unsigned order of weights: -0 counts as 0, NaN below every number.
__device__ __forceinline__ uint32_t weight_order(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// inclusive sum over the workgroup's threads; `part` holds one word per wave
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* part, uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t up = __shfl_up(v, off, 64);
    if (lane >= off) v += up;
  }
  __syncthreads();
  if (lane == 63) part[wave] = v;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelectThreads / 64; ++w) {
    const uint32_t p = part[w];
    all += p;
    before += w < wave ? p : 0u;
  }
  *total = all;
  return v + before;
}

struct SelectArgs {
  const float* weights;
  int64_t stride_b, stride_h;
  const int32_t* lengths;
  int32_t* kept;         // [B,KVH,budget]
  int32_t* new_lengths;  // [B]
  int32_t width;         // entries a row of weights has
  int32_t budget, sinks, recent;
};

__global__ __launch_bounds__(kSelectThreads) void paged_select_kernel(SelectArgs a) {
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t part[kSelectThreads / 64];
  __shared__ uint32_t found[2];
  const int tid = threadIdx.x;
  const int32_t b = (int32_t)blockIdx.y, h = (int32_t)blockIdx.x;
  const int32_t length = clamp_i32(a.lengths[b], 0, a.width);
  const float* w = a.weights + b * a.stride_b + h * a.stride_h;
  int32_t* kept = a.kept + ((int64_t)b * gridDim.x + h) * a.budget;
  const int32_t count = length < a.budget ? length : a.budget;
  if (h == 0 && tid == 0) a.new_lengths[b] = count;
  for (int32_t i = count + tid; i < a.budget; i += kSelectThreads) kept[i] = -1;
  if (length <= a.budget) {
    for (int32_t i = tid; i < count; i += kSelectThreads) kept[i] = i;
    return;
  }
  const int32_t first = a.sinks, last = length - a.recent;  // the entries that compete
  const int lane = tid & 63, wave = tid >> 6;
  // 16 entries a thread and round, entry base + 1,024 k + tid: up to 16,384 are
  // read once and stay in registers, longer rows are read again by every pass
  const int32_t rounds = (length + kRound - 1) / kRound;
  uint32_t u[16];
  auto load = [&](int32_t base) {
    float x[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int32_t i = base + 1024 * k + tid;
      x[k] = w[i < length ? i : 0];
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) u[k] = weight_order(x[k]);
  };
  if (rounds == 1) load(0);

  uint32_t need = (uint32_t)(a.budget - a.sinks - a.recent);
  uint32_t prefix = 0;  // of the order word of the last entry that stays
  if (need > 0) {
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      hist[tid] = 0u;
      hist[tid + 1024] = 0u;
      __syncthreads();
      for (int32_t round = 0; round < rounds; ++round) {
        if (rounds > 1) load(round * kRound);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int32_t i = round * kRound + 1024 * k + tid;
          const bool in = i >= first && i < last && (pass == 0 || (u[k] >> (shift + bits)) == prefix);
          const uint32_t digit = (u[k] >> shift) & ((1u << bits) - 1u);
          // equal weights meet in one digit: a wave that shares one counts once (64
          // adds to one word took 16,384 equal weights from 16 to 51 us)
          const uint64_t on = __ballot(in);
          if (on == 0) continue;
          const uint32_t lead = __builtin_amdgcn_readlane(digit, __builtin_ctzll(on));
          if (__ballot(in && digit == lead) == on) {
            if (lane == __builtin_ctzll(on)) atomicAdd(&hist[lead], (uint32_t)__builtin_popcountll(on));
          } else if (in) {
            atomicAdd(&hist[digit], 1u);
          }
        }
      }
      __syncthreads();
      // from the largest digit down, the one that holds the need-th
      const int d0 = 2047 - 2 * tid, d1 = d0 - 1;
      const uint32_t c0 = hist[d0], c1 = hist[d1];
      uint32_t all;
      const uint32_t upto = block_scan(c0 + c1, part, &all), above = upto - c0 - c1;
      if (above < need && need <= upto) {
        const bool lower = need > above + c0;
        found[0] = (uint32_t)(lower ? d1 : d0);
        found[1] = need - above - (lower ? c0 : 0u);
      }
      __syncthreads();
      prefix = (prefix << bits) | found[0];
      need = found[1];
      __syncthreads();
    }
  } else {
    prefix = 0xffffffffu;  // above every weight: none of them stays
  }

  // in order: those above the last one's word, and `need` of those at it.  The
  // waves' counts of every 1,024 entries meet in LDS (high half: at the word).
  uint32_t over_done = 0, ties_done = 0;
  for (int32_t round = 0; round < rounds; ++round) {
    if (rounds > 1) load(round * kRound);
    uint64_t over[16], at[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int32_t i = round * kRound + 1024 * k + tid;
      const bool in = i < length, forced = i < first || i >= last;
      over[k] = __ballot(in && (forced || u[k] > prefix));
      at[k] = __ballot(in && !forced && u[k] == prefix && need > 0);
      if (lane == 0)
        hist[16 * k + wave] = (uint32_t)__builtin_popcountll(over[k]) | ((uint32_t)__builtin_popcountll(at[k]) << 16);
    }
    __syncthreads();
    const uint32_t mine = tid < 256 ? hist[tid] : 0u;
    uint32_t all;
    const uint32_t upto = block_scan(mine, part, &all);
    if (tid < 256) hist[tid] = upto - mine;
    __syncthreads();
    const uint64_t below = (1ull << lane) - 1ull;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const uint32_t prior = hist[16 * k + wave];
      const uint32_t ties = ties_done + (prior >> 16) + (uint32_t)__builtin_popcountll(at[k] & below);
      const bool stays = (over[k] >> lane & 1ull) || ((at[k] >> lane & 1ull) && ties < need);
      const uint32_t to = over_done + (prior & 0xffffu) + (uint32_t)__builtin_popcountll(over[k] & below) +
                          (ties < need ? ties : need);
      if (stays && to < (uint32_t)a.budget) kept[to] = round * kRound + 1024 * k + tid;
    }
    over_done += all & 0xffffu;
    ties_done += all >> 16;
    __syncthreads();
  }
}

struct CompactArgs {
  PagedCache c;
  const int32_t* kept;  // [B,KVH,budget], -1: nothing
  int32_t budget, KVH;
  const int32_t* to_tables;
  int64_t to_stride, to_width;
  const float* weights;  // [B,KVH,width], or null
  int64_t w_sb, w_sh;
  float* moved;  // [B,KVH,width] contiguous
  int32_t width;
};

// 64 kept entries a workgroup: D/8 threads copy 16 bytes each of a key and a
// value, four rows of loads in flight a thread.
template <int D>
__global__ __launch_bounds__(256) void paged_compact_kernel(CompactArgs a) {
  constexpr int kParts = D / 8, kRows = 256 / kParts, kSteps = 64 / kRows;
  const int tid = threadIdx.x, part = tid % kParts, r = tid / kParts;
  const int32_t b = (int32_t)blockIdx.z, h = (int32_t)blockIdx.y, j0 = (int32_t)blockIdx.x * 64;
  const int32_t* kept = a.kept + ((int64_t)b * a.KVH + h) * a.budget;
  const int32_t mask = (1 << a.c.page_shift) - 1;
  const int64_t room = a.c.table_width << a.c.page_shift, to_room = a.to_width << a.c.page_shift;
  uint4 kx[kSteps], vx[kSteps];
  int64_t to[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int32_t j = j0 + i * kRows + r;
    const int32_t e = j < a.budget ? kept[j] : -1;
    const bool in = e >= 0 && e < room && j < to_room;
    int32_t src = -1, dst = -1;
    if (in) {
      src = a.c.tables[b * a.c.table_stride + (e >> a.c.page_shift)];
      dst = a.to_tables[b * a.to_stride + (j >> a.c.page_shift)];
    }
    // (an entry that stays where it is needs no copy: one of 16 sequences of 4,096
    // moving took 85 us with copies of the others, 13 without)
    const bool ok = (uint32_t)src < (uint32_t)a.c.n_pages && (uint32_t)dst < (uint32_t)a.c.n_pages &&
                    (src != dst || ((e ^ j) & mask) != 0);
    const int64_t from = src * a.c.page_bytes + h * a.c.head_bytes + (int64_t)(e & mask) * a.c.slot_bytes + 16 * part;
    to[i] = ok ? dst * a.c.page_bytes + h * a.c.head_bytes + (int64_t)(j & mask) * a.c.slot_bytes + 16 * part : -1;
    kx[i] = uint4{0u, 0u, 0u, 0u};
    vx[i] = uint4{0u, 0u, 0u, 0u};
    if (ok) {
      kx[i] = *(const uint4*)(a.c.k + from);
      vx[i] = *(const uint4*)(a.c.v + from);
    }
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    if (to[i] >= 0) {
      *(uint4*)(a.c.k + to[i]) = kx[i];
      *(uint4*)(a.c.v + to[i]) = vx[i];
    }
  if (a.weights != nullptr && tid < 64 && j0 + tid < a.width) {
    const int32_t j = j0 + tid, e = j < a.budget ? kept[j] : -1;
    a.moved[((int64_t)b * a.KVH + h) * a.width + j] =
        e >= 0 && e < a.width ? a.weights[b * a.w_sb + h * a.w_sh + e] : 0.f;
  }
}

}  // namespace jkv

extern "C" {

int jkv_paged_select(const float* weights, int64_t weight_stride_b, int64_t weight_stride_h, const int32_t* lengths,
                     int64_t B, int64_t KVH, int64_t width, int64_t budget, int64_t sinks, int64_t recent,
                     int32_t* kept, int32_t* new_lengths, jkv_stream_t stream_) {
  using namespace jkv;
  JKV_CHECK_ARG(B >= 0 && B < 65536 && KVH > 0 && KVH < ((int64_t)1 << 20), "invalid eviction geometry");
  JKV_CHECK_ARG(width >= 0 && width < ((int64_t)1 << 30) && budget > 0 && budget < ((int64_t)1 << 30),
                "the budget must be positive");
  JKV_CHECK_ARG(sinks >= 0 && recent >= 0 && sinks <= budget && recent <= budget - sinks,
                "the first and the last entries that stay must fit the budget");
  if (B == 0) return JKV_OK;
  JKV_CHECK_ARG((weights || width == 0) && lengths && kept && new_lengths, "null buffer");
  SelectArgs a = {};
  a.weights = weights; a.stride_b = weight_stride_b; a.stride_h = weight_stride_h;
  a.lengths = lengths; a.kept = kept; a.new_lengths = new_lengths;
  a.width = (int32_t)width; a.budget = (int32_t)budget; a.sinks = (int32_t)sinks; a.recent = (int32_t)recent;
  hipLaunchKernelGGL(paged_select_kernel, dim3((uint32_t)KVH, (uint32_t)B), dim3(kSelectThreads), 0,
                     (hipStream_t)stream_, a);
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

int jkv_paged_compact(void* key_pages, void* value_pages, int32_t dtype, int64_t page_stride, int64_t head_stride,
                      int64_t slot_stride, int64_t n_pages, int64_t page_size, const int32_t* block_tables,
                      int64_t table_stride, int64_t table_width, const int32_t* kept, int64_t budget,
                      const int32_t* new_tables, int64_t new_table_stride, int64_t new_table_width, int64_t B,
                      int64_t KVH, int64_t D, const float* weights, int64_t weight_stride_b, int64_t weight_stride_h,
                      int64_t width, float* moved, jkv_stream_t stream_) {
  using namespace jkv;
  CompactArgs a = {};
  int rc = paged_cache_args(&a.c, key_pages, value_pages, page_stride, head_stride, slot_stride, n_pages, page_size,
                            block_tables, table_stride, table_width, nullptr, nullptr, nullptr, 0, 0, KVH, D,
                            0x7fffffff, dtype);
  if (rc != JKV_OK) return rc;
  JKV_CHECK_ARG(B >= 0 && B < 65536 && KVH < 65536, "invalid eviction geometry");
  JKV_CHECK_ARG(budget >= 0 && budget < ((int64_t)1 << 30) && width >= 0 && width < ((int64_t)1 << 30),
                "invalid kept entries");
  JKV_CHECK_ARG(new_table_width >= 0 && new_table_width < ((int64_t)1 << 27), "invalid block table");
  const int64_t rows = weights != nullptr && width > budget ? width : budget;
  if (B == 0 || rows == 0) return JKV_OK;
  JKV_CHECK_ARG(key_pages && value_pages && block_tables && kept && new_tables && (!weights || moved), "null buffer");
  a.kept = kept; a.budget = (int32_t)budget; a.KVH = (int32_t)KVH;
  a.to_tables = new_tables; a.to_stride = new_table_stride; a.to_width = new_table_width;
  a.weights = weights; a.w_sb = weight_stride_b; a.w_sh = weight_stride_h; a.moved = moved; a.width = (int32_t)width;
  JKV_CHECK_GRID(ceil_div(rows, 64), 256);
  const dim3 grid((uint32_t)ceil_div(rows, 64), (uint32_t)KVH, (uint32_t)B), block(256);
  if (D == 128) hipLaunchKernelGGL((paged_compact_kernel<128>), grid, block, 0, (hipStream_t)stream_, a);
  else hipLaunchKernelGGL((paged_compact_kernel<64>), grid, block, 0, (hipStream_t)stream_, a);
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

}  // extern "C"
