// What the kernels over a paged K/V cache share: the cache's description, the
// sequences of a packed batch, and the rotary angles.
//
// Entry j of sequence b lies in slot j % page_size of page
// tables[b][j / page_size].  Keys are stored rotated.  A call's new tokens are
// packed: sequence b owns rows [starts[b], starts[b+1]) and they are its last
// entries, so token t of T sits at entry lengths[b] - T + t and at position
// positions[b] + t.  Entry counts and positions differ once entries have been
// evicted.
//
// Device integers are not trusted: starts are clamped to the rows there are,
// lengths to what a table row can list (and to the caller's bound), and a page number outside the pool
// is never followed (it reads as zeros, and nothing is written to it).
#pragma once

#include "jkv_common.h"

namespace jkv {

struct PagedCache {
  uint8_t* k;  // pools, addressed in bytes; K and V share their strides
  uint8_t* v;
  int64_t page_bytes, head_bytes, slot_bytes;
  int32_t n_pages, page_shift;
  const int32_t* tables;  // [B] rows table_stride apart, table_width pages each
  int64_t table_stride, table_width;
  const int32_t* lengths;    // [B] entries, the new tokens among them
  const int32_t* starts;     // [B+1] packed rows of each sequence, or null: one token a sequence
  const int32_t* positions;  // [B] position of each sequence's first new token, or null: its entry index
  int32_t N, B;              // packed rows, sequences
  int32_t top;               // entries a sequence can have: what its table row lists and the caller bounds
};

// one sequence of a batch
struct PagedSeq {
  int32_t row0, tokens;  // its packed rows
  int32_t length;        // entries
  int32_t pos0;          // position of its first new token
};

__device__ __forceinline__ int32_t clamp_i32(int32_t v, int32_t lo, int32_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

__device__ __forceinline__ int32_t paged_length(const PagedCache& c, int32_t b) {
  return clamp_i32(c.lengths[b], 0, c.top);
}

__device__ __forceinline__ void paged_rows(const PagedCache& c, int32_t b, int32_t* row0, int32_t* tokens) {
  if (c.starts == nullptr) {
    *row0 = b;
    *tokens = 1;
    return;
  }
  *row0 = clamp_i32(c.starts[b], 0, c.N);
  *tokens = clamp_i32(c.starts[b + 1], *row0, c.N) - *row0;
}

__device__ __forceinline__ PagedSeq paged_seq(const PagedCache& c, int32_t b) {
  PagedSeq s;
  paged_rows(c, b, &s.row0, &s.tokens);
  s.length = paged_length(c, b);
  s.pos0 = c.positions != nullptr ? c.positions[b] : s.length - s.tokens;
  return s;
}

// Turns (angle / 2 pi) per position of the D/2 frequencies, theta^(-2i/D) / 2 pi
// in 64 bits; by value in the kernel's arguments, so no table is kept.
struct RopeRates {
  double turns[64];
  int32_t on;
};

// cos and sin of position * frequency: the product and its fraction of a turn
// in 64 bits (32 lose the angle of far positions), the functions in 32.
__device__ __forceinline__ void rope_trig(double turns, int32_t pos, float* c, float* s) {
  const float f = (float)__builtin_amdgcn_fract(turns * (double)pos);
  *c = __builtin_amdgcn_cosf(f);
  *s = __builtin_amdgcn_sinf(f);
}

// Types of the cache and the queries: 16-bit floats.
template <int DT> struct Half16;
template <> struct Half16<JKV_F16> {
  typedef _Float16 T;
  typedef half8 V8;
  typedef half4 V4;
};
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
template <> struct Half16<JKV_BF16> {
  typedef __bf16 T;
  typedef bf16x8 V8;
  typedef bf16x4 V4;
};

// What the attention kernels of one call share.
struct PagedAttnArgs {
  PagedCache c;
  RopeRates rope;
  const uint8_t* q;
  int64_t qst, qsh;  // byte strides of a token and a head
  uint8_t* out;
  int64_t ost, osh;
  float* lse;      // [N,QH] natural log, or null
  float* weights;  // [B,KVH,..], or null
  int64_t wsb, wsh;
  int32_t accumulate;
  int32_t QH, KVH, per;   // per: query heads of a kv head
  int32_t window, sinks;  // at most kPagedMost
  int32_t max_new;
  // Base-2 scores are (q * q_mul) k * scale2.  q_mul is the softmax scale times
  // log2(e); where that passes a half, a power of two of it is left to scale2, so
  // that a rotated fp16 query (up to sqrt 2 of its size) cannot overflow.
  float q_mul, scale2;
  int32_t items;  // chunks: an upper bound of all sequences' row blocks
  int32_t item_rows;  // chunks: packed (token, head) rows of a block, 128 or 256
  int32_t fold;   // chunks: the item from which the order runs backwards
  // splits of the entries, joined by paged_join_kernel (one split: none)
  int32_t splits, split_tiles;
  int32_t waves;  // few rows: 1, or more waves a workgroup that join in LDS
  float2* part_ml;  // [splits][N*QH] reference maximum (base 2) and sum
  float* part_o;    // [splits][N*QH][D]
  float* lse2;      // [KVH][N][per] base-2 log-sum-exps for the weights, or null
  float* scores;    // few rows with weights: [B,KVH,max_new*per,score_width] base-2 scores, or null
  int64_t score_width;
  // what becomes of a score before its softmax (see ScoreShape), base 2
  float cap_mul, cap2;      // 2 scale log2(e) / cap and cap log2(e), or 0
  const float* slopes;      // [QH] a unit of distance, or null
  const int32_t* prefixes;  // [B] first entries that all of a sequence's rows see, or null
  int64_t v_head_bytes, v_slot_bytes;  // of values that lie without pages
  uint8_t* rest;  // [N,QH,D] of the output's type: what its rounding took off, or null
  uint8_t* q_parts;  // chunks with weights: [KVH][N][per] rotated queries, D of their leading and D of their trailing parts
};

// A score's form (a bit each; plain: the kernels without any of these).
enum { kFormPlain = 0, kFormShaped = 1, kFormCap = 2, kFormBias = 4 };

// A shaped score is cap * tanh(scale q k / cap) - slope * distance, in base 2.
// With E = exp(2x), tanh x = 1 - 2 / (1 + E): two transcendental instructions of
// 8 cycles each and three others of 4, where a rational function of x^2 as exact
// would take eleven and a reciprocal.  Of a cap c it is within 2e-7 c, and
// right at infinite scores.
struct ScoreShape {
  float mul, cap2, twice, slope2;
};
template <int FORM, typename Args> __device__ __forceinline__ ScoreShape score_shape(const Args& a, int32_t head) {
  ScoreShape s = {};
  if constexpr (FORM != kFormPlain) {
    s.mul = FORM & kFormCap ? a.cap_mul : a.scale2;
    s.cap2 = a.cap2;  // (0 without a cap)
    s.twice = -2.f * a.cap2;
    if constexpr (FORM & kFormBias) s.slope2 = a.slopes[head] * 1.4426950408889634f;
  }
  return s;
}
// In two steps, so that a caller can put other work between them.  The first, which
// with a cap leaves 1 + E, grows with the score (the host makes `mul` positive); the
// second adds `base`, cap2 less what the caller moves scores by.
template <int FORM> __device__ __forceinline__ float shape_first(const ScoreShape& s, float x) {
  if constexpr (FORM & kFormCap) x = 1.f + __builtin_amdgcn_exp2f(x * s.mul);
  return x;
}
template <int FORM> __device__ __forceinline__ float shape_second(const ScoreShape& s, float x, float distance, float base) {
  if constexpr (FORM & kFormCap) x = fmaf(s.twice, __builtin_amdgcn_rcpf(x), base);
  else x = fmaf(x, s.mul, base);
  if constexpr (FORM & kFormBias) x = fmaf(-s.slope2, fabsf(distance), x);
  return x;
}
template <int FORM> __device__ __forceinline__ float shape_score(const ScoreShape& s, float x, float distance) {
  return shape_second<FORM>(s, shape_first<FORM>(s, x), distance, s.cap2);
}
// What the first step of a masked score is: its second is -infinity.
template <int FORM> __device__ __forceinline__ float shape_masked() { return FORM & kFormCap ? 0.f : -INFINITY; }

// the first entries that all rows of a sequence see
__device__ __forceinline__ int32_t paged_prefix(const int32_t* prefixes, int32_t b, int32_t length) {
  return prefixes != nullptr ? clamp_i32(prefixes[b], 0, length) : 0;
}

// where lse2 holds row n * QH + head
__device__ __forceinline__ int64_t paged_lse2_at(int32_t N, int32_t per, int64_t row, int32_t QH) {
  const int32_t n = (int32_t)((uint32_t)row / (uint32_t)QH), head = (int32_t)(row - (int64_t)n * QH);
  const int32_t kvh = (int32_t)((uint32_t)head / (uint32_t)per);
  return ((int64_t)kvh * N + n) * per + (head - kvh * per);
}

static const int32_t kPagedMost = 0x3fffffff;  // entries of a sequence: sums of two of them stay in 32 bits

// launches; what they need of the workspace is in the arguments already
int paged_launch_few(const PagedAttnArgs& a, int32_t dtype, int64_t D, hipStream_t stream);
int paged_launch_few_weights(const PagedAttnArgs& a, hipStream_t stream);
int paged_launch_chunk(const PagedAttnArgs& a, int32_t dtype, int64_t D, hipStream_t stream);
int paged_launch_form_f16(const PagedAttnArgs& a, int form, bool few, int64_t D, hipStream_t stream);
int paged_launch_form_bf16(const PagedAttnArgs& a, int form, bool few, int64_t D, hipStream_t stream);
int paged_launch_join(const PagedAttnArgs& a, int32_t dtype, int64_t D, hipStream_t stream);

// The tiles of `size` entries that rows at entries first..last may see: `lead`
// tiles from entry 0 on that hold sinks, then those from tile `main` on.
struct PagedTiles {
  int32_t lead, main, count;
};
__host__ __device__ inline PagedTiles paged_tiles(int32_t first, int32_t last, int32_t window, int32_t sinks, int32_t size) {
  int32_t low = first - window + 1;  // the first entry of any row's window
  if (low < 0) low = 0;
  const int32_t seen = sinks < low ? sinks : low;
  PagedTiles t;
  t.main = low / size;
  t.lead = (seen + size - 1) / size;
  if (t.lead > t.main) t.lead = t.main;
  t.count = last < 0 ? 0 : t.lead + last / size - t.main + 1;
  return t;
}

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

// Transposing LDS read of 8-byte pieces at LDS byte address at: in each 16-lane
// block, lane 4j + e receives element e of the pieces that the block's lanes j,
// j+4, j+8, j+12 address (ds_read_b64_tr_b16).
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4_t lds_short4_t;
template <typename V4>
__device__ __forceinline__ V4 lds_read_tr(uint32_t at) {
  return __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)(size_t)at));
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(size_t)(const void __attribute__((address_space(3)))*)p;
}

// A masked weight is 0, but 0 times an infinite or NaN value is not.  Tiles with
// masked entries are therefore staged with such values as 0, and where one was
// met a second walk over those tiles adds it to the rows that do see it.  So are
// all tiles once a walk has ended in sums that are not finite: a visible weight
// is above 0 even where its 16 bits are not.

// w with the infinite and NaN halves 0; sets *found if there were any
template <int DT>
__device__ __forceinline__ uint4v finite_halves(uint4v w, bool* found) {
  constexpr uint32_t kExp = DT == JKV_F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool lo = (w[e] & kExp) == kExp, hi = ((w[e] >> 16) & kExp) == kExp;
    *found = *found || lo || hi;
    w[e] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu);
  }
  return w;
}
// v with the infinite and NaN elements 0
template <int DT, typename V8>
__device__ __forceinline__ V8 finite_part(V8 v) {
  bool found = false;
  return __builtin_bit_cast(V8, finite_halves<DT>(__builtin_bit_cast(uint4v, v), &found));
}
// `up`: 1 where v is +infinity or NaN; `down`: 1 where it is -infinity or NaN.
// Their products with the rows' visibility say which sums they belong to (both: NaN).
template <int DT, typename V8>
__device__ __forceinline__ void non_finite_marks(V8 v, V8* up, V8* down) {
  typedef typename Half16<DT>::T T;
  constexpr uint16_t kExp = DT == JKV_F16 ? 0x7c00 : 0x7f80;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint16_t u = __builtin_bit_cast(uint16_t, (T)v[e]);
    const bool bad = (u & kExp) == kExp, nan = (u & 0x7fff) > kExp, neg = u >> 15;
    (*up)[e] = bad && (nan || !neg) ? (T)1.f : (T)0.f;
    (*down)[e] = bad && (nan || neg) ? (T)1.f : (T)0.f;
  }
}
__device__ __forceinline__ float marked(float o, float up, float down) {
  return o + (up > 0.f ? INFINITY : 0.f) + (down > 0.f ? -INFINITY : 0.f);
}

// A launch's threads along x have to fit 32 bits.
#define JKV_CHECK_GRID(blocks, threads) \
  JKV_CHECK_ARG((int64_t)(blocks) * (threads) < ((int64_t)1 << 32), "grid too large")

// host side: fills c and the rates, or says what is wrong with them
int paged_cache_args(PagedCache* c, const void* k, const void* v, int64_t page_stride, int64_t head_stride,
                     int64_t slot_stride, int64_t n_pages, int64_t page_size, const int32_t* tables,
                     int64_t table_stride, int64_t table_width, const int32_t* lengths, const int32_t* starts,
                     const int32_t* positions, int64_t N, int64_t B, int64_t KVH, int64_t D, int64_t max_length,
                     int32_t dtype);
int paged_rope_args(RopeRates* r, double theta, int64_t D);
void paged_scale_args(PagedAttnArgs* a, float scale);
int paged_form_args(PagedAttnArgs* a, int* form, float scale, float softcap, const float* slopes, const int32_t* prefixes);

}  // namespace jkv
