// New tokens' keys and values into the pages of a K/V cache, keys rotated at
// their positions.
//
// One thread takes eight dims and their rotary partners of one key and the
// same dims of the value: 16-byte loads and stores throughout.  The rotation
// is fp32 products of the 16-bit key with fp32 cos/sin, rounded once to the
// cache's type.  Memory bounds it: 9,463 bf16 tokens of 8 heads of 128 in 15.6
// us, 5.0 TB/s; one token of 16 sequences in 3.1, a launch's latency.
#include <math.h>
#include <string.h>

#include "paged.h"

namespace jkv {

int paged_cache_args(PagedCache* c, const void* k, const void* v, int64_t page_stride, int64_t head_stride,
                     int64_t slot_stride, int64_t n_pages, int64_t page_size, const int32_t* tables,
                     int64_t table_stride, int64_t table_width, const int32_t* lengths, const int32_t* starts,
                     const int32_t* positions, int64_t N, int64_t B, int64_t KVH, int64_t D, int64_t max_length,
                     int32_t dtype) {
  JKV_CHECK_ARG(dtype == JKV_F16 || dtype == JKV_BF16, "paged caches hold fp16 or bf16, got dtype %d", dtype);
  JKV_CHECK_ARG(D == 64 || D == 128, "paged caches support head_dim 64 and 128, got %lld", (long long)D);
  JKV_CHECK_ARG(B >= 0 && N >= 0 && KVH > 0, "invalid paged geometry");
  JKV_CHECK_ARG(N < ((int64_t)1 << 30) && B < ((int64_t)1 << 24), "too many rows or sequences");
  JKV_CHECK_ARG(starts != nullptr || N == B, "without starts there is one new token a sequence");
  JKV_CHECK_ARG(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
                "the page size must be a power of two from 16 to 4096, got %lld", (long long)page_size);
  JKV_CHECK_ARG(n_pages >= 0 && n_pages < ((int64_t)1 << 31), "invalid page count");
  JKV_CHECK_ARG(table_width >= 0 && table_width < ((int64_t)1 << 27), "invalid block table");
  JKV_CHECK_ARG(page_stride >= 0 && head_stride >= 0, "page strides must not be negative");
  JKV_CHECK_ARG(page_stride % 8 == 0 && head_stride % 8 == 0 && slot_stride % 8 == 0 && slot_stride >= D &&
                    slot_stride < ((int64_t)1 << 22),
                "page strides must be multiples of 8 elements, slots at least a row apart");
  JKV_CHECK_ARG(((uintptr_t)k | (uintptr_t)v) % 16 == 0, "pages must be 16-byte aligned");
  if (B > 0 && N > 0) JKV_CHECK_ARG(k && v && tables && lengths, "null buffer");
  int shift = 4;
  while (((int64_t)1 << shift) < page_size) ++shift;
  c->k = (uint8_t*)k; c->v = (uint8_t*)v;
  c->page_bytes = 2 * page_stride; c->head_bytes = 2 * head_stride; c->slot_bytes = 2 * slot_stride;
  c->n_pages = (int32_t)n_pages; c->page_shift = shift;
  c->tables = tables; c->table_stride = table_stride; c->table_width = table_width;
  c->lengths = lengths; c->starts = starts; c->positions = positions;
  c->N = (int32_t)N; c->B = (int32_t)B;
  const int64_t room = table_width << shift, most = room < kPagedMost ? room : kPagedMost;
  c->top = (int32_t)(max_length < most ? max_length : most);
  return JKV_OK;
}

int paged_rope_args(RopeRates* r, double theta, int64_t D) {
  JKV_CHECK_ARG(theta == 0.0 || (theta > 0.0 && isfinite(theta)), "the rotary base must be positive, or 0 for none");
  r->on = theta > 0.0;
  if (!r->on) return JKV_OK;
  // a thread's last rates: 64 powers cost a small call a microsecond or two
  static thread_local double last_theta = 0.0;
  static thread_local int64_t last_dim = 0;
  static thread_local double last[64];
  if (last_theta != theta || last_dim != D) {
    for (int i = 0; i < 64; ++i)
      last[i] = i < D / 2 ? pow(theta, -2.0 * i / (double)D) / 6.283185307179586476925286766559 : 0.0;
    last_theta = theta;
    last_dim = D;
  }
  memcpy(r->turns, last, sizeof(last));
  return JKV_OK;
}

struct AppendArgs {
  PagedCache c;
  RopeRates rope;
  const uint8_t* key;
  const uint8_t* value;
  int64_t kst, ksh, vst, vsh;  // byte strides of a token and a head
  int32_t KVH;
};

template <int DT, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  typedef typename Half16<DT>::T T;
  typedef typename Half16<DT>::V8 V8;
  constexpr int kParts = D / 16;  // threads of one (token, head)
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t total = (int64_t)a.c.N * a.KVH * kParts;
  if (at >= total) return;
  const int part = (int)(at % kParts);
  const int64_t th = at / kParts;
  const int32_t n = (int32_t)(th / a.KVH), h = (int32_t)(th - (int64_t)n * a.KVH);
  // the sequence of row n: the last one that starts at or before it
  int32_t b = n;
  if (a.c.starts != nullptr) {
    int32_t lo = 0, hi = a.c.B;  // starts[lo] <= n < starts[hi]
    if (a.c.B == 0 || n < a.c.starts[0] || n >= a.c.starts[a.c.B]) return;
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (a.c.starts[mid] <= n) lo = mid; else hi = mid;
    }
    b = lo;
  }
  const PagedSeq s = paged_seq(a.c, b);
  const int32_t t = n - s.row0, entry = s.length - s.tokens + t;
  if (t < 0 || t >= s.tokens || entry < 0) return;
  const int32_t page = a.c.tables[b * a.c.table_stride + (entry >> a.c.page_shift)];
  if ((uint32_t)page >= (uint32_t)a.c.n_pages) return;
  const int64_t to = page * a.c.page_bytes + h * a.c.head_bytes +
                     (int64_t)(entry & ((1 << a.c.page_shift) - 1)) * a.c.slot_bytes + 16 * part;
  const uint8_t* kp = a.key + n * a.kst + h * a.ksh + 16 * part;
  const uint8_t* vp = a.value + n * a.vst + h * a.vsh + 16 * part;
  V8 x0 = *(const V8*)kp, x1 = *(const V8*)(kp + D);
  const V8 v0 = *(const V8*)vp, v1 = *(const V8*)(vp + D);
  if (a.rope.on) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float c, sn;
      rope_trig(a.rope.turns[8 * part + e], s.pos0 + t, &c, &sn);
      const float u = (float)x0[e], w = (float)x1[e];
      x0[e] = (T)(u * c - w * sn);
      x1[e] = (T)(w * c + u * sn);
    }
  }
  *(V8*)(a.c.k + to) = x0;
  *(V8*)(a.c.k + to + D) = x1;
  *(V8*)(a.c.v + to) = v0;
  *(V8*)(a.c.v + to + D) = v1;
}

}  // namespace jkv

extern "C" {

int jkv_paged_append(const void* key, int64_t key_stride_t, int64_t key_stride_h, const void* value,
                     int64_t value_stride_t, int64_t value_stride_h, int32_t dtype, void* key_pages,
                     void* value_pages, int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                     int64_t n_pages, int64_t page_size, const int32_t* block_tables, int64_t table_stride,
                     int64_t table_width, const int32_t* lengths, const int32_t* starts, const int32_t* positions,
                     int64_t N, int64_t B, int64_t KVH, int64_t D, double rope_theta, jkv_stream_t stream_) {
  using namespace jkv;
  hipStream_t stream = (hipStream_t)stream_;
  AppendArgs a = {};
  int rc = paged_cache_args(&a.c, key_pages, value_pages, page_stride, head_stride, slot_stride, n_pages, page_size,
                            block_tables, table_stride, table_width, lengths, starts, positions, N, B, KVH, D, 0x7fffffff,
                            dtype);
  if (rc != JKV_OK) return rc;
  rc = paged_rope_args(&a.rope, rope_theta, D);
  if (rc != JKV_OK) return rc;
  const int64_t strides[4] = {key_stride_t, key_stride_h, value_stride_t, value_stride_h};
  for (int i = 0; i < 4; ++i)
    JKV_CHECK_ARG(strides[i] % 8 == 0, "token and head strides must be multiples of 8 elements");
  JKV_CHECK_ARG(((uintptr_t)key | (uintptr_t)value) % 16 == 0, "keys and values must be 16-byte aligned");
  if (N == 0 || B == 0) return JKV_OK;
  JKV_CHECK_ARG(key && value, "null buffer");
  a.key = (const uint8_t*)key; a.kst = 2 * key_stride_t; a.ksh = 2 * key_stride_h;
  a.value = (const uint8_t*)value; a.vst = 2 * value_stride_t; a.vsh = 2 * value_stride_h;
  a.KVH = (int32_t)KVH;
  JKV_CHECK_ARG(KVH < ((int64_t)1 << 20), "too many kv heads");
  const int64_t blocks = ceil_div(N * KVH * (D / 16), 256);
  JKV_CHECK_GRID(blocks, 256);
  const dim3 grid((uint32_t)blocks), block(256);
  if (dtype == JKV_F16 && D == 128) hipLaunchKernelGGL((paged_append_kernel<JKV_F16, 128>), grid, block, 0, stream, a);
  else if (dtype == JKV_F16) hipLaunchKernelGGL((paged_append_kernel<JKV_F16, 64>), grid, block, 0, stream, a);
  else if (D == 128) hipLaunchKernelGGL((paged_append_kernel<JKV_BF16, 128>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((paged_append_kernel<JKV_BF16, 64>), grid, block, 0, stream, a);
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

}  // extern "C"
