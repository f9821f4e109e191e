// Pages of a K/V cache copied to other pages of its pools, in all layers: what
// a forked sequence needs before it writes to a page that it shares.
//
// Memory bounds it: each byte that counts is read and written once, in 16-byte
// pieces, of keys and values both.  A workgroup takes a run of one page's rows
// (head, slot) in one layer.  Only the rows below a pair's entry count move.  Loads
// and stores that the caches need not keep: 402 MB of whole pages 187 -> 140 us
// (5.7 TB/s of both), the used parts of eight pages in 32 layers, 33 MB, 28 -> 15;
// two pieces a thread 138 and 15.6, eight 247 and 36.
#include "paged.h"

namespace jkv {

static const int kCopyThreads = 256;
static const int kCopyEach = 4;  // pieces a thread has in flight, of keys and of values

struct CopyArgs {
  PagedCache c;
  int64_t layer_bytes;
  const int32_t *sources, *targets, *entries;
  int32_t pieces, row_shift, runs;  // 16-byte pieces of a page, log2 of a row's, workgroups of a page
};

__global__ __launch_bounds__(kCopyThreads) void paged_copy_kernel(CopyArgs a) {
  const uint32_t pair = blockIdx.x / (uint32_t)a.runs, run = blockIdx.x - pair * (uint32_t)a.runs;
  const int32_t src = a.sources[pair], dst = a.targets[pair], size = 1 << a.c.page_shift;
  if ((uint32_t)src >= (uint32_t)a.c.n_pages || (uint32_t)dst >= (uint32_t)a.c.n_pages || src == dst) return;
  const int32_t count = a.entries != nullptr ? clamp_i32(a.entries[pair], 0, size) : size;
  const int64_t layer = blockIdx.y * a.layer_bytes, from = layer + src * a.c.page_bytes, to = layer + dst * a.c.page_bytes;
  uint4v k[kCopyEach], v[kCopyEach];
  int64_t off[kCopyEach];
#pragma unroll
  for (int e = 0; e < kCopyEach; ++e) {
    // piece i of the page: head, slot, part
    const int32_t i = (int32_t)((run * kCopyEach + e) * kCopyThreads + threadIdx.x);
    const int32_t part = i & ((1 << a.row_shift) - 1), slot = (i >> a.row_shift) & (size - 1);
    const bool on = i < a.pieces && slot < count;
    off[e] = on ? (i >> (a.row_shift + a.c.page_shift)) * a.c.head_bytes + slot * a.c.slot_bytes + 16 * part : -1;
    if (on) {
      k[e] = __builtin_nontemporal_load((const uint4v*)(a.c.k + from + off[e]));
      v[e] = __builtin_nontemporal_load((const uint4v*)(a.c.v + from + off[e]));
    }
  }
#pragma unroll
  for (int e = 0; e < kCopyEach; ++e)
    if (off[e] >= 0) {
      __builtin_nontemporal_store(k[e], (uint4v*)(a.c.k + to + off[e]));
      __builtin_nontemporal_store(v[e], (uint4v*)(a.c.v + to + off[e]));
    }
}

}  // namespace jkv

extern "C" {

int jkv_paged_copy(void* key_pages, void* value_pages, int32_t dtype, int64_t layers, int64_t layer_stride,
                   int64_t page_stride, int64_t head_stride, int64_t slot_stride, int64_t n_pages, int64_t page_size,
                   int64_t KVH, int64_t D, const int32_t* sources, const int32_t* targets, const int32_t* entries,
                   int64_t pairs, jkv_stream_t stream_) {
  using namespace jkv;
  CopyArgs a = {};
  int rc = paged_cache_args(&a.c, key_pages, value_pages, page_stride, head_stride, slot_stride, n_pages, page_size,
                            nullptr, 0, 0, nullptr, nullptr, nullptr, 0, 0, KVH, D, 0x7fffffff, dtype);
  if (rc != JKV_OK) return rc;
  JKV_CHECK_ARG(layers >= 0 && layers < 65536 && layer_stride >= 0 && layer_stride % 8 == 0,
                "layers must be fewer than 65536, their stride a multiple of 8 elements");
  JKV_CHECK_ARG(pairs >= 0 && pairs < ((int64_t)1 << 24) && KVH < ((int64_t)1 << 16), "too many pages or heads");
  if (pairs == 0 || layers == 0 || n_pages == 0) return JKV_OK;
  JKV_CHECK_ARG(key_pages && value_pages && sources && targets, "null buffer");
  a.layer_bytes = 2 * layer_stride;
  a.sources = sources; a.targets = targets; a.entries = entries;
  const int64_t pieces = page_size * (D / 8) * KVH;
  JKV_CHECK_ARG(pieces < ((int64_t)1 << 30), "pages too large");
  a.pieces = (int32_t)pieces; a.row_shift = D == 128 ? 4 : 3;
  a.runs = (int32_t)ceil_div(pieces, kCopyThreads * kCopyEach);
  JKV_CHECK_GRID(pairs * a.runs, kCopyThreads);
  hipLaunchKernelGGL(paged_copy_kernel, dim3((uint32_t)(pairs * a.runs), (uint32_t)layers), dim3(kCopyThreads), 0,
                     (hipStream_t)stream_, a);
  JKV_CHECK_LAUNCH();
  return JKV_OK;
}

}  // extern "C"
