// Shared pieces of the paged-cache kernels: the cache as a kernel argument, its address arithmetic, and the two
// 16-bit element types.
#pragma once

#include "gwa_common.h"

namespace {

// gwa_paged_cache as the kernels take it (checked by paged_check); strides in elements
struct PagedArgs {
  uint16_t* k;
  uint16_t* v;
  float* w;
  const int32_t* table;
  const int32_t* q_start;
  const int32_t* kv_len;
  int64_t page_stride, head_stride, slot_stride, w_page_stride, w_head_stride, table_stride;
  int pages, batch, capacity;  // capacity: slots a table row can address
  int page_shift, kv_heads;
};

struct Bf16 {
  static __device__ __forceinline__ float load(uint16_t b) { return bf16_to_f32(b); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2_rn(a, b); }
};
struct Fp16 {
  static __device__ __forceinline__ float load(uint16_t b) { return f16_bits_to_f32(b); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_f16x2(a, b); }
};

// Keys of sequence b, held inside what its table row can address, and its new tokens' rows [t0, t0 + n)
__device__ __forceinline__ int paged_kv_len(const PagedArgs& c, int b) { return min(max(c.kv_len[b], 0), c.capacity); }
__device__ __forceinline__ void paged_new(const PagedArgs& c, int b, int tokens, int& t0, int& n) {
  t0 = min(max(c.q_start[b], 0), tokens);
  n = min(max(c.q_start[b + 1], t0), tokens) - t0;
}
// page holding slot (0 <= slot < capacity) of sequence b; an id outside the pool reads as its nearest page
__device__ __forceinline__ int paged_page(const PagedArgs& c, const int32_t* row, int slot) {
  return min(max(row[slot >> c.page_shift], 0), c.pages - 1);
}
__device__ __forceinline__ int64_t paged_at(const PagedArgs& c, int page, int head, int slot) {
  return page * c.page_stride + head * c.head_stride + (slot & ((1 << c.page_shift) - 1)) * c.slot_stride;
}
__device__ __forceinline__ int64_t paged_w_at(const PagedArgs& c, int page, int head, int slot) {
  return page * c.w_page_stride + head * c.w_head_stride + (slot & ((1 << c.page_shift) - 1));
}

// Host side: the checks every entry point shares, and the kernels' form of the cache.
inline int paged_check(const char* what, const gwa_paged_cache* c, bool need_q, bool need_w, PagedArgs* a) {
  GWA_REQUIRE(c, "%s: null cache", what);
  GWA_REQUIRE(c->page_size >= 8 && c->page_size <= 4096 && (c->page_size & (c->page_size - 1)) == 0,
              "%s: page_size %d must be a power of two, 8 to 4096", what, c->page_size);
  GWA_REQUIRE(c->dtype == GWA_DT_BF16 || c->dtype == GWA_DT_F16, "%s: cache dtype %d is neither bf16 nor fp16", what,
              c->dtype);
  GWA_REQUIRE(c->head_dim >= 8 && c->head_dim <= 256 && c->head_dim % 8 == 0,
              "%s: head_dim %d must be a multiple of 8, 8 to 256", what, c->head_dim);
  GWA_REQUIRE(c->kv_heads > 0 && c->kv_heads < 65536, "%s: kv_heads %d", what, c->kv_heads);
  GWA_REQUIRE(c->pages > 0 && c->pages < (1ll << 31), "%s: %lld pages", what, (long long)c->pages);
  GWA_REQUIRE(c->batch >= 0 && c->batch < 65536, "%s: batch %lld", what, (long long)c->batch);
  GWA_REQUIRE(c->table_width >= 0 && c->table_width * c->page_size < (1ll << 30) && c->table_stride >= c->table_width,
              "%s: table of %lld pages a row at stride %lld", what, (long long)c->table_width,
              (long long)c->table_stride);
  GWA_REQUIRE(c->page_stride % 8 == 0 && c->head_stride % 8 == 0 && c->slot_stride % 8 == 0 && c->page_stride > 0 &&
                  c->head_stride > 0 && c->slot_stride >= c->head_dim && c->page_stride < (1ll << 31) &&
                  c->head_stride < (1ll << 31) && c->slot_stride * c->page_size < (1ll << 31),
              "%s: page, head and slot strides must be positive multiples of 8 elements below 2^31", what);
  GWA_REQUIRE(c->k && c->v && (c->batch == 0 || (c->kv_len && (c->table || c->table_width == 0))),
              "%s: null pointer", what);
  GWA_REQUIRE(!need_q || c->q_start, "%s: null q_start", what);
  GWA_REQUIRE(!need_w || c->w, "%s: the cache has no gathered weights", what);
  GWA_REQUIRE(!c->w || (c->w_page_stride > 0 && c->w_head_stride >= c->page_size), "%s: weight strides", what);
  GWA_REQUIRE(GWA_ALIGNED(c->k, 16) && GWA_ALIGNED(c->v, 16) && GWA_ALIGNED(c->w, 4),
              "%s: k and v must be 16-byte aligned", what);
  int shift = 0;
  while ((1 << shift) < c->page_size) ++shift;
  *a = PagedArgs{(uint16_t*)c->k, (uint16_t*)c->v, c->w, c->table, c->q_start, c->kv_len, c->page_stride,
                 c->head_stride, c->slot_stride, c->w_page_stride, c->w_head_stride, c->table_stride, (int)c->pages,
                 (int)c->batch, (int)(c->table_width * c->page_size), shift, c->kv_heads};
  return GWA_OK;
}

}  // namespace
