// Shared pieces of the paged-cache kernels: the cache as a kernel argument, its address arithmetic, the two 16-bit
// element types, and 8-bit elements as either of them.
#pragma once

#include <type_traits>

#include "gwa_common.h"

namespace {

// gwa_paged_cache as the kernels take it (checked by paged_check); strides in elements. Of an 8-bit cache k and v point
// at bytes, and ks and vs hold its rows' scales.
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
  uint8_t* ks;
  uint8_t* vs;
  int64_t s_page_stride, s_head_stride;
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

__device__ __forceinline__ int64_t paged_s_at(const PagedArgs& c, int page, int head, int slot) {
  return page * c.s_page_stride + head * c.s_head_stride + (slot & ((1 << c.page_shift) - 1));
}

// Eight e4m3 codes under a row's scale as eight values of T, by the conversions that take a scale: its exponent field is
// the scale byte, value = code * 2^(byte - 127) (byte 255: NaN). Exact in bf16 under the bytes 3 (its least code stands for
// 2^-133) to 246; past them, and in fp16, rounded where the type's subnormals do not hold the value, or infinite.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
template <class T>
__device__ __forceinline__ v4i widen8(uint32_t lo, uint32_t hi, float s) {
  if constexpr (std::is_same_v<T, Bf16>) {
    return (v4i){__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true))};
  } else {
    return (v4i){__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, false)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, true)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, false)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, true))};
  }
}

// Eight elements, and one, from place `at` of a pool (paged_at), as values of T; E8: of an 8-bit cache, s the row's scale
template <class T, bool E8>
__device__ __forceinline__ v4i held8(const uint16_t* pool, int64_t at, float s) {
  if constexpr (E8) {
    const uint2 w = *(const uint2*)((const uint8_t*)pool + at);
    return widen8<T>(w.x, w.y, s);
  } else {
    return *(const v4i*)(pool + at);
  }
}
template <class T, bool E8>
__device__ __forceinline__ float held1(const uint16_t* pool, int64_t at, float s) {
  if constexpr (E8) return T::load((uint16_t)widen8<T>(((const uint8_t*)pool)[at], 0, s)[0]);
  else return T::load(pool[at]);
}
// the scale of a slot's row in ks or vs; 1 for a 16-bit cache, whose elements have none
template <bool E8>
__device__ __forceinline__ float held_scale(const PagedArgs& c, const uint8_t* scales, int page, int head, int slot) {
  if constexpr (E8) return scale_of(scales[paged_s_at(c, page, head, slot)]);
  else return 1.0f;
}

// Host side: the checks every entry point shares, and the kernels' form of the cache.
// `scales`: of an 8-bit cache (`dtype` is then the type of its calls' q, k, v and o), whose elements are bytes: a row's
// 16-byte pieces hold 16 of them.
inline int paged_check(const char* what, const gwa_paged_cache* c, bool need_q, bool need_w, PagedArgs* a,
                       const gwa_paged_scales* scales = nullptr) {
  const int piece = scales ? 16 : 8;
  GWA_REQUIRE(c, "%s: null cache", what);
  GWA_REQUIRE(c->page_size >= 8 && c->page_size <= 4096 && (c->page_size & (c->page_size - 1)) == 0,
              "%s: page_size %d must be a power of two, 8 to 4096", what, c->page_size);
  GWA_REQUIRE(c->dtype == GWA_DT_BF16 || c->dtype == GWA_DT_F16, "%s: cache dtype %d is neither bf16 nor fp16", what,
              c->dtype);
  GWA_REQUIRE(c->head_dim >= piece && c->head_dim <= 256 && c->head_dim % piece == 0,
              "%s: head_dim %d must be a multiple of %d, %d to 256", what, c->head_dim, piece, piece);
  GWA_REQUIRE(c->kv_heads > 0 && c->kv_heads < 65536, "%s: kv_heads %d", what, c->kv_heads);
  GWA_REQUIRE(c->pages > 0 && c->pages < (1ll << 31), "%s: %lld pages", what, (long long)c->pages);
  GWA_REQUIRE(c->batch >= 0 && c->batch < 65536, "%s: batch %lld", what, (long long)c->batch);
  GWA_REQUIRE(c->table_width >= 0 && c->table_width * c->page_size < (1ll << 30) && c->table_stride >= c->table_width,
              "%s: table of %lld pages a row at stride %lld", what, (long long)c->table_width,
              (long long)c->table_stride);
  GWA_REQUIRE(c->page_stride % piece == 0 && c->head_stride % piece == 0 && c->slot_stride % piece == 0 && c->page_stride > 0 &&
                  c->head_stride > 0 && c->slot_stride >= c->head_dim && c->page_stride < (1ll << 31) &&
                  c->head_stride < (1ll << 31) && c->slot_stride * c->page_size < (1ll << 31),
              "%s: page, head and slot strides must be positive multiples of %d elements below 2^31", what, piece);
  GWA_REQUIRE(c->k && c->v && (c->batch == 0 || (c->kv_len && (c->table || c->table_width == 0))),
              "%s: null pointer", what);
  GWA_REQUIRE(!need_q || c->q_start, "%s: null q_start", what);
  GWA_REQUIRE(!need_w || c->w, "%s: the cache has no gathered weights", what);
  GWA_REQUIRE(!c->w || (c->w_page_stride > 0 && c->w_head_stride >= c->page_size), "%s: weight strides", what);
  GWA_REQUIRE(GWA_ALIGNED(c->k, 16) && GWA_ALIGNED(c->v, 16) && GWA_ALIGNED(c->w, 4),
              "%s: k and v must be 16-byte aligned", what);
  GWA_REQUIRE(!scales || (scales->k && scales->v && scales->page_stride > 0 && scales->head_stride >= c->page_size &&
                          scales->page_stride < (1ll << 31) && scales->head_stride < (1ll << 31)),
              "%s: the scales' pointers or strides", what);
  int shift = 0;
  while ((1 << shift) < c->page_size) ++shift;
  *a = PagedArgs{(uint16_t*)c->k, (uint16_t*)c->v, c->w, c->table, c->q_start, c->kv_len, c->page_stride,
                 c->head_stride, c->slot_stride, c->w_page_stride, c->w_head_stride, c->table_stride, (int)c->pages,
                 (int)c->batch, (int)(c->table_width * c->page_size), shift, c->kv_heads, scales ? scales->k : nullptr,
                 scales ? scales->v : nullptr, scales ? scales->page_stride : 0, scales ? scales->head_stride : 0};
  return GWA_OK;
}

}  // namespace
