// Pieces of the matrix-core attention kernels over a paged cache: the direct-to-LDS copy from 64-bit addresses, the
// MFMA forms of the two element types, LDS swizzles and reads.
#pragma once

#include "fp6_gemm_common.h"
#include "paged_common.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

typedef short v4s_ __attribute__((ext_vector_type(4)));
typedef short v2s_ __attribute__((ext_vector_type(2)));
typedef _Float16 v8h_ __attribute__((ext_vector_type(8)));
typedef float v2f_pm __attribute__((ext_vector_type(2)));
typedef _Float16 v2h_pm __attribute__((ext_vector_type(2)));

template <class T>
struct Mfma;
template <>
struct Mfma<Bf16> {
  static __device__ __forceinline__ v16f wide(v4i a, v4i b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ v4f tall(v4i a, v4i b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ int pack(float a, float b) { return (int)pack_bf16x2_rn(a, b); }
  static constexpr uint32_t kExp = 0x7f80u;  // an element's exponent bits: all set in infinities and NaN
};
template <>
struct Mfma<Fp16> {
  static __device__ __forceinline__ v16f wide(v4i a, v4i b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h_, a), __builtin_bit_cast(v8h_, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ v4f tall(v4i a, v4i b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h_, a), __builtin_bit_cast(v8h_, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ int pack(float a, float b) {
    return __builtin_bit_cast(int, __builtin_convertvector((v2f_pm){a, b}, v2h_pm));
  }
  static constexpr uint32_t kExp = 0x7c00u;
};

// Direct-to-LDS copy of 16 bytes a lane from a 64-bit address: LDS [lds_addr + 16 lane, +16) <- [p, +16). As asm for
// dma16's reason: the waits are the kernel's, so the compiler's wait counts must not include it.
__device__ __forceinline__ void copy16(uint32_t lds_addr, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_addr), "v"(p) : "memory", "m0");
}

__device__ __forceinline__ v4s_ lds_read_tr(const uint8_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s_*)(uintptr_t)p);
}
__device__ __forceinline__ v4i two_halves(v4s_ a, v4s_ b) {
  return (v4i){__builtin_bit_cast(int, (v2s_){a[0], a[1]}), __builtin_bit_cast(int, (v2s_){a[2], a[3]}),
               __builtin_bit_cast(int, (v2s_){b[0], b[1]}), __builtin_bit_cast(int, (v2s_){b[2], b[3]})};
}

// Slot of 16-byte chunk ch in row r of an LDS tile of rows of D elements (CH = D / 8 chunks, 256 or 128 bytes). K: 16
// lanes that read one chunk of 16 consecutive rows touch all 16 chunk places of 256 bytes. V: the transposing
// reads take 64 bytes of 4 consecutive rows at once, which land in four different quarters of 256 bytes.
template <int D>
__device__ __forceinline__ int k_place(int ch, int r) {
  return D == 128 ? ch ^ (r & 15) : ch ^ ((r >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int v_place(int ch, int r) {
  return D == 128 ? ch ^ (4 * (r & 3)) : ch ^ (4 * ((r >> 1) & 1));
}

// Infinities and NaN among eight 16-bit elements become 0 in x; whether there were any.
template <class T>
__device__ __forceinline__ bool take_nonfinite(v4i& x) {
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (uint32_t)x[i];
    const bool lo = (w & Mfma<T>::kExp) == Mfma<T>::kExp, hi = ((w >> 16) & Mfma<T>::kExp) == Mfma<T>::kExp;
    any |= lo || hi;
    x[i] = (int)(w & (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu));
  }
  return any;
}

// Sequence b's part of a call for one kv head: its rows (new token i, query head of the group) flattened as i * group + g
struct Rows {
  int t0, n, len, group, total;
  __device__ __forceinline__ int limit(int row, bool causal) const {  // last key the row sees, -1 for none
    return causal ? max(len - n + row / group, -1) : len - 1;
  }
};
__device__ __forceinline__ Rows rows_of(const PagedArgs& c, int b, int tokens, int group) {
  Rows r;
  paged_new(c, b, tokens, r.t0, r.n);
  r.len = paged_kv_len(c, b);
  r.group = group;
  r.total = r.n * group;
  return r;
}

}  // namespace
