// Rotary positions as the paged-cache kernels apply them, and where a new token's row goes.
#pragma once

#include "paged_common.h"

namespace {

// 8 consecutive elements of the three element types as fp32, in 16-byte pieces
template <int DT>
__device__ __forceinline__ void unpack8(const v4i& r, float (&f)[8]) {  // of the two 16-bit types
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (uint32_t)r[i];
    f[2 * i] = DT == GWA_DT_BF16 ? bf16_lo(w) : f16_bits_to_f32((uint16_t)w);
    f[2 * i + 1] = DT == GWA_DT_BF16 ? bf16_hi(w) : f16_bits_to_f32((uint16_t)(w >> 16));
  }
}
template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&f)[8]) {
  if constexpr (DT == GWA_DT_F32) {
    const float4* p = (const float4*)((const float*)base + at);
    const float4 a = p[0], b = p[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    unpack8<DT>(*(const v4i*)((const uint16_t*)base + at), f);
  }
}
template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t at, const float (&f)[8]) {
  if constexpr (DT == GWA_DT_F32) {
    float4* p = (float4*)((float*)base + at);
    p[0] = make_float4(f[0], f[1], f[2], f[3]);
    p[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    v4i r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = (int)(DT == GWA_DT_BF16 ? Bf16::pack(f[2 * i], f[2 * i + 1]) : Fp16::pack(f[2 * i], f[2 * i + 1]));
    *(v4i*)((uint16_t*)base + at) = r;
  }
}
template <int DT>
__device__ __forceinline__ float load1(const void* base, int64_t at) {
  if constexpr (DT == GWA_DT_F32) return ((const float*)base)[at];
  else return DT == GWA_DT_BF16 ? Bf16::load(((const uint16_t*)base)[at]) : Fp16::load(((const uint16_t*)base)[at]);
}
template <int DT>
__device__ __forceinline__ void store1(void* base, int64_t at, float f) {
  if constexpr (DT == GWA_DT_F32) ((float*)base)[at] = f;
  else ((uint16_t*)base)[at] = DT == GWA_DT_BF16 ? f32_to_bf16(f) : f32_to_f16_bits(f);
}

struct Rotation {
  const float* cos_t;
  const float* sin_t;
  const int32_t* positions;
  int64_t table_rows;
  int rot, interleaved;
  float sign;  // -1 rotates back
};

__device__ __forceinline__ int64_t table_row(const Rotation& r, int64_t t) {
  int64_t p = r.positions ? r.positions[t] : t;
  p = min(max(p, (int64_t)0), r.table_rows - 1);
  return p * (r.rot / 2);
}

// Elements a unit of work covers: 16 with VEC (8 pairs, or 16 channels past the rotated ones; both halves of the
// half layout lie on 16-byte pieces then), else one pair / two channels: the channels c0 and c1 where each part of it
// begins, and whether it lies past the rotated ones.
template <bool VEC>
__device__ __forceinline__ bool unit_channels(const Rotation& r, int unit, int& c0, int& c1) {
  constexpr int N = VEC ? 8 : 1;
  const bool tail = 2 * N * unit >= r.rot;
  // first and second piece: the pairs' two halves, or neighbours
  c0 = tail || r.interleaved ? 2 * N * unit : N * unit;
  c1 = tail || r.interleaved ? c0 + N : c0 + r.rot / 2;
  return tail;
}
// a unit's pairs turned by their cosines and sines
template <int N>
__device__ __forceinline__ void turn_unit(const Rotation& r, float (&a)[N], float (&b)[N], const float (&c)[N],
                                          float (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] *= r.sign;
  if (N > 1 && r.interleaved) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float e = a[2 * i], o = a[2 * i + 1];
      a[2 * i] = fmaf(e, c[i], -o * s[i]);
      a[2 * i + 1] = fmaf(e, s[i], o * c[i]);
      const float e2 = b[2 * i], o2 = b[2 * i + 1];
      b[2 * i] = fmaf(e2, c[N / 2 + i], -o2 * s[N / 2 + i]);
      b[2 * i + 1] = fmaf(e2, s[N / 2 + i], o2 * c[N / 2 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = a[i], o = b[i];
      a[i] = fmaf(e, c[i], -o * s[i]);
      b[i] = fmaf(e, s[i], o * c[i]);
    }
  }
}
// A unit's rotated values
template <int DT, bool VEC>
__device__ __forceinline__ void rotated_unit(const void* x, int64_t xo, const Rotation& r, int64_t row, int unit, int& c0,
                                             int& c1, float (&a)[VEC ? 8 : 1], float (&b)[VEC ? 8 : 1]) {
  const bool tail = unit_channels<VEC>(r, unit, c0, c1);
  if constexpr (VEC) {
    if constexpr (DT == GWA_DT_F32) {
      load8<DT>(x, xo + c0, a);
      load8<DT>(x, xo + c1, b);
      if (!tail) {
        float c[8], s[8];
        load8<GWA_DT_F32>(r.cos_t, row + 8 * unit, c);
        load8<GWA_DT_F32>(r.sin_t, row + 8 * unit, s);
        turn_unit<8>(r, a, b, c, s);
      }
    } else {
      const v4i xa = *(const v4i*)((const uint16_t*)x + xo + c0), xb = *(const v4i*)((const uint16_t*)x + xo + c1);
      float c[8], s[8];
      if (!tail) {
        load8<GWA_DT_F32>(r.cos_t, row + 8 * unit, c);
        load8<GWA_DT_F32>(r.sin_t, row + 8 * unit, s);
      }
      __builtin_amdgcn_sched_barrier(0);
      unpack8<DT>(xa, a);
      unpack8<DT>(xb, b);
      if (!tail) turn_unit<8>(r, a, b, c, s);
    }
  } else {
    a[0] = load1<DT>(x, xo + c0), b[0] = load1<DT>(x, xo + c1);
    if (!tail) {
      float c[1] = {r.cos_t[row + unit]}, s[1] = {r.sin_t[row + unit]};
      turn_unit<1>(r, a, b, c, s);
    }
  }
}
// One unit from x to y; it reads all it writes before it writes, so x and y may be the same.
template <int DT, bool VEC>
__device__ __forceinline__ void rotate_unit(const void* x, int64_t xo, void* y, int64_t yo, const Rotation& r,
                                            int64_t row, int unit) {
  int c0, c1;
  float a[VEC ? 8 : 1], b[VEC ? 8 : 1];
  rotated_unit<DT, VEC>(x, xo, r, row, unit, c0, c1, a, b);
  if constexpr (VEC) {
    store8<DT>(y, yo + c0, a);
    store8<DT>(y, yo + c1, b);
  } else {
    store1<DT>(y, yo + c0, a[0]);
    store1<DT>(y, yo + c1, b[0]);
  }
}

// The sequence of a new token: how many end at or before it (q_start ascends; empty ones end where they start). The whole
// wave calls it, for one token.
__device__ __forceinline__ int token_sequence(const PagedArgs& c, int t) {
  const int lane = threadIdx.x & 63;
  int b = 0;
  for (int i = 0; i < c.batch; i += 64)
    b += __popcll(__ballot(i + lane < c.batch && c.q_start[min(i + lane, c.batch - 1) + 1] <= t));
  return b;
}
// The page and slot of a new token of sequence b; slot -1: none (a token of no sequence, a slot before the first or past the
// table)
struct TokenPlace {
  int page, slot;
};
__device__ __forceinline__ TokenPlace token_place(const PagedArgs& c, int b, int t, int tokens) {
  TokenPlace p = {0, -1};
  if (b < c.batch) {
    int t0, n;
    paged_new(c, b, tokens, t0, n);
    const int64_t place = (int64_t)c.kv_len[b] - n + (t - t0);
    if (t >= t0 && t - t0 < n && place >= 0 && place < c.capacity) {
      p.slot = (int)place;
      p.page = paged_page(c, c.table + b * c.table_stride, p.slot);
    }
  }
  return p;
}

inline int rotation_check(const char* what, const float* cos_t, const float* sin_t, int64_t table_rows, int64_t head_dim,
                   int64_t rot) {
  GWA_REQUIRE(rot >= 0 && rot <= head_dim && rot % 2 == 0, "%s: %lld rotated channels of %lld (an even number expected)",
              what, (long long)rot, (long long)head_dim);
  GWA_REQUIRE(rot == 0 || (cos_t && sin_t && table_rows > 0 && table_rows < (1ll << 31)),
              "%s: a table of %lld positions", what, (long long)table_rows);
  return GWA_OK;
}

// whether every unit of 16 elements lies on 16-byte pieces of x and y and of the tables
inline bool vector_units(int64_t head_dim, int64_t rot, const float* cos_t, const float* sin_t) {
  return head_dim % 16 == 0 && rot % 16 == 0 && (rot == 0 || (GWA_ALIGNED(cos_t, 16) && GWA_ALIGNED(sin_t, 16)));
}
inline bool vector_operand(const void* p, int64_t ldt, int64_t ldh, int elem) {
  return GWA_ALIGNED(p, 16) && ldt * elem % 16 == 0 && ldh * elem % 16 == 0;
}

}  // namespace
