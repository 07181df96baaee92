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

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)(uint32_t)(uint64_t)x) | (uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32);
}

// Direct-to-LDS copy of 16 bytes a lane: LDS [lds_addr + 16 lane, +16) <- [base + off, +16), base the same for the wave
// (a 64-bit address: pools pass 4 GiB). As asm for dma16's reason: the waits are the kernel's, so the compiler's wait
// counts must not include it.
__device__ __forceinline__ void copy16(uint32_t lds_addr, const void* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds_addr), "v"(off), "s"(base) : "memory", "m0");
}
// the same from an address of the lane's own
__device__ __forceinline__ void copy16(uint32_t lds_addr, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_addr), "v"(p) : "memory", "m0");
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

// What a row's softmax ends as, from its running maximum m (log2 domain) and sum l: the factor of its values and the log2
// of the whole sum. A row without keys, or all of whose scores are -inf, has m = -inf and l = 0: 0 and -inf. A NaN score raises no maximum but is in l,
// so that such a row's are NaN, whether or not it has seen other scores.
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
__device__ __forceinline__ float log2_sum(float m, float l) { return m + __builtin_amdgcn_logf(l); }
// the lse that a row's scores are measured against for the weights it gives; a row without a sum gives none
__device__ __forceinline__ float gather_lse2(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

// Sequence b's part of a call for one kv head: its rows (new token i, query head of the group) flattened as i * group + g
struct Rows {
  int t0, n, len, group, total;
  __device__ __forceinline__ int token_limit(int i, bool causal) const {  // last key new token i sees, -1 for none
    return causal ? max(len - n + i, -1) : len - 1;
  }
  __device__ __forceinline__ int limit(int row, bool causal) const { return token_limit(row / group, causal); }
};
__device__ __forceinline__ Rows rows_of(const PagedArgs& c, int b, int tokens, int group) {
  Rows r;
  paged_new(c, b, tokens, r.t0, r.n);
  r.len = paged_kv_len(c, b);
  r.group = group;
  r.total = r.n * group;
  return r;
}

// the same, for a sequence the whole wave works on: in scalar registers, which the copies' LDS addresses need
__device__ __forceinline__ Rows uniform_rows_of(const PagedArgs& c, int b, int tokens, int group) {
  const Rows r = rows_of(c, b, tokens, group);
  return Rows{uniform(r.t0), uniform(r.n), uniform(r.len), group, uniform(r.total)};
}

// The division of many-row work. A row tile is the rows of TT consecutive new tokens of one sequence and kv head; tiles
// are laid end to end (heads, then sequences, then tokens), each as long as the keys its last token sees plus a constant,
// and the line is cut into `shares` runs of equal length, one a workgroup. A cut inside a tile lies at the last whole
// BN keys before it. Lengths of tiles are linear in their index, so positions have closed forms; the last tile of a
// sequence counts as if it were whole.
struct TileLine {
  int first_keys, slope, none, tiles;  // keys of tile 0 (may be negative), keys more a tile, tiles without keys
  static constexpr int kFixed = 64;    // a tile's constant part, in keys: its queries, its first copies, its output
  // length of the first t tiles
  __device__ __forceinline__ int64_t before(int t) const {
    int64_t x = (int64_t)kFixed * t;
    if (t > none) x += (int64_t)(t - none) * first_keys + (int64_t)slope * ((int64_t)t * (t - 1) - (int64_t)none * (none - 1)) / 2;
    return x;
  }
  // the tile that position x < before(tiles) falls into; the whole wave calls it, 64 candidates at a time
  __device__ __forceinline__ int tile_at(int64_t x) const {
    int lo = 0, width = tiles;  // among tiles [lo, lo + width)
    while (width > 1) {
      const int step = (width + 63) / 64, mine = (int)(threadIdx.x & 63) * step;
      const int at = __popcll(__ballot(mine < width && before(lo + mine) <= x)) - 1;
      lo += at * step;
      width = min(step, width - at * step);
    }
    return lo;
  }
};
__device__ __forceinline__ TileLine tile_line(const Rows& r, int tt, bool causal) {
  TileLine l;
  l.tiles = (r.n + tt - 1) / tt;
  l.slope = causal ? tt : 0;
  l.first_keys = causal ? r.len - r.n + tt : r.len;
  // tile t has keys where first_keys + slope t > 0
  l.none = l.first_keys > 0 ? 0 : causal ? min(l.tiles, -l.first_keys / tt + 1) : l.tiles;
  return l;
}
// The sequences i .. i + 63 of a batch, one a lane: the lane's line, its length, and the length up to its end
struct LineLanes {
  TileLine line;
  int64_t own, upto;
};
__device__ __forceinline__ LineLanes line_lanes(const PagedArgs& c, int tokens, int tt, bool causal, int i) {
  const int lane = threadIdx.x & 63;
  LineLanes r = {};
  if (i + lane < c.batch) {
    r.line = tile_line(rows_of(c, i + lane, tokens, 1), tt, causal);
    r.own = r.line.before(r.line.tiles);
  }
  r.upto = r.own;
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) {
    const int64_t y = __shfl_up(r.upto, w);
    if (lane >= w) r.upto += y;
  }
  return r;
}
// A place on the line: a head's sequence, a tile of it, and how many whole BN keys of the tile lie before it (which may be
// more than the tile has)
struct Place {
  int h, b, tile, unit;
};
// One head's length, and the places of a share's start and of the next one's. The whole wave calls these; `first` are the
// lanes of the batch's first 64 sequences, which are all there are as a rule.
__device__ __forceinline__ int64_t head_line(const PagedArgs& c, int tokens, int tt, bool causal, const LineLanes& first) {
  int64_t all = uniform64(__shfl(first.upto, 63));
  for (int i = 64; i < c.batch; i += 64) all += uniform64(__shfl(line_lanes(c, tokens, tt, causal, i).upto, 63));
  return all;
}
template <int BN>
__device__ __forceinline__ Place place_of(const PagedArgs& c, int tokens, int tt, bool causal, int64_t per_head,
                                          const LineLanes& first, int64_t x) {
  Place p;
  // the head: as many as end at or before x
  p.h = 0;
  for (int i = 0; i < c.kv_heads; i += 64)
    p.h += __popcll(__ballot(i + (int)(threadIdx.x & 63) < c.kv_heads && (i + (int)(threadIdx.x & 63) + 1) * per_head <= x));
  p.h = uniform(p.h);
  p.b = c.batch, p.tile = p.unit = 0;
  if (p.h >= c.kv_heads) return p;  // the line's end
  x -= p.h * per_head;
  for (int i = 0; i < c.batch; i += 64) {
    LineLanes s = first;
    if (i > 0) s = line_lanes(c, tokens, tt, causal, i);
    const uint64_t past = __ballot(s.upto > x);
    if (past) {
      const int at = uniform(__ffsll((unsigned long long)past) - 1);
      x = uniform64(x - __shfl(s.upto - s.own, at));
      TileLine l;
      l.first_keys = uniform(__shfl(s.line.first_keys, at));
      l.slope = uniform(__shfl(s.line.slope, at));
      l.none = uniform(__shfl(s.line.none, at));
      l.tiles = uniform(__shfl(s.line.tiles, at));
      p.b = i + at;
      p.tile = uniform(l.tile_at(x));
      p.unit = (int)(x - l.before(p.tile)) / BN;
      break;
    }
    x = uniform64(x - __shfl(s.upto, 63));
  }
  p.b = uniform(p.b), p.tile = uniform(p.tile), p.unit = uniform(p.unit);
  return p;
}
// start of share i of n, a power of two
__device__ __forceinline__ int64_t share_start(int64_t all, int i, int n) { return all * i >> (__ffs(n) - 1); }

}  // namespace
