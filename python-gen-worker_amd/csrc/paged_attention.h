// Attention of new tokens over a paged key/value cache, with the keys' attention weight gathered on request: the kernels
// and the choice among them, of a 16-bit cache and (E8) of an 8-bit one, whose e4m3 codes become values of the call's
// 16-bit type T on their way to the matrix cores (widen8).
#pragma once
#include <algorithm>
#include <type_traits>

#include "paged_mfma.h"

namespace {

constexpr int kCus = 256;  // MI355X

// One call's operands, as the matrix-core kernels take them. Partial results (fp32, each normalised by its own sum, with
// the log2 of that sum) of key split s in o_part [s][tokens * heads][D] and lse_part [s][tokens * heads]; of a share
// (many rows) in [2 * shares][rows of a tile].
struct AttnArgs {
  PagedArgs c;
  const uint16_t* q;
  int64_t ldqt, ldqh;
  uint16_t* o;
  float* lse;
  float* o_part;
  float* lse_part;
  int4* cuts;             // [shares]: a share's cut tiles, see Cut
  float* scores;          // [tokens * heads][score_stride] in the log2 domain, or NULL
  float* w_part;
  int64_t score_stride;
  int tokens, heads, splits, split_keys, tiles, shares;
  float c_log2;
  int causal;
};

// s + the dot product of eight 16-bit elements each, fp32
template <class T>
__device__ __forceinline__ float dot8(v4i x, v4i y, float s) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    s = fmaf(T::load((uint16_t)x[e]), T::load((uint16_t)y[e]), s);
    s = fmaf(T::load((uint16_t)((uint32_t)x[e] >> 16)), T::load((uint16_t)((uint32_t)y[e] >> 16)), s);
  }
  return s;
}

// What a share says of the row tiles that its ends cut, for the join: x: 0, 1 or 2: no part of a tile that an earlier share
// began, one that later shares continue, one that ends the tile; y: rows of a tile that it begins and later shares
// continue (0: none), which start at token z, kv head w. Every share's workgroup sets its own; thread 0 writes.
__device__ __forceinline__ void no_cuts(const AttnArgs& a, int share) {
  if (threadIdx.x == 0) a.cuts[share] = make_int4(0, 0, 0, 0);
}
__device__ __forceinline__ void set_cut(const AttnArgs& a, int share, bool begun, bool ends, int rows, int token, int h) {
  if (threadIdx.x != 0) return;
  if (begun) {
    a.cuts[share].x = ends ? 2 : 1;
  } else {
    a.cuts[share].y = rows, a.cuts[share].z = token, a.cuts[share].w = h;
  }
}

// ---------------------------------------------------------------------------
// any head_dim: one wave per (new token, query head)
// ---------------------------------------------------------------------------
constexpr int RW_WAVES = 4, RW_MAX_D = 256;

// q . key of one lane's key, fp32; q in LDS, the key's row read in 16-byte pieces
template <class T, bool E8>
__device__ __forceinline__ float row_dot(const float* q, const uint16_t* pool, int64_t at, float scale, int d) {
  float s = 0.0f;
  for (int i = 0; i < d; i += 8) {
    const v4i r = held8<T, E8>(pool, at + i, scale);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s = fmaf(q[i + 2 * e], T::load((uint16_t)r[e]), s);
      s = fmaf(q[i + 2 * e + 1], T::load((uint16_t)((uint32_t)r[e] >> 16)), s);
    }
  }
  return s;
}

// The form for head sizes without a matrix kernel, right rather than fast: every row reads K and V for itself, on scalar
// products, and a row's keys are not split. One token over 701 keys, 32 heads of 96 over 8: 232 us (floor 0.4); 32
// sequences of up to 32768 keys 24.3 ms (241 us); 1021 and 866 tokens over 6007 and 2367 keys, 24 heads of 96 over 4: 13 ms,
// 25 with the weights (55 us).
//
// 64 keys a step, one a lane: scores, the running maximum m and sum l of the softmax over all keys so far (in the
// log2 domain, p = 2^(s c - m)), then the outputs, which lie over the lanes (channel lane + 64 i).
template <class T, bool E8>
__global__ __launch_bounds__(64 * RW_WAVES) void paged_attn_rows_kernel(PagedArgs c, const uint16_t* q, int64_t ldqt,
                                                                        int64_t ldqh, uint16_t* o, float* lse,
                                                                        int tokens, int heads, int d, float c_log2,
                                                                        int causal) {
  __shared__ float qs[RW_WAVES][RW_MAX_D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * RW_WAVES + wave;
  if (row >= (int64_t)tokens * heads) return;  // no barriers below: a wave reads only what it wrote
  const int t = (int)(row / heads), x = (int)(row - (int64_t)t * heads), h = x / (heads / c.kv_heads);
  for (int i = lane; i < d; i += 64) qs[wave][i] = T::load(q[t * ldqt + x * ldqh + i]);
  __builtin_amdgcn_wave_barrier();
  int b = 0;
  for (int i = 0; i < c.batch; i += 64)
    b += __popcll(__ballot(i + lane < c.batch && c.q_start[min(i + lane, c.batch - 1) + 1] <= t));
  int keys = 0;
  if (b < c.batch) {
    int t0, n;
    paged_new(c, b, tokens, t0, n);
    const int len = paged_kv_len(c, b);
    if (t >= t0 && t - t0 < n) keys = causal ? min(max(len - n + (t - t0) + 1, 0), len) : len;
  }
  const int32_t* pages = c.table + (int64_t)b * c.table_stride;
  float m = -INFINITY, l = 0.0f, acc[RW_MAX_D / 64] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j0 = 0; j0 < keys; j0 += 64) {
    const int j = j0 + lane, nj = min(64, keys - j0);
    float s = -INFINITY;
    if (j < keys) {
      const int page = paged_page(c, pages, j);
      s = row_dot<T, E8>(qs[wave], c.k, paged_at(c, page, h, j), held_scale<E8>(c, c.ks, page, h, j), d) * c_log2;
    }
    float mx = s;
    for (int w = 32; w; w >>= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
    const float m_new = fmaxf(m, mx);
    const float ref = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - ref), p = __builtin_amdgcn_exp2f(s - ref);
    float sum = p;
    for (int w = 32; w; w >>= 1) sum += __shfl_xor(sum, w);
    l = fmaf(l, alpha, sum);
    m = m_new;
#pragma unroll
    for (int i = 0; i < RW_MAX_D / 64; ++i) acc[i] *= alpha;
    for (int k = 0; k < nj; ++k) {
      const float pk = __shfl(p, k);
      const int page = paged_page(c, pages, j0 + k);
      const int64_t vr = paged_at(c, page, h, j0 + k) + lane;
      const float vs = held_scale<E8>(c, c.vs, page, h, j0 + k);
#pragma unroll
      for (int i = 0; i < RW_MAX_D / 64; ++i)
        if (lane + 64 * i < d) acc[i] = fmaf(pk, held1<T, E8>(c.v, vr + 64 * i, vs), acc[i]);
    }
  }
  const float inv = inverse_sum(l);
  for (int i = 0; i < RW_MAX_D / 64; ++i)
    if (lane + 64 * i < d) o[row * d + lane + 64 * i] = (uint16_t)T::pack(acc[i] * inv, 0.0f);
  if (lane == 0) lse[row] = log2_sum(m, l) * kLn2;
}

// w[key] += sum of 2^(s c - lse) over the rows that see the key: one lane a key, 64 keys of one kv head a wave
template <class T, bool E8>
__global__ __launch_bounds__(64) void paged_gather_rows_kernel(PagedArgs c, const uint16_t* q, int64_t ldqt,
                                                               int64_t ldqh, const float* lse, int tokens, int heads,
                                                               int d, float c_log2, int causal) {
  __shared__ float qs[RW_MAX_D];
  const int lane = threadIdx.x, b = blockIdx.y / c.kv_heads, h = blockIdx.y % c.kv_heads, g = heads / c.kv_heads;
  const int len = paged_kv_len(c, b);
  int t0, n;
  paged_new(c, b, tokens, t0, n);
  for (int j0 = blockIdx.x * 64; j0 < len; j0 += gridDim.x * 64) {
    const int j = min(j0 + lane, len - 1);
    const int page = paged_page(c, c.table + b * c.table_stride, j);
    const int64_t key = paged_at(c, page, h, j);
    const float ks = held_scale<E8>(c, c.ks, page, h, j);
    float sum = 0.0f;
    for (int i = 0; i < n * g; ++i) {
      const int t = t0 + i / g, x = h * g + i % g;
      const int seen = causal ? len - n + i / g : len - 1;
      if (seen < j0) continue;  // the same for the whole wave
      __syncthreads();
      for (int e = lane; e < d; e += 64) qs[e] = T::load(q[t * ldqt + x * ldqh + e]);
      __syncthreads();
      const float s = row_dot<T, E8>(qs, c.k, key, ks, d) * c_log2;
      if (j <= seen) sum += __builtin_amdgcn_exp2f(s - gather_lse2(lse[(int64_t)t * heads + x]));
    }
    if (j0 + lane < len) c.w[paged_w_at(c, page, h, j)] += sum;
  }
}

// ---------------------------------------------------------------------------
// head_dim 64 and 128, many rows: MFMA 32x32x16, 32 rows a wave
// ---------------------------------------------------------------------------
// One pass over the keys with a running softmax. A workgroup of NW waves owns 32 NW rows (new token, query head of the
// group) of one sequence and kv head and walks its keys in tiles of BN, double buffered in LDS by direct copies
// whose lanes look their key's page up a tile ahead. Per tile a wave computes, with fp32 accumulators:
//   S^T = K q^T           (keys x rows: a lane holds one row, 16 keys of each 32)
//   p   = 2^(S c - m)     (m: the row's running maximum; O and the sum l are rescaled where it moves)
//   O^T = O^T + V^T p^T   (V^T by transposing reads, in the key order S^T leaves p in, so p stays in registers)
// p is rounded to the cache's type, as the MFMA's operands are 16 bits wide, and summed into l before: O is off by 1.1 to
// 1.3 times what one rounding of the output costs. m, l, S and O are fp32.
// A tile takes two slots, each ended by a barrier: the matrix slot (O of the tile before, S of this one) and the softmax
// slot. With 8 waves the SIMD's second wave runs one slot behind the first, so that one has the matrix cores while
// the other has the vector unit.
// Tiles that every row of the workgroup sees whole run without a mask; the others compare each score's key with the
// lane's limit. There 0 * v of a hidden key must not reach O: whoever copied a part of the tile sets values that are not
// finite to 0 and says so, and rows that do see such a key get its values added one by one at the end.
//
// Measured on 4096 new tokens over 16500 keys, 32 heads of 128 over 8 (981 GFLOP): 883 to 950 us, 1.03 to 1.11 PFLOP/s,
// where an 8192^3 library product reaches 1.22 to 1.26. The matrix cores are busy 49 % of the time and the vector unit 51 %, at
// a clock that falls to 1.65 to 1.8 GHz; without the copies it takes 849 us (of 965 then), without the exponentials 891. Before the fixed operand order
// every MFMA waited for the LDS read issued just ahead of it (1057 us); both waves of a SIMD in the same phase take 1013;
// 128-key tiles spill and take 1710. Of an 8-bit cache (E8) the rows pass through registers, where they become 16-bit values
// on their way to LDS, a tile ahead: one conversion for two values, again for each row tile; 2048 tokens over 16500 keys
// (525 GFLOP) take 550 to 567 us where a 16-bit cache takes 500 in the same run. Those registers come on top: at head_dim
// 128 the form of 4 waves spills 30 of a lane (16 tokens for each of 32 sequences over up to 8192 keys, 32 heads over 8: 100
// us, a 16-bit cache 102), that of 8 waves 3. Five sequences of up to 509 tokens over up to 4001 keys, 16 heads of 64: 34 us,
// in which nothing is busy (matrix cores 11 %, vector unit 27 %, LDS 7 %): a tile has half the work between the same two
// barriers, and 2 waves a SIMD do not cover what each waits for (37 us of an 8-bit cache).
template <int D, int BN, int NW>
struct TileShape {
  static constexpr int kRow = 2 * D, kRun = 1024 / kRow;  // row bytes; rows a 1 KB copy covers
  static constexpr int kRuns = BN / kRun / NW;            // copies a wave, per K and per V tile
  static constexpr int kTile = BN * kRow;                 // LDS: K tiles 0 and 1, then V tiles 0 and 1
  static constexpr int kNSB = BN / 32, kNC = BN / 16, kND = D / 32, kNQ = D / 16;
};

template <class T, int D, int BN, int NW, bool E8>
__global__ __launch_bounds__(64 * NW, 2) void paged_attn_tile_kernel(AttnArgs a) {
  using S = TileShape<D, BN, NW>;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * S::kTile];
  __shared__ uint32_t aside;  // whether any value of a masked tile was set aside
  const PagedArgs& c = a.c;
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63;
  const int behind = wave >> 2;             // slots this wave runs behind the workgroup's first
  const int j = lane & 31, hf = lane >> 5;  // MFMA column (row of the call, key or channel) and half
  constexpr int BM = 32 * NW;
  const int g = a.heads / c.kv_heads;
  const bool causal = a.causal != 0;
  constexpr int kElem = E8 ? 1 : 2;  // bytes
  const uint32_t page_bytes = (uint32_t)(kElem * c.page_stride), slot_bytes = (uint32_t)(kElem * c.slot_stride);
  const uint32_t slot_mask = (1u << c.page_shift) - 1;

  // read offsets in a tile: K row j, chunk hf (chunk 2 cd + hf: the address xor 32 cd; rows 32 sb + j: a constant
  // more). V^T operand (channel block db, 16-key step cc): lane p = lane % 16 of column half dh points at key 4 hf + p / 4
  // (16 cc and 8 more: constants), channels 16 dh + 4 (p % 4) .. + 4 (block db: the address xor 64 db)
  const uint32_t kro = (uint32_t)(j * S::kRow + 16 * k_place<D>(hf, j));
  const int vr = 4 * hf + ((lane & 15) >> 2), vc = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  const uint32_t vro = (uint32_t)(vr * S::kRow + 16 * v_place<D>(vc >> 3, vr) + 2 * (vc & 7));
  constexpr int CH = D / 8;
  const int crow = lane / CH, cpl = lane % CH;  // the lane's row and chunk place in a 1 KB copy
  // (a wave's copies are a multiple of 4 KB apart, so the swizzles of the lane's row are the same in all)
  const uint32_t klane = crow * slot_bytes + 8 * kElem * k_place<D>(cpl, wave * S::kRun + crow);
  const uint32_t vlane = crow * slot_bytes + 8 * kElem * v_place<D>(cpl, wave * S::kRun + crow);

  const int tt = BM / g;  // new tokens a row tile holds
  const bool shared = a.shares > 0;
  int share = 0;
  Place at, end;
  if (shared) {
    // this workgroup's share. An XCD's workgroups (every 8th) take neighbouring shares, which are of one head where
    // there are 8 (or 16, ...), so that K and V are shared in its L2
    share = blockIdx.x % kXcds * (a.shares / kXcds) + blockIdx.x / kXcds;
    const LineLanes lanes = line_lanes(c, a.tokens, tt, causal, 0);
    const int64_t per_head = head_line(c, a.tokens, tt, causal, lanes), all = per_head * c.kv_heads;
    const int64_t x0 = share_start(all, share, a.shares), x1 = share_start(all, share + 1, a.shares);
    no_cuts(a, share);
    if (x0 >= x1) return;
    at = place_of<BN>(c, a.tokens, tt, causal, per_head, lanes, x0);
    end = place_of<BN>(c, a.tokens, tt, causal, per_head, lanes, x1);
  } else {  // a workgroup a row tile, all of its keys; the tiles that see the most start first
    const int groups = c.batch * c.kv_heads, grp = blockIdx.x % groups;
    at = Place{grp % c.kv_heads, grp / c.kv_heads, a.tiles - 1 - (int)(blockIdx.x / groups), 0};
    end = at;
  }
  Rows R = uniform_rows_of(c, at.b, a.tokens, g);
  if (!shared && at.tile * tt >= R.n) return;

  while (true) {  // one part of a row tile's keys: BN-key units [at.unit, to)
    const int h = at.h, i0 = at.tile * tt, i1 = min(i0 + tt, R.n);
    const bool last = shared && at.h == end.h && at.b == end.b && at.tile == end.tile;
    const int lim_lo = R.token_limit(i0, causal), lim_hi = R.token_limit(i1 - 1, causal);
    const int units = max(1, (lim_hi + BN) / BN), to = last ? min(end.unit, units) : units;
    if (at.unit < to) {
      const int32_t* pages = c.table + (int64_t)at.b * c.table_stride;
      const uint8_t* kbase = (const uint8_t*)c.k + kElem * h * c.head_stride;
      const uint8_t* vbase = (const uint8_t*)c.v + kElem * h * c.head_stride;
      const int r = 32 * wave + j, ri = i0 + r / g, rc = min(ri, i1 - 1);  // the lane's row, its token
      const int tok = R.t0 + rc, head = h * g + r % g;
      const int lim = R.token_limit(rc, causal);
      // the part's keys [k_lo, k_hi) and the tiles of them that every row sees whole
      const int k_lo = at.unit * BN, k_hi = min(to * BN, lim_hi + 1);
      const int ntiles = k_hi > k_lo ? to - at.unit : 0;
      const int nfull = min(max(lim_lo + 1 - k_lo, 0) / BN, k_hi > k_lo ? (k_hi - k_lo) / BN : 0);

      v4i qop[S::kNQ];  // q^T operand: q[row][16 cd + 8 hf .. + 8]
      const uint16_t* qp = a.q + tok * a.ldqt + head * a.ldqh + 8 * hf;
#pragma unroll
      for (int cd = 0; cd < S::kNQ; ++cd) qop[cd] = *(const v4i*)(qp + 16 * cd);

      // Copies of 1 KB cover kRun rows from a multiple of kRun on, which lie in one page (page_size >= 8), so a copy's page
      // and address are the wave's, and a lane adds a constant. Ids of the tile whose values are copied next, and of the
      // one after it, whose keys are; copies wholly past the last key repeat that key's.
      int pgv[S::kRuns], pgk[S::kRuns];
      auto run_key = [&](int t, int u) __attribute__((always_inline)) {
        return min(k_lo + t * BN + (wave + NW * u) * S::kRun, (k_hi - 1) & ~(S::kRun - 1));
      };
      auto place = [&](int t, int u, int page) __attribute__((always_inline)) {
        return (uint64_t)(uint32_t)min(max(uniform(page), 0), c.pages - 1) * page_bytes +
               ((uint32_t)run_key(t, u) & slot_mask) * slot_bytes;
      };
      auto look_up = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < S::kRuns; ++u) pgk[u] = pages[run_key(t, u) >> c.page_shift];
      };
      // of an 8-bit cache the copies go through registers, which hold the lane's 8 codes of a copy and its row's scale
      // until they land
      uint2 kraw[S::kRuns], vraw[S::kRuns];
      uint32_t kscale[S::kRuns], vscale[S::kRuns];
      auto scale_at = [&](int t, int u, int page) __attribute__((always_inline)) {
        return min(max(uniform(page), 0), c.pages - 1) * c.s_page_stride + h * c.s_head_stride +
               ((uint32_t)run_key(t, u) & slot_mask);
      };
      auto copy_keys = [&](int t) __attribute__((always_inline)) {
        const uint32_t st = (uint32_t)(uintptr_t)(lds + (t & 1) * S::kTile);
#pragma unroll
        for (int u = 0; u < S::kRuns; ++u) {
          if constexpr (E8) {
            kraw[u] = *(const uint2*)(kbase + place(t, u, pgk[u]) + klane);
            kscale[u] = c.ks[scale_at(t, u, pgk[u]) + crow];
          } else {
            copy16(st + (wave + NW * u) * 1024, kbase + place(t, u, pgk[u]), klane);
          }
        }
      };
      auto copy_values = [&](int t) __attribute__((always_inline)) {
        const uint32_t st = (uint32_t)(uintptr_t)(lds + (2 + (t & 1)) * S::kTile);
#pragma unroll
        for (int u = 0; u < S::kRuns; ++u) {
          if constexpr (E8) {
            vraw[u] = *(const uint2*)(vbase + place(t, u, pgv[u]) + vlane);
            vscale[u] = c.vs[scale_at(t, u, pgv[u]) + crow];
          } else {
            copy16(st + (wave + NW * u) * 1024, vbase + place(t, u, pgv[u]), vlane);
          }
        }
      };
      // E8: tile t's keys from the registers into LDS
      auto land_keys = [&](int t) __attribute__((always_inline)) {
        uint8_t* st = lds + (t & 1) * S::kTile;
#pragma unroll
        for (int u = 0; u < S::kRuns; ++u)
          *(v4i*)(st + (wave + NW * u) * 1024 + lane * 16) = widen8<T>(kraw[u].x, kraw[u].y, scale_of(kscale[u]));
      };
      // the copies that go out in tile t's first slot: its values and the next tile's keys, into the places of the
      // tiles read up to the slot before
      auto copies = [&](int t) __attribute__((always_inline)) {
        copy_values(t);
        if (t + 1 < ntiles) copy_keys(t + 1);
#pragma unroll
        for (int u = 0; u < S::kRuns; ++u) pgv[u] = pgk[u];
        if (t + 2 < ntiles) look_up(t + 2);
      };
      // the end of its second slot: they have landed, here and (after the barrier) everywhere
      auto landed = [&](int t) __attribute__((always_inline)) {
        if constexpr (E8) {
          uint8_t* vb = lds + (2 + (t & 1)) * S::kTile;
          const bool masked = t >= nfull;
          bool bad = false;
#pragma unroll
          for (int u = 0; u < S::kRuns; ++u) {
            v4i x = widen8<T>(vraw[u].x, vraw[u].y, scale_of(vscale[u]));
            if (masked) {
              if (k_lo + t * BN + (wave + NW * u) * S::kRun + crow >= k_hi) x = (v4i){};  // whatever a page holds past the end
              else bad |= take_nonfinite<T>(x);
            }
            *(v4i*)(vb + (wave + NW * u) * 1024 + lane * 16) = x;
          }
          if (bad) aside = 1;
          if (t + 1 < ntiles) land_keys(t + 1);
          __syncthreads();
          return;
        }
        wait_vm_lgkm0<0>();
        if (t >= nfull && t < ntiles) {  // a masked tile
          uint8_t* vb = lds + (2 + (t & 1)) * S::kTile;
          bool bad = false;
#pragma unroll
          for (int u = 0; u < S::kRuns; ++u) {
            v4i* p = (v4i*)(vb + (wave + NW * u) * 1024 + lane * 16);
            v4i x = *p;
            if (k_lo + t * BN + (wave + NW * u) * S::kRun + crow >= k_hi) *p = (v4i){};  // whatever a page holds past the end
            else if (take_nonfinite<T>(x)) *p = x, bad = true;
          }
          if (bad) aside = 1;
        }
        __syncthreads();
      };

      v16f oacc[S::kND], sc[S::kNSB];
      v4i pop[S::kNC];
#pragma unroll
      for (int db = 0; db < S::kND; ++db) oacc[db] = (v16f){};
      float m_run = -INFINITY, l_run = 0.0f;

      // matrix slot: O of tile t - 1 (VALUES), then S of tile t (KEYS). The operands are read from LDS kAhead MFMAs ahead
      // of their use, in an order the scheduler may not change: left to itself, short of registers, it waits for
      // each operand right after asking for it
      auto matrix = [&](int t, auto values_c, auto keys_c) __attribute__((always_inline)) {
        constexpr bool VALUES = decltype(values_c)::value, KEYS = decltype(keys_c)::value;
        constexpr int kAhead = 6, kV = VALUES ? S::kND * S::kNC : 0, kAll = kV + (KEYS ? S::kNQ * S::kNSB : 0);
        const uint8_t* vb = lds + (2 + ((t - 1) & 1)) * S::kTile;
        const uint8_t* kb = lds + (t & 1) * S::kTile;
        v4i ring[kAhead];
        auto read = [&](int i) __attribute__((always_inline)) {
          if (i < kV) {
            const uint8_t* p = vb + (vro ^ (uint32_t)(64 * (i / S::kNC))) + 16 * (i % S::kNC) * S::kRow;
            ring[i % kAhead] = two_halves(lds_read_tr(p), lds_read_tr(p + 8 * S::kRow));
          } else {
            const int k = i - kV;
            ring[i % kAhead] = *(const v4i*)(kb + (kro ^ (uint32_t)(32 * (k / S::kNSB))) + k % S::kNSB * 32 * S::kRow);
          }
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) read(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kAll; ++i) {
          if (i < kV) {
            oacc[i / S::kNC] = Mfma<T>::wide(ring[i % kAhead], pop[i % S::kNC], oacc[i / S::kNC]);
          } else {
            const int k = i - kV;
            sc[k % S::kNSB] = Mfma<T>::wide(ring[i % kAhead], qop[k / S::kNSB], k < S::kNSB ? (v16f){} : sc[k % S::kNSB]);
          }
          if (i + kAhead < kAll) read(i + kAhead);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      const std::true_type yes;
      const std::false_type no;
      auto softmax_of = [&](int t, auto mask_c) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask_c)::value;
        if (MASK) {
          const int vis = lim - (k_lo + t * BN) - 4 * hf;  // the lane's last visible key of the tile, less its keys' common part
#pragma unroll
          for (int sb = 0; sb < S::kNSB; ++sb)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (32 * sb + 8 * (i >> 2) + (i & 3) > vis) sc[sb][i] = -INFINITY;
        }
        // the lane's maximum; the first level as med3(a, b, 3e38), which is max for scores below that and, unlike
        // fmaxf, needs no quieting of raw MFMA results first
        float m8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          m8[i] = __builtin_amdgcn_fmed3f(sc[0][i], sc[0][i + 8], 3.0e38f);
#pragma unroll
          for (int sb = 1; sb < S::kNSB; ++sb)
            m8[i] = fmaxf(m8[i], __builtin_amdgcn_fmed3f(sc[sb][i], sc[sb][i + 8], 3.0e38f));
        }
#pragma unroll
        for (int w = 4; w >= 1; w >>= 1)
#pragma unroll
          for (int i = 0; i < w; ++i) m8[i] = fmaxf(m8[i], m8[i + w]);
        const float x_max = fmaxf(m8[0], __shfl_xor(m8[0], 32)) * a.c_log2;
        const bool bump = x_max > m_run;
        const float m_new = bump ? x_max : m_run;
        // a row whose scores so far are all -inf (behind the mask, or by themselves) subtracts 0: its p are all 0
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m_run - ref);  // 0 on the first tile
        m_run = m_new;
        float ps[S::kNC];
#pragma unroll
        for (int cc = 0; cc < S::kNC; ++cc) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[cc >> 1][8 * (cc & 1) + e], a.c_log2, -ref));
          ps[cc] = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
          pop[cc] = (v4i){Mfma<T>::pack(p[0], p[1]), Mfma<T>::pack(p[2], p[3]), Mfma<T>::pack(p[4], p[5]),
                          Mfma<T>::pack(p[6], p[7])};
        }
#pragma unroll
        for (int w = S::kNC / 2; w >= 1; w >>= 1)
#pragma unroll
          for (int i = 0; i < w; ++i) ps[i] += ps[i + w];
        l_run = __builtin_fmaf(l_run, alpha, ps[0]);
        if (__builtin_amdgcn_ballot_w64(bump) != 0) {  // alpha is 1 in lanes whose maximum stayed
#pragma unroll
          for (int db = 0; db < S::kND; ++db) oacc[db] *= alpha;
        }
      };
      auto softmax = [&](int t) __attribute__((always_inline)) {
        if (t < nfull) softmax_of(t, no);
        else softmax_of(t, yes);
      };

      if (ntiles > 0) {
        if (tid == 0) aside = 0;
        look_up(0);
        copy_keys(0);
#pragma unroll
        for (int u = 0; u < S::kRuns; ++u) pgv[u] = pgk[u];
        if (ntiles > 1) look_up(1);
        if constexpr (E8) land_keys(0);
        wait_vm_lgkm0<0>();
        __syncthreads();
        // tile t: slots 2 t and 2 t + 1 of the waves that run ahead, one later of those behind; all pass the same barriers
        if (behind == 0) {
          copies(0);
          matrix(0, no, yes);
          barrier_lds();
          for (int t = 0; t + 1 < ntiles; ++t) {
            softmax(t);
            landed(t);
            copies(t + 1);
            matrix(t + 1, yes, yes);
            barrier_lds();
          }
          softmax_of(ntiles - 1, yes);
          landed(ntiles - 1);
          matrix(ntiles, yes, no);
          barrier_lds();
          __syncthreads();
        } else {
          copies(0);
          barrier_lds();
          matrix(0, no, yes);
          landed(0);
          for (int t = 0; t + 1 < ntiles; ++t) {
            copies(t + 1);
            softmax(t);
            barrier_lds();
            matrix(t + 1, yes, yes);
            landed(t + 1);
          }
          softmax_of(ntiles - 1, yes);
          barrier_lds();
          matrix(ntiles, yes, no);
          __syncthreads();
        }
        if (aside) {  // rows that see keys whose values were set aside: those values, one by one
          for (int key = k_lo + nfull * BN; key < k_hi; ++key) {
            const int page = paged_page(c, pages, key);
            const int64_t at_key = paged_at(c, page, h, key);
            const float ks = held_scale<E8>(c, c.ks, page, h, key), vs = held_scale<E8>(c, c.vs, page, h, key);
            float s = 0.0f;
#pragma unroll
            for (int cd = 0; cd < S::kNQ; ++cd) s = dot8<T>(qop[cd], held8<T, E8>(c.k, at_key + 8 * hf + 16 * cd, ks), s);
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s + __shfl_xor(s, 32), a.c_log2, -m_run));
            if (key <= lim) {
#pragma unroll
              for (int db = 0; db < S::kND; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float v = held1<T, E8>(c.v, at_key + 32 * db + 8 * (i >> 2) + 4 * hf + (i & 3), vs);
                  if (!(fabsf(v) < INFINITY)) oacc[db][i] = fmaf(p, v, oacc[db][i]);
                }
            }
          }
        }
        __syncthreads();  // `aside` has been read
      }

      const float l_tot = l_run + __shfl_xor(l_run, 32);
      const float inv = inverse_sum(l_tot), lse2 = log2_sum(m_run, l_tot);
      if (at.unit > 0 || to < units) {
        // a part: into the share's slot, the first for a tile that an earlier share began, else the second
        set_cut(a, share, at.unit > 0, to == units, (i1 - i0) * g, R.t0 + i0, h);
        const int64_t prow = (int64_t)(2 * share + (at.unit > 0 ? 0 : 1)) * BM + r;
        float* op = a.o_part + prow * D + 4 * hf;
#pragma unroll
        for (int db = 0; db < S::kND; ++db)
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *(float4*)(op + 32 * db + 2 * i) = make_float4(oacc[db][i] * inv, oacc[db][i + 1] * inv,
                                                           oacc[db][i + 2] * inv, oacc[db][i + 3] * inv);
        if (hf == 0) a.lse_part[prow] = lse2;
      } else if (r < tt * g && ri < i1) {
        const int64_t out_row = (int64_t)tok * a.heads + head;
        uint16_t* op = a.o + out_row * D + 4 * hf;
#pragma unroll
        for (int db = 0; db < S::kND; ++db)
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *(uint2*)(op + 32 * db + 2 * i) =
                make_uint2((uint32_t)Mfma<T>::pack(oacc[db][i] * inv, oacc[db][i + 1] * inv),
                           (uint32_t)Mfma<T>::pack(oacc[db][i + 2] * inv, oacc[db][i + 3] * inv));
        if (hf == 0) a.lse[out_row] = lse2 * kLn2;
      }
    }
    if (last) break;
    at.unit = 0;
    if (!shared) {
      at.tile += a.tiles;  // more tiles than the host knew of
      if (at.tile * tt >= R.n) break;
    } else if (i1 < R.n) {
      ++at.tile;
    } else {
      at.tile = 0;
      do {  // the next sequence with new tokens, of the next head after the last
        if (++at.b == c.batch) at.b = 0, ++at.h;
        if (at.h == c.kv_heads) return;  // the line's end
        R = uniform_rows_of(c, at.b, a.tokens, g);
      } while (R.n == 0);
    }
  }
}

// Joins the parts of row tiles that the shares' ends cut, in the shares' order: a workgroup for JT rows of the tile that
// its share begins and others continue. All parts' sums are read at once and turned into their factors in LDS, so that a
// part's values wait for nothing (read in turn, 12 parts of a tile of 28 rows took 14 us, so 6).
constexpr int JT = 16;

template <class T, int D, int BM>
__global__ __launch_bounds__(256) void paged_attn_join_parts_kernel(AttnArgs a) {
  constexpr int kAtOnce = 64, kItems = JT * D / 4 / 256;  // parts whose factors are held; a thread's pieces of 4 channels
  __shared__ float factor[kAtOnce][JT];
  __shared__ int slots[2 * kCus + 1];  // the slots of the tile's parts, in order
  __shared__ int nslots;
  const int share = blockIdx.x / (BM / JT), r0 = blockIdx.x % (BM / JT) * JT;
  const int4 cut = a.cuts[share];
  if (cut.y <= r0) return;
  if (threadIdx.x < 64) {
    int n = 1;
    bool ended = false;
    for (int s = share + 1; s < a.shares && !ended; s += 64) {
      const int mine = s + threadIdx.x, kind = mine < a.shares ? a.cuts[mine].x : 0;
      const uint64_t ends = __ballot(kind == 2);
      // up to the first share that ends a tile: the parts before it are all of this one
      const uint64_t upto = ends ? ends ^ (ends - 1) : ~0ull;
      const uint64_t parts = __ballot(kind != 0) & upto;
      if (parts >> threadIdx.x & 1) slots[n + __popcll(parts & ((1ull << threadIdx.x) - 1))] = 2 * mine;
      n += __popcll(parts);
      ended = ends != 0;
    }
    if (threadIdx.x == 0) slots[0] = 2 * share + 1, nslots = n;
  }
  __syncthreads();
  const int parts = nslots, g = a.heads / a.c.kv_heads, rows = min(JT, cut.y - r0);
  const int fr = threadIdx.x / 16, lane = threadIdx.x % 16;  // 16 lanes a row find its factors
  auto sum_of = [&](int k) { return fr < rows ? a.lse_part[(int64_t)slots[k] * BM + r0 + fr] : 0.0f; };
  float m = -INFINITY;
  for (int k = lane; k < parts; k += 16) m = fmaxf(m, sum_of(k));
#pragma unroll
  for (int w = 8; w; w >>= 1) m = fmaxf(m, __shfl_xor(m, w));
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  for (int k = lane; k < parts; k += 16) l += __builtin_amdgcn_exp2f(sum_of(k) - ref);
#pragma unroll
  for (int w = 8; w; w >>= 1) l += __shfl_xor(l, w);
  const float inv = inverse_sum(l);
  auto out_row = [&](int r) { return (int64_t)(cut.z + (r0 + r) / g) * a.heads + cut.w * g + (r0 + r) % g; };
  if (lane == 0 && fr < rows) a.lse[out_row(fr)] = log2_sum(m, l) * kLn2;
  v4f o[kItems] = {};
  for (int k0 = 0; k0 < parts; k0 += kAtOnce) {
    const int n = min(kAtOnce, parts - k0);
    if (k0 > 0) __syncthreads();
    for (int k = lane; k < n; k += 16) factor[k][fr] = __builtin_amdgcn_exp2f(sum_of(k0 + k) - ref) * inv;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kItems; ++e) {
      const int i = threadIdx.x + 256 * e, r = i / (D / 4), d = i % (D / 4) * 4;
      if (r >= rows) continue;
#pragma unroll 8
      for (int k = 0; k < n; ++k) o[e] += *(const v4f*)(a.o_part + ((int64_t)slots[k0 + k] * BM + r0 + r) * D + d) * factor[k][r];
    }
  }
#pragma unroll
  for (int e = 0; e < kItems; ++e) {
    const int i = threadIdx.x + 256 * e, r = i / (D / 4), d = i % (D / 4) * 4;
    if (r < rows)
      *(uint2*)(a.o + out_row(r) * D + d) = make_uint2((uint32_t)Mfma<T>::pack(o[e][0], o[e][1]),
                                                       (uint32_t)Mfma<T>::pack(o[e][2], o[e][3]));
  }
}

// ---------------------------------------------------------------------------
// head_dim 64 and 128, few rows: MFMA 16x16x32, 16 RB rows a workgroup, every wave its own keys
// ---------------------------------------------------------------------------
// Bound by reading K and V. A workgroup owns a run of one sequence's and kv head's keys; wave w takes its tiles w,
// w + NW, ... of 32 keys through two LDS stages of its own (no barriers in the loop; the next tile is in flight
// while one is computed), and the waves' O, m and l are joined at the end. The run's page ids are read into LDS
// first, so that no ordinary load's wait falls among the copies'.
// Runs: with SHARES the line of all keys is cut into one equal share for each CU, as for many rows: a workgroup's start
// costs a few microseconds, so one round of workgroups that all end together reads fastest (32 sequences of up to
// 32768 keys: runs of 4096 keys, 866 workgroups, took 321 us, of 16384 keys, 328 workgroups, 303). Where the keys are so few
// that runs of 256 are all there at once, a run is a split of that length, which a workgroup finds without the line.
// Measured: the 32 sequences 276 us, 5.7 TB/s (a copy reaches 4.94; the copies alone, without the products, took 296 with
// their join before the shares); 4 tokens each over up to 8192 keys 88 us with the join, 8 tokens 101 (floors 76 and 85); one
// sequence of 701 keys, 32 heads over 8, 9 to 10 us and 3.9 for the join (medians): launch and four dependent loads.
// Of an 8-bit cache (E8) two tiles are in flight in registers, K's codes as the operands need them and V's on to LDS as
// 16-bit values. The 32 sequences of up to 32768 keys: 163 us, 4.9 TB/s (170 a call with the join); the same loads
// without any work on them 153. One scale byte a lane, given out by lane moves, and places found by the wave: 179 us of a
// call with every lane loading its rows' own. The sequence of 701 keys: 9.0 us and 3.1; a workgroup of 8 waves for all its
// keys, with no join: 11.6 to 12.5, so there is none.
// Two row blocks (17 to 32 rows) at head_dim 128 do not fit an 8-bit cache's registers: two tiles in flight, V's operands read
// ahead and O spill 125 to 128 of a lane (one block 5 to 15, heads of 64 at most 6, the 16-bit form none). 8 tokens for each of
// 32 sequences over up to 8192 keys, 32 heads over 8: 240 us where a 16-bit cache takes 101; 4 tokens, one block: 58 and 80.
constexpr int FW_KEYS = 32, FW_PAGES = 512;  // keys a tile; page ids staged at a time (whole tiles: page_size >= 8)
constexpr int FW_WAVES = 4, FW_UNIT = FW_KEYS * FW_WAVES;
// Where the segment of a run that starts at key s_lo ends, at k_hi at the latest: behind the FW_PAGES-th page from that of
// s_lo on, which may lie inside its page (runs start at multiples of 128 keys, pages hold up to 4096). The next
// segment starts on a page, whole tiles later.
constexpr __host__ __device__ int segment_end(int s_lo, int k_hi, int page_shift) {
  const int end = ((s_lo >> page_shift) + FW_PAGES) << page_shift;
  return end < k_hi ? end : k_hi;
}
constexpr bool segment_fits(int s_lo, int k_hi, int page_shift) {
  const int end = segment_end(s_lo, k_hi, page_shift);
  return ((end - 1) >> page_shift) - (s_lo >> page_shift) < FW_PAGES && (end == k_hi || (end - s_lo) % FW_KEYS == 0);
}
static_assert(segment_fits(0, 1 << 30, 3) && segment_fits(128, 1 << 30, 4) && segment_fits(128, 1 << 30, 8) &&
              segment_fits(256, 1 << 30, 9) && segment_fits(384, 131200, 8) && segment_fits(128 * 33, 1 << 30, 12));

template <int D, int RB, bool E8>
struct FewShape {
  static constexpr int kRow = 2 * D, kRun = 1024 / kRow;
  static constexpr int kRuns = FW_KEYS / kRun;  // copies a tile, per K and per V
  static constexpr int kTile = FW_KEYS * kRow;
  static constexpr int kStages = E8 ? kTile : 4 * kTile;  // K and V of two tiles; V of one
  static constexpr int kND = D / 16, kNQ = D / 32;
  static constexpr int kOut = 16 * RB * (D + 4) * 4;  // a wave's O at the end (rows padded against bank conflicts)
  static constexpr int kWave = kStages > kOut ? kStages : kOut;
};
// A lane's part of a tile of an 8-bit cache, in registers from its loads to its use: of keys i16 and 16 + i16 the D / 4 codes
// from channel D / 4 q4 on, which are the lane's operands as they lie (the queries' chunks follow that order); of the
// values 16 codes of every (1024 / D)th row, which go through LDS to be read across keys. A lane loads one scale byte and gets
// those it needs from others.
template <int D>
struct FewRaw {
  static constexpr int kK = D / 64, kV = D / 32, kRows = 1024 / D;
  v4i k[2][kK], v[kV];
  uint32_t scale;  // of the key `lane`, in the upper half of its value 32 lanes below
};

template <class T, int D, int RB, bool SHARES, bool E8>
__global__ __launch_bounds__(64 * FW_WAVES, E8 ? 2 : 1) void paged_attn_few_kernel(AttnArgs a) {
  using S = FewShape<D, RB, E8>;
  constexpr int NW = FW_WAVES, BM = 16 * RB;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NW * S::kWave];
  __shared__ float stat[NW][2][BM];  // m and l by wave
  __shared__ int page_ids[FW_PAGES];
  const PagedArgs& c = a.c;
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63;
  const int i16 = lane & 15, q4 = lane >> 4;  // MFMA column (row of the call, key or channel) and quarter
  const int g = a.heads / c.kv_heads, tt = BM / g;  // new tokens a row tile holds
  const bool causal = a.causal != 0;
  constexpr int kElem = E8 ? 1 : 2;  // bytes
  const uint32_t page_bytes = (uint32_t)(kElem * c.page_stride), slot_bytes = (uint32_t)(kElem * c.slot_stride);
  const uint32_t slot_mask = (1u << c.page_shift) - 1;
  uint8_t* const mine = lds + wave * S::kWave;

  // K operand: key 16 x + i16, chunk q4 (chunk 4 cd + q4: the address xor 64 cd). V^T operand (channels 16 db ..): lane
  // p = i16 of quarter q4 points at key 4 q4 + p / 4 (and + 16), channels 16 db + 4 (p % 4) .. + 4
  const uint32_t kro = (uint32_t)(i16 * S::kRow + 16 * k_place<D>(q4, i16));
  uint32_t vro[S::kND];
#pragma unroll
  for (int db = 0; db < S::kND; ++db) {
    const int r = 4 * q4 + (i16 >> 2), col = 16 * db + 4 * (lane & 3);
    vro[db] = (uint32_t)((E8 ? 0 : S::kTile) + r * S::kRow + 16 * v_place<D>(col >> 3, r) + 2 * (col & 7));
  }
  constexpr int CH = D / 8;
  const int crow = lane / CH, cpl = lane % CH;
  uint32_t klane[S::kRuns], vlane[S::kRuns];  // the lane's part of each copy's addresses
#pragma unroll
  for (int u = 0; u < S::kRuns; ++u) {
    klane[u] = crow * slot_bytes + 16 * k_place<D>(cpl, u * S::kRun + crow);
    vlane[u] = crow * slot_bytes + 16 * v_place<D>(cpl, u * S::kRun + crow);
  }

  // the rows of tokens [i0, i1) of sequence b and kv head h over keys [k_lo, k_hi); `slot`: where the partial result
  // goes, -1 for a whole one
  auto run = [&](const Rows& R, int b, int h, int i0, int i1, int k_lo, int k_hi, int slot) __attribute__((always_inline)) {
    const int32_t* pages = c.table + (int64_t)b * c.table_stride;
    const uint8_t* kbase = (const uint8_t*)c.k + kElem * h * c.head_stride;
    const uint8_t* vbase = (const uint8_t*)c.v + kElem * h * c.head_stride;
    const int nrows = (i1 - i0) * g;
    int lim[RB];
    int64_t out_row[RB];
    v4i qop[RB][S::kNQ];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int r = min(16 * rb + i16, nrows - 1), tok = R.t0 + i0 + r / g, head = h * g + r % g;
      lim[rb] = R.token_limit(i0 + r / g, causal);
      out_row[rb] = (int64_t)tok * a.heads + head;
      // operand cd's channels: 32 cd + 8 q4 .. + 8, of an 8-bit cache D / 4 q4 + 8 cd .. + 8
      const uint16_t* qp = a.q + tok * a.ldqt + head * a.ldqh + (E8 ? D / 4 : 8) * q4;
#pragma unroll
      for (int cd = 0; cd < S::kNQ; ++cd) qop[rb][cd] = *(const v4i*)(qp + (E8 ? 8 : 32) * cd);
    }
    const int lim_lo = R.token_limit(i0, causal);

    v4f oacc[RB][S::kND];
    float m_run[RB], l_run[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m_run[rb] = -INFINITY, l_run[rb] = 0.0f;
#pragma unroll
      for (int db = 0; db < S::kND; ++db) oacc[rb][db] = (v4f){};
    }

    for (int s_lo = k_lo, s_hi; s_lo < k_hi; s_lo = s_hi) {  // keys whose page ids are staged at a time
      const int p0 = s_lo >> c.page_shift;
      s_hi = segment_end(s_lo, k_hi, c.page_shift);
      if (s_lo > k_lo) __syncthreads();  // the ids of the last segment are no longer read
      for (int i = tid; i <= ((s_hi - 1) >> c.page_shift) - p0; i += 64 * NW)
        page_ids[i] = min(max(pages[p0 + i], 0), c.pages - 1);
      __syncthreads();
      const int ntiles = (s_hi - s_lo + FW_KEYS - 1) / FW_KEYS;
      bool aside = false;  // whether values of a masked tile were set aside (see the many-rows kernel)
      auto whole = [&](int t) {  // every row sees the whole tile
        return s_lo + (t + 1) * FW_KEYS <= min(lim_lo + 1, s_hi);
      };
      // a copy's rows lie in one page (page_size >= 8): its address is the wave's; copies wholly past the last key repeat
      // that key's
      auto issue = [&](int t) __attribute__((always_inline)) {
        const uint32_t st = (uint32_t)(uintptr_t)(mine + ((t / NW) & 1) * 2 * S::kTile);
#pragma unroll
        for (int u = 0; u < S::kRuns; ++u) {
          const uint32_t key = (uint32_t)min(s_lo + t * FW_KEYS + u * S::kRun, (s_hi - 1) & ~(S::kRun - 1));
          const uint64_t off = (uint64_t)(uint32_t)uniform(page_ids[(key >> c.page_shift) - p0]) * page_bytes +
                               (key & slot_mask) * slot_bytes;
          copy16(st + u * 1024, kbase + off, klane[u]);
          copy16(st + S::kTile + u * 1024, vbase + off, vlane[u]);
        }
      };
      // E8: the loads of a tile, by runs of 8 rows, which lie in one page: their places are the wave's. Runs wholly past the
      // last key repeat that key's.
      auto load = [&](int t, FewRaw<D>& w) __attribute__((always_inline)) {
        int64_t at[4], sat[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = min(s_lo + t * FW_KEYS + 8 * r, (s_hi - 1) & ~7);
          const int page = uniform(page_ids[(key >> c.page_shift) - p0]);
          at[r] = (int64_t)((uint64_t)(uint32_t)page * page_bytes + (key & slot_mask) * slot_bytes);
          sat[r] = page * c.s_page_stride + h * c.s_head_stride + (key & slot_mask);
        }
        const uint32_t k_lane = (i16 & 7) * slot_bytes + D / 4 * q4;
        const uint32_t v_lane = (lane / (D / 16) & 7) * slot_bytes + 16 * (lane % (D / 16));
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint8_t* p = kbase + (i16 < 8 ? at[2 * x] : at[2 * x + 1]) + k_lane;
#pragma unroll
          for (int i = 0; i < FewRaw<D>::kK; ++i) w.k[x][i] = *(const v4i*)(p + 16 * i);
        }
#pragma unroll
        for (int u = 0; u < FewRaw<D>::kV; ++u)
          w.v[u] = *(const v4i*)(vbase + (D == 128 ? at[u] : lane < 32 ? at[2 * u] : at[2 * u + 1]) + v_lane);
        const int run = lane >> 3 & 3;
        w.scale = (lane < 32 ? c.ks : c.vs)[(run < 2 ? run == 0 ? sat[0] : sat[1] : run == 2 ? sat[2] : sat[3]) + (lane & 7)];
      };
      auto step = [&](int t, const FewRaw<D>& w, auto mask_c) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask_c)::value;
        uint8_t* kb = E8 ? mine : mine + ((t / NW) & 1) * 2 * S::kTile;
        const int k0 = s_lo + t * FW_KEYS;
        v4i pop[RB];
        float ks[2], vs[FewRaw<D>::kV];
        if constexpr (E8) {
#pragma unroll
          for (int u = 0; u < FewRaw<D>::kV; ++u)
            vs[u] = scale_of((uint32_t)__shfl((int)w.scale, 32 + FewRaw<D>::kRows * u + lane / (D / 16)));
          ks[0] = scale_of((uint32_t)__shfl((int)w.scale, i16)), ks[1] = scale_of((uint32_t)__shfl((int)w.scale, 16 + i16));
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int u = 0; u < FewRaw<D>::kV; ++u) {
            const int row = FewRaw<D>::kRows * u + lane / (D / 16);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              v4i x = widen8<T>(w.v[u][2 * e], w.v[u][2 * e + 1], vs[u]);
              if (MASK) {
                if (k0 + row >= s_hi) x = (v4i){};  // whatever a page holds past the end
                else if (take_nonfinite<T>(x)) aside = true;
              }
              *(v4i*)(kb + row * S::kRow + 16 * v_place<D>(2 * (lane % (D / 16)) + e, row)) = x;
            }
          }
        } else if (MASK) {
#pragma unroll
          for (int u = 0; u < S::kRuns; ++u) {
            v4i* at = (v4i*)(kb + S::kTile + u * 1024 + lane * 16);
            v4i x = *at;
            if (k0 + u * S::kRun + crow >= s_hi) *at = (v4i){};  // whatever a page holds past the end
            else if (take_nonfinite<T>(x)) *at = x, aside = true;
          }
        }
        v4f sc[RB][2];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) sc[rb][0] = sc[rb][1] = (v4f){};
#pragma unroll
        for (int cd = 0; cd < S::kNQ; ++cd)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            v4i kop;
            if constexpr (E8) {
              kop = widen8<T>(w.k[x][cd / 2][2 * (cd & 1)], w.k[x][cd / 2][2 * (cd & 1) + 1], ks[x]);
            } else {
              kop = *(const v4i*)(kb + 16 * x * S::kRow + (kro ^ (uint32_t)(64 * cd)));
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) sc[rb][x] = Mfma<T>::tall(kop, qop[rb][cd], sc[rb][x]);
          }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          // the lane's scores: its row, keys 16 x + 4 q4 + r
          if (a.scores && 16 * rb + i16 < nrows) {
            float* sp = a.scores + out_row[rb] * a.score_stride + k0 + 4 * q4;
#pragma unroll
            for (int x = 0; x < 2; ++x)
              if (k0 + 16 * x + 4 * q4 < a.score_stride)
                *(float4*)(sp + 16 * x) = make_float4(sc[rb][x][0] * a.c_log2, sc[rb][x][1] * a.c_log2,
                                                      sc[rb][x][2] * a.c_log2, sc[rb][x][3] * a.c_log2);
          }
          float mx = -INFINITY;
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              if (MASK && 16 * x + r > lim[rb] - k0 - 4 * q4) sc[rb][x][r] = -INFINITY;
              mx = fmaxf(mx, sc[rb][x][r]);
            }
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32)) * a.c_log2;
          const bool bump = mx > m_run[rb];
          const float m_new = bump ? mx : m_run[rb];
          const float ref = m_new == -INFINITY ? 0.0f : m_new;
          const float alpha = __builtin_amdgcn_exp2f(m_run[rb] - ref);
          m_run[rb] = m_new;
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[rb][e >> 2][e & 3], a.c_log2, -ref));
          l_run[rb] = __builtin_fmaf(l_run[rb], alpha, ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])));
          pop[rb] = (v4i){Mfma<T>::pack(p[0], p[1]), Mfma<T>::pack(p[2], p[3]), Mfma<T>::pack(p[4], p[5]),
                          Mfma<T>::pack(p[6], p[7])};
          if (__builtin_amdgcn_ballot_w64(bump) != 0) {
#pragma unroll
            for (int db = 0; db < S::kND; ++db) oacc[rb][db] *= alpha;
          }
        }
        if constexpr (E8) {  // all reads ahead of the products: one at a time each waits for its own
          v4i vop[S::kND];
#pragma unroll
          for (int db = 0; db < S::kND; ++db)
            vop[db] = two_halves(lds_read_tr(kb + vro[db]), lds_read_tr(kb + vro[db] + 16 * S::kRow));
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int db = 0; db < S::kND; ++db)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) oacc[rb][db] = Mfma<T>::tall(vop[db], pop[rb], oacc[rb][db]);
        } else {
#pragma unroll
          for (int db = 0; db < S::kND; ++db) {
            const v4s_ lo = lds_read_tr(kb + vro[db]), hi = lds_read_tr(kb + vro[db] + 16 * S::kRow);
            const v4i vop = two_halves(lo, hi);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) oacc[rb][db] = Mfma<T>::tall(vop, pop[rb], oacc[rb][db]);
          }
        }
      };
      if constexpr (E8) {
        // tiles wave, wave + NW, ...: two in flight, in registers of their own. The loads go out whether or not there is such
        // a tile (past the end they repeat the last key), so that how many are outstanding is known wherever one is waited
        // for: with conditions around them every wait is for all. (Two tiles' loads a wave are repeated so: next to nothing of
        // a long run, half of all of a split of 256 keys, whose lines are in the caches then)
        FewRaw<D> w0, w1;
        auto tile = [&](int t, FewRaw<D>& w) __attribute__((always_inline)) {
          if (whole(t)) step(t, w, std::false_type{});
          else step(t, w, std::true_type{});
          load(t + 2 * NW, w);
        };
        load(wave, w0);
        load(wave + NW, w1);
        for (int t = wave; t < ntiles; t += 2 * NW) {
          tile(t, w0);
          if (t + NW >= ntiles) break;
          tile(t + NW, w1);
        }
      } else {
        // tiles wave, wave + NW, ...: the next one's copies go out before this one's are waited for
        if (wave < ntiles) issue(wave);
        for (int t = wave; t < ntiles; t += NW) {
          if (t + NW < ntiles) {
            issue(t + NW);
            wait_vm_lgkm0<2 * S::kRuns>();
          } else {
            wait_vm_lgkm0<0>();
          }
          asm volatile("" ::: "memory");
          if (whole(t)) step(t, {}, std::false_type{});
          else step(t, {}, std::true_type{});
          wait_vm_lgkm0<63>();  // this tile's LDS reads are done before its stage is copied into again
          asm volatile("" ::: "memory");
        }
      }
      if (__builtin_amdgcn_ballot_w64(aside) != 0) {  // rows that see keys whose values were set aside: those values
        for (int t = wave; t < ntiles; t += NW) {
          if (whole(t)) continue;
          for (int key = s_lo + t * FW_KEYS; key < min(s_lo + (t + 1) * FW_KEYS, s_hi); ++key) {
            const int page = paged_page(c, pages, key);
            const int64_t at_key = paged_at(c, page, h, key);
            const float ks = held_scale<E8>(c, c.ks, page, h, key), vs = held_scale<E8>(c, c.vs, page, h, key);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
              float s = 0.0f;
#pragma unroll
              for (int cd = 0; cd < S::kNQ; ++cd)
                s = dot8<T>(qop[rb][cd], held8<T, E8>(c.k, at_key + (E8 ? D / 4 * q4 + 8 * cd : 8 * q4 + 32 * cd), ks), s);
              s += __shfl_xor(s, 16);
              s += __shfl_xor(s, 32);
              const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s, a.c_log2, -m_run[rb]));
              if (key <= lim[rb]) {
#pragma unroll
                for (int db = 0; db < S::kND; ++db)
#pragma unroll
                  for (int r = 0; r < 4; ++r) {
                    const float v = held1<T, E8>(c.v, at_key + 16 * db + 4 * q4 + r, vs);
                    if (!(fabsf(v) < INFINITY)) oacc[rb][db][r] = fmaf(p, v, oacc[rb][db][r]);
                  }
              }
            }
          }
        }
      }
    }

    // join the waves: each leaves its O [row][channel] with its m and l, thread by thread they are summed in wave order
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      float* op = (float*)mine + (16 * rb + i16) * (D + 4);
#pragma unroll
      for (int db = 0; db < S::kND; ++db) *(v4f*)(op + 16 * db + 4 * q4) = oacc[rb][db];
      l_run[rb] += __shfl_xor(l_run[rb], 16);
      l_run[rb] += __shfl_xor(l_run[rb], 32);
      if (q4 == 0) stat[wave][0][16 * rb + i16] = m_run[rb], stat[wave][1][16 * rb + i16] = l_run[rb];
    }
    __syncthreads();
    for (int i = tid; i < nrows * (D / 4); i += 64 * NW) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, stat[w][0][r]);
      const float ref = m == -INFINITY ? 0.0f : m;
      float l = 0.0f;
      v4f o = {};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = __builtin_amdgcn_exp2f(stat[w][0][r] - ref);
        l = __builtin_fmaf(stat[w][1][r], f, l);
        o += *(const v4f*)((const float*)(lds + w * S::kWave) + r * (D + 4) + d) * f;
      }
      const float inv = inverse_sum(l), lse2 = log2_sum(m, l);
      const int64_t row = (int64_t)(R.t0 + i0 + r / g) * a.heads + h * g + r % g;
      if (slot < 0) {
        *(uint2*)(a.o + row * D + d) = make_uint2((uint32_t)Mfma<T>::pack(o[0] * inv, o[1] * inv),
                                                  (uint32_t)Mfma<T>::pack(o[2] * inv, o[3] * inv));
        if (d == 0) a.lse[row] = lse2 * kLn2;
      } else {
        const int64_t prow = SHARES ? (int64_t)slot * BM + r : (int64_t)slot * a.tokens * a.heads + row;
        // a split without keys leaves only its lse
        if (SHARES || k_hi > k_lo) *(v4f*)(a.o_part + prow * D + d) = o * inv;
        if (d == 0) a.lse_part[prow] = lse2;
      }
    }
  };

  if constexpr (!SHARES) {
    const int groups = c.batch * c.kv_heads;
    const int grp = blockIdx.x % groups, split = blockIdx.x / groups, b = grp / c.kv_heads, h = grp % c.kv_heads;
    const Rows R = uniform_rows_of(c, b, a.tokens, g);
    for (int i0 = 0; i0 < R.n; i0 += tt) {
      const int i1 = min(i0 + tt, R.n), lim_hi = R.token_limit(i1 - 1, causal), k_lo = split * a.split_keys;
      const int k_hi = split + 1 < a.splits ? min(k_lo + a.split_keys, lim_hi + 1) : lim_hi + 1;
      if (i0 > 0) __syncthreads();  // the stages are copied into again
      run(R, b, h, i0, i1, k_lo, k_hi, a.splits > 1 ? split : -1);
    }
  } else {
    const int share = blockIdx.x % kXcds * (a.shares / kXcds) + blockIdx.x / kXcds;
    const LineLanes lanes = line_lanes(c, a.tokens, tt, causal, 0);
    const int64_t per_head = head_line(c, a.tokens, tt, causal, lanes), all = per_head * c.kv_heads;
    const int64_t x0 = share_start(all, share, a.shares), x1 = share_start(all, share + 1, a.shares);
    no_cuts(a, share);
    if (x0 >= x1) return;
    Place at = place_of<FW_UNIT>(c, a.tokens, tt, causal, per_head, lanes, x0);
    const Place end = place_of<FW_UNIT>(c, a.tokens, tt, causal, per_head, lanes, x1);
    Rows R = uniform_rows_of(c, at.b, a.tokens, g);
    while (true) {
      const int i0 = at.tile * tt, i1 = min(i0 + tt, R.n), lim_hi = R.token_limit(i1 - 1, causal);
      const bool last = at.h == end.h && at.b == end.b && at.tile == end.tile;
      const int units = max(1, (lim_hi + FW_UNIT) / FW_UNIT), to = last ? min(end.unit, units) : units;
      if (at.unit < to) {
        // a part goes into the share's slot: the first for a tile that an earlier share began, else the second
        const bool part = at.unit > 0 || to < units;
        if (part) set_cut(a, share, at.unit > 0, to == units, (i1 - i0) * g, R.t0 + i0, at.h);
        run(R, at.b, at.h, i0, i1, at.unit * FW_UNIT, min(to * FW_UNIT, lim_hi + 1),
            part ? 2 * share + (at.unit > 0 ? 0 : 1) : -1);
        __syncthreads();  // the stages are copied into again
      }
      if (last) break;
      at.unit = 0;
      if (i1 < R.n) {
        ++at.tile;
      } else {
        at.tile = 0;
        do {  // the next sequence with new tokens, of the next head after the last
          if (++at.b == c.batch) at.b = 0, ++at.h;
          if (at.h == c.kv_heads) return;  // the line's end
          R = uniform_rows_of(c, at.b, a.tokens, g);
        } while (R.n == 0);
      }
    }
  }
}

// Joins a row's splits, in their order: D / 4 lanes a row, 4 channels each, 4 splits' loads in flight.
template <class T, int D>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnArgs a) {
  constexpr int L = D / 4;
  const int64_t rows = (int64_t)a.tokens * a.heads, row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (row >= rows) return;
  const int d = threadIdx.x % L * 4;
  float m = -INFINITY;
  for (int s = 0; s < a.splits; s += 4) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = a.lse_part[min(s + e, a.splits - 1) * rows + row];
    m = fmaxf(fmaxf(fmaxf(m, x[0]), fmaxf(x[1], x[2])), x[3]);
  }
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  v4f o = {};
  for (int s = 0; s < a.splits; s += 4) {
    float f[4];
    v4f x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = s + e < a.splits ? __builtin_amdgcn_exp2f(a.lse_part[min(s + e, a.splits - 1) * rows + row] - ref) : 0.0f;
      x[e] = (v4f){};
      // a split without keys for the row has not written its part
      if (f[e] != 0.0f) x[e] = *(const v4f*)(a.o_part + ((s + e) * rows + row) * D + d);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) l += f[e], o += x[e] * f[e];
  }
  const float inv = inverse_sum(l);
  *(uint2*)(a.o + row * D + d) = make_uint2((uint32_t)Mfma<T>::pack(o[0] * inv, o[1] * inv),
                                            (uint32_t)Mfma<T>::pack(o[2] * inv, o[3] * inv));
  if (d == 0) a.lse[row] = log2_sum(m, l) * kLn2;
}

// ---------------------------------------------------------------------------
// gathered weights: w[key] += sum over the rows that see it of 2^(s c - lse)
// ---------------------------------------------------------------------------

// From the scores that the few-rows kernel left (a sixteenth of the keys' bytes at 4 heads of 128 to a kv head, where
// recomputing them would read the keys again): 4 keys a thread, the rows in order. 16 sequences of up to 8192 keys: 6.8 us.
__global__ __launch_bounds__(256) void paged_gather_scores_kernel(AttnArgs a) {
  const PagedArgs& c = a.c;
  const int b = blockIdx.y / c.kv_heads, h = blockIdx.y % c.kv_heads, g = a.heads / c.kv_heads;
  const Rows R = rows_of(c, b, a.tokens, g);
  for (int j0 = (blockIdx.x * 256 + threadIdx.x) * 4; j0 < R.len; j0 += gridDim.x * 1024) {
    float sum[4] = {};
    for (int r = 0; r < R.total; ++r) {
      const int lim = R.limit(r, a.causal != 0);
      if (j0 > lim) continue;
      const int64_t row = (int64_t)(R.t0 + r / g) * a.heads + h * g + r % g;
      const float lse2 = gather_lse2(a.lse[row]);
      const float4 s = *(const float4*)(a.scores + row * a.score_stride + j0);
      const float x[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j0 + e <= lim) sum[e] += __builtin_amdgcn_exp2f(x[e] - lse2);
    }
    const int page = paged_page(c, c.table + (int64_t)b * c.table_stride, j0);  // page_size >= 8: all four in one page
    float* w = c.w + paged_w_at(c, page, h, j0);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j0 + e < R.len) w[e] += sum[e];
  }
}

// Recomputed: a wave holds 32 keys as the MFMA's A operand and walks the rows in tiles of 64 (64 / group new tokens with
// all heads of the group), which a workgroup of 4 waves (128 keys) copies to LDS, double buffered (q^T as B). A lane sums
// its row's probabilities for 16 keys; the lanes of the 32 rows are joined at the end. The tokens are divided over
// `splits` workgroups where the keys alone are too few to fill the chip: each leaves its sums in w_part
// [split][group][score_stride], joined in order. Two sequences of 1021 and 866 tokens over 6007 and 2367 keys, 24 heads of
// 128 over 4: 112 us. It waits rather than computes (vector unit busy 32 % of the time, matrix cores 17 %, LDS 11 %): a wave
// has its scores and then their exponentials in turn, between two barriers a tile. With a division a row in the copies and a
// mask on every tile of such odd groups 157.
constexpr int GT_WAVES = 4, GT_ROWS = 64, GT_KEYS = 32 * GT_WAVES;

template <class T, int D, bool E8>
__global__ __launch_bounds__(64 * GT_WAVES, 3) void paged_gather_tile_kernel(AttnArgs a) {
  constexpr int NQ = D / 16, kRow = 2 * D, kRun = 1024 / kRow, kRuns = GT_ROWS / kRun / GT_WAVES, kStage = GT_ROWS * kRow;
  constexpr int kAhead = 4;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kStage];
  const PagedArgs& c = a.c;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, j = lane & 31, hf = lane >> 5;
  const int groups = c.batch * c.kv_heads;
  const int grp = blockIdx.x % groups, rest = blockIdx.x / groups, split = rest % a.splits;
  const int b = grp / c.kv_heads, h = grp % c.kv_heads, g = a.heads / c.kv_heads, tt = GT_ROWS / g;
  const Rows R = uniform_rows_of(c, b, a.tokens, g);
  const bool causal = a.causal != 0;
  const int32_t* pages = c.table + (int64_t)b * c.table_stride;
  constexpr int CH = D / 8;
  const int crow = lane / CH, cpl = lane % CH;
  const uint32_t qro = (uint32_t)(j * kRow + 16 * k_place<D>(hf, j));  // chunk 2 cd + hf: xor 32 cd
  const uint16_t* q0 = a.q + R.t0 * a.ldqt + h * g * a.ldqh;
  const float* lse0 = a.lse + (int64_t)R.t0 * a.heads + h * g;
  int64_t qoff[kRuns];  // the lane's part of a whole tile's copies
#pragma unroll
  for (int u = 0; u < kRuns; ++u) {
    const int place = (wave + GT_WAVES * u) * kRun + crow, r = min(place, tt * g - 1);
    qoff[u] = r / g * a.ldqt + r % g * a.ldqh + 8 * k_place<D>(cpl, place);
  }

  for (int w0 = rest / a.splits * GT_KEYS; w0 < R.len; w0 += a.tiles * GT_KEYS) {
    const int j0 = w0 + 32 * wave, key = min(j0 + j, R.len - 1);
    const int kpage = paged_page(c, pages, key);
    const int64_t kat = paged_at(c, kpage, h, key);
    const float ks = held_scale<E8>(c, c.ks, kpage, h, key);
    v4i kop[NQ];
#pragma unroll
    for (int cd = 0; cd < NQ; ++cd) kop[cd] = held8<T, E8>(c.k, kat + 8 * hf + 16 * cd, ks);
    // tokens that see a key of this workgroup's come last; this split's share of their tiles
    const int first = causal ? max(w0 - (R.len - R.n), 0) : 0;
    const int all = first < R.n ? (R.n - first + tt - 1) / tt : 0;
    const int t_lo = (int)((int64_t)all * split / a.splits), t_hi = (int)((int64_t)all * (split + 1) / a.splits);
    // row r of a tile: its token i + r / g (the last of the sequence where that is past it), head r % g; rows past the
    // tile's tokens repeat its last
    auto issue = [&](int t) __attribute__((always_inline)) {
      const uint32_t st = (uint32_t)(uintptr_t)(lds + (t & 1) * kStage);
      const int i = first + t * tt, most = R.n - 1 - i;
#pragma unroll
      for (int u = 0; u < kRuns; ++u) {
        const int run = wave + GT_WAVES * u, r = min(run * kRun + crow, tt * g - 1);
        const int64_t off = most >= tt - 1 ? qoff[u] : min(r / g, most) * a.ldqt + r % g * a.ldqh + 8 * k_place<D>(cpl, run * kRun + crow);
        copy16(st + run * 1024, q0 + i * a.ldqt + off);
      }
    };
    float sum[16] = {}, lse2[2], next2[2];
    auto lse_of = [&](int t) __attribute__((always_inline)) {
      const int i = first + t * tt, most = R.n - 1 - i;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = 32 * x + j;  // rows past the tile's tokens: a probability of 0
        next2[x] = r < tt * g ? gather_lse2(lse0[(int64_t)(i + min(r / g, most)) * a.heads + r % g]) : INFINITY;
      }
    };
    if (t_lo < t_hi) {
      lse_of(t_lo);
      issue(t_lo);
    }
    for (int t = t_lo; t < t_hi; ++t) {
      wait_vm_lgkm0<0>();
      __syncthreads();  // tile t is there; everyone is done with the other stage
      lse2[0] = next2[0], lse2[1] = next2[1];
      if (t + 1 < t_hi) {
        lse_of(t + 1);
        issue(t + 1);
      }
      const uint8_t* st = lds + (t & 1) * kStage;
      const int i0 = first + t * tt;
      v16f s[2];
      v4i ring[kAhead];  // operands read ahead of their MFMAs, in this order
      auto read = [&](int k) __attribute__((always_inline)) {
        ring[k % kAhead] = *(const v4i*)(st + 32 * (k % 2) * kRow + (qro ^ (uint32_t)(32 * (k / 2))));
      };
#pragma unroll
      for (int k = 0; k < kAhead; ++k) read(k);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 2 * NQ; ++k) {
        s[k % 2] = Mfma<T>::wide(kop[k / 2], ring[k % kAhead], k < 2 ? (v16f){} : s[k % 2]);
        if (k + kAhead < 2 * NQ) read(k + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
      // tiles all of whose tokens see all of the wave's keys need no mask
      if (i0 + tt <= R.n && R.token_limit(i0, causal) >= j0 + 31) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[i] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][i], a.c_log2, -lse2[x]));
      } else {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = 32 * x + j, i = i0 + r / g;
          const int vis = r < tt * g && i < R.n ? R.token_limit(i, causal) - j0 - 4 * hf : -64;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][e], a.c_log2, -lse2[x]));
            sum[e] += 8 * (e >> 2) + (e & 3) <= vis ? p : 0.0f;
          }
        }
      }
    }
    __syncthreads();  // the next keys' first tile is copied into a stage that this one's last may still be read from
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int w = 16; w; w >>= 1) sum[i] += __shfl_xor(sum[i], w);
    if (j == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int at = j0 + 8 * (i >> 2) + 4 * hf + (i & 3);
        if (at >= R.len) continue;
        if (a.splits > 1) a.w_part[((int64_t)split * groups + grp) * a.score_stride + at] = sum[i];
        else c.w[paged_w_at(c, paged_page(c, pages, at), h, at)] += sum[i];
      }
    }
  }
}

__global__ __launch_bounds__(256) void paged_gather_join_kernel(AttnArgs a) {
  const PagedArgs& c = a.c;
  const int grp = blockIdx.y, b = grp / c.kv_heads, h = grp % c.kv_heads, groups = c.batch * c.kv_heads;
  const int len = paged_kv_len(c, b);
  for (int j = blockIdx.x * 256 + threadIdx.x; j < len; j += gridDim.x * 256) {
    float sum = 0.0f;
    for (int s = 0; s < a.splits; ++s) sum += a.w_part[((int64_t)s * groups + grp) * a.score_stride + j];
    c.w[paged_w_at(c, paged_page(c, c.table + (int64_t)b * c.table_stride, j), h, j)] += sum;
  }
}

// ---------------------------------------------------------------------------
// the choice of kernel and splits
// ---------------------------------------------------------------------------
constexpr int64_t kScoreBytes = 256ll << 20;  // most workspace spent on kept scores

struct Plan {
  bool matrix, few, keep_scores;
  int64_t tile_rows;  // rows a workgroup: 16 or 32 (few), 128 or 256
  int splits, split_keys, shares, tiles;
  int row_splits, key_tiles;  // of the recomputing gather
  int64_t score_stride, gathered, part_floats, bytes;
};

template <bool E8>
Plan plan_of(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t d, int64_t max_q, int64_t max_kv,
             int64_t capacity, bool gather) {
  Plan p = {};
  // a row tile holds a token's whole group of query heads
  p.matrix = (d == 64 || d == 128) && heads / kv_heads <= 256;
  p.splits = 1, p.split_keys = 1 << 30;
  if (!p.matrix || batch == 0 || tokens == 0) return p;
  const int64_t group = heads / kv_heads, rows = (max_q < 1 ? 1 : max_q) * group, groups = batch * kv_heads;
  max_kv = max_kv < 1 ? 1 : max_kv;
  p.few = rows <= 32;
  p.tile_rows = p.few ? (rows <= 16 ? 16 : 32) : rows <= 128 ? 128 : 256;
  if (p.few) p.keep_scores = gather && tokens * heads * ((capacity + 3) / 4 * 4) * 4 <= kScoreBytes;
  // few splits only: their join reads them in turn (72 of 2 sequences of 18361 keys: 39 us in all, as shares 19)
  if (p.few && groups * ((max_kv + 255) / 256) <= kCus && max_kv <= 8 * 256) {
    p.split_keys = 256;
    p.splits = (int)((max_kv + 255) / 256);
    if (p.splits > 1) p.part_floats = p.splits * tokens * heads * (d + 1);
  } else {
    // as many workgroups as fit at once, but no more than 32 to a row tile: 2 sequences of 95 tokens over 5619 keys, 6
    // heads over 2, cut into 64 parts a tile take 26 us, into 32 23, into 8 32; the join reads every part
    const int64_t tt = p.tile_rows / group, tiles = ((max_q < 1 ? 1 : max_q) + tt - 1) / tt;
    const int64_t row_tiles = kv_heads * std::min(batch * tiles, tokens / tt + batch), units = (max_kv + 63) / 64;
    // (two workgroups a CU where they fit; 8-bit rows leave fewer bytes in flight a wave: 16 rows over up to 32768 keys of 32
    // sequences take 170 us with two and 178 with one, heads of 64 90 and 124)
    p.shares = p.tile_rows == 128 || (E8 && p.tile_rows == 16) ? 2 * kCus : kCus;
    // Many rows: a workgroup a row tile where that takes no longer. 64 keys take it about 2 us, and it goes through
    // whole rounds of workgroups; shares always end together, but take 8 us to find and to join and 6 % more for
    // their cut tiles (4096 tokens over 16500 keys, 32 heads over 8, 512 tiles: 894 us against 965; 150 tokens over 152
    // keys, 8 heads over 4: 16.9 against 20.3)
    const int64_t rounds = (row_tiles + p.shares - 1) / p.shares;
    if (!p.few && 200 * units * rounds * p.shares < 212 * units * row_tiles + 800 * p.shares && groups * tiles < (1ll << 31)) {
      p.tiles = (int)tiles;
      p.shares = 0;
    } else {
      while (p.shares > 8 && p.shares > 32 * row_tiles) p.shares /= 2;
      p.part_floats = 2 * p.shares * p.tile_rows * (d + 1);
    }
  }
  p.score_stride = (capacity + 3) / 4 * 4;
  if (p.keep_scores) {
    p.gathered = tokens * heads * p.score_stride;
  } else if (gather) {
    p.key_tiles = (int)(max_kv > 0 ? (max_kv + GT_KEYS - 1) / GT_KEYS : 1);
    // six workgroups a CU, of at least 2 row tiles each
    int64_t want = (1536 + p.key_tiles * groups - 1) / (p.key_tiles * groups), most = rows / (2 * GT_ROWS);
    if (want > most) want = most;
    if (want < 1 || want * groups * p.score_stride * 4 > kScoreBytes) want = 1;
    p.row_splits = (int)want;
    if (want > 1) p.gathered = want * groups * p.score_stride;
  }
  p.bytes = (p.gathered + p.part_floats) * 4 + p.shares * 16;
  return p;
}

template <class T, int D, bool E8>
void launch_matrix(const Plan& p, AttnArgs a, int64_t max_kv, bool gather, hipStream_t st) {
  const unsigned groups = (unsigned)(a.c.batch * a.c.kv_heads);
  if (p.few && p.shares == 0) {
    const dim3 grid(groups * (unsigned)p.splits), block(64 * FW_WAVES);
    if (p.tile_rows == 16) hipLaunchKernelGGL((paged_attn_few_kernel<T, D, 1, false, E8>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((paged_attn_few_kernel<T, D, 2, false, E8>), grid, block, 0, st, a);
    if (p.splits > 1)
      hipLaunchKernelGGL((paged_attn_join_kernel<T, D>), dim3((unsigned)(((int64_t)a.tokens * a.heads * D + 1023) / 1024)),
                         dim3(256), 0, st, a);
  } else if (p.shares == 0) {
    const dim3 grid(groups * (unsigned)p.tiles);
    if (p.tile_rows == 128) hipLaunchKernelGGL((paged_attn_tile_kernel<T, D, 64, 4, E8>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_attn_tile_kernel<T, D, 64, 8, E8>), grid, dim3(512), 0, st, a);
  } else {
    const dim3 grid((unsigned)p.shares);
    const dim3 jgrid((unsigned)(p.shares * (p.tile_rows / JT)));
    if (p.tile_rows == 16) {
      hipLaunchKernelGGL((paged_attn_few_kernel<T, D, 1, true, E8>), grid, dim3(64 * FW_WAVES), 0, st, a);
      hipLaunchKernelGGL((paged_attn_join_parts_kernel<T, D, 16>), jgrid, dim3(256), 0, st, a);
    } else if (p.tile_rows == 32) {
      hipLaunchKernelGGL((paged_attn_few_kernel<T, D, 2, true, E8>), grid, dim3(64 * FW_WAVES), 0, st, a);
      hipLaunchKernelGGL((paged_attn_join_parts_kernel<T, D, 32>), jgrid, dim3(256), 0, st, a);
    } else if (p.tile_rows == 128) {
      hipLaunchKernelGGL((paged_attn_tile_kernel<T, D, 64, 4, E8>), grid, dim3(256), 0, st, a);
      hipLaunchKernelGGL((paged_attn_join_parts_kernel<T, D, 128>), jgrid, dim3(256), 0, st, a);
    } else {
      hipLaunchKernelGGL((paged_attn_tile_kernel<T, D, 64, 8, E8>), grid, dim3(512), 0, st, a);
      hipLaunchKernelGGL((paged_attn_join_parts_kernel<T, D, 256>), jgrid, dim3(256), 0, st, a);
    }
  }
  if (!gather) return;
  if (p.keep_scores) {
    const unsigned blocks = (unsigned)((max_kv + 1023) / 1024);
    hipLaunchKernelGGL(paged_gather_scores_kernel, dim3(blocks ? blocks : 1, groups), dim3(256), 0, st, a);
  } else {
    a.tiles = p.key_tiles, a.splits = p.row_splits;
    if (a.heads / a.c.kv_heads > GT_ROWS) {
      hipLaunchKernelGGL((paged_gather_rows_kernel<T, E8>), dim3((unsigned)((max_kv + 63) / 64 > 0 ? (max_kv + 63) / 64 : 1), groups),
                         dim3(64), 0, st, a.c, a.q, a.ldqt, a.ldqh, a.lse, a.tokens, a.heads, D, a.c_log2, a.causal);
      return;
    }
    hipLaunchKernelGGL((paged_gather_tile_kernel<T, D, E8>), dim3(groups * (unsigned)(a.tiles * a.splits)),
                       dim3(64 * GT_WAVES), 0, st, a);
    if (a.splits > 1)
      hipLaunchKernelGGL(paged_gather_join_kernel, dim3((unsigned)(max_kv > 0 ? (max_kv + 255) / 256 : 1), groups), dim3(256),
                         0, st, a);
  }
}

// The entry points' bodies; `scales`: of an 8-bit cache
template <bool E8>
int64_t workspace_of(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_q,
                     int64_t max_kv, int64_t capacity, int gather) {
  if (batch < 0 || tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_q < 0 || max_kv < 0) return 0;
  return plan_of<E8>(batch, tokens, heads, kv_heads, head_dim, max_q, max_kv, capacity, gather != 0).bytes;
}

template <bool E8>
int attention_call(const char* what, const gwa_paged_cache* cache, const gwa_paged_scales* scales, const void* q,
                   int64_t ldqt, int64_t ldqh, void* o, float* lse, int64_t tokens, int64_t heads, int64_t max_q,
                   int64_t max_kv, float scale, int causal, int gather, void* workspace, int64_t workspace_bytes,
                   void* stream) {
  PagedArgs c;
  const int bad = paged_check(what, cache, true, gather != 0, &c, scales);
  if (bad != GWA_OK) return bad;
  const int64_t d = cache->head_dim;
  GWA_REQUIRE(tokens >= 0 && tokens < (1ll << 31) && heads > 0 && heads < 65536 && heads % c.kv_heads == 0,
              "%s: %lld tokens, %lld query heads over %d kv heads", what, (long long)tokens, (long long)heads,
              c.kv_heads);
  GWA_REQUIRE(max_q >= 0 && max_q <= tokens && max_kv >= 0 && max_kv <= c.capacity,
              "%s: max_q %lld of %lld tokens, max_kv %lld in a table of %d slots", what, (long long)max_q,
              (long long)tokens, (long long)max_kv, c.capacity);
  GWA_REQUIRE(scale > 0.0f && scale < INFINITY, "%s: scale must be positive and finite", what);
  GWA_REQUIRE(ldqt % 8 == 0 && ldqh % 8 == 0 && ldqt > 0 && ldqh > 0 && tokens * ldqt < (1ll << 46),
              "%s: q's token and head strides must be positive multiples of 8", what);
  const int64_t rows = tokens * heads, groups = (int64_t)c.batch * c.kv_heads;
  GWA_REQUIRE(rows < (1ll << 31) && groups < 65536, "%s: %lld rows of %lld sequences' heads are too many", what,
              (long long)rows, (long long)groups);
  if (tokens == 0) return GWA_OK;
  GWA_REQUIRE(q && o && lse, "%s: null pointer", what);
  GWA_REQUIRE(GWA_ALIGNED(q, 16) && GWA_ALIGNED(o, 16) && GWA_ALIGNED(lse, 4),
              "%s: q and o must be 16-byte aligned", what);
  hipStream_t st = (hipStream_t)stream;
  const float c_log2 = scale * kLog2e;
  const Plan p = plan_of<E8>(c.batch, tokens, heads, c.kv_heads, d, max_q, max_kv, c.capacity, gather != 0);
  if (p.matrix && c.batch > 0) {
    GWA_REQUIRE(rows * p.splits < (1ll << 31) && groups * (p.key_tiles + 1) * (p.row_splits + 1) < (1ll << 31),
                "%s: %lld rows over %lld sequences' heads are too many", what, (long long)rows, (long long)groups);
    GWA_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && GWA_ALIGNED(workspace, 16)),
                "%s: a workspace of %lld bytes, %lld are needed (16-byte aligned)", what, (long long)workspace_bytes,
                (long long)p.bytes);
    float* ws = (float*)workspace;
    const int64_t n_o = p.part_floats / (d + 1) * d;
    // scores or gathered parts first: scores' rows are read and written 16 bytes at a time
    const int64_t n_s = p.gathered;
    const AttnArgs a = {c, (const uint16_t*)q, ldqt, ldqh, (uint16_t*)o, lse, ws + n_s, ws + n_s + n_o,
                        (int4*)(ws + n_s + p.part_floats),
                        p.keep_scores ? ws : nullptr, ws, p.score_stride, (int)tokens, (int)heads, p.splits, p.split_keys,
                        p.tiles, p.shares, c_log2, causal};
    if (cache->dtype == GWA_DT_BF16) {
      if (d == 128) launch_matrix<Bf16, 128, E8>(p, a, max_kv, gather != 0, st);
      else launch_matrix<Bf16, 64, E8>(p, a, max_kv, gather != 0, st);
    } else {
      if (d == 128) launch_matrix<Fp16, 128, E8>(p, a, max_kv, gather != 0, st);
      else launch_matrix<Fp16, 64, E8>(p, a, max_kv, gather != 0, st);
    }
    return gwa_check_launch(what);
  }
  const dim3 grid((unsigned)((rows + RW_WAVES - 1) / RW_WAVES)), block(64 * RW_WAVES);
  const dim3 ggrid((unsigned)((max_kv + 63) / 64 > 0 ? (max_kv + 63) / 64 : 1), (unsigned)groups);
  auto run = [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((paged_attn_rows_kernel<T, E8>), grid, block, 0, st, c, (const uint16_t*)q, ldqt, ldqh,
                       (uint16_t*)o, lse, (int)tokens, (int)heads, (int)d, c_log2, causal);
    if (gather && groups > 0)
      hipLaunchKernelGGL((paged_gather_rows_kernel<T, E8>), ggrid, dim3(64), 0, st, c, (const uint16_t*)q, ldqt, ldqh, lse,
                         (int)tokens, (int)heads, (int)d, c_log2, causal);
  };
  if (cache->dtype == GWA_DT_BF16) run(Bf16{});
  else run(Fp16{});
  return gwa_check_launch(what);
}

}  // namespace
