// New tokens into a paged cache of e4m3 codes under a power of two a row, and rows of it read back. Both move each value
// once: they are bound by memory, small calls by their launch.
#include "paged_rotary.h"

namespace {

constexpr int W8_THREADS = 512, R8_THREADS = 256;  // of a workgroup at most; of one that reads

// A row's scale byte b from its largest finite magnitude (fp32 bits), 2^(127 - b), and the largest code magnitude. 448 * 2^e
// >= amax holds from e = floor(log2 amax) - 8 on, or one more where amax's fraction passes that of 448 = 1.75 * 2^8. At
// the type's last binade 256 * 2^e would be infinite: there codes end at 240. A rotation may take a key past the type's
// range, by tables longer than 1; it counts as the type's largest value then, whose byte is kTop.
struct RowScale {
  uint32_t byte;
  float inverse, most;
};
template <int DT>
__device__ __forceinline__ RowScale row_scale(uint32_t amax) {
  constexpr int kTop = DT == GWA_DT_BF16 ? 247 : 135;
  const int b = min(max((int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u), 1), kTop);
  return {(uint32_t)b, __uint_as_float((uint32_t)(254 - b) << 23), b == kTop ? 240.0f : 448.0f};
}
// x under its row's scale, for the conversion, which rounds to nearest (ties to even) and takes infinities and NaN to NaN.
// No finite value of the row passes 448 (held_to).
__device__ __forceinline__ float scaled(float x, const RowScale& s) { return x * s.inverse; }
__device__ __forceinline__ uint2 codes8(const float (&x)[8], const RowScale& s) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(scaled(x[4 * i], s), scaled(x[4 * i + 1], s), 0, false);
    w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(scaled(x[4 * i + 2], s), scaled(x[4 * i + 3], s), r, true);
  }
  return make_uint2(w[0], w[1]);
}
// x, if finite, held to the largest code of a row whose codes end below 448
__device__ __forceinline__ float held_to(float x, const RowScale& s) {
  const float top = s.most / s.inverse;
  return fabsf(x) < INFINITY ? fminf(fmaxf(x, -top), top) : x;
}
// the larger of `most` and |x|, NaN and (with FINITE) infinities left out
template <bool FINITE>
__device__ __forceinline__ float larger(float most, float x) {
  return FINITE && fabsf(x) == INFINITY ? most : fmaxf(most, fabsf(x));
}

// x's maximum over groups of n neighbouring lanes, n a power of two up to 64
__device__ __forceinline__ float group_max(float x, int n) {
  auto moved = [](float v, auto move_c) __attribute__((always_inline)) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), decltype(move_c)::value, 0xf, 0xf, true));
  };
  if (n > 1) x = fmaxf(x, moved(x, std::integral_constant<int, 0xb1>{}));   // the neighbour's, within four
  if (n > 2) x = fmaxf(x, moved(x, std::integral_constant<int, 0x4e>{}));   // the other pair's
  if (n > 4) x = fmaxf(x, moved(x, std::integral_constant<int, 0x141>{}));  // eight lanes mirrored
  if (n > 8) x = fmaxf(x, moved(x, std::integral_constant<int, 0x140>{}));  // sixteen
  if (n > 16) x = fmaxf(x, __shfl_xor(x, 16)), x = fmaxf(x, __shfl_xor(x, 32));
  return x;
}

// One workgroup a token: its query heads into q_out, its key and value heads into the slot, each row by 2^lane_bits lanes
// (the units of 16 channels of a row; with odd sizes, strides or places (not VEC) a wave, whose lanes take two pairs at
// most), which find the row's largest value between them. A row is read once and held in registers meanwhile. Every XCD
// has a run of neighbouring tokens, whose codes and scale bytes share lines in its L2.
// Bytes bound it, and on the way there the chain of dependent loads: the slot's three are scalar loads that no wait for a row
// falls among (as vector loads behind the row's: 4 us more), and the tables' go out before the row's are waited for.
// Measured: 10475 prompt tokens, 16 / 16 heads of 64, half of each rotated, fp16: 27 to 28 us, 3.9 TB/s; 8192 tokens, 32 / 8
// heads of 128: 37.5 us, 4.9 TB/s, without VEC 100; 48 tokens of as many sequences 4.5 us, without VEC 8.0. Workgroups
// of 256 threads whatever the rows are: 34.5 us of the prompts where this form then took 31; two or four
// tokens a workgroup: 31 to 38; a limit of 64 registers, for 8 waves a SIMD: spills, 30.
template <int DT, bool VEC>
__global__ __launch_bounds__(W8_THREADS) void paged_write_fp8_kernel(PagedArgs c, const uint16_t* q, int64_t ldqt,
                                                                     int64_t ldqh, const uint16_t* k, int64_t ldkt,
                                                                     int64_t ldkh, const uint16_t* v, int64_t ldvt,
                                                                     int64_t ldvh, uint16_t* q_out, Rotation r, int tokens,
                                                                     int heads, int head_dim, int lane_bits) {
  constexpr int N = VEC ? 8 : 1, kHeld = VEC ? 1 : 2;
  const int t = blockIdx.x % kXcds * (gridDim.x / kXcds) + blockIdx.x / kXcds;
  if (t >= tokens) return;
  const int64_t row = r.rot ? table_row(r, t) : 0;
  const TokenPlace place = token_place(c, token_sequence(c, t), t, tokens);
  const int hk = c.kv_heads, rows = heads + 2 * hk, units = head_dim / (2 * N);
  const int lanes = 1 << lane_bits, u0 = threadIdx.x & (lanes - 1), step = blockDim.x >> lane_bits;
  for (int h0 = 0; h0 < rows; h0 += step) {
    const int h = h0 + (threadIdx.x >> lane_bits);
    const bool is_q = h < heads, is_k = !is_q && h < heads + hk, is_v = !is_q && !is_k && h < rows;
    const int kh = is_k ? h - heads : h - heads - hk;
    const uint16_t* from = is_q ? q + t * ldqt + h * ldqh : is_k ? k + t * ldkt + kh * ldkh : v + t * ldvt + kh * ldvh;
    const Rotation turn = {r.cos_t, r.sin_t, nullptr, 0, is_v ? 0 : r.rot, r.interleaved, 1.0f};
    float a[kHeld][N], b[kHeld][N];
    int c0[kHeld], c1[kHeld];
    auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (u0 + i * lanes < units && h < rows) f(i);
    };
    each([&](int i) __attribute__((always_inline)) {
      rotated_unit<DT, VEC>(from, 0, turn, row, u0 + i * lanes, c0[i], c1[i], a[i], b[i]);
    });
    if (is_q) {
      uint16_t* out = q_out + ((int64_t)t * heads + h) * head_dim;
      each([&](int i) __attribute__((always_inline)) {
        if constexpr (VEC) {
          store8<DT>(out, c0[i], a[i]);
          store8<DT>(out, c1[i], b[i]);
        } else {
          store1<DT>(out, c0[i], a[i][0]);
          store1<DT>(out, c1[i], b[i][0]);
        }
      });
    }
    auto row_max = [&](auto finite_c) __attribute__((always_inline)) {
      float most = 0.0f;
      each([&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          most = larger<decltype(finite_c)::value>(larger<decltype(finite_c)::value>(most, a[i][e]), b[i][e]);
      });
      return group_max(most, lanes);
    };
    float most = row_max(std::false_type{});
    // (all lanes take part in both; what is not a row's has 0)
    if (__ballot(most == INFINITY)) most = row_max(std::true_type{});
    if (place.slot < 0 || !(is_k || is_v)) continue;
    const RowScale s = row_scale<DT>(__float_as_uint(most));
    if (s.most < 448.0f)  // a row at the top of the type's range
      each([&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < N; ++e) a[i][e] = held_to(a[i][e], s), b[i][e] = held_to(b[i][e], s);
      });
    uint8_t* out = (uint8_t*)(is_k ? c.k : c.v) + paged_at(c, place.page, kh, place.slot);
    each([&](int i) __attribute__((always_inline)) {
      if constexpr (VEC) {
        *(uint2*)(out + c0[i]) = codes8(a[i], s);
        *(uint2*)(out + c1[i]) = codes8(b[i], s);
      } else {
        const uint32_t pair = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(scaled(a[i][0], s), scaled(b[i][0], s), 0, false);
        out[c0[i]] = (uint8_t)pair;
        out[c1[i]] = (uint8_t)(pair >> 8);
      }
    });
    if (u0 == 0) {
      (is_k ? c.ks : c.vs)[paged_s_at(c, place.page, kh, place.slot)] = (uint8_t)s.byte;
      if (is_k && c.w) c.w[paged_w_at(c, place.page, kh, place.slot)] = 0.0f;
    }
  }
}

// A thread the same 16 channels of a key's and its value's row; a token's place is found by the thread, in a few dependent
// loads that neighbours share. Bound by memory: 39236 keys of 6 sequences, 8 heads of 128: 49 us, 4.9 TB/s (a large copy:
// 5.1); 700 keys 3.8 us, a launch and that chain.
template <class T>
__global__ __launch_bounds__(R8_THREADS) void paged_read_fp8_kernel(PagedArgs c, uint16_t* k_out, uint16_t* v_out,
                                                                    int tokens, int pieces) {
  const int64_t i = (int64_t)blockIdx.x * R8_THREADS + threadIdx.x;
  const uint32_t per = (uint32_t)c.kv_heads * (uint32_t)pieces;
  const int64_t t64 = i / per;
  if (t64 >= tokens) return;
  const int t = (int)t64;
  const uint32_t in = (uint32_t)(i - t64 * per), h = in / (uint32_t)pieces, p = in - h * (uint32_t)pieces;
  int b = 0, n_b = c.batch;  // the first sequence that ends behind the token, among [b, b + n_b]
  while (n_b > 0) {
    const int half = n_b >> 1;
    if (c.q_start[b + half + 1] <= t) b += half + 1, n_b -= half + 1;
    else n_b = half;
  }
  if (b >= c.batch) return;
  int t0, n;
  paged_new(c, b, tokens, t0, n);
  const int64_t place = (int64_t)c.kv_len[b] - n + (t - t0);
  if (t < t0 || t - t0 >= n || place < 0 || place >= c.capacity) return;
  const int slot = (int)place, page = paged_page(c, c.table + b * c.table_stride, slot);
  const int64_t at = paged_at(c, page, (int)h, slot) + 16 * p, sat = paged_s_at(c, page, (int)h, slot);
  const v4i kk = *(const v4i*)((const uint8_t*)c.k + at), vv = *(const v4i*)((const uint8_t*)c.v + at);
  const float ks = scale_of(c.ks[sat]), vs = scale_of(c.vs[sat]);
  const int64_t o = i * 16;
  *(v4i*)(k_out + o) = widen8<T>(kk[0], kk[1], ks);
  *(v4i*)(k_out + o + 8) = widen8<T>(kk[2], kk[3], ks);
  *(v4i*)(v_out + o) = widen8<T>(vv[0], vv[1], vs);
  *(v4i*)(v_out + o + 8) = widen8<T>(vv[2], vv[3], vs);
}

}  // namespace

extern "C" int gwa_paged_write_fp8(const gwa_paged_cache* cache, const gwa_paged_scales* scales, const void* q,
                                   int64_t ldqt, int64_t ldqh, const void* k, int64_t ldkt, int64_t ldkh, const void* v,
                                   int64_t ldvt, int64_t ldvh, const float* cos_t, const float* sin_t,
                                   int64_t table_rows, const int32_t* positions, void* q_out, int64_t tokens,
                                   int64_t heads, int64_t rot, int interleaved, void* stream) {
  const char* what = "paged_write_fp8";
  GWA_REQUIRE(scales, "%s: null scales", what);
  PagedArgs c;
  int bad = paged_check(what, cache, true, false, &c, scales);
  if (bad != GWA_OK) return bad;
  const int64_t d = cache->head_dim;
  GWA_REQUIRE(tokens >= 0 && tokens < (1ll << 31) && heads >= 0 && heads < (1 << 16), "%s: %lld tokens, %lld heads",
              what, (long long)tokens, (long long)heads);
  bad = rotation_check(what, cos_t, sin_t, table_rows, d, rot);
  if (bad != GWA_OK) return bad;
  if (tokens == 0) return GWA_OK;
  GWA_REQUIRE((heads == 0 || (q && q_out)) && k && v, "%s: null pointer", what);
  GWA_REQUIRE(GWA_ALIGNED(q, 2) && GWA_ALIGNED(k, 2) && GWA_ALIGNED(v, 2) && GWA_ALIGNED(q_out, 2) &&
                  GWA_ALIGNED(cos_t, 4) && GWA_ALIGNED(sin_t, 4) && GWA_ALIGNED(positions, 4),
              "%s: misaligned pointer", what);
  const Rotation r = {cos_t, sin_t, positions, table_rows, (int)rot, interleaved != 0, 1.0f};
  const bool vec = vector_units(d, rot, cos_t, sin_t) && vector_operand(q, ldqt, ldqh, 2) &&
                   vector_operand(k, ldkt, ldkh, 2) && vector_operand(v, ldvt, ldvh, 2) && GWA_ALIGNED(q_out, 16);
  int lane_bits = 6;
  if (vec)
    for (lane_bits = 0; 1 << lane_bits < d / 16; ++lane_bits) {}
  // whole waves, as many as a token's rows need, in as few turns as W8_THREADS allows
  const int64_t needed = (heads + 2 * c.kv_heads) << lane_bits, turns = (needed + W8_THREADS - 1) / W8_THREADS;
  const dim3 grid((unsigned)((tokens + kXcds - 1) / kXcds * kXcds));
  const dim3 block((unsigned)(((needed + turns - 1) / turns + 63) / 64 * 64));
  GWA_REQUIRE((int64_t)grid.x * block.x < (1ll << 32), "%s: %lld tokens are too many", what, (long long)tokens);
#define GWA_WRITE8(DT, VEC)                                                                                        \
  hipLaunchKernelGGL((paged_write_fp8_kernel<DT, VEC>), grid, block, 0, (hipStream_t)stream, c, (const uint16_t*)q, \
                     ldqt, ldqh, (const uint16_t*)k, ldkt, ldkh, (const uint16_t*)v, ldvt, ldvh, (uint16_t*)q_out, r, \
                     (int)tokens, (int)heads, (int)d, lane_bits)
  if (cache->dtype == GWA_DT_BF16) { if (vec) GWA_WRITE8(GWA_DT_BF16, true); else GWA_WRITE8(GWA_DT_BF16, false); }
  else { if (vec) GWA_WRITE8(GWA_DT_F16, true); else GWA_WRITE8(GWA_DT_F16, false); }
#undef GWA_WRITE8
  return gwa_check_launch(what);
}

extern "C" int gwa_paged_read_fp8(const gwa_paged_cache* cache, const gwa_paged_scales* scales, void* k_out, void* v_out,
                                  int64_t tokens, void* stream) {
  const char* what = "paged_read_fp8";
  GWA_REQUIRE(scales, "%s: null scales", what);
  PagedArgs c;
  const int bad = paged_check(what, cache, true, false, &c, scales);
  if (bad != GWA_OK) return bad;
  GWA_REQUIRE(tokens >= 0 && tokens < (1ll << 31), "%s: %lld tokens", what, (long long)tokens);
  if (tokens == 0 || c.batch == 0) return GWA_OK;
  GWA_REQUIRE(k_out && v_out && GWA_ALIGNED(k_out, 16) && GWA_ALIGNED(v_out, 16),
              "%s: the outputs must be there, 16-byte aligned", what);
  const int pieces = cache->head_dim / 16;
  const int64_t blocks = (tokens * c.kv_heads * pieces + R8_THREADS - 1) / R8_THREADS;
  GWA_REQUIRE(blocks * R8_THREADS < (1ll << 32), "%s: %lld tokens are too many", what, (long long)tokens);
  const dim3 grid((unsigned)blocks), block(R8_THREADS);
  if (cache->dtype == GWA_DT_BF16)
    hipLaunchKernelGGL((paged_read_fp8_kernel<Bf16>), grid, block, 0, (hipStream_t)stream, c, (uint16_t*)k_out,
                       (uint16_t*)v_out, (int)tokens, pieces);
  else
    hipLaunchKernelGGL((paged_read_fp8_kernel<Fp16>), grid, block, 0, (hipStream_t)stream, c, (uint16_t*)k_out,
                       (uint16_t*)v_out, (int)tokens, pieces);
  return gwa_check_launch(what);
}
