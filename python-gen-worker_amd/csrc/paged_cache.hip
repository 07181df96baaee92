// Rotary positions, the write of new tokens into a paged key/value cache, and the eviction of its least attended
// keys. All three move each value once and compute next to nothing: they are bound by memory, small calls by their
// launch. A copy of 2 GiB on this card runs at 4.94 TB/s (read and written bytes).
#include <algorithm>
#include <type_traits>

#include "paged_rotary.h"

namespace {

constexpr int RT_THREADS = 256;

// A thread a unit; the tables' rows are shared by a token's heads in L1. 16411 tokens, 24 heads of 128, half of each head
// rotated, bf16: 38 to 39 us for 202 MB, 5.2 TB/s; fp32 91 us for 403 MB, 4.4 TB/s.
template <int DT, bool VEC>
__global__ __launch_bounds__(RT_THREADS) void rotary_kernel(const void* x, int64_t ldxt, int64_t ldxh, void* y,
                                                            int64_t ldyt, int64_t ldyh, Rotation r, int64_t tokens,
                                                            int heads, int units) {
  const uint32_t per = (uint32_t)heads * (uint32_t)units;  // units a token
  const int64_t i = (int64_t)blockIdx.x * RT_THREADS + threadIdx.x;
  const int64_t t = i / per;
  if (t >= tokens) return;
  const uint32_t in = (uint32_t)(i - t * per), h = in / (uint32_t)units, u = in - h * (uint32_t)units;
  rotate_unit<DT, VEC>(x, t * ldxt + h * ldxh, y, t * ldyt + h * ldyh, r, r.rot ? table_row(r, t) : 0, (int)u);
}

// One workgroup a token: its query heads into q_out, its key and value heads into the token's slot, which the whole
// workgroup looks up once. 10475 tokens with 16 + 2 x 16 heads of 64: 22 us for 130 MB, 5.9 TB/s, on the same
// inputs again and again; on three sets in turn 27 to 28. 48 tokens 4.3 us.
template <int DT, bool VEC>
__global__ __launch_bounds__(RT_THREADS) void paged_write_kernel(PagedArgs c, const uint16_t* q, int64_t ldqt,
                                                                 int64_t ldqh, const uint16_t* k, int64_t ldkt,
                                                                 int64_t ldkh, const uint16_t* v, int64_t ldvt,
                                                                 int64_t ldvh, uint16_t* q_out, Rotation r, int tokens,
                                                                 int heads, int head_dim, int units) {
  const int t = blockIdx.x;
  const TokenPlace place = token_place(c, token_sequence(c, t), t, tokens);
  int64_t at = -1, wat = 0;
  if (place.slot >= 0) {
    at = paged_at(c, place.page, 0, place.slot);
    wat = paged_w_at(c, place.page, 0, place.slot);
  }
  const int64_t row = r.rot ? table_row(r, t) : 0;
  const Rotation none = {nullptr, nullptr, nullptr, 0, 0, 0, 1.0f};
  const int hk = c.kv_heads, items = (heads + (at >= 0 ? 2 * hk : 0)) * units;
  for (int i = threadIdx.x; i < items; i += RT_THREADS) {
    const int h = (int)((uint32_t)i / (uint32_t)units), u = i - h * units;
    if (h < heads)
      rotate_unit<DT, VEC>(q, t * ldqt + h * ldqh, q_out, ((int64_t)t * heads + h) * head_dim, r, row, u);
    else if (h < heads + hk)
      rotate_unit<DT, VEC>(k, t * ldkt + (h - heads) * ldkh, c.k, at + (h - heads) * c.head_stride, r, row, u);
    else
      rotate_unit<DT, VEC>(v, t * ldvt + (h - heads - hk) * ldvh, c.v, at + (h - heads - hk) * c.head_stride, none, 0,
                           u);
  }
  if (at >= 0 && c.w)
    for (int h = threadIdx.x; h < hk; h += RT_THREADS) c.w[wat + h * c.w_head_stride] = 0.0f;
}

}  // namespace

extern "C" int gwa_rotary_embed(const void* x, int64_t ldxt, int64_t ldxh, const float* cos_t, const float* sin_t,
                                int64_t table_rows, const int32_t* positions, void* y, int64_t ldyt, int64_t ldyh,
                                int64_t tokens, int64_t heads, int64_t head_dim, int64_t rot, int interleaved,
                                int inverse, int dtype, void* stream) {
  const char* what = "rotary_embed";
  GWA_REQUIRE(tokens >= 0 && heads >= 0 && heads < (1 << 20) && head_dim >= 2 && head_dim % 2 == 0 && head_dim <= 1024,
              "%s: %lld tokens, %lld heads of %lld (an even head_dim up to 1024)", what, (long long)tokens,
              (long long)heads, (long long)head_dim);
  GWA_REQUIRE(dtype >= GWA_DT_BF16 && dtype <= GWA_DT_F32, "%s: dtype %d", what, dtype);
  const int bad = rotation_check(what, cos_t, sin_t, table_rows, head_dim, rot);
  if (bad != GWA_OK) return bad;
  if (tokens == 0 || heads == 0) return GWA_OK;
  GWA_REQUIRE(x && y, "%s: null pointer", what);
  const int elem = dtype == GWA_DT_F32 ? 4 : 2;
  GWA_REQUIRE(GWA_ALIGNED(x, elem) && GWA_ALIGNED(y, elem) && GWA_ALIGNED(cos_t, 4) && GWA_ALIGNED(sin_t, 4) &&
                  GWA_ALIGNED(positions, 4), "%s: misaligned pointer", what);
  const Rotation r = {cos_t, sin_t, positions, table_rows, (int)rot, interleaved != 0, inverse ? -1.0f : 1.0f};
  const bool vec = vector_units(head_dim, rot, cos_t, sin_t) && vector_operand(x, ldxt, ldxh, elem) &&
                   vector_operand(y, ldyt, ldyh, elem);
  const int units = (int)(head_dim / (vec ? 16 : 2));
  const int64_t blocks = (tokens * heads * units + RT_THREADS - 1) / RT_THREADS;
  GWA_REQUIRE(tokens < (1ll << 40) && blocks < (1ll << 31), "%s: %lld tokens are too many", what, (long long)tokens);
#define GWA_ROTARY(DT, VEC)                                                                                        \
  hipLaunchKernelGGL((rotary_kernel<DT, VEC>), dim3((unsigned)blocks), dim3(RT_THREADS), 0, (hipStream_t)stream, x, \
                     ldxt, ldxh, y, ldyt, ldyh, r, tokens, (int)heads, units)
  if (dtype == GWA_DT_BF16) { if (vec) GWA_ROTARY(GWA_DT_BF16, true); else GWA_ROTARY(GWA_DT_BF16, false); }
  else if (dtype == GWA_DT_F16) { if (vec) GWA_ROTARY(GWA_DT_F16, true); else GWA_ROTARY(GWA_DT_F16, false); }
  else { if (vec) GWA_ROTARY(GWA_DT_F32, true); else GWA_ROTARY(GWA_DT_F32, false); }
#undef GWA_ROTARY
  return gwa_check_launch(what);
}

extern "C" int gwa_paged_write(const gwa_paged_cache* cache, const void* q, int64_t ldqt, int64_t ldqh, const void* k,
                               int64_t ldkt, int64_t ldkh, const void* v, int64_t ldvt, int64_t ldvh,
                               const float* cos_t, const float* sin_t, int64_t table_rows, const int32_t* positions,
                               void* q_out, int64_t tokens, int64_t heads, int64_t rot, int interleaved,
                               void* stream) {
  const char* what = "paged_write";
  PagedArgs c;
  int bad = paged_check(what, cache, true, false, &c);
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
  const int units = (int)(d / (vec ? 16 : 2));
#define GWA_WRITE(DT, VEC)                                                                                         \
  hipLaunchKernelGGL((paged_write_kernel<DT, VEC>), dim3((unsigned)tokens), dim3(RT_THREADS), 0,                   \
                     (hipStream_t)stream, c, (const uint16_t*)q, ldqt, ldqh, (const uint16_t*)k, ldkt, ldkh,       \
                     (const uint16_t*)v, ldvt, ldvh, (uint16_t*)q_out, r, (int)tokens, (int)heads, (int)d, units)
  if (cache->dtype == GWA_DT_BF16) { if (vec) GWA_WRITE(GWA_DT_BF16, true); else GWA_WRITE(GWA_DT_BF16, false); }
  else { if (vec) GWA_WRITE(GWA_DT_F16, true); else GWA_WRITE(GWA_DT_F16, false); }
#undef GWA_WRITE
  return gwa_check_launch(what);
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------
namespace {

constexpr int EV_THREADS = 1024, EV_WAVES = EV_THREADS / 64, EV_BINS = 2048;

// Weights as integers of the same order: -0 counts as 0, a NaN above every number
__device__ __forceinline__ uint32_t weight_rank(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the waves before this one and over all, of one value a wave (lane 0 holds it); two barriers.
__device__ __forceinline__ uint32_t wave_scan(uint32_t mine, uint32_t* cells, uint32_t& total) {
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) cells[wave] = mine;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (int i = 0; i < EV_WAVES; ++i) {
    const uint32_t x = cells[i];
    if (i < wave) before += x;
    all += x;
  }
  total = all;
  return before;
}

// One workgroup per (sequence, kv head). The rank of the last kept weight among the keys before the recent ones is
// found digit by digit (11 + 11 + 10 bits, a histogram each: 11 bits hold the sign, the exponent and two bits of the
// mantissa, so weights of one magnitude still spread over several counters); keys above it and, from the lowest
// slot on, as many equal to it as are still wanted are kept. Each wave owns a run of slots, so that after one sum
// over the waves every wave knows where its kept slots go: `kept` ascends and no order depends on timing. Bound by
// latency and, at many keys, by the few instructions a key takes on one CU: the first EV_HELD ranks are read once, up to
// 8 loads of 4 slots a thread in flight (24.9 -> 21.5 us over 16 of one slot, at 8 caches of 32768), and held in LDS for
// all passes (read again in every pass they took 76 us, held in registers, whose passes are unrolled code, 38 us and
// 13 for 640 keys). EV_AHEAD LDS reads go before what a pass does with them (2 us of 30 over one at a time; 8 and 16
// the same).
constexpr int EV_HELD = 32768;
constexpr int EV_AHEAD = 4;

__global__ __launch_bounds__(EV_THREADS) void evict_select_kernel(PagedArgs c, int budget, int recent, int held,
                                                                  int32_t* kept, int32_t* new_len) {
  extern __shared__ __attribute__((aligned(16))) uint32_t ranks[];  // held
  __shared__ uint32_t bins[EV_BINS];
  __shared__ uint32_t cells[EV_WAVES];
  __shared__ uint32_t found[2];
  const int h = blockIdx.x % c.kv_heads, b = blockIdx.x / c.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = paged_kv_len(c, b);
  int32_t* out = kept + (int64_t)blockIdx.x * budget;
  if (h == 0 && tid == 0) new_len[b] = min(n, budget);
  if (n <= budget) {
    for (int i = tid; i < budget; i += EV_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const int32_t* row = c.table + b * c.table_stride;
  // Only the `first` keys before the recent ones are ranked: more than budget - recent of them. Rank 0, which no
  // weight has, fills their last 64 slots up.
  const int first = n - recent, padded = (first + 63) & ~63;
  for (int i = tid; i < recent; i += EV_THREADS) out[budget - recent + i] = first + i;
  uint32_t want = (uint32_t)(budget - recent);
  if (want == 0) return;
  const int run = ((first + EV_WAVES - 1) / EV_WAVES + 63) & ~63;
  const int j0 = min(wave * run, padded), j1 = min(j0 + run, padded);
  auto rank_of = [&](int j) __attribute__((always_inline)) {
    const int at = min(j, first - 1);
    const uint32_t u = weight_rank(c.w[paged_w_at(c, paged_page(c, row, at), h, at)]);
    return j < first ? u : 0;
  };
  const int in_lds = min(padded, held);
  // a thread takes 4 neighbouring slots, which lie in one page (page_size >= 8), G times, all of them in flight together
  auto fill = [&](auto group_c) __attribute__((always_inline)) {
    constexpr int G = decltype(group_c)::value;
    typedef float v4u __attribute__((ext_vector_type(4), aligned(4)));
    for (int j = 4 * tid; j < in_lds; j += 4 * G * EV_THREADS) {
      int from[G], page[G];
      v4u w[G];
#pragma unroll
      for (int k = 0; k < G; ++k) from[k] = min(j + 4 * k * EV_THREADS, (first - 1) & ~3), page[k] = paged_page(c, row, from[k]);
#pragma unroll
      for (int k = 0; k < G; ++k) w[k] = *(const v4u*)(c.w + paged_w_at(c, page[k], h, from[k]));
#pragma unroll
      for (int k = 0; k < G; ++k) {
        const int s = j + 4 * k * EV_THREADS;
        if (s >= in_lds) break;
        v4i u;
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = s + i < first ? (int)weight_rank(w[k][i]) : 0;
        *(v4i*)(ranks + s) = u;
      }
    }
  };
  if (in_lds > 4 * EV_THREADS) fill(std::integral_constant<int, 8>{});
  else fill(std::integral_constant<int, 1>{});
  // f(slot of the wave's first lane, the lane's rank) over the wave's run, 64 slots at a time
  auto each = [&](auto f) __attribute__((always_inline)) {
    const int mid = min(j1, in_lds);
    int j = j0;
    for (; j + 64 * EV_AHEAD <= mid; j += 64 * EV_AHEAD) {
      uint32_t u[EV_AHEAD];
#pragma unroll
      for (int k = 0; k < EV_AHEAD; ++k) u[k] = ranks[j + 64 * k + lane];
#pragma unroll
      for (int k = 0; k < EV_AHEAD; ++k) f(j + 64 * k, u[k]);
    }
    for (; j < mid; j += 64) f(j, ranks[j + lane]);
    for (; j < j1; j += 64) f(j, rank_of(j + lane));
  };

  uint32_t prefix = 0;
  int shift = 21;
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < EV_BINS; i += EV_THREADS) bins[i] = 0;
    __syncthreads();
    // a slot of rank 0 counts below every key, so the place looked for never lies on one
    each([&](int, uint32_t u) __attribute__((always_inline)) {
      if (pass == 0 || (u >> (shift + bits)) == prefix) atomicAdd(&bins[(u >> shift) & ((1u << bits) - 1)], 1u);
    });
    __syncthreads();
    // counters from the top, two a thread: the one at which the count reaches `want`
    const int i1 = EV_BINS - 1 - 2 * tid, i0 = i1 - 1;
    const uint32_t c1 = bins[i1], c0 = bins[i0];
    uint32_t inc = c1 + c0;
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t x = __shfl_up(inc, o);
      if (lane >= o) inc += x;
    }
    uint32_t all;
    const uint32_t last = __shfl(inc, 63);
    const uint32_t above = wave_scan(last, cells, all) + inc - c1 - c0;
    if (above < want && above + c1 >= want) found[0] = (uint32_t)i1, found[1] = above;
    if (above + c1 < want && above + c1 + c0 >= want) found[0] = (uint32_t)i0, found[1] = above + c1;
    __syncthreads();
    prefix = (prefix << bits) | found[0];
    want -= found[1];  // still wanted among the keys of this prefix
    shift = pass == 0 ? 10 : 0;
    __syncthreads();
  }
  // now: the keys ranked above `prefix` are kept, and the first `want` equal to it
  uint32_t above = 0, equal = 0;  // of the wave's run
  each([&](int, uint32_t u) __attribute__((always_inline)) {
    above += (uint32_t)__popcll(__ballot(u > prefix));
    equal += (uint32_t)__popcll(__ballot(u == prefix));
  });
  uint32_t all;
  uint32_t eq = wave_scan(equal, cells, all);  // equal ones before this wave's run, of which at most `want` are kept
  uint32_t at = wave_scan(above, cells, all) + min(eq, want);
  auto lanes_below = [](uint64_t m) __attribute__((always_inline)) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
  };
  each([&](int j, uint32_t u) __attribute__((always_inline)) {
    bool keep = u > prefix;
    const uint64_t eqs = __ballot(u == prefix);
    if (eqs) {  // the same for the whole wave
      keep |= (eqs >> lane & 1) && eq + lanes_below(eqs) < want;
      eq += __popcll(eqs);
    }
    const uint64_t keeps = __ballot(keep);
    if (keep) out[at + lanes_below(keeps)] = j + lane;
    at += __popcll(keeps);
  });
}

constexpr int EC_THREADS = 256;

// Kept rows into the new pages: a row of k and v is head_dim / 8 pieces of 16 bytes (16 of an 8-bit cache), one piece of both
// a thread. 252 k rows of 128 (257 MB read and written), the same ones again and again: 44 to 46 us, 5.6 to 5.8 TB/s; three
// sets in turn: 55, of an 8-bit cache 32.
__global__ __launch_bounds__(EC_THREADS) void evict_copy_kernel(PagedArgs c, const int32_t* new_table,
                                                                int64_t new_stride, int new_capacity,
                                                                const int32_t* kept, int budget, int pieces) {
  const int h = blockIdx.y % c.kv_heads, b = blockIdx.y / c.kv_heads;
  const int rows = min(min(paged_kv_len(c, b), budget), new_capacity);
  // one step where the host's max_kv holds
  for (int64_t i = (int64_t)blockIdx.x * EC_THREADS + threadIdx.x; i < (int64_t)rows * pieces; i += (int64_t)gridDim.x * EC_THREADS) {
    const int r = (int)(i / pieces), p = (int)(i - (int64_t)r * pieces);
    const int j = min(max(kept[(int64_t)blockIdx.y * budget + r], 0), paged_kv_len(c, b) - 1);
    const int from = paged_page(c, c.table + b * c.table_stride, j);
    const int to = paged_page(c, new_table + b * new_stride, r);
    const int64_t src = paged_at(c, from, h, j) + 8 * p, dst = paged_at(c, to, h, r) + 8 * p;
    const v4i kk = *(const v4i*)(c.k + src), vv = *(const v4i*)(c.v + src);
    *(v4i*)(c.k + dst) = kk;
    *(v4i*)(c.v + dst) = vv;
    if (p == 0) {
      c.w[paged_w_at(c, to, h, r)] = c.w[paged_w_at(c, from, h, j)];
      if (c.ks) {
        c.ks[paged_s_at(c, to, h, r)] = c.ks[paged_s_at(c, from, h, j)];
        c.vs[paged_s_at(c, to, h, r)] = c.vs[paged_s_at(c, from, h, j)];
      }
    }
  }
}

// The entry points' body; `scales`: of an 8-bit cache, whose rows the copy takes as 16-bit elements of half as many
int evict_call(const char* what, const gwa_paged_cache* cache, const gwa_paged_scales* scales, const int32_t* new_table,
               int64_t new_stride, int64_t new_width, int64_t max_kv, int64_t budget, int64_t recent, int32_t* kept,
               int32_t* new_len, void* stream) {
  PagedArgs c;
  const int bad = paged_check(what, cache, false, true, &c, scales);
  if (bad != GWA_OK) return bad;
  if (scales) c.page_stride /= 2, c.head_stride /= 2, c.slot_stride /= 2;
  GWA_REQUIRE(budget > 0 && budget < (1ll << 30) && recent >= 0 && recent <= budget,
              "%s: a budget of %lld keys, %lld of them recent", what, (long long)budget, (long long)recent);
  GWA_REQUIRE(max_kv >= 0 && max_kv <= c.capacity, "%s: max_kv %lld in a table of %d slots", what, (long long)max_kv,
              c.capacity);
  const int64_t most = max_kv < budget ? max_kv : budget;
  GWA_REQUIRE(new_width * cache->page_size >= most && new_width * cache->page_size < (1ll << 30) &&
                  new_stride >= new_width,
              "%s: new_table has %lld pages a row, %lld keys are kept", what, (long long)new_width, (long long)most);
  if (c.batch == 0) return GWA_OK;
  GWA_REQUIRE(kept && new_len && (new_table || new_width == 0), "%s: null pointer", what);
  const int64_t groups = (int64_t)c.batch * c.kv_heads;
  const int pieces = cache->head_dim / (scales ? 16 : 8);
  const int64_t blocks = (std::max<int64_t>(most, 1) * pieces + EC_THREADS - 1) / EC_THREADS;
  GWA_REQUIRE(groups < 65536 && blocks < (1ll << 31), "%s: %lld heads of sequences are too many", what,
              (long long)groups);
  const int held = (int)std::min<int64_t>((max_kv + 63) / 64 * 64, EV_HELD);
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)groups), dim3(EV_THREADS), (size_t)held * 4,
                     (hipStream_t)stream, c, (int)budget, (int)recent, held, kept, new_len);
  const int rc = gwa_check_launch(what);
  if (rc != GWA_OK || new_width == 0) return rc;
  hipLaunchKernelGGL(evict_copy_kernel, dim3((unsigned)blocks, (unsigned)groups), dim3(EC_THREADS), 0,
                     (hipStream_t)stream, c, new_table, new_stride, (int)(new_width * cache->page_size), kept,
                     (int)budget, pieces);
  return gwa_check_launch(what);
}

}  // namespace

extern "C" int gwa_paged_evict(const gwa_paged_cache* cache, const int32_t* new_table, int64_t new_stride,
                               int64_t new_width, int64_t max_kv, int64_t budget, int64_t recent, int32_t* kept,
                               int32_t* new_len, void* stream) {
  return evict_call("paged_evict", cache, nullptr, new_table, new_stride, new_width, max_kv, budget, recent, kept, new_len,
                    stream);
}

extern "C" int gwa_paged_evict_fp8(const gwa_paged_cache* cache, const gwa_paged_scales* scales,
                                   const int32_t* new_table, int64_t new_stride, int64_t new_width, int64_t max_kv,
                                   int64_t budget, int64_t recent, int32_t* kept, int32_t* new_len, void* stream) {
  const char* what = "paged_evict_fp8";
  GWA_REQUIRE(scales, "%s: null scales", what);
  return evict_call(what, cache, scales, new_table, new_stride, new_width, max_kv, budget, recent, kept, new_len, stream);
}
