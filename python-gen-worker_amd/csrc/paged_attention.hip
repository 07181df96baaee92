// Attention of new tokens over a paged key/value cache, with the keys' attention weight gathered on request.
#include "paged_common.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// ---------------------------------------------------------------------------
// any head_dim: one wave per (new token, query head)
// ---------------------------------------------------------------------------
constexpr int RW_WAVES = 4, RW_MAX_D = 256;

// q . key of one lane's key, fp32; q in LDS, the key's row read in 16-byte pieces
template <class T>
__device__ __forceinline__ float row_dot(const float* q, const uint16_t* key, int d) {
  float s = 0.0f;
  for (int i = 0; i < d; i += 8) {
    const v4i r = *(const v4i*)(key + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s = fmaf(q[i + 2 * e], T::load((uint16_t)r[e]), s);
      s = fmaf(q[i + 2 * e + 1], T::load((uint16_t)((uint32_t)r[e] >> 16)), s);
    }
  }
  return s;
}

// 64 keys a step, one a lane: scores, the running maximum m and sum l of the softmax over all keys so far (in the
// log2 domain, p = 2^(s c - m)), then the outputs, which lie over the lanes (channel lane + 64 i).
template <class T>
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
    if (j < keys) s = row_dot<T>(qs[wave], c.k + paged_at(c, paged_page(c, pages, j), h, j), d) * c_log2;
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
      const uint16_t* vr = c.v + paged_at(c, paged_page(c, pages, j0 + k), h, j0 + k);
#pragma unroll
      for (int i = 0; i < RW_MAX_D / 64; ++i)
        if (lane + 64 * i < d) acc[i] = fmaf(pk, T::load(vr[lane + 64 * i]), acc[i]);
    }
  }
  const float inv = keys > 0 ? 1.0f / l : 0.0f;
  for (int i = 0; i < RW_MAX_D / 64; ++i)
    if (lane + 64 * i < d) o[row * d + lane + 64 * i] = (uint16_t)T::pack(acc[i] * inv, 0.0f);
  if (lane == 0) lse[row] = keys > 0 ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
}

// w[key] += sum of 2^(s c - lse) over the rows that see the key: one lane a key, 64 keys of one kv head a wave
template <class T>
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
    const uint16_t* key = c.k + paged_at(c, page, h, j);
    float sum = 0.0f;
    for (int i = 0; i < n * g; ++i) {
      const int t = t0 + i / g, x = h * g + i % g;
      const int seen = causal ? len - n + i / g : len - 1;
      if (seen < j0) continue;  // the same for the whole wave
      __syncthreads();
      for (int e = lane; e < d; e += 64) qs[e] = T::load(q[t * ldqt + x * ldqh + e]);
      __syncthreads();
      const float s = row_dot<T>(qs, key, d) * c_log2;
      if (j <= seen) sum += __builtin_amdgcn_exp2f(s - lse[(int64_t)t * heads + x] * kLog2e);
    }
    if (j0 + lane < len) c.w[paged_w_at(c, page, h, j)] += sum;
  }
}

}  // namespace

extern "C" int64_t gwa_paged_attention_workspace(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int) {
  return 0;
}

extern "C" int gwa_paged_attention(const gwa_paged_cache* cache, const void* q, int64_t ldqt, int64_t ldqh, void* o,
                                   float* lse, int64_t tokens, int64_t heads, int64_t max_q, int64_t max_kv,
                                   float scale, int causal, int gather, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
  const char* what = "paged_attention";
  PagedArgs c;
  const int bad = paged_check(what, cache, true, gather != 0, &c);
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
  const dim3 grid((unsigned)((rows + RW_WAVES - 1) / RW_WAVES)), block(64 * RW_WAVES);
  const dim3 ggrid((unsigned)((max_kv + 63) / 64 > 0 ? (max_kv + 63) / 64 : 1), (unsigned)groups);
  auto run = [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((paged_attn_rows_kernel<T>), grid, block, 0, st, c, (const uint16_t*)q, ldqt, ldqh,
                       (uint16_t*)o, lse, (int)tokens, (int)heads, (int)d, c_log2, causal);
    if (gather && groups > 0)
      hipLaunchKernelGGL((paged_gather_rows_kernel<T>), ggrid, dim3(64), 0, st, c, (const uint16_t*)q, ldqt, ldqh, lse,
                         (int)tokens, (int)heads, (int)d, c_log2, causal);
  };
  if (cache->dtype == GWA_DT_BF16) run(Bf16{});
  else run(Fp16{});
  return gwa_check_launch(what);
}
