// Attention over a paged key/value cache of e4m3 codes under a power of two a row: the entry points.
#include "paged_attention.h"

extern "C" int64_t gwa_paged_attention_fp8_workspace(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                                                     int64_t head_dim, int64_t max_q, int64_t max_kv, int64_t capacity,
                                                     int gather) {
  return workspace_of<true>(batch, tokens, heads, kv_heads, head_dim, max_q, max_kv, capacity, gather);
}

extern "C" int gwa_paged_attention_fp8(const gwa_paged_cache* cache, const gwa_paged_scales* scales, const void* q,
                                       int64_t ldqt, int64_t ldqh, void* o, float* lse, int64_t tokens, int64_t heads,
                                       int64_t max_q, int64_t max_kv, float scale, int causal, int gather,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "paged_attention_fp8";
  GWA_REQUIRE(scales, "%s: null scales", what);
  return attention_call<true>(what, cache, scales, q, ldqt, ldqh, o, lse, tokens, heads, max_q, max_kv, scale, causal,
                              gather, workspace, workspace_bytes, stream);
}
