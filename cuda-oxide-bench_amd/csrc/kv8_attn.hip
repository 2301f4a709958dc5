// Attention over the paged 8-bit cache where a row sees the tokens up to its own place, or all.
#include "kv8_attn.h"

extern "C" size_t mx_gqa_kv8_workspace(int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d) {
  using namespace mx::kv8;
  if (!sizes_ok(B, T, max_q, max_kv, n_q, n_kv, d)) return 0;
  return workspace_of(plan(B, T, max_q, max_kv, n_q, n_kv, d), T, n_q, d);
}

extern "C" int mx_gqa_kv8(const void* q, const void* k_cache, const void* v_cache, const float* k_scale,
                          const float* v_scale, const int* page_table, const int* kv_lens, const int* cu, void* O, int B,
                          int T, int max_q, int max_kv, int n_q, int n_kv, int d, int page, int pages, int max_pages,
                          int q_stride, float scale, int causal, int dtype, void* workspace, size_t ws_bytes,
                          void* stream) {
  using namespace mx::kv8;
  const int rc = check_call(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, cu, O, B, T, max_q, max_kv, n_q,
                            n_kv, d, page, pages, max_pages, q_stride, dtype);
  if (rc != MX_OK) return rc;
  const Plan p = plan(B, T, max_q, max_kv, n_q, n_kv, d);
  const Args a{(const uint16_t*)q, (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, page_table, kv_lens,
               cu, (uint16_t*)O, (float*)workspace, B, T, n_q, n_kv, pages, max_pages, q_stride, log2_page(page),
               causal ? 1 : 0, p.splits, p.chunk, scale * kLog2e, 0, 0, nullptr, 0};
  return launch<PLAIN>(a, p, d, dtype, ws_bytes, stream);
}
