// Attention over the paged 8-bit cache for drafted tokens that form a tree: a row sees the tokens before the drafted
// ones, and of those the ones that its mask names.
#include "kv8_attn.h"

extern "C" size_t mx_gqa_kv8_tree_workspace(int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d) {
  using namespace mx::kv8;
  if (!sizes_ok(B, T, max_q, max_kv, n_q, n_kv, d)) return 0;
  return workspace_of(tree_plan(B, T, max_q, max_kv, n_q, n_kv, d), T, n_q, d);
}

extern "C" int mx_gqa_kv8_tree(const void* q, const void* k_cache, const void* v_cache, const float* k_scale,
                               const float* v_scale, const int* page_table, const int* kv_lens, const int* cu,
                               const void* tree, void* O, int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d,
                               int page, int pages, int max_pages, int q_stride, float scale, int words, int dtype,
                               void* workspace, size_t ws_bytes, void* stream) {
  using namespace mx::kv8;
  if (!tree) return MX_ERR_NULL;
  const int rc = check_call(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, cu, O, B, T, max_q, max_kv, n_q,
                            n_kv, d, page, pages, max_pages, q_stride, dtype);
  if (rc != MX_OK) return rc;
  if (words < 1 || words > kMostWords / 2) return MX_ERR_SHAPE;
  if ((uintptr_t)tree & 7) return MX_ERR_ALIGN;
  const Plan p = tree_plan(B, T, max_q, max_kv, n_q, n_kv, d);
  const Args a{(const uint16_t*)q, (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, page_table, kv_lens,
               cu, (uint16_t*)O, (float*)workspace, B, T, n_q, n_kv, pages, max_pages, q_stride, log2_page(page), 1,
               p.splits, p.chunk, scale * kLog2e, 0, 0, (const uint32_t*)tree, 2 * words};
  return launch<TREE>(a, p, d, dtype, ws_bytes, stream);
}
