// Attention over the paged 8-bit cache where a row sees the last tokens up to its own place and the sequence's first.
#include "kv8_attn.h"

namespace mx {
namespace kv8 {

// The split of the keys goes by the most tokens of a sequence that a block of the rows kernel's rows visits, in whole tiles
// (a block of the tile kernel's rows visits up to 192 more, in the last split).  Windows of 1024 tokens of 64
// channels keep to one workgroup, their sinks' and their cut tile with them (one sequence, window 1000: 15.4 us an
// eager call in 5 splits and 11.6 in one).
static Plan window_plan(int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d, int window, int sinks) {
  const long long rows = std::min(max_q, 32);
  const int kv = (int)std::min((long long)max_kv, 64 * (up(sinks, 64) + up(window + rows + 62, 64)));
  Plan p = plan(B, T, max_q, kv, n_q, n_kv, d);
  side_by_side(p, (long long)std::min(max_q, T) * (n_q / n_kv), (long long)B * n_kv, kv, d);
  if (p.nr && (long long)kv * d <= 1152 * 64) {
    p.splits = 1;
    p.chunk = kv;
  }
  return p;
}

}  // namespace kv8
}  // namespace mx

extern "C" size_t mx_gqa_kv8_window_workspace(int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d, int window,
                                              int sinks) {
  using namespace mx::kv8;
  if (!sizes_ok(B, T, max_q, max_kv, n_q, n_kv, d) || window < 1 || sinks < 0) return 0;
  return workspace_of(window_plan(B, T, max_q, max_kv, n_q, n_kv, d, window, sinks), T, n_q, d);
}

extern "C" int mx_gqa_kv8_window(const void* q, const void* k_cache, const void* v_cache, const float* k_scale,
                                 const float* v_scale, const int* page_table, const int* kv_lens, const int* cu, void* O,
                                 int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d, int page, int pages,
                                 int max_pages, int q_stride, float scale, int window, int sinks, int dtype,
                                 void* workspace, size_t ws_bytes, void* stream) {
  using namespace mx::kv8;
  const int rc = check_call(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, cu, O, B, T, max_q, max_kv, n_q,
                            n_kv, d, page, pages, max_pages, q_stride, dtype);
  if (rc != MX_OK) return rc;
  if (window < 1 || sinks < 0) return MX_ERR_SHAPE;
  const Plan p = window_plan(B, T, max_q, max_kv, n_q, n_kv, d, window, sinks);
  // no row of the page table holds more tokens
  const Args a{(const uint16_t*)q, (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, page_table, kv_lens,
               cu, (uint16_t*)O, (float*)workspace, B, T, n_q, n_kv, pages, max_pages, q_stride, log2_page(page), 1,
               p.splits, p.chunk, scale * kLog2e, (int)std::min<long long>(window, kMostTokens),
               (int)std::min<long long>(sinks, kMostTokens), nullptr, 0};
  return launch<WINDOW>(a, p, d, dtype, ws_bytes, stream);
}
