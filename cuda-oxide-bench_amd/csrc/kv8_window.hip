// Attention over the paged 8-bit cache where a row sees the last tokens up to its own place and the sequence's first.
#include "kv8_attn.h"

namespace mx {
namespace kv8 {

// The split of the keys goes by the most tokens of a sequence that a block of the rows kernel's rows visits, in whole tiles.
// (A block of the tile kernel's rows visits up to 256 more: its 224 more rows may cross 4 borders of tiles.  They go to the
// last split.)
//
// One workgroup where plan() would take it, and up to 8 KB of a head's K codes past that: the sinks' tile and the one that a
// window's cut adds on 64 channels, one of them on 128.  It saves the second launch, which counts where the host launches
// each call, and loses where it does not.  Split and in one workgroup, us, windows with 4 sinks, 4 queries a KV head, 1 or
// 4 rows a sequence: on 64 channels, 1000 tokens (5 tiles a wave), 1 sequence in a graph 8.6..9.2 and 9.7..11.4, eager
// 14.5..15.7 and 10.3..11.3; 16 of 8 heads in a graph 10.6 and 11.5, 64 18.3 either way.  On 128 channels, 440 tokens, 1
// sequence in a graph 10.6..11.1 and 9.5..9.9, 4 11.0 and 13.1, eager 15.3 and 10.4..13.1.  Past it one workgroup loses in
// eager calls too or gains less: 128 channels, 1000 tokens in a graph 10.9 and 14.1, eager 15.0 and 14.0.
static Plan window_plan(int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d, int window, int sinks) {
  const long long rows = std::min(max_q, 32);
  const int kv = (int)std::min((long long)max_kv, 64 * (up(sinks, 64) + up(window + rows + 62, 64)));
  Plan p = plan(B, T, max_q, kv, n_q, n_kv, d);
  side_by_side(p, (long long)std::min(max_q, T) * (n_q / n_kv), (long long)B * n_kv, kv, d);
  if (p.nr && (long long)kv * d <= 65536 + 8192) {
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
